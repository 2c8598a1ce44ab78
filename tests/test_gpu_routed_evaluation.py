"""Documents evaluated by models of their own, and the operators on scores and rows around it, against the oracle. Needs an MI355X."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import catboost_amd as cb
from oracle import model_builder as mb
from oracle.oracle import OracleModel

pytestmark = pytest.mark.gpu


def model(seed, n_float, dim, trees=30, depth=5, one_hot=False):
    rng = np.random.default_rng(seed)
    floats = [mb.float_feature(i, i) for i in range(n_float)]
    cats = [mb.cat_feature(0, n_float)] if one_hot else []
    out = []
    for t in range(trees):
        splits = [("float", int(rng.integers(n_float)), float(np.float32(rng.normal()))) for _ in range(1 + t % depth)]
        if one_hot and t % 3 == 0:
            splits[-1] = ("onehot", 0, 1 + t % 4)
        out.append((splits, rng.normal(size=(1 << len(splits)) * dim)))
    d = mb.build_oblivious(floats, cats, dim, out, scale=1.25, bias=list(rng.normal(size=dim)))
    m = cb.ModelCalcer()
    m.load_from_dict(d)
    m.enable_gpu_evaluation(0)
    return m, OracleModel(d)


def mixed(models, x, dim, ids, weights):
    """Definition: values of the models that a document names, added in order."""
    values = [np.reshape(o.calc(x), (len(x), dim)) for _, o in models]
    out = np.zeros((len(x), dim))
    for j in range(ids.shape[1]):
        for e in range(len(models)):
            at = ids[:, j] == e
            out[at] += (1.0 if weights is None else weights[at, j, None]) * values[e][at]
    return out


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a)).cuda()


def routed(models, layout, features, docs, ids, weights, dim, stream=None):
    evaluators = [m.evaluator() for m, _ in models]
    size = cb.eval_routed_bytes(evaluators, layout, docs, ids.shape[1])
    workspace = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    results = torch.full((docs * dim + 1,), 7.0, dtype=torch.float64, device="cuda")
    d, w = dev(ids.astype(np.int32)), None if weights is None else dev(weights)
    torch.cuda.synchronize()
    cb.eval_routed(evaluators, features, docs, ids.shape[1], d.data_ptr(), 0 if w is None else w.data_ptr(), results.data_ptr(), workspace.data_ptr(), size,
                   stream)
    assert float(results[-1]) == 7.0 and bool((workspace[size:] == 255).all())
    return results[:-1].cpu().numpy().reshape(docs, dim)


# one pass in tree order gives the oracle's sums; a product and an addition for each model are rounded the same way in both
@pytest.mark.parametrize("docs", [1, 2, 63, 700, 20_000])
@pytest.mark.parametrize("dim,per_doc,weighted", [(1, 1, False), (1, 2, True), (3, 1, True), (3, 3, True), (10, 2, False)])
def test_flat_rows(docs, dim, per_doc, weighted):
    rng = np.random.default_rng(docs + dim)
    models = [model(s, n, dim) for s, n in enumerate((7, 12, 3, 20, 9))]
    stride = 24  # wider than what any model reads
    x = rng.normal(size=(docs, stride)).astype(np.float32)
    ids = rng.integers(-1, 6, size=(docs, per_doc))
    ids[ids == 3] = 4  # model 3 has no document
    ids[rng.random(docs) < 0.1] = 1  # the same model several times
    weights = rng.normal(size=(docs, per_doc)) if weighted else None
    d = dev(x)
    f = cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), stride)
    np.testing.assert_array_equal(routed(models, cb.LAYOUT_FLAT_ROWS, f, docs, ids, weights, dim), mixed(models, x, dim, ids, weights))


@pytest.mark.parametrize("docs", [5, 3001])
def test_split_rows_with_categories(docs):
    rng = np.random.default_rng(docs)
    models = [model(1, 8, 2, one_hot=True), model(2, 8, 2), model(3, 8, 2, one_hot=True)]
    x = rng.normal(size=(docs, 9)).astype(np.float32)
    cats = rng.integers(0, 6, size=(docs, 2)).astype(np.int32)
    ids = rng.integers(0, 3, size=(docs, 2))
    d, c = dev(x), dev(cats)
    f = cb.DeviceEvaluator.features(cb.LAYOUT_SPLIT_ROWS, d.data_ptr(), 9, c.data_ptr(), 2)
    flat = np.concatenate([x[:, :8], cats[:, :1].view(np.float32)], 1)
    np.testing.assert_array_equal(routed(models, cb.LAYOUT_SPLIT_ROWS, f, docs, ids, None, 2), mixed(models, flat, 2, ids, None))


def test_on_a_stream_with_slices_and_no_documents():
    rng = np.random.default_rng(3)
    models = [model(s, 10, 1) for s in range(2)] + [model(0, 10, 1)]
    for m, _ in models:
        m.set_small_batch_slicing(True)
    docs = 4000
    x = rng.normal(size=(docs, 10)).astype(np.float32)
    ids = rng.integers(0, 3, size=(docs, 1))
    stream = torch.cuda.Stream()
    d = dev(x)
    f = cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), 10)
    got = routed(models, cb.LAYOUT_FLAT_ROWS, f, docs, ids, None, 1, stream.cuda_stream)
    np.testing.assert_allclose(got, mixed(models, x, 1, ids, None), rtol=1e-9, atol=1e-12)  # the slices' own bar
    cb.eval_routed([m.evaluator() for m, _ in models], f, 0, 1, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("docs", [4001, 300_000])
def test_models_rows_at_any_address(docs):
    """An odd number of features and a workspace at a multiple of 8: a model's first document is at any multiple of 4."""
    rng = np.random.default_rng(docs)
    models = [model(s, n, 1, trees=60) for s, n in enumerate((51, 37, 51))]
    x = rng.normal(size=(docs, 53)).astype(np.float32)
    ids = rng.integers(0, 3, size=(docs, 1)).astype(np.int32)
    ids[rng.random(docs) < 0.3] = 2
    d, i = dev(x), dev(ids)
    evaluators = [m.evaluator() for m, _ in models]
    size = cb.eval_routed_bytes(evaluators, cb.LAYOUT_FLAT_ROWS, docs, 1)
    results = torch.full((docs,), 7.0, dtype=torch.float64, device="cuda")
    f = cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), 53)
    expected = mixed(models, x, 1, ids, None)[:, 0]
    for at in (8, 24, 0):
        workspace = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        cb.eval_routed(evaluators, f, docs, 1, i.data_ptr(), 0, results.data_ptr(), workspace.data_ptr() + at, size)
        np.testing.assert_allclose(results.cpu().numpy(), expected, rtol=1e-9, atol=1e-12)  # the models' own bar
        assert bool((workspace[:at] == 255).all()) and bool((workspace[at + size:] == 255).all())


def test_the_most_evaluators_and_the_most_for_a_document():
    """1024 of them, most of a few models again and again, 64 for each document, the same ones several times."""
    rng = np.random.default_rng(5)
    models = [model(s, 10, 2) for s in range(3)]
    docs, count, per_doc = 150, 1024, 64
    x = rng.normal(size=(docs, 10)).astype(np.float32)
    ids = rng.integers(-1, count + 1, size=(docs, per_doc))
    weights = rng.normal(size=(docs, per_doc))
    d = dev(x)
    f = cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), 10)
    inside = np.where((ids >= 0) & (ids < count), ids % 3, -1)
    got = routed([models[e % 3] for e in range(count)], cb.LAYOUT_FLAT_ROWS, f, docs, ids, weights, 2)
    np.testing.assert_array_equal(got, mixed(models, x, 2, inside, weights))


def test_from_two_threads_at_once():
    rng = np.random.default_rng(6)
    models = [model(s, 10, 2) for s in range(3)]
    docs = 3000
    x = rng.normal(size=(2, docs, 10)).astype(np.float32)
    ids = rng.integers(0, 3, size=(2, docs, 2))
    data = [dev(a) for a in x]
    features = [cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), 10) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    evaluators = [m.evaluator() for m, _ in models]
    size = cb.eval_routed_bytes(evaluators, cb.LAYOUT_FLAT_ROWS, docs, 2)
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    indexes = [dev(i.astype(np.int32)) for i in ids]
    results = [torch.empty(docs, 2, dtype=torch.float64, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            for _ in range(10):
                cb.eval_routed(evaluators, features[i], docs, 2, indexes[i].data_ptr(), 0, results[i].data_ptr(), spaces[i].data_ptr(), size,
                               streams[i].cuda_stream)
        except Exception as e:
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for i in range(2):
        np.testing.assert_array_equal(results[i].cpu().numpy(), mixed(models, x[i], 2, ids[i], None))


def test_refusals():
    models = [model(1, 6, 1), model(2, 9, 1), model(3, 6, 2)]
    one, wide, other = (m.evaluator() for m, _ in models)
    x, ids, out = torch.zeros(10, 9, device="cuda"), torch.zeros(10, dtype=torch.int32, device="cuda"), torch.zeros(10, dtype=torch.float64, device="cuda")
    size = cb.eval_routed_bytes([one, wide], cb.LAYOUT_FLAT_ROWS, 10, 1)
    workspace = torch.zeros(size, dtype=torch.uint8, device="cuda")

    def call(evaluators=(one, wide), layout=cb.LAYOUT_FLAT_ROWS, stride=9, docs=10, per_doc=1, ids_ptr=ids.data_ptr(), space=workspace.data_ptr(), room=size,
             results=out.data_ptr()):
        cb.eval_routed(list(evaluators), cb.DeviceEvaluator.features(layout, x.data_ptr(), stride), docs, per_doc, ids_ptr, 0, results, space, room)

    call()
    for arguments, message in [
            (dict(evaluators=[]), "evaluators: 0"), (dict(evaluators=[one] * 1025), "evaluators: 1025"), (dict(evaluators=[one, other]), "different dimensions"),
            (dict(layout=cb.LAYOUT_FLAT_COLUMNS, stride=10), "features in rows"), (dict(layout=7), "unknown feature layout"), (dict(stride=8), "expected: 9"),
            (dict(per_doc=0), "evaluators per document: 0"), (dict(per_doc=65), "evaluators per document: 65"), (dict(docs=1 << 31), "too many documents"),
            (dict(ids_ptr=0), "pointer is null"), (dict(results=0), "pointer is null"), (dict(space=0), "are needed"), (dict(room=size - 1), "are needed"),
            (dict(space=workspace.data_ptr() + 4), "multiple of 8")]:
        with pytest.raises(cb.CatBoostError, match=message):
            call(**arguments)
    with pytest.raises(cb.CatBoostError, match="different dimensions"):
        cb.eval_routed_bytes([one, other], cb.LAYOUT_FLAT_ROWS, 10, 1)
    library = cb.load_library()
    null = (ctypes.c_void_p * 2)(one._h, None)
    assert not library.CbHipEvalRouted(null, 2, ctypes.byref(cb.DeviceEvaluator.features(0, x.data_ptr(), 9)), 10, 1, ids.data_ptr(), None, out.data_ptr(),
                                       workspace.data_ptr(), size, None)
    assert "handle is null" in cb.last_error()


def test_a_gated_mixture_from_features_to_classes():
    """A gate model's values choose each document's two models among those that are on; their classes' values are mixed, classes
    that the document has had are made less likely, the three best ones and their probabilities are the answer."""
    rng = np.random.default_rng(11)
    docs, experts, dim, per_doc = 5000, 4, 6, 2
    gate, gate_oracle = model(100, 10, experts)
    models = [model(200 + e, 10, dim) for e in range(experts)]
    x = rng.normal(size=(docs, 10)).astype(np.float32)
    d = dev(x)
    f = cb.DeviceEvaluator.features(cb.LAYOUT_FLAT_ROWS, d.data_ptr(), 10)
    on, prior = np.array([[0b1011]], np.uint32), rng.normal(size=experts).astype(np.float32)  # the third model is off
    seen = rng.integers(0, dim, size=(docs, 2)).astype(np.int32)
    offsets = np.arange(docs + 1) * 2
    presence = np.full(docs, 1.5, np.float32)
    t = {k: dev(v) for k, v in dict(on=on.view(np.int32), rows=np.zeros(docs, np.int32), prior=prior, seen=seen.ravel(), offsets=offsets, presence=presence).items()}

    def empty(*shape, dtype=torch.float64):
        return torch.empty(shape, dtype=dtype, device="cuda")

    scores, ids, weights = empty(docs, experts), empty(docs, per_doc, dtype=torch.int32), empty(docs, per_doc)
    torch.cuda.synchronize()
    gate.evaluator().eval_data(f, docs, scores.data_ptr())
    cb.adjust_scores(cb.FLOAT64, docs, experts, scores.data_ptr(), experts,
                     cb.score_adjustment(class_bias_ptr=t["prior"].data_ptr(), allowed_ptr=t["on"].data_ptr(), allowed_stride=1, allowed_count=1,
                                         allowed_rows_ptr=t["rows"].data_ptr()), scores.data_ptr(), experts)
    cb.select_top(cb.FLOAT64, docs, experts, scores.data_ptr(), experts, per_doc, True, ids.data_ptr(), weights.data_ptr())
    evaluators = [m.evaluator() for m, _ in models]
    size = cb.eval_routed_bytes(evaluators, cb.LAYOUT_FLAT_ROWS, docs, per_doc)
    values, workspace = empty(docs, dim), empty(size, dtype=torch.uint8)
    torch.cuda.synchronize()  # the evaluators run on streams of their own
    cb.eval_routed(evaluators, f, docs, per_doc, ids.data_ptr(), weights.data_ptr(), values.data_ptr(), workspace.data_ptr(), size)
    cb.adjust_scores(cb.FLOAT64, docs, dim, values.data_ptr(), dim,
                     cb.score_adjustment(history_offsets_ptr=t["offsets"].data_ptr(), history_ptr=t["seen"].data_ptr(), history_count=2 * docs,
                                         presence_ptr=t["presence"].data_ptr()), values.data_ptr(), dim)
    best, probabilities = empty(docs, 3, dtype=torch.int32), empty(docs, 3)
    cb.select_top(cb.FLOAT64, docs, dim, values.data_ptr(), dim, 3, False, best.data_ptr(), probabilities.data_ptr())

    g = np.reshape(gate_oracle.calc(x), (docs, experts)) + prior
    g[:, 2] = -np.inf
    order = np.argsort(-g, axis=1, kind="stable")[:, :per_doc]
    np.testing.assert_array_equal(ids.cpu().numpy(), order)
    w = np.exp(np.take_along_axis(g, order, 1) - g.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    np.testing.assert_allclose(weights.cpu().numpy(), w, rtol=1e-14)
    v = mixed(models, x, dim, order, w)
    had = np.zeros((docs, dim), bool)
    np.put_along_axis(had, seen.astype(np.int64), True, 1)
    v -= 1.5 * had
    np.testing.assert_allclose(values.cpu().numpy(), v, rtol=1e-12, atol=1e-12)
    p = np.exp(v - v.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    top = np.argsort(-v, axis=1, kind="stable")[:, :3]
    np.testing.assert_array_equal(best.cpu().numpy(), top)
    np.testing.assert_allclose(probabilities.cpu().numpy(), np.take_along_axis(p, top, 1), rtol=1e-11)
    # and the evaluator's own probabilities of the same values
    own = empty(docs, dim)
    evaluators[0].apply_prediction_type(cb.APT_PROBABILITY, docs, values.data_ptr(), own.data_ptr())
    evaluators[0].synchronize()
    np.testing.assert_allclose(own.cpu().numpy(), p, rtol=1e-9, atol=1e-12)
