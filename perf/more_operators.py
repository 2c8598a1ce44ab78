"""The experts' products and the draw of a class, as cases that can be timed: their inputs, one pass through each, in plain
torch operations and through the library's entry points, and the bytes and operations that a pass cannot do without.

  sample   a class of every row drawn by the softmax of its scores: temperature, the k best, the likeliest that make up p,
           those of at least a share of the best one's probability, from given random numbers
  gated    rows sorted by expert through their experts' gated projections, act(x G^T) * (x U^T) (and every gradient)
  product  rows sorted by expert times their experts' weights, x W^T (and both gradients)
"""
import math

import numpy as np
import torch

own = False  # True: the library's kernels; False: the plain form

DEVICE = "cuda:0"
TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}  # the library's names of the types
SIZES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def _sample(**k):
    return dict(dict(op="sample", type="bf16", rows=1, classes=10, pad=0, spread=4.0, closed=0.0, top_k=0, top_p=0.0, min_p=0.0), **k)


def _gated(**k):
    return dict(dict(op="gated", type="bf16", rows=1, width=8, hidden=8, experts=1, activation="silu", idle=0.0, dropped=0.0,
                     backward=False), **k)


def _product(**k):
    return dict(dict(op="product", type="bf16", rows=1, width=8, hidden=8, experts=1, idle=0.0, dropped=0.0, backward=False), **k)


def listed():
    return [
        # one row that is answered step by step
        dict(_sample(type="f16", rows=1, classes=50021, top_k=50, top_p=0.9), name="sample_one_row"),
        # a server's batch: every row with parameters of its own, some without; rows padded to whole lines, classes masked
        dict(_sample(type="bf16", rows=64, classes=131000, pad=72, closed=0.3, top_k=100, top_p=0.9, min_p=0.02), name="sample_serving"),
        # a large batch of single-precision scores, no bound on how many classes take part
        dict(_sample(type="f32", rows=384, classes=100003, spread=2.0, top_p=0.95), name="sample_large"),
        # a class for every document of a table, by the raw values of a ten-class model
        dict(_sample(type="f64", rows=2_000_000, classes=10, spread=2.0, top_p=0.95, min_p=0.01), name="sample_ten_classes"),
        # seven rows that wait for an answer, at two experts each
        dict(_gated(type="bf16", rows=14, width=4096, hidden=1024, experts=64), name="gated_few_rows"),
        # the rows of a long prompt, some experts without any
        dict(_gated(type="f16", rows=8192, width=4096, hidden=4096, experts=8, activation="gelu_tanh", idle=0.1), name="gated_prompt"),
        # single precision, odd sizes
        dict(_gated(type="f32", rows=5003, width=1001, hidden=699, experts=5, activation="gelu"), name="gated_single"),
        # the rows of a training step at four experts each, with all gradients
        dict(_gated(type="bf16", rows=65536, width=4096, hidden=1024, experts=64, dropped=0.02, backward=True), name="gated_training"),
        # the second product of the seven rows
        dict(_product(type="bf16", rows=14, width=1024, hidden=4096, experts=64), name="product_few_rows"),
        # a batch's scores of every class of a vocabulary: one expert
        dict(_product(type="bf16", rows=64, width=4096, hidden=131000), name="product_scores"),
        # documents times the linear model of their segment, ten raw values
        dict(_product(type="f32", rows=500_009, width=200, hidden=10, experts=37, dropped=0.01), name="product_documents"),
        # the second product of the training step, with its gradients
        dict(_product(type="bf16", rows=65536, width=1024, hidden=4096, experts=64, dropped=0.02, backward=True), name="product_training"),
    ]


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    def size(lo, hi):
        """Mostly a multiple of 64 or 8, now and then any."""
        unit = rng.choice([64, 64, 8, 1])
        return max(1, log_int(lo, hi) // unit) * unit

    family = rng.choice(["vocabulary", "vocabulary", "classes", "few", "few", "prompt", "training", "scores", "documents"])
    if family in ("vocabulary", "classes"):
        limits = dict(top_k=rng.choice([0, 0, 1, log_int(2, 1000)]), top_p=rng.choice([0.0, 0.5, 0.9, 0.99]),
                      min_p=rng.choice([0.0, 0.0, 0.001, 0.1]), closed=rng.choice([0.0, 0.0, 0.5]), spread=rng.choice([0.5, 2.0, 4.0]),
                      pad=rng.choice([0, 0, 5, 64]))
        if family == "vocabulary":
            classes = log_int(2000, 131072)
            return _sample(type=rng.choice(["f32", "f16", "bf16"]), rows=log_int(1, max(1, min(384, 32_000_000 // classes))),
                           classes=classes, **limits)
        classes = log_int(2, 1000)
        return _sample(type=rng.choice(["f64", "f64", "f32", "bf16"]), rows=log_int(100, 16_000_000 // classes), classes=classes, **limits)
    experts = rng.choice([1, rng.randint(2, 8), log_int(8, 128)])
    routes = dict(experts=experts, idle=rng.choice([0.0, 0.2]), dropped=rng.choice([0.0, 0.05]))
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    make = rng.choice([_gated, _product])
    more = dict(activation=rng.choice(list(ACTIVATIONS))) if make is _gated else {}
    if family == "documents":
        return _product(type=rng.choice(["f32", "f64"]), rows=log_int(1000, 500_000), width=rng.randint(5, 200),
                        hidden=rng.randint(1, 10), **routes)
    if family == "scores":
        return _product(type=kind, rows=log_int(1, 200), width=size(512, 4096), hidden=size(2000, 131072))
    width = size(256, 8192)
    hidden = size(128, max(128, min(8192, 600_000_000 // (width * experts))))
    if family == "few":
        return make(type=kind, rows=log_int(1, 256), width=width, hidden=hidden, **routes, **more)
    backward = family == "training"
    rows = log_int(200, max(200, min(65536, (250_000_000_000 if kind == "f32" else 500_000_000_000) // (width * hidden * (3 if backward else 1)))))
    return make(type=kind, rows=rows, width=width, hidden=hidden, backward=backward, **routes, **more)


# ---- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = TYPES[case["type"]]
    made = torch.float64 if kind == torch.float64 else torch.float32

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=made)

    rows, s = case["rows"], dict(case=case)
    if case["op"] == "sample":
        wide = torch.full((rows, case["classes"] + case["pad"]), float("nan"), dtype=kind, device=DEVICE)
        s["scores"] = wide[:, :case["classes"]]
        scores = randn(rows, case["classes"]) * case["spread"]
        if case["closed"]:  # what a mask has left out
            scores[rand(rows, case["classes"]) < case["closed"]] = float("-inf")
        s["scores"].copy_(scores)
        s["temperature"], s["uniform"] = 0.6 + 0.8 * rand(rows), rand(rows)
        # every request has limits of its own; a fifth of them leaves each out
        if case["top_k"]:
            s["top_k"] = torch.where(rand(rows) < 0.2, 0, 1 + (rand(rows) * case["top_k"]).to(torch.int32)).to(torch.int32)
        if case["top_p"]:
            s["top_p"] = torch.where(rand(rows) < 0.2, 1.0, case["top_p"] * (1 - 0.1 * rand(rows)))
        if case["min_p"]:
            s["min_p"] = torch.where(rand(rows) < 0.2, 0.0, case["min_p"] * rand(rows))
        return s
    width, hidden, experts = case["width"], case["hidden"], case["experts"]
    if experts > 1 or case["dropped"]:
        # experts that are asked for more or less often, some not at all; rows behind the last sorted one belong to none
        liked = 0.25 + rand(experts)
        liked[1:][rand(experts - 1) < case["idle"]] = 0
        count = rows - int(rows * case["dropped"])
        chosen = torch.multinomial(liked, count, replacement=True, generator=g)
        counts = torch.zeros(experts + 1, dtype=torch.int64, device=DEVICE).index_add_(0, chosen + 1, torch.ones_like(chosen))
        s["offsets"] = torch.cumsum(counts, 0).to(torch.int32)
    s["source"] = randn(rows, width).to(kind)
    for name in ("gate", "up") if case["op"] == "gated" else ("weights",):
        s[name] = torch.empty(experts, hidden, width, dtype=kind, device=DEVICE)
        for part in torch.split(s[name], max(1, 100_000_000 // (hidden * width))):  # in parts: the wide copies are large
            part.copy_(randn(*part.shape) * width ** -0.5)
    # the program's buffers: rows that belong to no expert stay as they are
    s["result"] = torch.zeros(rows, hidden, dtype=kind, device=DEVICE)
    if case["backward"]:
        s["gradients"] = randn(rows, hidden).to(kind)
        s["source_gradients"] = torch.zeros(rows, width, dtype=kind, device=DEVICE)
    return s


# ---- the plain form

def _plain_sample(s):
    x = s["scores"].to(torch.float64)  # an index is a border between sums
    rows, classes = x.shape
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(classes, device=DEVICE)[None, :]
    e = torch.exp((ordered - ordered[:, :1]) / s["temperature"].to(torch.float64)[:, None])
    e = torch.where(ordered > float("-inf"), e, 0)
    if "top_k" in s:
        k = s["top_k"][:, None]
        e = torch.where((k <= 0) | (rank < k), e, 0)
    keep = e > 0
    if "top_p" in s:
        p = s["top_p"].to(torch.float64)[:, None]
        sums = torch.cumsum(e, 1)
        keep &= (p >= 1) | (rank == 0) | (sums - e < p * sums[:, -1:])
    if "min_p" in s:
        keep &= e >= s["min_p"].to(torch.float64)[:, None]
    e = torch.where(keep, e, 0)
    sums = torch.cumsum(e, 1)
    total = sums[:, -1:]
    at = (sums <= s["uniform"].to(torch.float64)[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, keep.sum(1, keepdim=True) - 1)
    weights = torch.gather(e, 1, at) / total
    return [torch.gather(order, 1, at).view(rows).to(torch.int32), weights.view(rows).to(torch.float64 if s["scores"].dtype == torch.float64 else torch.float32)]


def _parts(s):
    """Where each row goes when every expert has as many places as the largest needs, and how many those are."""
    case = s["case"]
    if "offsets" not in s:
        return torch.arange(case["rows"], device=DEVICE), case["rows"]
    offsets = s["offsets"].to(torch.int64)
    most = int((offsets[1:] - offsets[:-1]).max())
    row = torch.arange(int(offsets[-1]), device=DEVICE)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    return expert * most + row - offsets[expert], most


def _spread(rows, places, most, experts, acc):
    wide = torch.zeros(experts * most, rows.shape[1], dtype=acc, device=DEVICE)
    wide[places] = rows[:places.numel()].to(acc)
    return wide.view(experts, most, -1)


def _together(wide, places, out):
    out[:places.numel()] = wide.reshape(-1, wide.shape[2])[places].to(out.dtype)
    return out


def _activation(name, x):
    """act(x) and its derivative."""
    if name == "silu":
        y = 1 / (1 + torch.exp(-x))
        return x * y, y * (1 + x * (1 - y))
    if name == "gelu":
        y = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * y, y + x * torch.exp(-0.5 * x * x) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    return torch.where(x > 0, x, 0), (x > 0).to(x.dtype)


def _plain_gated(s):
    case, kind = s["case"], s["source"].dtype
    acc = torch.float64 if kind == torch.float64 else torch.float32
    places, most = _parts(s)
    x = _spread(s["source"], places, most, case["experts"], acc)
    gate, up = s["gate"].to(acc), s["up"].to(acc)
    g, u = torch.bmm(x, gate.transpose(1, 2)), torch.bmm(x, up.transpose(1, 2))
    a, da = _activation(case["activation"], g)
    out = [_together(a * u, places, s["result"])]
    if case["backward"]:
        d = _spread(s["gradients"], places, most, case["experts"], acc)
        dg, du = d * u * da, d * a
        out.append(_together(torch.bmm(dg, gate) + torch.bmm(du, up), places, s["source_gradients"]))
        out.append(torch.bmm(dg.transpose(1, 2), x).to(kind))
        out.append(torch.bmm(du.transpose(1, 2), x).to(kind))
    return out


def _plain_product(s):
    case, kind = s["case"], s["source"].dtype
    acc = torch.float64 if kind == torch.float64 else torch.float32
    places, most = _parts(s)
    x, w = _spread(s["source"], places, most, case["experts"], acc), s["weights"].to(acc)
    out = [_together(torch.bmm(x, w.transpose(1, 2)), places, s["result"])]
    if case["backward"]:
        d = _spread(s["gradients"], places, most, case["experts"], acc)
        out.append(_together(torch.bmm(d, w), places, s["source_gradients"]))
        out.append(torch.bmm(d.transpose(1, 2), x).to(kind))
    return out


# ---- the library's calls

def _at(s, name):
    return s[name].data_ptr() if name in s else 0


def _own_sample(s, cb, code, stream):
    scores = s["scores"]
    rows, classes = scores.shape
    indexes = torch.empty(rows, dtype=torch.int32, device=DEVICE)
    weights = torch.empty(rows, dtype=torch.float64 if scores.dtype == torch.float64 else torch.float32, device=DEVICE)
    sampling = cb.sampling(temperature_ptr=_at(s, "temperature"), top_k_ptr=_at(s, "top_k"), top_p_ptr=_at(s, "top_p"), min_p_ptr=_at(s, "min_p"))
    size = cb.sample_classes_bytes(code, rows, classes)
    workspace = torch.empty(size, dtype=torch.uint8, device=DEVICE)
    cb.sample_classes(code, rows, classes, scores.data_ptr(), scores.stride(0), sampling, s["uniform"].data_ptr(), indexes.data_ptr(), weights.data_ptr(),
                      workspace.data_ptr(), size, stream)
    return [indexes, weights]


def _own_gated(s, cb, code, stream):
    case, x = s["case"], s["source"]
    rows, width, hidden, experts = case["rows"], case["width"], case["hidden"], case["experts"]
    activation, offsets, of_expert = ACTIVATIONS[case["activation"]], _at(s, "offsets"), hidden * width
    # what the backward pass needs of the forward one: the rows' gate and up values, in 32 bits at least
    kept = torch.empty(rows, 2 * hidden, dtype=torch.promote_types(x.dtype, torch.float32), device=DEVICE) if case["backward"] else None
    cb.gated_rows(code, activation, rows, width, hidden, experts, offsets, x.data_ptr(), width, s["gate"].data_ptr(), s["up"].data_ptr(), of_expert,
                  s["result"].data_ptr(), hidden, 0 if kept is None else kept.data_ptr(), stream)
    out = [s["result"]]
    if kept is not None:
        dgate, dup = torch.empty_like(s["gate"]), torch.empty_like(s["up"])
        pre = torch.empty(rows, 2 * hidden, dtype=x.dtype, device=DEVICE)  # the gradients of those values
        cb.gated_rows_backward(code, activation, rows, width, hidden, experts, offsets, s["gradients"].data_ptr(), hidden, x.data_ptr(), width,
                               s["gate"].data_ptr(), s["up"].data_ptr(), of_expert, kept.data_ptr(), pre.data_ptr(),
                               s["source_gradients"].data_ptr(), width, dgate.data_ptr(), dup.data_ptr(), of_expert, stream)
        out += [s["source_gradients"], dgate, dup]
    return out


def _own_product(s, cb, code, stream):
    case, x = s["case"], s["source"]
    rows, width, hidden, experts = case["rows"], case["width"], case["hidden"], case["experts"]
    offsets, of_expert = _at(s, "offsets"), hidden * width
    cb.multiply_rows(code, rows, width, hidden, experts, offsets, x.data_ptr(), width, s["weights"].data_ptr(), of_expert, s["result"].data_ptr(), hidden,
                     stream)
    out = [s["result"]]
    if case["backward"]:
        dw = torch.empty_like(s["weights"])
        cb.multiply_rows_backward(code, rows, width, hidden, experts, offsets, s["gradients"].data_ptr(), hidden, x.data_ptr(), width,
                                  s["weights"].data_ptr(), of_expert, s["source_gradients"].data_ptr(), width, dw.data_ptr(), of_expert, stream)
        out += [s["source_gradients"], dw]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        import catboost_amd as cb

        call = {"sample": _own_sample, "gated": _own_gated, "product": _own_product}[op]
        return call(state, cb, CODES[state["case"]["type"]], torch.cuda.current_stream().cuda_stream)
    return {"sample": _plain_sample, "gated": _plain_gated, "product": _plain_product}[op](state)


# ---- what a pass cannot do without

def work(case):
    size, rows = SIZES[case["type"]], case["rows"]
    if case["op"] == "sample":
        limits = 4 * rows * (2 + sum(bool(case[k]) for k in ("top_k", "top_p", "min_p")))
        return {"bytes": rows * case["classes"] * size + limits + rows * (12 if size == 8 else 8), "flops": 3 * rows * case["classes"]}
    matrices = 2 if case["op"] == "gated" else 1
    there = rows - int(rows * case["dropped"])
    # few rows do not reach every expert
    experts = case["experts"] if there >= 8 * case["experts"] else case["experts"] * (1 - (1 - 1 / case["experts"]) ** there)
    weights = matrices * experts * case["hidden"] * case["width"] * size
    source, result = there * case["width"] * size, there * case["hidden"] * size
    product = 2 * there * case["width"] * case["hidden"] * matrices
    if not case["backward"]:
        return {"bytes": source + weights + result, "flops": product}
    return {"bytes": source + weights + result + result + source + weights * case["experts"] / experts, "flops": 3 * product}


# ---- the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "sample":
        return None if case["rows"] * case["classes"] > 45_000_000 else _exact_sample(prepare(case, seed))
    return _exact_routed(prepare(case, seed), case)


def _exact_sample(s):
    x = s["scores"].to(torch.float64).cpu().numpy()
    rows, classes = x.shape
    take = {k: s[k].cpu().numpy() for k in ("temperature", "uniform", "top_k", "top_p", "min_p") if k in s}
    indexes, weights = np.empty(rows, np.int32), np.empty(rows, np.float64)
    step = max(1, 4_000_000 // classes)
    for begin in range(0, rows, step):  # some rows at a time
        part = slice(begin, min(rows, begin + step))
        at = {k: v[part, None] for k, v in take.items()}
        order = np.argsort(-x[part], axis=1, kind="stable")
        z = np.take_along_axis(x[part], order, 1).astype(np.longdouble)
        e = np.exp((z - z[:, :1]) / at["temperature"].astype(np.longdouble))
        if "top_k" in at:
            e[(np.arange(classes) >= at["top_k"]) & (at["top_k"] > 0)] = 0
        cut = np.zeros(e.shape, bool)
        if "top_p" in at:
            sums = np.cumsum(e, 1)
            cut[:, 1:] = (sums[:, :-1] >= at["top_p"].astype(np.longdouble) * sums[:, -1:]) & (at["top_p"] < 1)
        if "min_p" in at:
            cut |= e < at["min_p"].astype(np.longdouble)
        e[cut] = 0
        sums = np.cumsum(e, 1)
        found = np.argmax(sums > at["uniform"].astype(np.longdouble) * sums[:, -1:], axis=1)[:, None]
        indexes[part] = np.take_along_axis(order, found, 1)[:, 0]
        weights[part] = (np.take_along_axis(e, found, 1) / sums[:, -1:])[:, 0].astype(np.float64)
    return [torch.from_numpy(indexes), torch.from_numpy(weights)]


def _exact_routed(s, case):
    rows, hidden, f64 = case["rows"], case["hidden"], torch.float64
    bounds = s["offsets"].tolist() if "offsets" in s else [0, rows]
    names = ("gate", "up") if case["op"] == "gated" else ("weights",)
    result = torch.zeros(rows, hidden, dtype=f64, device=DEVICE)
    back = [torch.zeros(rows, case["width"], dtype=f64, device=DEVICE)] + [torch.zeros(s[n].shape, dtype=f64, device=DEVICE) for n in names] if case["backward"] else []
    for e in range(case["experts"]):
        part = slice(bounds[e], bounds[e + 1])
        if part.start == part.stop:
            continue
        x = s["source"][part].to(f64).requires_grad_(case["backward"])
        w = [s[n][e].to(f64).requires_grad_(case["backward"]) for n in names]
        y = torch.nn.functional.linear(x, w[0])
        if len(w) == 2:
            act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
                   "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["activation"]]
            y = act(y) * torch.nn.functional.linear(x, w[1])
        result[part] = y.detach()
        if back:
            gradients = torch.autograd.grad(y, [x] + w, s["gradients"][part].to(f64))
            back[0][part] = gradients[0]
            for to, g in zip(back[1:], gradients[1:]):
                to[e] = g
    return [result] + back
