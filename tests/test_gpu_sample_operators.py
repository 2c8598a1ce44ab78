"""A class drawn by the softmax of a row's scores, against the definition by sorted rows in extended precision. Needs an MI355X."""
import numpy as np
import pytest
import torch

import catboost_amd as cb

pytestmark = pytest.mark.gpu

TYPES = {cb.FLOAT64: torch.float64, cb.FLOAT32: torch.float32, cb.FLOAT16: torch.float16, cb.BFLOAT16: torch.bfloat16}
NAMES = {cb.FLOAT64: "f64", cb.FLOAT32: "f32", cb.FLOAT16: "f16", cb.BFLOAT16: "bf16"}
ALL = pytest.mark.parametrize("kind", list(TYPES), ids=NAMES.get)


def drawn(x, temperature, top_k, top_p, min_p, uniform):
    """One row by the definition: index, weight, and how near the draw is to a border (as a share of the sum)."""
    there = np.flatnonzero(x > -np.inf)
    if not len(there):
        return -1, 0.0, 1.0
    order = there[np.argsort(-x[there], kind="stable")]
    z = x[order].astype(np.longdouble)
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    if z[0] == np.inf:
        e = (z == np.inf).astype(np.longdouble)
    else:
        e = np.exp((z - z[0]) / np.longdouble(temperature))
    if top_k > 0:
        e = np.where(np.arange(len(e)) < top_k, e, 0)
    near = np.longdouble(1.0)
    keep = np.ones(len(e), bool)
    total = e.sum()
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(e)[:-1]])
        share = np.longdouble(max(top_p, 0)) * total
        keep = before < share
        keep[0] = True
        near = min(near, np.min(np.abs(before[1:] - share), initial=1.0) / total)
    least = np.longdouble(min(min_p, 1.0)) if min_p > 0 else np.longdouble(0)
    keep &= e >= least
    e = np.where(keep, e, 0)
    sums = np.cumsum(e)
    share = np.longdouble(min(max(np.nan_to_num(uniform), 0), 1)) * sums[-1]
    at = int(np.argmax(sums > share)) if sums[-1] > share else int(np.max(np.flatnonzero(e)))
    near = min(near, np.min(np.abs(sums - share)) / sums[-1])
    return int(order[at]), float(e[at] / sums[-1]), float(near)


class Draw:
    def __init__(self, kind, scores, uniform, temperature=None, top_k=None, top_p=None, min_p=None, pad=0, weights=True):
        rows, classes = scores.shape
        wide = torch.full((rows, classes + pad), float("nan"), dtype=TYPES[kind], device="cuda")
        self.scores = wide[:, :classes]
        self.scores.copy_(torch.from_numpy(scores))
        self.kind = kind

        def dev(a, t):
            return None if a is None else torch.as_tensor(np.asarray(a, t)).cuda()

        self.parts = [dev(temperature, np.float32), dev(top_k, np.int32), dev(top_p, np.float32), dev(min_p, np.float32)]
        self.uniform = dev(uniform, np.float32)
        self.indexes = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        self.weights = torch.full((rows,), -7, dtype=torch.float64 if kind == cb.FLOAT64 else torch.float32, device="cuda") if weights else None
        self.size = cb.sample_classes_bytes(kind, rows, classes)
        self.workspace = torch.empty(max(self.size, 8), dtype=torch.uint8, device="cuda")
        self()

    def __call__(self):
        rows, classes = self.scores.shape
        ptr = [0 if t is None else t.data_ptr() for t in self.parts]
        cb.sample_classes(self.kind, rows, classes, self.scores.data_ptr(), self.scores.stride(0), cb.sampling(*ptr), self.uniform.data_ptr(),
                          self.indexes.data_ptr(), 0 if self.weights is None else self.weights.data_ptr(), self.workspace.data_ptr(), self.size,
                          torch.cuda.current_stream().cuda_stream)

    def check(self):
        """Classes are equal unless a border is nearer than the roundings of the sums; weights to one rounding of their type more."""
        x = self.scores.to(torch.float64).cpu().numpy()
        rows, classes = x.shape
        got, weights = self.indexes.cpu().numpy(), None if self.weights is None else self.weights.to(torch.float64).cpu().numpy()
        given = [np.full(rows, d) if t is None else t.cpu().numpy() for t, d in zip(self.parts, (1.0, 0, 1.0, 0.0))]
        uniform = self.uniform.cpu().numpy()
        sure = 0
        for r in range(rows):
            index, weight, near = drawn(x[r], given[0][r], given[1][r], given[2][r] if not np.isnan(given[2][r]) else 1.0, given[3][r], uniform[r])
            # each class's weight is off by half a whole number (2^-45 of the best one's at most for these sizes) and the exponential's rounding
            if near > classes * 2.0 ** -45 + 2.0 ** -45:
                sure += 1
                assert got[r] == index, (r, got[r], index, near)
                if weights is not None:
                    step = 2.0 ** -53 if self.kind == cb.FLOAT64 else 2.0 ** -24
                    assert abs(weights[r] - weight) <= weight * (step + classes * 2.0 ** -45 + 2.0 ** -44), (r, weights[r], weight)
        assert sure >= 0.9 * rows


SIZES = [(1, 1), (5, 2), (40, 3), (64, 10), (33, 17), (20, 64), (12, 100), (9, 257), (6, 1000), (4, 4097), (3, 20011), (2, 131000)]


def scores_of(rng, rows, classes, kind, spread=3.0):
    return rng.standard_normal((rows, classes)) * spread


@ALL
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_plain_draw(kind, size):
    rng = np.random.default_rng(size[1])
    Draw(kind, scores_of(rng, *size, kind), rng.random(size[0])).check()


@ALL
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("limits", ["k", "p", "m", "kp", "kpm"])
def test_limits(kind, size, limits):
    rng = np.random.default_rng(size[1] + len(limits))
    rows, classes = size
    scores = scores_of(rng, rows, classes, kind)
    scores[rng.random(size) < 0.2] = -np.inf
    more = {}
    if "k" in limits:
        more["top_k"] = rng.integers(-1, max(2, min(classes + 3, 60)), rows)
    if "p" in limits:
        more["top_p"] = rng.random(rows) * 1.1
    if "m" in limits:
        more["min_p"] = np.where(rng.random(rows) < 0.2, 0, 10.0 ** -rng.uniform(0, 5, rows))
    Draw(kind, scores, rng.random(rows), temperature=rng.uniform(0.3, 2.0, rows), pad=3, **more).check()


@ALL
def test_ties_go_to_the_lowest_class(kind):
    """Equal scores: every sum is a whole number of equal weights, so borders are exact."""
    classes = 8
    scores = np.zeros((16, classes))
    uniform = np.repeat(np.arange(8) / 8, 2)
    d = Draw(kind, scores, uniform)
    assert d.indexes.tolist() == [i // 2 for i in range(16)]
    assert torch.all(d.weights == 0.125)
    # half of the sum, whether asked for by number or by share: the four lowest
    for more in (dict(top_k=[4] * 16), dict(top_p=[0.5] * 16)):
        d = Draw(kind, scores, uniform, **more)
        assert d.indexes.tolist() == [i // 2 // 2 for i in range(16)] and torch.all(d.weights == 0.25)
    # both zeros are equal
    signs = scores.copy()
    signs[:, ::2] = -0.0
    assert Draw(kind, signs, uniform).indexes.tolist() == [i // 2 for i in range(16)]


@ALL
@pytest.mark.parametrize("classes", [10, 300, 70001])
def test_ties_among_many(kind, classes):
    """Few different scores: the class is found by its place among equals."""
    rng = np.random.default_rng(classes)
    rows = 6
    scores = rng.integers(-2, 3, (rows, classes)) * 0.5
    Draw(kind, scores, rng.random(rows), top_k=[0, 0, 7, classes // 2, 0, 3], top_p=[1, 0.4, 1, 1, 0.9, 0.5]).check()
    scores[:] = 1.5  # all alike: the draw is uniform * classes
    d = Draw(kind, scores, [0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1])
    expected = [0, classes // 4, classes // 2, int(classes * 0.75), int(classes * (1 - 2.0 ** -24)), classes - 1]
    assert d.indexes.tolist() == expected


@ALL
@pytest.mark.parametrize("value", [0.0, 1.5, -1.5])
def test_a_score_that_most_of_many_classes_have(kind, value):
    """More classes with one score than 16 bits count, under and over it a few others, zeros of both signs among them."""
    rng = np.random.default_rng(9)
    classes, rows = 140001, 8
    scores = np.full((rows, classes), value)
    scores[rng.random((rows, classes)) < 0.01] = -0.0
    scores[rng.random((rows, classes)) < 0.01] = 0.0
    scores[:, 5:4000:7] = rng.standard_normal((rows, 571)) * 3
    Draw(kind, scores, rng.random(rows), top_k=[0, 0, 100, 90000, 0, 300, 0, 139000], top_p=[1, 0.8, 1, 0.9, 0.01, 0.5, 0.99, 1], min_p=[0, 0.01, 0, 0, 0, 0, 0.5, 0]).check()


@ALL
@pytest.mark.parametrize("classes", [3, 12, 40, 700, 9000])
def test_values_at_the_ends(kind, classes):
    """Infinities and NaN, rows without any class, temperatures, numbers and limits outside their ranges."""
    inf, nan = float("inf"), float("nan")
    rng = np.random.default_rng(classes)
    big = {cb.FLOAT64: 1.7e308, cb.FLOAT32: 3.3e38, cb.FLOAT16: 6e4, cb.BFLOAT16: 3.3e38}[kind]
    rows = 14
    x = scores_of(rng, rows, classes, kind)
    x[0] = -inf
    x[1] = nan
    x[2, 1] = nan
    x[3, [0, 2]] = inf
    x[4] = -inf
    x[4, 2] = -big
    x[5, 0], x[5, 1] = big, -big
    temperature, uniform = np.ones(rows), rng.random(rows)
    temperature[6], temperature[7], temperature[8], temperature[9], temperature[10] = 0, -1, nan, inf, 1e-30
    uniform[11], uniform[12], uniform[13] = -3, 2, nan
    uniform[3] = 0.7
    top_p, min_p, top_k = np.ones(rows), np.zeros(rows), np.zeros(rows, int)
    top_p[2], min_p[12], top_k[13] = nan, nan, -5
    d = Draw(kind, x, uniform, temperature, top_k, top_p, min_p)
    d.check()
    got = d.indexes.tolist()
    assert got[:2] == [-1, -1] and d.weights[:2].tolist() == [0, 0]
    assert got[2] != 1 and got[3] == 2 and d.weights[3] == 0.5 and got[4] == 2 and d.weights[4] == 1 and got[5] == 0
    best = d.scores.to(torch.float64).cpu().numpy().argmax(1)
    for r in (6, 7, 8, 10):
        assert got[r] == best[r] and d.weights[r] == 1
    assert got[13] == best[13]
    # one class by each of the limits
    for more in (dict(top_k=[1] * rows), dict(top_p=[0] * rows), dict(top_p=[-1] * rows), dict(min_p=[1] * rows), dict(min_p=[5] * rows)):
        d = Draw(kind, x, [0.99] * rows, **more)
        for r in range(6, rows):
            if (d.scores[r] == d.scores[r].max()).sum() == 1:
                assert d.indexes[r] == best[r] and d.weights[r] == 1


@ALL
def test_shares_of_many_draws(kind):
    """10000 rows with the same four scores, numbers in steps: each class comes as often as its weight says, to one step."""
    rows = 10000
    scores = np.tile(np.log([4.0, 1.0, 3.0, 2.0]), (rows, 1))
    d = Draw(kind, scores, (np.arange(rows) + 0.5) / rows, weights=False)
    e = torch.exp(d.scores[0].to(torch.float64)).cpu().numpy()
    counts = np.bincount(d.indexes.cpu().numpy(), minlength=4)
    assert np.all(np.abs(counts - rows * e / e.sum()) <= 1.01)


@ALL
@pytest.mark.parametrize("classes", [10, 500, 40000])
def test_replays(kind, classes):
    """A captured draw gives what the eager one gives, replay after replay."""
    rng = np.random.default_rng(3)
    d = Draw(kind, scores_of(rng, 7, classes, kind), rng.random(7), top_p=[0.9] * 7, top_k=[0, 5, 0, 9, 0, 0, 40])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        d()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            d()
    for step in range(3):
        d.uniform.copy_(torch.rand(7, device="cuda"))
        d.scores.mul_(0.9)
        d()
        expected = d.indexes.clone(), d.weights.clone()
        d.indexes.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d.indexes, expected[0]) and torch.equal(d.weights, expected[1])
        d.check()


@pytest.mark.parametrize("kind", [cb.FLOAT32, cb.BFLOAT16], ids=NAMES.get)
@pytest.mark.parametrize("classes", [10, 100, 2000, 20000])
def test_rows_past_32_bits(kind, classes):
    """Rows that begin more than 2^32 bytes, and 2^31 values, behind the first."""
    rows, stride = 3, (1 << 31) + 1
    rng = np.random.default_rng(classes)
    d = Draw(kind, scores_of(rng, rows, classes, kind), rng.random(rows), top_p=[0.9] * rows)
    expected = d.indexes.clone()
    wide = torch.empty((rows - 1) * stride + classes, dtype=TYPES[kind], device="cuda").as_strided((rows, classes), (stride, 1))
    wide.copy_(d.scores)
    d.scores = wide
    d.indexes.fill_(-7)
    d()
    assert torch.equal(d.indexes, expected)


@ALL
@pytest.mark.parametrize("classes", [16, 33, 512, 3000, 33333])
def test_rows_at_any_address(kind, classes):
    """Rows that begin anywhere, next to others of NaN."""
    rng = np.random.default_rng(1)
    d = Draw(kind, scores_of(rng, 5, classes, kind), rng.random(5), top_k=[0, 9, 0, 200, 0], top_p=[1, 1, 0.5, 0.9, 0.2])
    expected = d.indexes.clone(), d.weights.clone()
    values = d.scores.clone()
    for shift in (1, 2, 3, 5):
        flat = torch.full((shift + 5 * (classes + 1) + 8,), float("nan"), dtype=TYPES[kind], device="cuda")
        d.scores = flat[shift:shift + 5 * (classes + 1)].view(5, classes + 1)[:, :classes]
        d.scores.copy_(values)
        d()
        assert torch.equal(d.indexes, expected[0]) and torch.equal(d.weights, expected[1])


def test_two_threads_at_once():
    """Calls from two threads on streams of their own do not disturb each other."""
    import threading

    rng = np.random.default_rng(6)
    draws = [Draw(cb.BFLOAT16, scores_of(rng, 20, 30000, 0), rng.random(20)), Draw(cb.FLOAT32, scores_of(rng, 20, 9000, 0), rng.random(20))]
    expected = [d.indexes.clone() for d in draws]
    torch.cuda.synchronize()
    failed = []

    def work(d, e):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                d.indexes.fill_(-1)
                d()
                s.synchronize()
                if not torch.equal(d.indexes, e):
                    failed.append(d.kind)

    threads = [threading.Thread(target=work, args=a) for a in zip(draws, expected)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
