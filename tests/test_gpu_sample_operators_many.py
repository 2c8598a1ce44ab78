"""A class drawn from rows of very many classes, and from many long rows, against the definition in 64 bits and more. Needs an MI355X."""
import numpy as np
import pytest
import torch

import catboost_amd as cb

pytestmark = pytest.mark.gpu

TYPES = {cb.FLOAT64: torch.float64, cb.FLOAT32: torch.float32, cb.FLOAT16: torch.float16, cb.BFLOAT16: torch.bfloat16}
NAMES = {cb.FLOAT64: "f64", cb.FLOAT32: "f32", cb.FLOAT16: "f16", cb.BFLOAT16: "bf16"}
ALL = pytest.mark.parametrize("kind", list(TYPES), ids=NAMES.get)


def draw(kind, scores, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    rows, classes = scores.shape
    parts = [None if a is None else torch.as_tensor(np.asarray(a, t)).cuda()
             for a, t in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    numbers = torch.as_tensor(np.asarray(uniform, np.float32)).cuda()
    indexes = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((rows,), -7, dtype=torch.float64 if kind == cb.FLOAT64 else torch.float32, device="cuda")
    cb.sample_classes(kind, rows, classes, scores.data_ptr(), scores.stride(0), cb.sampling(*(0 if t is None else t.data_ptr() for t in parts)),
                      numbers.data_ptr(), indexes.data_ptr(), weights.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return indexes.cpu().numpy(), weights.cpu().to(torch.float64).numpy()


class Row:
    """A row in its order: best score first, of equal ones the lowest class."""

    def __init__(self, scores, temperature=1.0):
        z, order = torch.sort(scores.to(torch.float64), descending=True, stable=True)
        z = z.cpu().numpy().astype(np.longdouble)
        self.order, self.e = order.cpu().numpy(), np.exp((z - z[0]) / np.longdouble(temperature))

    def share(self, index, top_k=0, top_p=1.0, min_p=0.0):
        """By the definition: the sums before and up to the class, its own, and that of the class where top_p ends, as shares of the sum of
        what takes part."""
        e = self.e.copy()
        if top_k > 0:
            e[top_k:] = 0
        sums = np.cumsum(e)
        keep, edge = e >= np.longdouble(min_p), 0
        if top_p < 1:
            keep[1:] &= sums[:-1] < np.longdouble(top_p) * sums[-1]
            edge = e[min(int(np.searchsorted(sums, np.longdouble(top_p) * sums[-1])), len(e) - 1)]
        total = e[keep].sum()
        at = int(np.flatnonzero(self.order == index)[0])
        return (sums[at] - e[at]) / total, sums[at] / total, e[at] / total, edge / total


# Sums of whole numbers are off by under 2^-28 of a row's sum: once for a class's place and once for the whole. Where that moves the end of top_p
# by a class, the whole is off by that class's share too.
OFF = 2.0 ** -27


def check(row, index, weight, uniform, **limits):
    before, upto, share, edge = row.share(index, **limits)
    off = OFF + float(edge)
    assert before - off <= uniform <= upto + off, (index, float(before), float(upto))
    assert abs(weight - share) <= off * share + 2.0 ** -24 * share, (index, weight, float(share))


# Classes whose weights are small, but not all of them together: 2^-19 to 2^-25.5 of the best one's
@ALL
@pytest.mark.parametrize("classes,low,high", [(1 << 22, -29.0, -29.0), (1 << 22, -31.0, -28.0), (1_000_003, -33.0, -30.5), ((1 << 24) - 5, -31.0, -27.0)],
                         ids=["alike", "4M", "1M", "16M"])
def test_many_classes_of_small_weights(kind, classes, low, high):
    rng = np.random.default_rng(classes & 1023)
    rows, best = 4, classes // 3
    x = rng.uniform(low, high, classes)
    x[best] = 0
    scores = torch.from_numpy(x).cuda().to(TYPES[kind])[None].repeat(rows, 1)
    uniform = [1 - 2.0 ** -24, 1 - 2.0 ** -22, 1.0, 0.5]
    limits = dict(top_k=[0, classes // 2, 0, 0], top_p=[1, 1, 1, 0.75], min_p=[0, 0, 2.0 ** -46, 0])
    indexes, weights = draw(kind, scores, uniform, **limits)
    row = Row(scores[0])
    for r in range(rows):
        given = {k: v[r] for k, v in limits.items()}
        if r < 3:
            check(row, indexes[r], weights[r], uniform[r], **given)
        else:
            assert indexes[r] == best and weights[r] == 1


@ALL
def test_many_classes_of_all_weights(kind):
    """Scores from the best one's down to those that weigh nothing, at every limit."""
    rng = np.random.default_rng(7)
    rows, classes = 6, 700_001
    scores = torch.from_numpy(rng.standard_normal((rows, classes)) * np.array([[0.01], [1], [3], [6], [3], [3]])).cuda().to(TYPES[kind])
    uniform = rng.random(rows).astype(np.float32)
    temperature = np.array([1, 0.5, 1, 2, 1, 0.7], np.float32)
    limits = dict(top_k=[0, 1000, 0, 600_000, 50, 0], top_p=[1, 1, 0.9, 0.99, 0.5, 1], min_p=[0, 0, 0, 0, 0, 1e-3])
    limits = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in limits.items()}
    indexes, weights = draw(kind, scores, uniform, temperature, **limits)
    for r in range(rows):
        check(Row(scores[r], temperature[r]), indexes[r], weights[r], uniform[r], **{k: v[r] for k, v in limits.items()})


# ---- more long rows than compute units

def chunked(kind, scores, uniform, limits, step):
    """The same rows, some at a time."""
    got = [draw(kind, scores[b:b + step], uniform[b:b + step], **{k: v[b:b + step] for k, v in limits.items()}) for b in range(0, scores.shape[0], step)]
    return np.concatenate([g[0] for g in got]), np.concatenate([g[1] for g in got])


@ALL
@pytest.mark.parametrize("rows,classes", [(257, 9001), (300, 4097), (1000, 6000)])
def test_many_long_rows(kind, rows, classes):
    """Every limit, masked classes, rows of infinities, of NaN, of nothing, of equals and of the best class alone, at any address."""
    rng = np.random.default_rng(classes)
    x = rng.standard_normal((rows, classes)) * rng.uniform(0.1, 5, (rows, 1))
    x[rng.random((rows, classes)) < 0.2] = -np.inf
    x[rng.random((rows, classes)) < 0.001] = np.nan
    x[5::40] = np.round(x[5::40])  # more equals than are listed
    x[6::40] = 1.5
    x[7::40] = -np.inf
    x[8::40] = np.nan
    x[9::40, 7::50] = np.inf
    x[10::40] = np.where(np.isfinite(x[10::40]), x[10::40] * 1e-4, x[10::40])  # all in the first step
    wide = torch.full((rows, classes + 3), float("nan"), dtype=TYPES[kind], device="cuda")
    scores = wide[:, :classes]
    scores.copy_(torch.from_numpy(x))
    uniform = rng.random(rows).astype(np.float32)
    limits = dict(temperature=np.where(rng.random(rows) < 0.1, 0, rng.uniform(0.3, 2, rows)).astype(np.float32),
                  top_k=np.where(rng.random(rows) < 0.5, 0, rng.integers(1, classes, rows)).astype(np.int32),
                  top_p=np.where(rng.random(rows) < 0.5, 1, rng.random(rows)).astype(np.float32),
                  min_p=np.where(rng.random(rows) < 0.7, 0, 10.0 ** -rng.uniform(0, 5, rows)).astype(np.float32))
    indexes, weights = draw(kind, scores, uniform, **limits)
    for step in (rows, 256, 100):
        again = chunked(kind, scores, uniform, limits, step)
        assert np.array_equal(indexes, again[0]) and np.array_equal(weights, again[1])
    for r in range(rows):
        row = scores[r].to(torch.float64)
        row = torch.where(torch.isnan(row), -float("inf"), row)
        best, at = row.max().item(), int(row.argmax())
        if best == -np.inf:
            assert indexes[r] == -1 and weights[r] == 0
        elif not limits["temperature"][r] > 0:
            assert row[indexes[r]] == best and indexes[r] == int(torch.nonzero(row == best)[0, 0]) and weights[r] == 1, at
        elif best == np.inf:
            assert row[indexes[r]] == np.inf
        else:
            check(Row(row, limits["temperature"][r]), indexes[r], weights[r], uniform[r], **{k: v[r] for k, v in limits.items() if k != "temperature"})
