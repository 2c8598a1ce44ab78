"""Operators on scores and on routed rows against their definitions in 64 bits and more. Needs an MI355X.

Tolerances count roundings of half a step: U is half a step of what a kernel computes in (2^-24, 2^-53 for 64-bit values),
HALF half a step of the type that it stores (with half of the smallest subnormal where values are that small)."""
import ctypes

import numpy as np
import pytest
import torch

import catboost_amd as cb

pytestmark = pytest.mark.gpu

TYPES = {cb.FLOAT64: torch.float64, cb.FLOAT32: torch.float32, cb.FLOAT16: torch.float16, cb.BFLOAT16: torch.bfloat16}
NAMES = {cb.FLOAT64: "f64", cb.FLOAT32: "f32", cb.FLOAT16: "f16", cb.BFLOAT16: "bf16"}
ALL = pytest.mark.parametrize("kind", list(TYPES), ids=NAMES.get)
HALF = {cb.FLOAT64: 2.0 ** -53, cb.FLOAT32: 2.0 ** -24, cb.FLOAT16: 2.0 ** -11, cb.BFLOAT16: 2.0 ** -8}
TINY = {cb.FLOAT64: 0.0, cb.FLOAT32: 2.0 ** -150, cb.FLOAT16: 2.0 ** -25, cb.BFLOAT16: 2.0 ** -134}


def u(kind):
    return 2.0 ** -53 if kind == cb.FLOAT64 else 2.0 ** -24


def acc(kind):
    return torch.float64 if kind == cb.FLOAT64 else torch.float32


def ptr(t):
    return 0 if t is None else t.data_ptr()


def dev(a, dtype=None):
    return None if a is None else torch.as_tensor(np.ascontiguousarray(a)).to("cuda", dtype)


def table(values, kind, pad=0, fill=7.0):
    """The values rounded to the type, as the first columns of a wider table of `fill`."""
    rows, width = values.shape
    wide = torch.full((rows, width + pad), fill, dtype=TYPES[kind], device="cuda")
    wide[:, :width] = torch.from_numpy(values).cuda().to(TYPES[kind])
    return wide[:, :width]


def exactly(t):
    return t.detach().to(torch.float64).cpu().numpy().astype(np.longdouble)


def compare(got, expected, bound, kind):
    """|got - expected| <= bound + one rounding to the type; infinities and NaN at the same places."""
    got, expected = np.asarray(got, np.longdouble), np.asarray(expected, np.longdouble)
    assert np.array_equal(np.isnan(got), np.isnan(expected))
    finite = np.isfinite(expected)
    assert np.array_equal(got[~finite & ~np.isnan(expected)], expected[~finite & ~np.isnan(expected)])
    bound = np.broadcast_to(bound, expected.shape)[finite]
    off = np.abs(got[finite] - expected[finite])
    allowed = bound + HALF[kind] * (np.abs(expected[finite]) + bound) + TINY[kind]
    worst = np.max(off - allowed, initial=-1.0)
    assert worst <= 0, "off by %g where %g is allowed" % (off[np.argmax(off - allowed)], allowed[np.argmax(off - allowed)])


# ---------------------------------------------------------------- penalties, biases, masks

def history(rng, rows, classes, most, outside=True):
    lengths = rng.integers(0, most + 1, rows)
    lengths[rng.random(rows) < 0.2] = 0
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = (classes * rng.random(int(offsets[-1])) ** 3).astype(np.int32)
    if outside and len(ids):
        ids[rng.random(len(ids)) < 0.05] = -1
        ids[rng.random(len(ids)) < 0.03] = classes
        ids[rng.random(len(ids)) < 0.02] = np.iinfo(np.int32).min
    return offsets, ids


def adjusted(x, p):
    """The definition, row by row; and the largest of the values on the way to each result."""
    rows, classes = x.shape
    x, big = x.copy(), np.abs(np.where(np.isfinite(x), x, 0))
    for r in range(rows):
        if p.get("offsets") is not None:
            entries = p["ids"][p["offsets"][r]:p["offsets"][r + 1]]
            prompt = p["prompts"][r] if p.get("prompts") is not None else 0
            given = set(int(c) for c in entries if 0 <= c < classes)
            counts = {}
            for c in entries[max(prompt, 0):]:
                if 0 <= c < classes:
                    counts[int(c)] = counts.get(int(c), 0) + 1
            for c in given:
                v = x[r, c]
                if p.get("repetition") is not None:
                    rep = np.longdouble(p["repetition"][r])
                    v = v / rep if v > 0 else v * rep
                    big[r, c] = max(big[r, c], abs(v) if np.isfinite(v) else 0)
                n = counts.get(c, 0)
                if n and p.get("frequency") is not None:
                    v = v - np.longdouble(p["frequency"][r]) * n
                    big[r, c] = max(big[r, c], abs(v) if np.isfinite(v) else 0) + abs(np.longdouble(p["frequency"][r]) * n)
                if n and p.get("presence") is not None:
                    v = v - np.longdouble(p["presence"][r])
                    big[r, c] = max(big[r, c], abs(v) if np.isfinite(v) else 0)
                x[r, c] = v
        if p.get("class_bias") is not None:
            x[r] += p["class_bias"][r if p["class_bias"].shape[0] > 1 else 0].astype(np.longdouble)
            big[r] = np.maximum(big[r], np.abs(np.where(np.isfinite(x[r]), x[r], 0)))
        if p.get("bias_offsets") is not None:
            wanted = {}
            for e in range(p["bias_offsets"][r], p["bias_offsets"][r + 1]):
                wanted[int(p["bias_classes"][e])] = np.longdouble(p["bias_values"][e])
            for c, v in wanted.items():
                if 0 <= c < classes:
                    x[r, c] += v
                    big[r, c] = max(big[r, c], abs(x[r, c]) if np.isfinite(x[r, c]) else 0)
        if p.get("allowed") is not None:
            m = p["allowed_rows"][r] if p.get("allowed_rows") is not None else r
            if 0 <= m < p["allowed"].shape[0]:
                c = np.arange(classes)
                x[r, (p["allowed"][m, c >> 5] >> (c & 31).astype(np.uint32)) & 1 == 0] = -np.inf
    return x, big


class Adjustment:
    """The parts on the GPU, and the struct that points at them."""

    def __init__(self, p):
        d = {k: dev(v) for k, v in p.items() if v is not None and k != "allowed"}
        if p.get("allowed") is not None:
            d["allowed"] = dev(p["allowed"].view(np.int32))
        self.keep = d
        g = d.get
        self.struct = cb.score_adjustment(
            history_offsets_ptr=ptr(g("offsets")), history_ptr=ptr(g("ids")), history_count=len(p["ids"]) if "ids" in p else 0,
            prompt_lengths_ptr=ptr(g("prompts")), repetition_ptr=ptr(g("repetition")), frequency_ptr=ptr(g("frequency")), presence_ptr=ptr(g("presence")),
            class_bias_ptr=ptr(g("class_bias")), class_bias_stride=p["class_bias"].shape[1] if p.get("class_bias") is not None and p["class_bias"].shape[0] > 1 else 0,
            bias_offsets_ptr=ptr(g("bias_offsets")), bias_classes_ptr=ptr(g("bias_classes")), bias_values_ptr=ptr(g("bias_values")),
            bias_count=len(p["bias_classes"]) if "bias_classes" in p else 0, allowed_ptr=ptr(g("allowed")),
            allowed_stride=p["allowed"].shape[1] if p.get("allowed") is not None else 0,
            allowed_count=p["allowed"].shape[0] if p.get("allowed") is not None else 0, allowed_rows_ptr=ptr(g("allowed_rows")))


def parts(rng, rows, classes, which, most=40):
    p = {}
    if "h" in which:
        p["offsets"], p["ids"] = history(rng, rows, classes, most)
        if "p" in which:
            p["prompts"] = rng.integers(0, most, rows).astype(np.int32)
        if "r" in which:
            p["repetition"] = (1 + rng.random(rows)).astype(np.float32)
        if "f" in which:
            p["frequency"] = rng.normal(size=rows).astype(np.float32)
        if "s" in which:
            p["presence"] = rng.normal(size=rows).astype(np.float32)
    if "c" in which:
        p["class_bias"] = rng.normal(size=(1, classes)).astype(np.float32)
    if "C" in which:
        p["class_bias"] = rng.normal(size=(max(rows, 2), classes)).astype(np.float32)[:max(rows, 2)]
    if "b" in which:
        p["bias_offsets"], p["bias_classes"] = history(rng, rows, classes, 6)
        p["bias_values"] = (rng.normal(size=len(p["bias_classes"])) * 10).astype(np.float32)
    if "m" in which:
        masks = rows if "M" not in which else 3
        p["allowed"] = rng.integers(0, 1 << 32, (masks, (classes + 31) // 32), dtype=np.uint32)
        p["allowed"][rng.random(masks) < 0.3] = 0  # nothing left
        if "M" in which:
            p["allowed_rows"] = rng.integers(-1, 5, rows).astype(np.int32)  # 3 and 4: behind the last mask
    return p


SHAPES = [(1, 1, 0), (3, 2, 1), (701, 10, 0), (1300, 10, 3), (5, 33, 0), (2, 4095, 0), (3, 4096, 0), (2, 4097, 5), (4, 20003, 0), (2, 70001, 7), (1, 131072, 0)]


@ALL
@pytest.mark.parametrize("rows,classes,pad", SHAPES)
@pytest.mark.parametrize("which", ["", "hprfs", "hfs", "hr", "cb", "C", "mM", "m", "hprfscbmM"])
def test_adjust_scores(kind, rows, classes, pad, which):
    rng = np.random.default_rng(rows * 1000 + classes + len(which))
    scores = table(rng.normal(size=(rows, classes)) * 4, kind, pad)
    p = parts(rng, rows, classes, which)
    a = Adjustment(p)
    wide = torch.full((rows, classes + pad + 2), 3.0, dtype=TYPES[kind], device="cuda")
    result = wide[:, :classes]
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), scores.stride(0), a.struct, result.data_ptr(), result.stride(0))
    expected, big = adjusted(exactly(scores), p)
    # at most six roundings on the way, each of a value of at most `big`
    compare(exactly(result), expected, 6.01 * u(kind) * big, kind)
    assert bool((wide[:, classes:] == 3.0).all())


@ALL
@pytest.mark.parametrize("rows,classes,most", [(40, 3, 5), (2000, 7, 2), (700, 12, 30), (300, 100, 3), (30, 2047, 900), (8, 4097, 20), (600, 4500, 4), (513, 8200, 40),
                                               (270, 16400, 10), (90, 100003, 60_000)])
def test_adjust_scores_in_place(kind, rows, classes, most):
    """Every length of slices and tiles, histories of every length beside them, a result where the scores were."""
    rng = np.random.default_rng(rows + classes)
    scores = table(rng.normal(size=(rows, classes)) * 4, kind)
    if rows * classes > 1_000_000:  # a few rows with what the others lack keep the definition quick
        p = parts(rng, rows, classes, "hprfsbmM", 1)
        few = np.concatenate([[0], np.cumsum(np.where(np.arange(rows) % 29 == 3, rng.integers(most // 2, most + 1, rows), 0))]).astype(np.int64)
        p["offsets"], p["ids"] = few, (classes * rng.random(int(few[-1])) ** 3).astype(np.int32)
        p["prompts"] = rng.integers(0, most, rows).astype(np.int32)
    else:
        p = parts(rng, rows, classes, "hprfscbmM", most)
    a = Adjustment(p)
    before = exactly(scores)
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), classes, a.struct, scores.data_ptr(), classes)
    expected, big = adjusted(before, p)
    compare(exactly(scores), expected, 6.01 * u(kind) * big, kind)


@ALL
@pytest.mark.parametrize("classes,pad", [(517, 3), (1024, 0), (2049, 0), (4099, 3)])
def test_adjust_scores_of_slices_in_plenty(kind, classes, pad):
    """Rows enough for the smaller workgroups, some with a history longer than a slice, some with more biases than names."""
    rng = np.random.default_rng(classes + pad)
    rows = 1030
    scores = table(rng.normal(size=(rows, classes)) * 4, kind, pad)
    p = parts(rng, rows, classes, "hprfscmM", 5)
    few = np.where(np.arange(rows) % 97 == 5, rng.integers(1025, 1400, rows), rng.integers(0, 4, rows))
    p["bias_offsets"] = np.concatenate([[0], np.cumsum(few)]).astype(np.int64)
    p["bias_classes"] = rng.integers(-1, classes + 1, int(p["bias_offsets"][-1])).astype(np.int32)
    p["bias_values"] = rng.normal(size=len(p["bias_classes"])).astype(np.float32)
    long = np.where(np.arange(rows) % 101 == 7, rng.integers(classes, 6000, rows), np.diff(p["offsets"]))
    p["offsets"] = np.concatenate([[0], np.cumsum(long)]).astype(np.int64)
    p["ids"] = (classes * rng.random(int(p["offsets"][-1])) ** 3).astype(np.int32)
    a = Adjustment(p)
    wide = torch.full((rows, classes + pad + 2), 3.0, dtype=TYPES[kind], device="cuda")
    result = wide[:, :classes]
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), scores.stride(0), a.struct, result.data_ptr(), result.stride(0))
    expected, big = adjusted(exactly(scores), p)
    compare(exactly(result), expected, 6.01 * u(kind) * big, kind)
    assert bool((wide[:, classes:] == 3.0).all())


@ALL
def test_adjust_scores_of_slices_in_plenty_with_histories_longer_than_they_are(kind):
    """As many threads as a slice may have, more than it has scores for: they look through the histories."""
    rng = np.random.default_rng(3)
    rows, classes = 1025, 517
    scores = table(rng.normal(size=(rows, classes)) * 4, kind, 1)
    p = parts(rng, rows, classes, "hprfsbm", 700)
    assert len(p["ids"]) > rows * 272
    a = Adjustment(p)
    result = torch.empty(rows, classes, dtype=TYPES[kind], device="cuda")
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), scores.stride(0), a.struct, result.data_ptr(), classes)
    expected, big = adjusted(exactly(scores), p)
    compare(exactly(result), expected, 6.01 * u(kind) * big, kind)


def test_adjust_scores_of_the_most_classes():
    """One row of 2^31 - 1: what is adjusted is at both ends, in the middle and around slices; everything else stays."""
    classes = (1 << 31) - 1
    scores = torch.empty(classes, dtype=torch.float16, device="cuda")
    for begin in range(0, classes, 1 << 28):
        scores[begin:begin + (1 << 28)].normal_()
    at = np.array([0, 1, 16383, 16384, 1 << 24, (1 << 30) + 5, classes - 16384, classes - 2, classes - 1])
    ids = np.concatenate([at, at[::2], [-1, np.iinfo(np.int32).min]]).astype(np.int32)
    p = dict(offsets=np.array([0, len(ids)]), ids=ids, frequency=np.array([0.5], np.float32), bias_offsets=np.array([0, 3]),
             bias_classes=np.array([classes - 1, 7, 1 << 30], np.int32), bias_values=np.array([4, 2, 1], np.float32),
             allowed=np.full((1, (classes + 31) // 32), 0xffffffff, np.uint32))
    off = np.array([5, 1 << 29, classes - 3])
    for c in off:
        p["allowed"][0, c >> 5] &= np.uint32(0xffffffff ^ 1 << (c & 31))
    a = Adjustment(p)
    result = torch.full_like(scores, 9.0)
    cb.adjust_scores(cb.FLOAT16, 1, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    changed = np.concatenate([at, [7, 1 << 30], off])
    expected = scores[torch.from_numpy(changed).cuda()].float().cpu().numpy()
    expected[:len(at)] -= 0.5 * (1 + (np.arange(len(at)) % 2 == 0))
    expected[len(at) - 1] += 4
    expected[len(at):len(at) + 2] += [2, 1]
    expected[len(at) + 2:] = -np.inf
    where = torch.from_numpy(changed).cuda()
    np.testing.assert_array_equal(result[where].float().cpu().numpy(), torch.from_numpy(expected).half().float().numpy())
    result[where] = scores[where]
    assert torch.equal(result, scores)


@pytest.mark.parametrize("classes", [10, 3000, 50_000])
def test_adjust_scores_with_many_biases(classes):
    """More bias entries than threads, most of them overridden by later ones, with values whose bits are small numbers."""
    rng = np.random.default_rng(classes)
    rows = 5
    lengths = np.array([20_000, 0, 1, 7000, 300])
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = rng.integers(0, classes, offsets[-1]).astype(np.int32)
    values = rng.integers(1, 5000, offsets[-1]).astype(np.int32).view(np.float32)  # below the smallest normal number
    values[::2] = rng.normal(size=len(values[::2]))
    scores = torch.zeros(rows, classes, device="cuda")
    a = Adjustment(dict(bias_offsets=offsets, bias_classes=ids, bias_values=values))
    cb.adjust_scores(cb.FLOAT32, rows, classes, scores.data_ptr(), classes, a.struct, scores.data_ptr(), classes)
    expected = np.zeros((rows, classes), np.float32)
    for r in range(rows):
        for e in range(offsets[r], offsets[r + 1]):
            expected[r, ids[e]] = values[e]
    np.testing.assert_array_equal(scores.cpu().numpy().view(np.int32), expected.view(np.int32))


@ALL
@pytest.mark.parametrize("classes", [2048, 5003, 40_001])
@pytest.mark.parametrize("with_history", [False, True])
def test_adjust_scores_with_named_biases_or_a_table(kind, classes, with_history):
    """Up to 1024 biases of a row are named: rows around that many, classes next to each other and the same ones again."""
    rng = np.random.default_rng(classes)
    lengths = np.array([64, 1025, 0, 1023, 1, 1024, 200, 2])
    rows = len(lengths)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = (rng.choice([0, 1000, 2040, classes - 12], offsets[-1]) + rng.integers(0, 12, offsets[-1])).astype(np.int32)
    ids[rng.random(len(ids)) < 0.1] = -1
    ids[rng.random(len(ids)) < 0.1] = classes
    p = dict(bias_offsets=offsets, bias_classes=ids, bias_values=(rng.normal(size=offsets[-1]) * 4).astype(np.float32))
    if with_history:
        p.update(offsets=np.arange(rows + 1) * 30, ids=rng.integers(0, classes, 30 * rows).astype(np.int32), presence=np.full(rows, 0.5, np.float32))
    scores = table(rng.normal(size=(rows, classes)), kind, classes % 2)
    a = Adjustment(p)
    result = torch.empty(rows, classes, dtype=TYPES[kind], device="cuda")
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), scores.stride(0), a.struct, result.data_ptr(), classes)
    expected, size = adjusted(exactly(scores), p)
    compare(exactly(result), expected, 8 * u(kind) * size, kind)


@ALL
@pytest.mark.parametrize("classes", [10, 100, 5003])
@pytest.mark.parametrize("with_history", [False, True])
def test_adjust_scores_of_a_row_is_the_same_beside_other_rows(kind, classes, with_history):
    """Bit for bit, zeros' signs too: classes without a bias keep -0, whether the rows around have biases enough for a table or not."""
    rng = np.random.default_rng(classes)
    lengths = np.array([3, 1100, 0, 2, 5])  # more than 1024: of the second row, and of a tile that has it
    rows = len(lengths)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = rng.integers(0, classes // 2, offsets[-1]).astype(np.int32)  # the other half has none
    values = rng.normal(size=offsets[-1]).astype(np.float32)
    values[::3], values[1::7] = 0.0, -0.0
    x = rng.normal(size=(rows, classes))
    x[rng.random((rows, classes)) < 0.5] = -0.0
    scores = table(x, kind)

    def run(first, n, biases):
        p = dict(bias_offsets=offsets[first:first + n + 1], bias_classes=ids[:biases], bias_values=values[:biases])
        if with_history:
            p.update(offsets=np.arange(first, first + n + 1) * 4, ids=(np.arange(4 * rows) % classes).astype(np.int32), presence=np.zeros(n, np.float32))
        a = Adjustment(p)
        result = torch.empty(n, classes, dtype=TYPES[kind], device="cuda")
        cb.adjust_scores(kind, n, classes, scores[first:].data_ptr(), classes, a.struct, result.data_ptr(), classes)
        return exactly(result)

    together = run(0, rows, offsets[-1])
    for r in range(rows):
        alone = run(r, 1, offsets[-1])[0]
        assert np.array_equal(alone, together[r]) and np.array_equal(np.signbit(alone), np.signbit(together[r])), r
    untouched = np.signbit(exactly(scores)[:, classes // 2:])
    assert np.array_equal(np.signbit(together[:, classes // 2:]), untouched)


@pytest.mark.parametrize("classes", [60, 5000])
def test_adjust_scores_with_a_history_too_long_for_named_biases(classes):
    """Some 2^19 entries, the most that leave room for names, and one more; counted exactly, with a few biases beside them."""
    rng = np.random.default_rng(4)
    lengths = np.array([(1 << 19) - 1, 1 << 19, 3])
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = rng.integers(0, classes, offsets[-1]).astype(np.int32)
    ids[:(1 << 19) - 1] = 7  # the largest count that a word with a name holds
    bias_ids = np.array([7, 8, 7, classes - 1, 8, 7, 0, 7], np.int32)
    values = np.array([9, 9, 1 / 4, -1, 2, 1 / 2, 3, 1], np.float32)
    p = dict(offsets=offsets, ids=ids, frequency=np.full(3, 2.0 ** -6, np.float32), bias_offsets=np.array([0, 3, 6, 8]), bias_classes=bias_ids, bias_values=values)
    a = Adjustment(p)
    scores = torch.zeros(3, classes, device="cuda")
    result = torch.empty_like(scores)
    cb.adjust_scores(cb.FLOAT32, 3, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    expected = np.zeros((3, classes))
    for r in range(3):
        expected[r] -= np.bincount(ids[offsets[r]:offsets[r + 1]], minlength=classes) * 2.0 ** -6
        for c in {7, 8, classes - 1, 0}:
            at = [e for e in range(p["bias_offsets"][r], p["bias_offsets"][r + 1]) if bias_ids[e] == c]
            expected[r, c] += values[at[-1]] if at else 0
    np.testing.assert_array_equal(result.cpu().numpy(), expected.astype(np.float32))  # every sum has few enough bits
    result.fill_(5)
    cb.adjust_scores(cb.FLOAT32, 1, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    np.testing.assert_array_equal(result[:1].cpu().numpy(), expected[:1].astype(np.float32))


@ALL
@pytest.mark.parametrize("rows,classes,most,biases", [(3000, 1, 3, 0), (3000, 1, 3, 3), (700, 2, 9, 4), (64, 40, 2, 3), (64, 40, 30, 30), (5, 7, 700, 300), (300, 9, 40, 2), (1, 10, 5000, 900),
                                                      (1, 10, 30, 2000), (33, 64, 65, 33)])
def test_adjust_scores_of_short_rows_with_histories_and_biases_of_all_lengths(kind, rows, classes, most, biases):
    """A row's own lanes count up to four entries each, all threads of the tile the others; more biases than names."""
    rng = np.random.default_rng(rows + classes + most)
    p = parts(rng, rows, classes, "hpfrs", most)
    if biases:
        p["bias_offsets"], p["bias_classes"] = history(rng, rows, classes, biases)
        p["bias_values"] = rng.normal(size=len(p["bias_classes"])).astype(np.float32)
    scores = table(rng.normal(size=(rows, classes)), kind)
    a = Adjustment(p)
    result = torch.empty_like(scores)
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    expected, big = adjusted(exactly(scores), p)
    compare(exactly(result), expected, 6.01 * u(kind) * big, kind)


@ALL
def test_adjust_scores_of_infinite_and_undefined_values(kind):
    rng = np.random.default_rng(5)
    rows, classes = 6, 5001
    x = rng.normal(size=(rows, classes))
    low = float(torch.finfo(TYPES[kind]).min)
    for value in (np.inf, -np.inf, np.nan, low, -low, 0.0, -0.0):
        x[rng.random((rows, classes)) < 0.05] = value
    scores = table(x, kind)
    p = parts(rng, rows, classes, "hprfmM", 3000)
    p["repetition"][:] = 1.0  # the largest value stays in range
    a = Adjustment(p)
    result = torch.empty_like(scores)
    cb.adjust_scores(kind, rows, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    expected, big = adjusted(exactly(scores), p)
    got = exactly(result)
    # values next to the type's largest may round to it or to infinity: both are compared at the type's largest
    most = np.longdouble(torch.finfo(TYPES[kind]).max)
    near = np.isfinite(expected) & (np.abs(expected) >= most * (1 - HALF[kind] * 4))
    assert np.array_equal(np.sign(got[near]), np.sign(expected[near])) and bool((np.abs(got[near]) >= most * (1 - HALF[kind] * 4)).all())
    compare(got[~near], expected[~near], 6.01 * u(kind) * big[~near], kind)


def test_adjust_scores_counts_and_last_biases():
    """Many times the same class, in one row and in rows next to each other; the last of equal biases counts."""
    rows, classes = 3, 100
    lengths = [70_000, 0, 65_536]
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    ids = np.full(offsets[-1], 99, np.int32)
    ids[::2] = 0
    bias_classes = np.tile(np.array([5, 6, 5], np.int32), 1000)
    p = dict(offsets=offsets, ids=ids, prompts=np.array([10, 5, 65_536], np.int32), frequency=np.ones(rows, np.float32),
             bias_offsets=np.array([0, 3000, 3000, 3000]), bias_classes=bias_classes, bias_values=np.arange(3000, dtype=np.float32))
    scores = torch.zeros(rows, classes, device="cuda")
    a = Adjustment(p)
    cb.adjust_scores(cb.FLOAT32, rows, classes, scores.data_ptr(), classes, a.struct, scores.data_ptr(), classes)  # in place
    expected = np.zeros((rows, classes))
    expected[0, 0], expected[0, 99] = -(35_000 - 5), -(35_000 - 5)
    expected[0, 5], expected[0, 6] = 2999, 2998
    np.testing.assert_array_equal(scores.cpu().numpy(), expected)


def test_adjust_scores_of_offsets_that_lead_nowhere():
    """Entries behind HistoryCount and BiasCount are not read, whatever the offsets say."""
    rows, classes = 2, 40
    p = dict(offsets=np.array([-5, 3, 1 << 40]), ids=np.array([1, 2, 3, 4], np.int32), presence=np.ones(rows, np.float32),
             bias_offsets=np.array([0, 1, 1 << 50]), bias_classes=np.array([7, 8], np.int32), bias_values=np.array([1, 2], np.float32))
    scores = torch.zeros(rows, classes, device="cuda")
    a = Adjustment(p)
    cb.adjust_scores(cb.FLOAT32, rows, classes, scores.data_ptr(), classes, a.struct, scores.data_ptr(), classes)
    expected = np.zeros((rows, classes))
    expected[0, [1, 2, 3]] = -1
    expected[1, 4] = -1
    expected[0, 7], expected[1, 8] = 1, 2
    np.testing.assert_array_equal(scores.cpu().numpy(), expected)


# ---------------------------------------------------------------- the best classes

def best(x, count, among):
    rows, classes = x.shape
    index = np.full((rows, count), -1, np.int32)
    weight = np.zeros((rows, count), np.longdouble)
    p = np.zeros((rows, classes), np.longdouble)
    for r in range(rows):
        usable = [c for c in range(classes) if x[r, c] > -np.inf]  # (not for NaN)
        order = sorted(usable, key=lambda c: (-x[r, c], c))[:count]
        over = order if among else usable
        if not usable:
            continue
        most = x[r, order[0]]
        e = {c: np.longdouble(1) if x[r, c] == most else np.exp(x[r, c] - most) for c in over}
        total = sum(e.values())
        for c in over:
            p[r, c] = e[c] / total
        index[r, :len(order)] = order
        weight[r, :len(order)] = [p[r, c] for c in order]
    return index, weight, p


def spread(x):
    finite = x[np.isfinite(x)]
    return float(finite.max() - finite.min()) if finite.size else 0.0


def weight_error(kind, x):
    """Relative: the difference to the largest is off by U times itself, the exponential by two, the sum by one for each of at
    most `classes` additions; numerator and total alike, and a division."""
    return u(kind) * (2 * (spread(x) + 2) + x.shape[1] + 2)


@ALL
@pytest.mark.parametrize("rows,classes,count,pad", [
    (1, 1, 1, 0), (5, 2, 2, 0), (9, 3, 8, 0), (6, 20, 32, 1), (70, 3, 4, 1), (1001, 10, 3, 0), (300, 10, 10, 2), (9, 16, 8, 0), (9, 17, 8, 0), (130, 33, 32, 0), (7, 64, 2, 0), (65, 65, 8, 0), (33, 128, 8, 0),
    (6, 129, 5, 0), (11, 256, 6, 0), (4, 300, 8, 3), (3, 512, 1, 0), (5, 513, 9, 0), (2, 1023, 32, 1), (3, 1024, 16, 0)])
@pytest.mark.parametrize("among", [False, True])
def test_select_top(kind, rows, classes, count, pad, among):
    rng = np.random.default_rng(classes * 100 + count)
    x = rng.normal(size=(rows, classes)) * 3
    x[rng.random((rows, classes)) < 0.2] = 1.5  # equal ones
    x[rng.random((rows, classes)) < 0.1] = -np.inf
    x[rng.random((rows, classes)) < 0.02] = np.nan
    if rows > 4:
        x[1] = -np.inf
        x[2, 1:] = np.nan
        x[3] = float(torch.finfo(TYPES[kind]).min)  # the lowest value is a score like any other
    scores = table(x, kind, pad)
    indexes = torch.full((rows * count + 1,), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((rows * count + 1,), 77, dtype=acc(kind), device="cuda")
    cb.select_top(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr())
    exact = exactly(scores)
    index, weight, p = best(exact, count, among)
    np.testing.assert_array_equal(indexes[:-1].cpu().numpy().reshape(rows, count), index)
    plain = np.delete(exact, 3, 0) if rows > 4 else exact
    error = weight_error(kind, plain)
    # weights below the smallest normal number may be lost
    compare(exactly(weights[:-1]).reshape(rows, count), weight, error * weight + 2.0 ** -125, kind if kind == cb.FLOAT64 else cb.FLOAT32)
    assert int(indexes[-1]) == 77 and float(weights[-1]) == 77

    g = rng.normal(size=(rows, count))
    gradients = torch.from_numpy(g).cuda().to(acc(kind))
    wide = torch.full((rows, classes + pad + 1), 5.0, dtype=TYPES[kind], device="cuda")
    cb.select_top_backward(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr(),
                           gradients.data_ptr(), wide.data_ptr(), wide.stride(0))
    g = np.where(index >= 0, exactly(gradients), 0)
    mean = (g * weight).sum(1, keepdims=True)
    sizes = (np.abs(g) * weight).sum(1, keepdims=True)
    expected, bound = -p * mean, np.zeros_like(p)
    # the mean is a sum of `count` products of weights that are off themselves
    off_mean = sizes * (error + u(kind) * (count + 2))
    bound = p * off_mean + np.abs(expected) * (error + 3 * u(kind))
    for r in range(rows):
        for k in range(count):
            if index[r, k] >= 0:
                c = index[r, k]
                expected[r, c] += weight[r, k] * g[r, k]
                bound[r, c] += weight[r, k] * abs(g[r, k]) * (error + 3 * u(kind)) + weight[r, k] * abs(mean[r, 0]) * 3 * u(kind)
    compare(exactly(wide[:, :classes]), expected, bound + 2.0 ** -120, kind)
    assert bool((wide[:, classes:] == 5.0).all())


@ALL
@pytest.mark.parametrize("classes", range(1, 18))
@pytest.mark.parametrize("among", [False, True])
def test_select_top_of_few_classes_for_many_rows(kind, classes, among):
    rng = np.random.default_rng(classes)
    rows, count, pad = 16384 + 77, 8 if classes % 5 == 0 else min(8, 1 + classes // 2), classes % 3
    x = rng.normal(size=(rows, classes)) * 3
    x[rng.random((rows, classes)) < 0.2] = 1.5
    x[rng.random((rows, classes)) < 0.05] = -0.0
    x[rng.random((rows, classes)) < 0.05] = 0.0
    x[rng.random((rows, classes)) < 0.1] = -np.inf
    x[rng.random((rows, classes)) < 0.02] = np.nan
    scores = table(x, kind, pad)
    indexes = torch.full((rows * count + 1,), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((rows * count + 1,), 77, dtype=acc(kind), device="cuda")
    cb.select_top(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr())
    exact = exactly(scores)
    usable = np.where(np.isnan(exact), -np.inf, exact)
    order = np.argsort(-usable, axis=1, kind="stable")[:, :count]
    taken = np.take_along_axis(usable, order, 1) > -np.inf
    if count > classes:  # what is not there: index -1, weight 0
        assert bool((indexes[:-1].view(rows, count)[:, classes:] == -1).all()) and bool((weights[:-1].view(rows, count)[:, classes:] == 0).all())
    there = order.shape[1]
    picked = np.zeros(usable.shape, bool)
    np.put_along_axis(picked, order, taken, 1)
    most = usable.max(1, keepdims=True)
    e = np.where(picked if among else usable > -np.inf, np.exp(usable - np.where(most > -np.inf, most, 0)), 0)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total > 0, total, 1)
    weight = np.where(taken, np.take_along_axis(p, order, 1), 0)
    np.testing.assert_array_equal(indexes[:-1].cpu().numpy().reshape(rows, count)[:, :there], np.where(taken, order, -1))
    error = weight_error(kind, exact)
    compare(exactly(weights[:-1]).reshape(rows, count)[:, :there], weight, error * weight + 2.0 ** -125, kind if kind == cb.FLOAT64 else cb.FLOAT32)
    assert int(indexes[-1]) == 77 and float(weights[-1]) == 77

    gradients = torch.from_numpy(rng.normal(size=(rows, count))).cuda().to(acc(kind))
    wide = torch.full((rows, classes + pad + 1), 5.0, dtype=TYPES[kind], device="cuda")
    cb.select_top_backward(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr(),
                           gradients.data_ptr(), wide.data_ptr(), wide.stride(0))
    g = np.where(taken, exactly(gradients)[:, :there], 0)
    mean, sizes = (g * weight).sum(1, keepdims=True), (np.abs(g) * weight).sum(1, keepdims=True)
    part, part_size = np.zeros(p.shape, np.longdouble), np.zeros(p.shape, np.longdouble)
    np.put_along_axis(part, order, weight * g, 1)
    np.put_along_axis(part_size, order, weight * np.abs(g) * (error + 3 * u(kind)) + weight * np.abs(mean) * 3 * u(kind), 1)
    expected = part - p * mean
    bound = p * sizes * (error + u(kind) * (count + 2)) + np.abs(p * mean) * (error + 3 * u(kind)) + part_size
    compare(exactly(wide[:, :classes]), expected, bound + 2.0 ** -120, kind)
    assert bool((wide[:, classes:] == 5.0).all())


def of_few_classes(kind, rows, classes, count, pad, among):
    """The first rows against the definition; what has rows enough is these rows again and again, all with the same results."""
    rng = np.random.default_rng(classes * 10 + count)
    different = 1001
    x = rng.normal(size=(different, classes)) * 3
    x[rng.random(x.shape) < 0.2] = 1.5
    x[rng.random(x.shape) < 0.05] = -0.0
    x[rng.random(x.shape) < 0.05] = 0.0
    x[rng.random(x.shape) < 0.1] = -np.inf
    x[rng.random(x.shape) < 0.02] = np.nan
    x[1], x[2], x[3, 1:] = -np.inf, np.nan, np.nan
    again = torch.arange(rows, device="cuda") % different
    wide = torch.full((rows, classes + pad), 7.0, dtype=TYPES[kind], device="cuda")
    wide[:, :classes] = dev(x).to(TYPES[kind])[again]
    scores = wide[:, :classes]
    g = rng.normal(size=(different, count))
    g[rng.random(g.shape) < 0.1] = 0.0
    gradients = dev(g).to(acc(kind))[again].contiguous()
    indexes = torch.full((rows * count + 1,), 77, dtype=torch.int32, device="cuda")
    weights = torch.full((rows * count + 1,), 77, dtype=acc(kind), device="cuda")
    out = torch.full((rows, classes + pad + 1), 5.0, dtype=TYPES[kind], device="cuda")
    cb.select_top(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr())
    cb.select_top_backward(kind, rows, classes, scores.data_ptr(), scores.stride(0), count, among, indexes.data_ptr(), weights.data_ptr(),
                           gradients.data_ptr(), out.data_ptr(), out.stride(0))
    assert int(indexes[-1]) == 77 and float(weights[-1]) == 77 and bool((out[:, classes:] == 5.0).all())
    indexes, weights = indexes[:-1].view(rows, count), weights[:-1].view(rows, count)
    for got in (indexes, weights, out[:, :classes]):
        assert torch.equal(got, got[:different][again])

    index, weight, p = best(exactly(scores[:different]), count, among)
    np.testing.assert_array_equal(indexes[:different].cpu().numpy(), index)
    error = weight_error(kind, exactly(scores[:different]))
    compare(exactly(weights[:different]), weight, error * weight + 2.0 ** -125, kind if kind == cb.FLOAT64 else cb.FLOAT32)
    # as in test_select_top
    g = np.where(index >= 0, exactly(gradients[:different]), 0)
    mean, sizes = (g * weight).sum(1, keepdims=True), (np.abs(g) * weight).sum(1, keepdims=True)
    expected = -p * mean
    if among:
        expected[:] = 0
    bound = p * sizes * (error + u(kind) * (count + 2)) + np.abs(expected) * (error + 3 * u(kind))
    for k in range(count):
        r = np.nonzero(index[:, k] >= 0)[0]
        part = weight[r, k] * (g[r, k] - mean[r, 0] if among else g[r, k])
        expected[r, index[r, k]] += part
        bound[r, index[r, k]] += weight[r, k] * (np.abs(g[r, k]) * (error + 3 * u(kind)) + np.abs(mean[r, 0]) * (error + 3 * u(kind)))
    compare(exactly(out[:different, :classes]), expected, bound + 2.0 ** -120, kind)


@ALL
@pytest.mark.parametrize("classes", range(1, 17))
@pytest.mark.parametrize("among", [False, True])
def test_select_top_of_few_classes_by_threads(kind, classes, among):
    """Rows enough that every row has a thread to itself: forward with 8 classes selected, forward and backward with fewer."""
    of_few_classes(kind, 32768 + 77, classes, 8, classes % 3, among)
    of_few_classes(kind, 131072 + 77, classes, 4 if classes % 4 == 1 else 1 + classes % 4, classes % 2, among)


@ALL
@pytest.mark.parametrize("rows", [32767, 32768, 131071, 131072])
@pytest.mark.parametrize("count", [4, 5, 8, 9])
def test_select_top_of_few_classes_around_the_rows_for_threads(kind, rows, count):
    of_few_classes(kind, rows, 10, count, 0, count % 2 == 0)


@ALL
def test_select_top_of_infinite_scores(kind):
    x = np.array([[np.inf, 1, np.inf, 0], [np.inf, np.inf, np.inf, np.inf], [1, np.inf, -np.inf, np.nan]])
    scores = table(x, kind)
    indexes = torch.empty(3, 3, dtype=torch.int32, device="cuda")
    weights = torch.empty(3, 3, dtype=acc(kind), device="cuda")
    for among in (False, True):
        cb.select_top(kind, 3, 4, scores.data_ptr(), 4, 3, among, indexes.data_ptr(), weights.data_ptr())
        assert indexes.tolist() == [[0, 2, 1], [0, 1, 2], [1, 0, -1]]
        third = [1 / 3] * 3 if among else [0.25] * 3
        np.testing.assert_allclose(weights.cpu().numpy(), [[0.5, 0.5, 0], third, [1, 0, 0]], rtol=2.0 ** -22)


@pytest.mark.parametrize("among", [False, True])
@pytest.mark.parametrize("classes,count", [(7, 3), (40, 5), (200, 8)])
def test_select_top_gradient_by_differences(classes, count, among):
    """Central differences in 64 bits: off by the third derivative (below 1 in size, over 6) times the step squared, and by
    the weights' rounding over the step."""
    rng = np.random.default_rng(classes)
    rows, step = 3, 2.0 ** -17
    x = rng.permutation(rows * classes).reshape(rows, classes) * (4.0 / classes)  # no two nearer than the steps
    g = rng.normal(size=(rows, count))

    def run(values):
        scores = table(values, cb.FLOAT64)
        i, w = torch.empty(rows, count, dtype=torch.int32, device="cuda"), torch.empty(rows, count, dtype=torch.float64, device="cuda")
        cb.select_top(cb.FLOAT64, rows, classes, scores.data_ptr(), classes, count, among, i.data_ptr(), w.data_ptr())
        return scores, i, w

    scores, i, w = run(x)
    dx = torch.empty(rows, classes, dtype=torch.float64, device="cuda")
    gradients = dev(g)
    cb.select_top_backward(cb.FLOAT64, rows, classes, 0 if among else scores.data_ptr(), classes, count, among, i.data_ptr(), w.data_ptr(),
                           gradients.data_ptr(), dx.data_ptr(), classes)
    size = np.abs(g).sum(1).max()
    for c in range(0, classes, max(1, classes // 9)):
        lower, upper = x.copy(), x.copy()
        lower[:, c] -= step
        upper[:, c] += step
        difference = ((run(upper)[2] - run(lower)[2]).cpu().numpy() * g).sum(1) / (2 * step)
        allowed = size * (step * step + weight_error(cb.FLOAT64, x) / step)
        assert np.max(np.abs(difference - dx[:, c].cpu().numpy())) <= allowed


# ---------------------------------------------------------------- rows sorted by expert and back

def sort(ids, experts):
    ids = dev(np.asarray(ids, np.int32).reshape(-1))
    places = torch.full((ids.numel() + 1,), 123, dtype=torch.int32, device="cuda")
    offsets = torch.full((experts + 2,), 123, dtype=torch.int32, device="cuda")
    size = cb.sort_by_expert_bytes(ids.numel(), experts)
    workspace = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")
    cb.sort_by_expert(ids.numel(), experts, ids.data_ptr(), places.data_ptr(), offsets.data_ptr(), workspace.data_ptr(), size)
    assert int(places[-1]) == 123 and int(offsets[-1]) == 123 and bool((workspace[size:] == 255).all())
    return places[:-1], offsets[:-1]


@pytest.mark.parametrize("slots", [0, 1, 2, 63, 64, 65, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8192, 8193, 16384, 16385, 70_001, 1_200_000])
@pytest.mark.parametrize("experts", [1, 2, 7, 64, 255, 256, 257, 1024])
def test_sort_by_expert(slots, experts):
    rng = np.random.default_rng(slots + experts)
    ids = (experts * rng.random(slots) ** 2).astype(np.int32)
    ids[rng.random(slots) < 0.05] = -1
    ids[rng.random(slots) < 0.02] = experts
    ids[rng.random(slots) < 0.01] = np.iinfo(np.int32).min
    places, offsets = sort(ids, experts)
    valid = (ids >= 0) & (ids < experts)
    order = np.argsort(np.where(valid, ids, experts), kind="stable")
    expected = np.empty(slots, np.int32)
    expected[order] = np.arange(slots)
    np.testing.assert_array_equal(places.cpu().numpy(), np.where(valid, expected, -1))
    np.testing.assert_array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(ids[valid], minlength=experts))]))


@pytest.mark.parametrize("experts", [900, 909, 910, 911, 1000])  # tables of 64 KB more or less
def test_sort_by_expert_around_64_kb(experts):
    for slots in (300, 20_000):
        ids = np.random.default_rng(slots).integers(0, experts, slots).astype(np.int32)
        places, offsets = sort(ids, experts)
        np.testing.assert_array_equal(places.cpu().numpy()[np.argsort(ids, kind="stable")], np.arange(slots))
        assert int(offsets[-1]) == slots


@pytest.mark.parametrize("slots", [500, 50_000])
def test_sort_by_one_of_many_experts(slots):
    for ids in (np.full(slots, 5), np.full(slots, -1), np.arange(slots) % 2 * 1023):
        places, offsets = sort(ids, 1024)
        valid = ids >= 0
        order = np.argsort(ids, kind="stable")
        expected = np.empty(slots, np.int32)
        expected[order] = np.arange(slots)
        np.testing.assert_array_equal(places.cpu().numpy(), np.where(valid, expected, -1))
        assert int(offsets[-1]) == valid.sum()


def routed(rng, rows, per_row, spare=3):
    """Places as a sort gives them, some of none, some behind the last row; with room for more rows."""
    slots = rows * per_row
    places = rng.permutation(slots + spare)[:slots].astype(np.int32)
    places[rng.random(slots) < 0.1] = -1
    if slots > 3:
        places[2] = slots + spare + 4
        places[3] = np.iinfo(np.int32).max
    return places.reshape(rows, per_row), slots + spare


ROWS = [(1, 1, 1, 0), (1, 2, 5, 0), (3, 64, 8, 0), (700, 1, 200, 0), (501, 3, 7, 2), (40, 4, 1000, 0), (9, 2, 4096, 0), (5, 8, 4099, 1), (2, 5, 16384, 0), (1000, 2, 10, 0),
        (33, 6, 63, 0), (20, 7, 65, 0), (300, 2, 1, 0), (64, 9, 514, 6), (3000, 2, 64, 0)]


@ALL
@pytest.mark.parametrize("rows,per_row,width,pad", ROWS)
def test_dispatch_rows(kind, rows, per_row, width, pad):
    rng = np.random.default_rng(rows + width)
    places, sorted_rows = routed(rng, rows, per_row)
    x = rng.normal(size=(rows, width))
    x[rng.random((rows, width)) < 0.01] = np.nan
    source = table(x, kind, pad)
    wide = torch.full((sorted_rows, width + pad + 1), 9.0, dtype=TYPES[kind], device="cuda")
    d = dev(places)
    cb.dispatch_rows(kind, rows, width, per_row, source.data_ptr(), source.stride(0), d.data_ptr(), wide.data_ptr(), sorted_rows, wide.stride(0))
    expected = torch.full_like(wide, 9.0)
    there = (places >= 0) & (places < sorted_rows)
    expected[torch.from_numpy(places[there].astype(np.int64)).cuda(), :width] = source[torch.from_numpy(np.nonzero(there)[0]).cuda()]
    bits = torch.int64 if kind == cb.FLOAT64 else torch.int32 if kind == cb.FLOAT32 else torch.int16
    assert torch.equal(wide.view(bits), expected.view(bits))


@ALL
@pytest.mark.parametrize("rows,per_row,width,pad", ROWS)
@pytest.mark.parametrize("weighted", [True, False])
def test_combine_rows_and_gradients(kind, rows, per_row, width, pad, weighted):
    rng = np.random.default_rng(rows + width + 1)
    places, sorted_rows = routed(rng, rows, per_row)
    y = table(rng.normal(size=(sorted_rows, width)), kind, pad, fill=float("nan"))
    unused = np.setdiff1d(np.arange(sorted_rows), places)
    y[torch.from_numpy(unused).cuda()] = float("nan")  # what no place names is not read
    there = (places >= 0) & (places < sorted_rows)
    weights = rng.normal(size=(rows, per_row))
    weights[~there] = np.nan  # nor is the weight of none
    w = dev(weights, acc(kind)) if weighted else None
    d = dev(places)
    wide = torch.full((rows, width + pad + 1), 9.0, dtype=TYPES[kind], device="cuda")
    cb.combine_rows(kind, rows, width, per_row, y.data_ptr(), sorted_rows, y.stride(0), d.data_ptr(), ptr(w), wide.data_ptr(), wide.stride(0))
    exact_y, exact_w = exactly(y), exactly(w) if weighted else np.ones((rows, per_row), np.longdouble)
    expected, size = np.zeros((rows, width), np.longdouble), np.zeros((rows, width), np.longdouble)
    for k in range(per_row):
        rs = np.nonzero(there[:, k])[0]
        part = exact_w[rs, k, None] * exact_y[places[rs, k]]
        expected[rs] += part
        size[rs] += np.abs(part)
    compare(exactly(wide[:, :width]), expected, u(kind) * (per_row + 1) * size, kind)  # a product and up to per_row additions each
    assert bool((wide[:, width:] == 9.0).all())

    g = table(rng.normal(size=(rows, width)), kind, pad, fill=float("nan"))
    dy = torch.full((sorted_rows, width + pad + 2), 9.0, dtype=TYPES[kind], device="cuda")
    dw = torch.full((rows * per_row + 1,), 9.0, dtype=acc(kind), device="cuda")
    cb.combine_rows_backward(kind, rows, width, per_row, g.data_ptr(), g.stride(0), y.data_ptr(), sorted_rows, y.stride(0), d.data_ptr(), ptr(w),
                             dy.data_ptr(), dy.stride(0), dw.data_ptr())
    exact_g = exactly(g)
    expected = np.full((sorted_rows, width), 9.0, np.longdouble)
    product, size = np.zeros((rows, per_row), np.longdouble), np.zeros((rows, per_row), np.longdouble)
    for k in range(per_row):
        rs = np.nonzero(there[:, k])[0]
        expected[places[rs, k]] = exact_w[rs, k, None] * exact_g[rs]
        product[rs, k] = (exact_y[places[rs, k]] * exact_g[rs]).sum(1)
        size[rs, k] = np.abs(exact_y[places[rs, k]] * exact_g[rs]).sum(1)
    compare(exactly(dy[:, :width]), expected, u(kind) * np.abs(expected), kind)
    assert bool((dy[:, width:] == 9.0).all())
    # the columns are added in chains of at most width / 32 + 32 additions, whatever they are split into, after one product
    compare(exactly(dw[:-1]).reshape(rows, per_row), product, u(kind) * (width // 32 + 33) * size, kind if kind == cb.FLOAT64 else cb.FLOAT32)
    assert float(dw[-1]) == 9.0

    # either alone
    dy2, dw2 = torch.full_like(dy, 9.0), torch.full_like(dw, 9.0)
    cb.combine_rows_backward(kind, rows, width, per_row, g.data_ptr(), g.stride(0), 0, sorted_rows, y.stride(0), d.data_ptr(), ptr(w), dy2.data_ptr(),
                             dy2.stride(0), 0)
    cb.combine_rows_backward(kind, rows, width, per_row, g.data_ptr(), g.stride(0), y.data_ptr(), sorted_rows, y.stride(0), d.data_ptr(), ptr(w), 0,
                             0, dw2.data_ptr())
    assert torch.equal(dy, dy2) and torch.equal(dw, dw2)


@ALL
@pytest.mark.parametrize("rows,per_row,pieces", [(16383, 2, 20), (16384, 2, 20), (16400, 1, 17), (16390, 3, 32), (4095, 2, 70), (4096, 2, 70), (4100, 1, 100), (4097, 2, 255), (4100, 1, 256)])
def test_combine_rows_and_gradients_of_many_rows(kind, rows, per_row, pieces):
    """Around the numbers of rows from which eight threads and a wave have a row's gradients; rows that end inside a piece."""
    in_piece = 2 if kind == cb.FLOAT64 else 4 if kind == cb.FLOAT32 else 8
    test_combine_rows_and_gradients(kind, rows, per_row, pieces * in_piece - 1, per_row % 2, True)


@ALL
def test_no_sorted_rows(kind):
    places = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    result = torch.full((4, 8), 9.0, dtype=TYPES[kind], device="cuda")
    cb.combine_rows(kind, 4, 8, 2, 0, 0, 8, places.data_ptr(), 0, result.data_ptr(), 8)
    assert bool((result == 0).all())
    dw = torch.full((4, 2), 9.0, dtype=acc(kind), device="cuda")
    cb.combine_rows_backward(kind, 4, 8, 2, result.data_ptr(), 8, 0, 0, 8, places.data_ptr(), 0, 0, 8, dw.data_ptr())
    assert bool((dw == 0).all())


# ---------------------------------------------------------------- together, streams, graphs

def mixture(kind, x, gate, bias, experts, per_row, stream, buffers):
    """A layer of experts: gate scores with biases, the best experts, rows to them and back. Every expert doubles its rows."""
    rows, width = x.shape
    b = buffers
    cb.adjust_scores(cb.FLOAT32, rows, experts, gate.data_ptr(), experts, bias.struct, b["scores"].data_ptr(), experts, stream)
    cb.select_top(cb.FLOAT32, rows, experts, b["scores"].data_ptr(), experts, per_row, True, b["ids"].data_ptr(), b["weights"].data_ptr(), stream)
    cb.sort_by_expert(rows * per_row, experts, b["ids"].data_ptr(), b["places"].data_ptr(), b["offsets"].data_ptr(), b["workspace"].data_ptr(),
                      b["workspace"].numel(), stream)
    cb.dispatch_rows(kind, rows, width, per_row, x.data_ptr(), width, b["places"].data_ptr(), b["sorted"].data_ptr(), rows * per_row, width, stream)
    torch.mul(b["sorted"], 2, out=b["sorted"])
    cb.combine_rows(kind, rows, width, per_row, b["sorted"].data_ptr(), rows * per_row, width, b["places"].data_ptr(), b["weights"].data_ptr(),
                    b["result"].data_ptr(), width, stream)
    cb.combine_rows_backward(kind, rows, width, per_row, x.data_ptr(), width, b["sorted"].data_ptr(), rows * per_row, width, b["places"].data_ptr(),
                             b["weights"].data_ptr(), b["sorted_gradients"].data_ptr(), width, b["weight_gradients"].data_ptr(), stream)
    cb.select_top_backward(cb.FLOAT32, rows, experts, b["scores"].data_ptr(), experts, per_row, True, b["ids"].data_ptr(), b["weights"].data_ptr(),
                           b["weight_gradients"].data_ptr(), b["gate_gradients"].data_ptr(), experts, stream)
    return b


def mixture_buffers(kind, rows, width, experts, per_row):
    def empty(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    slots = rows * per_row
    return dict(scores=empty(rows, experts), ids=empty(rows, per_row, dtype=torch.int32), weights=empty(rows, per_row), places=empty(slots, dtype=torch.int32),
                offsets=empty(experts + 1, dtype=torch.int32), workspace=empty(cb.sort_by_expert_bytes(slots, experts), dtype=torch.uint8),
                sorted=empty(slots, width, dtype=TYPES[kind]), result=empty(rows, width, dtype=TYPES[kind]),
                sorted_gradients=empty(slots, width, dtype=TYPES[kind]), weight_gradients=empty(rows, per_row), gate_gradients=empty(rows, experts))


def check_mixture(kind, x, b):
    # weights add up to 1 (five roundings), experts double: the result is twice the input
    exact = exactly(x)
    compare(exactly(b["result"]), 2 * exact, 16 * u(kind) * np.abs(exact), kind)
    # the product of a row and twice itself
    norm = 2 * (exact * exact).sum(1, keepdims=True)
    compare(exactly(b["weight_gradients"]), np.broadcast_to(norm, b["weight_gradients"].shape), u(kind) * (x.shape[1] // 32 + 33) * norm, cb.FLOAT32)


@pytest.mark.parametrize("kind", [cb.FLOAT32, cb.BFLOAT16], ids=NAMES.get)
@pytest.mark.parametrize("rows,width", [(3, 100), (2500, 64)])
def test_a_layer_of_experts_on_a_stream_and_in_graphs(kind, rows, width):
    experts, per_row = 9, 3
    rng = np.random.default_rng(rows)
    allowed = np.full((1, 1), 0b111011011, np.uint32)
    bias = Adjustment(dict(class_bias=rng.normal(size=(1, experts)).astype(np.float32), allowed=allowed, allowed_rows=np.zeros(rows, np.int32)))
    inputs = [(table(rng.normal(size=(rows, width)), kind), dev(rng.normal(size=(rows, experts)).astype(np.float32))) for _ in range(3)]
    eager = []
    for x, gate in inputs:
        b = mixture(kind, x, gate, bias, experts, per_row, None, mixture_buffers(kind, rows, width, experts, per_row))
        check_mixture(kind, x, b)
        ids = b["ids"].cpu().numpy()
        assert not np.isin(ids, [2, 5]).any() and (ids >= 0).all()
        eager.append({k: v.clone() for k, v in b.items() if k != "workspace"})
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b = mixture(kind, *inputs[1], bias, experts, per_row, side.cuda_stream, mixture_buffers(kind, rows, width, experts, per_row))
    side.synchronize()
    for k, v in eager[1].items():
        assert torch.equal(b[k], v), k
    # two graphs with buffers of their own, replayed in turn with eager work between
    graphs = []
    for _ in range(2):
        x, gate = torch.zeros_like(inputs[0][0]), torch.zeros_like(inputs[0][1])
        buffers = mixture_buffers(kind, rows, width, experts, per_row)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mixture(kind, x, gate, bias, experts, per_row, torch.cuda.current_stream().cuda_stream, buffers)
        graphs.append((graph, x, gate, buffers))
    for turn in range(6):
        at = turn % 3
        graph, x, gate, buffers = graphs[turn % 2]
        x.copy_(inputs[at][0])
        gate.copy_(inputs[at][1])
        graph.replay()
        mixture(kind, *inputs[(at + 1) % 3], bias, experts, per_row, None, mixture_buffers(kind, rows, width, experts, per_row))
        torch.cuda.synchronize()
        for k, v in eager[at].items():
            assert torch.equal(buffers[k], v), (turn, k)


def test_a_first_call_with_large_tables_is_captured():
    """More than 64 KB of LDS, which a kernel has to be allowed once for each device (in a process that runs this test alone, in the capture)."""
    slots, experts, rows, classes = 3000, 1021, 200, 90_001
    rng = np.random.default_rng(2)
    ids = rng.integers(0, experts, slots).astype(np.int32)
    d, places, offsets = dev(ids), torch.empty(slots, dtype=torch.int32, device="cuda"), torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    size = cb.sort_by_expert_bytes(slots, experts)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    scores = table(rng.normal(size=(rows, classes)), cb.BFLOAT16)
    p = parts(rng, rows, classes, "hsb", 3)
    a = Adjustment(p)
    result = torch.zeros_like(scores)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        cb.sort_by_expert(slots, experts, d.data_ptr(), places.data_ptr(), offsets.data_ptr(), workspace.data_ptr(), size, stream)
        cb.adjust_scores(cb.BFLOAT16, rows, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes, stream)
    eager = torch.zeros_like(scores)
    cb.adjust_scores(cb.BFLOAT16, rows, classes, scores.data_ptr(), classes, a.struct, eager.data_ptr(), classes)
    for _ in range(3):
        result.zero_()
        places.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(result, eager)
        np.testing.assert_array_equal(places.cpu().numpy()[np.argsort(ids, kind="stable")], np.arange(slots))


def test_offsets_that_pass_32_bits():
    """Histories and biases that lie behind 2^32 entries, rows that lie 2^32 values apart."""
    far, rows, classes = (1 << 32) + 10, 3, 700
    rng = np.random.default_rng(1)
    scores = table(rng.normal(size=(rows, classes)), cb.FLOAT32)
    p = dict(offsets=np.array([0, 4, 4, 9]), ids=rng.integers(0, classes, 9).astype(np.int32), frequency=np.ones(rows, np.float32))
    expected, _ = adjusted(exactly(scores), p)
    a = Adjustment(p)
    entries = torch.empty(far + 16, dtype=torch.int32, device="cuda")
    entries[far:far + 9] = a.keep["ids"]
    a.keep["offsets"] += far
    a.struct.History, a.struct.HistoryCount = entries.data_ptr(), far + 9
    result = torch.empty_like(scores)
    for few in (classes, 500):  # in tiles of rows and as slices
        cb.adjust_scores(cb.FLOAT32, rows, few, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
        kept = [i for i in range(9) if p["ids"][i] < few]
        assert kept
        np.testing.assert_allclose(result[:, :few].cpu().numpy(), expected[:, :few].astype(np.float64), rtol=0, atol=16 * 2.0 ** -24)
    del entries

    stride = (1 << 32) + 3
    wide = torch.empty(2 * stride + 64, dtype=torch.float16, device="cuda")
    source = table(rng.normal(size=(3, 50)), cb.FLOAT16)
    places = dev(np.array([[2], [0], [1]], np.int32))
    cb.dispatch_rows(cb.FLOAT16, 3, 50, 1, source.data_ptr(), 50, places.data_ptr(), wide.data_ptr(), 3, stride)
    for row, place in enumerate((2, 0, 1)):
        assert torch.equal(wide[place * stride:place * stride + 50], source[row])
    back = torch.empty_like(source)
    cb.combine_rows(cb.FLOAT16, 3, 50, 1, wide.data_ptr(), 3, stride, places.data_ptr(), 0, back.data_ptr(), 50)
    assert torch.equal(back, source)
    doubled = torch.empty(3, dtype=torch.float32, device="cuda")
    cb.combine_rows_backward(cb.FLOAT16, 3, 50, 1, source.data_ptr(), 50, wide.data_ptr(), 3, stride, places.data_ptr(), 0, 0, 50, doubled.data_ptr())
    np.testing.assert_allclose(doubled.cpu().numpy(), (exactly(source) ** 2).sum(1).astype(np.float64), rtol=40 * 2.0 ** -24)
    cb.adjust_scores(cb.FLOAT16, 3, 50, wide.data_ptr(), stride, cb.score_adjustment(), back.data_ptr(), 50)
    assert torch.equal(back[torch.tensor([2, 0, 1])], source)
    index, weight = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
    cb.select_top(cb.FLOAT16, 3, 50, wide.data_ptr(), stride, 1, True, index.data_ptr(), weight.data_ptr())
    assert torch.equal(index.long()[torch.tensor([2, 0, 1], device="cuda")], source.argmax(1))


@pytest.mark.parametrize("classes", [3, 20])
def test_more_rows_to_select_from_than_one_launch_takes(classes):
    rows, count = (1 << 24) + 77, 2
    scores = torch.randn(rows, classes, device="cuda").half()
    gradients = torch.randn(rows, count, device="cuda")

    def run(begin, end):
        n = end - begin
        indexes, weights = torch.empty(n, count, dtype=torch.int32, device="cuda"), torch.empty(n, count, device="cuda")
        cb.select_top(cb.FLOAT16, n, classes, scores[begin:].data_ptr(), classes, count, False, indexes.data_ptr(), weights.data_ptr())
        out = torch.full((n, classes), 5.0, dtype=torch.float16, device="cuda")
        cb.select_top_backward(cb.FLOAT16, n, classes, scores[begin:].data_ptr(), classes, count, False, indexes.data_ptr(), weights.data_ptr(),
                               gradients[begin:].data_ptr(), out.data_ptr(), classes)
        return indexes, weights, out

    for whole, first, second in zip(run(0, rows), run(0, 8_000_000), run(8_000_000, rows)):
        assert torch.equal(whole[:8_000_000], first) and torch.equal(whole[8_000_000:], second)


def test_more_slices_than_one_launch_takes():
    rows, classes = (1 << 21) + 9, 600
    scores = torch.randn(rows, classes, device="cuda").half()
    ids = torch.randint(0, classes, (rows,), dtype=torch.int32, device="cuda")
    a = Adjustment(dict(offsets=np.arange(rows + 1), ids=ids.cpu().numpy(), presence=np.full(rows, 2.5, np.float32)))
    result = torch.full_like(scores, 5.0)
    cb.adjust_scores(cb.FLOAT16, rows, classes, scores.data_ptr(), classes, a.struct, result.data_ptr(), classes)
    at = ids.long()[:, None]
    expected = scores.scatter(1, at, (scores.gather(1, at).float() - 2.5).half())
    assert torch.equal(result, expected)


def test_more_tiles_of_rows_than_one_launch_takes():
    rows = (1 << 30) + 700
    scores = torch.randn(rows, device="cuda", dtype=torch.float16)
    a = Adjustment(dict(class_bias=np.full((1, 1), 0.25, np.float32)))
    result = torch.full_like(scores, 5.0)
    cb.adjust_scores(cb.FLOAT16, rows, 1, scores.data_ptr(), 1, a.struct, result.data_ptr(), 1)
    assert torch.equal(result, (scores.float() + 0.25).half())


def test_more_pieces_of_rows_than_one_launch_takes():
    width = 7
    rows = (1 << 31) // width + 100
    source = torch.randn(rows, width, device="cuda", dtype=torch.float16)
    places = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda")
    moved = torch.full_like(source, 5.0)
    cb.dispatch_rows(cb.FLOAT16, rows, width, 1, source.data_ptr(), width, places.data_ptr(), moved.data_ptr(), rows, width)
    assert torch.equal(moved.flip(0), source)
    result = torch.full_like(source, 5.0)
    cb.combine_rows(cb.FLOAT16, rows, width, 1, moved.data_ptr(), rows, width, places.data_ptr(), 0, result.data_ptr(), width)
    assert torch.equal(result, source)
    result.fill_(5.0)
    products = torch.full((rows,), 5.0, device="cuda")
    cb.combine_rows_backward(cb.FLOAT16, rows, width, 1, source.data_ptr(), width, moved.data_ptr(), rows, width, places.data_ptr(), 0, result.data_ptr(),
                             width, products.data_ptr())
    assert torch.equal(result, moved)
    for begin in range(0, rows, 1 << 26):  # 7 products, 7 sums
        exact = source[begin:begin + (1 << 26)].double().square().sum(1)
        assert bool(((products[begin:begin + (1 << 26)].double() - exact).abs() <= 14 * 2.0 ** -24 * exact).all())


def test_the_most_slots():
    slots = (1 << 31) - 1
    ids = torch.empty(slots, dtype=torch.int32, device="cuda")
    for begin in range(0, slots, 1 << 28):
        part = ids[begin:begin + (1 << 28)]
        part.copy_(torch.arange(begin, begin + part.numel(), device="cuda") % 3)
    places, offsets = torch.empty_like(ids), torch.empty(3, dtype=torch.int32, device="cuda")
    size = cb.sort_by_expert_bytes(slots, 2)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    cb.sort_by_expert(slots, 2, ids.data_ptr(), places.data_ptr(), offsets.data_ptr(), workspace.data_ptr(), size)
    zeros = (slots + 2) // 3
    assert offsets.tolist() == [0, zeros, zeros + (slots + 1) // 3]
    for begin in range(0, slots, 1 << 28):
        i = torch.arange(begin, min(begin + (1 << 28), slots), device="cuda")
        expected = torch.where(i % 3 == 2, -1, i // 3 + (i % 3) * zeros)
        assert torch.equal(places[begin:begin + (1 << 28)].long(), expected)


def test_two_streams_at_once():
    """Calls of all kinds on two streams side by side, with buffers of their own."""
    kind, rows, width, experts, per_row = cb.FLOAT32, 3000, 256, 40, 2
    rng = np.random.default_rng(8)
    bias = Adjustment(dict(class_bias=rng.normal(size=(1, experts)).astype(np.float32)))
    inputs = [(table(rng.normal(size=(rows, width)), kind), dev(rng.normal(size=(rows, experts)).astype(np.float32))) for _ in range(2)]
    alone = [mixture(kind, *i, bias, experts, per_row, None, mixture_buffers(kind, rows, width, experts, per_row)) for i in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    buffers = [mixture_buffers(kind, rows, width, experts, per_row) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s, b in zip(inputs, streams, buffers):
            with torch.cuda.stream(s):
                mixture(kind, *i, bias, experts, per_row, s.cuda_stream, b)
    torch.cuda.synchronize()
    for a, b in zip(alone, buffers):
        for k in a:
            assert k == "workspace" or torch.equal(a[k], b[k]), k


def test_a_stream_that_is_not_given_is_the_default_one():
    x = torch.ones(1000, 100, device="cuda")
    a = Adjustment(dict(class_bias=np.ones((1, 100), np.float32)))
    for _ in range(5):
        x.mul_(2)
        cb.adjust_scores(cb.FLOAT32, 1000, 100, x.data_ptr(), 100, a.struct, x.data_ptr(), 100)
    assert bool((x == 63).all())


@pytest.mark.parametrize("stream", [1, 2])  # hipStreamLegacy, hipStreamPerThread
def test_named_streams(stream):
    x = torch.ones(1000, 100, device="cuda")
    a = Adjustment(dict(class_bias=np.ones((1, 100), np.float32)))
    torch.cuda.synchronize()
    for _ in range(5):
        cb.adjust_scores(cb.FLOAT32, 1000, 100, x.data_ptr(), 100, a.struct, x.data_ptr(), 100, stream)
    torch.cuda.synchronize()
    assert bool((x == 6).all())


def test_host_memory_is_refused():
    x = torch.ones(4, 4)
    with pytest.raises(cb.CatBoostError, match="memory that a GPU can write"):
        cb.adjust_scores(cb.FLOAT32, 4, 4, x.data_ptr(), 4, cb.score_adjustment(), x.data_ptr(), 4)
    # and leaves no error behind for the next call
    y = torch.ones(4, 4, device="cuda")
    cb.adjust_scores(cb.FLOAT32, 4, 4, y.data_ptr(), 4, cb.score_adjustment(), y.data_ptr(), 4)
    torch.cuda.synchronize()
