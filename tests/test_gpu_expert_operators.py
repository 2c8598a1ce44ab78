"""The experts' products and their gradients against their definitions in 64 bits and more. Needs an MI355X.

Tolerances count roundings of half a step: U is half a step of what sums are held in (2^-24, 2^-53 for 64-bit values), HALF half a
step of the type that is stored. A sum of K products, each and each addition rounded, is off by at most (K + 1) U times the sum of
the products' sizes (and a little more than that many times over: K U is far under 1)."""
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
ACTIVATIONS = {cb.SILU: "silu", cb.GELU: "gelu", cb.GELU_TANH: "gelu_tanh", cb.RELU: "relu"}
KEPT = {cb.FLOAT64: cb.FLOAT64, cb.FLOAT32: cb.FLOAT32, cb.FLOAT16: cb.FLOAT32, cb.BFLOAT16: cb.FLOAT32}  # what values for a gradient are held in
SENTINEL = 7.0


def held_in(kind):
    return TYPES[KEPT[kind]]


def u(kind):
    return 2.0 ** -53 if kind == cb.FLOAT64 else 2.0 ** -24


def exactly(t):
    """In a type whose roundings do not show: more than 64 bits for 64-bit values, which costs numpy its fast products."""
    values = t.detach().to(torch.float64).cpu().numpy()
    return values.astype(np.longdouble) if t.dtype == torch.float64 else values


def padded(values, kind, pad=0, fill=SENTINEL):
    """The values rounded to the type, as the first columns of a wider table of `fill`."""
    values = torch.as_tensor(np.asarray(values, np.float64))
    wide = torch.full(values.shape[:-1] + (values.shape[-1] + pad,), fill, dtype=TYPES[kind], device="cuda")
    wide[..., :values.shape[-1]] = values.cuda().to(TYPES[kind])
    return wide[..., :values.shape[-1]]


def within(got, expected, bound, kind):
    """|got - expected| <= bound + one rounding to the type."""
    assert got.shape == expected.shape
    if not got.size:
        return
    off = np.abs(got - expected)
    allowed = bound + HALF[kind] * (np.abs(expected) + bound) + TINY[kind]
    worst = np.argmax(off - allowed)
    assert np.all(off <= allowed), "off by %g where %g is allowed" % (off.flat[worst], allowed.flat[worst])


class Rows:
    """Rows sorted by expert: some of each, none of some, some behind the last."""

    def __init__(self, rng, rows, experts, behind=0, empty=0.3):
        share = rng.random(experts) + 0.1
        share[rng.random(experts) < empty] = 0
        if share.sum() == 0:
            share[:] = 1
        counts = rng.multinomial(rows - behind, share / share.sum())
        self.bounds = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.offsets = torch.from_numpy(self.bounds).cuda()

    def of(self, e):
        return slice(int(self.bounds[e]), int(self.bounds[e + 1]))


def product_bound(a, b, kind, extra=0):
    """(K + 1) U sum |a||b| for a [m, k] times b [n, k]"""
    k = a.shape[1]
    return (k + 1 + extra) * u(kind) * 1.01 * (np.abs(a) @ np.abs(b).T)


# rows, width, outputs, experts, rows behind the last
SHAPES = [(1, 1, 1, 1, 0), (3, 8, 16, 2, 0), (5, 3, 7, 2, 1), (17, 33, 31, 3, 2), (64, 64, 64, 1, 0), (131, 65, 130, 3, 5), (300, 128, 272, 4, 0),
          (700, 40, 10, 37, 20), (257, 96, 520, 70, 3), (40, 264, 129, 5, 0), (14, 1024, 96, 16, 2), (150, 24, 2, 2, 0),
          (520, 64, 256, 1, 0), (600, 200, 264, 3, 7), (1100, 56, 328, 2, 0), (260, 136, 8, 1, 0),
          (90, 200, 1100, 2, 0), (70, 72, 3000, 1, 0), (100, 72, 10008, 1, 0), (130, 64, 8200, 1, 0), (50, 40, 20000, 2, 0), (40, 1000, 12, 2, 0)]


def multiply(kind, x, w, offsets, result, rows=None):
    rows = x.shape[0] if rows is None else rows
    cb.multiply_rows(kind, rows, x.shape[1], w.shape[1], w.shape[0], offsets, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), result.data_ptr(),
                     result.stride(0), torch.cuda.current_stream().cuda_stream)


def weights_of(rng, kind, experts, outputs, width, gap=0):
    """Experts' weights with `gap` values between them."""
    flat = torch.full((experts, outputs * width + gap), SENTINEL, dtype=TYPES[kind], device="cuda")
    w = flat[:, :outputs * width].view(experts, outputs, width) if not gap else flat.as_strided((experts, outputs, width), (outputs * width + gap, width, 1))
    w.copy_(torch.from_numpy(rng.standard_normal((experts, outputs, width))).to(TYPES[kind]))
    return w


def not_for_64_bits(kind, shape):
    if kind == cb.FLOAT64 and shape[1] * shape[2] > 50_000:
        pytest.skip("the products of more than 64 bits take too long")


@ALL
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("pad", [0, 5])
def test_multiply_rows(kind, shape, pad):
    not_for_64_bits(kind, shape)
    rows, width, outputs, experts, behind = shape
    rng = np.random.default_rng(rows * 31 + width + pad)
    routes = Rows(rng, rows, experts, behind)
    x, w = padded(rng.standard_normal((rows, width)), kind, pad), weights_of(rng, kind, experts, outputs, width, pad)
    d = padded(rng.standard_normal((rows, outputs)), kind, pad)
    y, dx, dw = (padded(np.full(s, SENTINEL), kind, pad) for s in ((rows, outputs), (rows, width), (1, 1)))
    dw = torch.full((experts, outputs * width + pad), SENTINEL, dtype=TYPES[kind], device="cuda").as_strided(w.shape, w.stride())
    multiply(kind, x, w, routes.offsets.data_ptr(), y)
    cb.multiply_rows_backward(kind, rows, width, outputs, experts, routes.offsets.data_ptr(), d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0),
                              w.data_ptr(), w.stride(0), dx.data_ptr(), dx.stride(0), dw.data_ptr(), dw.stride(0), torch.cuda.current_stream().cuda_stream)
    X, W, D, Y, DX, DW = (exactly(t) for t in (x, w, d, y, dx, dw))
    for e in range(experts):
        part = routes.of(e)
        within(Y[part], X[part] @ W[e].T, product_bound(X[part], W[e], kind), kind)
        within(DX[part], D[part] @ W[e], product_bound(D[part], W[e].T, kind), kind)
        within(DW[e], D[part].T @ X[part], product_bound(D[part].T, X[part].T, kind), kind)
    # rows behind the last one, and what lies between rows
    assert np.all(Y[routes.bounds[-1]:] == SENTINEL) and np.all(DX[routes.bounds[-1]:] == SENTINEL)
    if pad:
        for t in (y, dx):
            assert torch.all(t.as_strided((t.shape[0] - 1, pad), (t.stride(0), 1), t.storage_offset() + t.shape[1]) == SENTINEL)
        assert torch.all(dw.as_strided((experts, pad), (dw.stride(0), 1), outputs * width) == SENTINEL)


def act(name, x):
    """act(x) and its derivative, in the type of x."""
    from scipy.special import erfc

    if name == "silu":
        y = 1 / (1 + np.exp(-x))
        return x * y, y * (1 + x * (1 - y))
    if name == "gelu":
        y = erfc((-x * np.sqrt(np.longdouble(0.5))).astype(np.float64)).astype(np.longdouble) / 2
        return x * y, y + x * np.exp(-x * x / 2) / np.sqrt(2 * np.longdouble(np.pi))
    if name == "gelu_tanh":
        c = np.sqrt(2 / np.longdouble(np.pi))
        t = np.tanh(c * (x + np.longdouble("0.044715") * x ** 3))
        return x * (1 + t) / 2, (1 + t) / 2 + x * (1 - t * t) / 2 * c * (1 + 3 * np.longdouble("0.044715") * x * x)
    return np.where(x > 0, x, 0), (x > 0).astype(np.longdouble)


def gated(kind, activation, x, gate, up, offsets, result, kept):
    cb.gated_rows(kind, activation, x.shape[0], x.shape[1], gate.shape[1], gate.shape[0], offsets, x.data_ptr(), x.stride(0), gate.data_ptr(), up.data_ptr(),
                  gate.stride(0), result.data_ptr(), result.stride(0), 0 if kept is None else kept.data_ptr(), torch.cuda.current_stream().cuda_stream)


def gated_backward(kind, activation, d, x, gate, up, offsets, kept, pre, dx, dgate, dup):
    cb.gated_rows_backward(kind, activation, d.shape[0], x.shape[1], d.shape[1], gate.shape[0], offsets, d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0),
                           gate.data_ptr(), up.data_ptr(), gate.stride(0), kept.data_ptr(), pre.data_ptr(), 0 if dx is None else dx.data_ptr(),
                           0 if dx is None else dx.stride(0), 0 if dgate is None else dgate.data_ptr(), 0 if dup is None else dup.data_ptr(),
                           gate.stride(0) if dgate is None else dgate.stride(0), torch.cuda.current_stream().cuda_stream)


@ALL
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("pad", [0, 3])
def test_gated_rows(kind, shape, pad):
    not_for_64_bits(kind, shape)
    rows, width, hidden, experts, behind = shape
    rng = np.random.default_rng(rows * 17 + width + pad)
    activation = rows % 4
    routes = Rows(rng, rows, experts, behind)
    x, d = padded(rng.standard_normal((rows, width)), kind, pad), padded(rng.standard_normal((rows, hidden)), kind, pad)
    gate, up = (weights_of(rng, kind, experts, hidden, width, pad) for _ in range(2))
    gate.mul_(width ** -0.5)
    up.mul_(width ** -0.5)
    offsets = routes.offsets.data_ptr()
    h, dx = padded(np.full((rows, hidden), SENTINEL), kind, pad), padded(np.full((rows, width), SENTINEL), kind, pad)
    kept = torch.full((rows, 2 * hidden), SENTINEL, dtype=held_in(kind), device="cuda")
    gated(kind, activation, x, gate, up, offsets, h, kept)
    alone = torch.full((rows, hidden), SENTINEL, dtype=TYPES[kind], device="cuda")
    gated(kind, activation, x, gate, up, offsets, alone, None)
    assert torch.equal(alone, h)
    X, G, U, H, K, D = (exactly(t) for t in (x, gate, up, h, kept, d))
    last = routes.bounds[-1]
    assert np.all(H[last:] == SENTINEL) and np.all(K[last:] == SENTINEL)
    step = u(kind)
    for e in range(experts):
        part = routes.of(e)
        g, v = X[part] @ G[e].T, X[part] @ U[e].T
        g_off, v_off = product_bound(X[part], G[e], kind), product_bound(X[part], U[e], kind)
        within(K[part, :hidden], g, g_off, KEPT[kind])
        within(K[part, hidden:], v, v_off, KEPT[kind])
        # no activation's slope is over 1.13; its own value is off by the exponential's and erfc's few steps: 16, of a value of at most |g|
        a, _ = act(ACTIVATIONS[activation], g)
        a_off = 1.13 * g_off + 16 * step * np.abs(g)
        within(H[part], a * v, a_off * (np.abs(v) + v_off) + (np.abs(a)) * v_off + 2 * step * np.abs(a * v), kind)
    # the gradients, step by step from what the step before left
    for in_place in (False, True) if kind in (cb.FLOAT32, cb.FLOAT64) else (False,):
        held = kept.clone()
        pre = held if in_place else torch.full((rows, 2 * hidden), SENTINEL, dtype=TYPES[kind], device="cuda")
        dgate, dup = (torch.full((experts, hidden * width + pad), SENTINEL, dtype=TYPES[kind], device="cuda").as_strided(gate.shape, gate.stride()) for _ in range(2))
        gated_backward(kind, activation, d, x, gate, up, offsets, held, pre, dx, dgate, dup)
        P, DX, DG, DU = (exactly(t) for t in (pre, dx, dgate, dup))
        g, v = K[:last, :hidden], K[:last, hidden:]
        a, slope = act(ACTIVATIONS[activation], g)
        # a slope's terms are under 1 + |g| and 2 g^2, each a few steps off
        slope_off = 24 * step * (1 + np.abs(g) + g * g)
        within(P[:last, :hidden], D[:last] * v * slope, np.abs(D[:last] * v) * (slope_off + 2 * step * np.abs(slope)), kind)
        within(P[:last, hidden:], D[:last] * a, np.abs(D[:last]) * (16 * step * np.abs(g) + step * np.abs(a)), kind)
        assert np.all(P[last:] == SENTINEL) and np.all(DX[last:] == SENTINEL)
        for e in range(experts):
            part = routes.of(e)
            dg, du = P[part, :hidden], P[part, hidden:]
            both = np.concatenate([dg, du], 1)
            within(DX[part], dg @ G[e] + du @ U[e], product_bound(both, np.concatenate([G[e], U[e]]).T, kind, 64), kind)
            within(DG[e], dg.T @ X[part], product_bound(dg.T, X[part].T, kind), kind)
            within(DU[e], du.T @ X[part], product_bound(du.T, X[part].T, kind), kind)


@pytest.mark.parametrize("activation", ACTIVATIONS, ids=ACTIVATIONS.get)
def test_gated_gradients_against_differences(activation):
    """In 64 bits: a step of 1e-5 in a direction changes the loss by its product with the gradients, to 1e-10 and the rounding of a
    difference of two sums of some thousand terms over 2e-5, 1e-8 of the loss's size."""
    rng = np.random.default_rng(activation)
    kind, rows, width, hidden, experts = cb.FLOAT64, 40, 30, 20, 3
    routes = Rows(rng, rows, experts, 0, 0)
    x, c = padded(rng.standard_normal((rows, width)), kind), padded(rng.standard_normal((rows, hidden)), kind)
    gate, up = (weights_of(rng, kind, experts, hidden, width) * width ** -0.5 for _ in range(2))
    offsets = routes.offsets.data_ptr()

    def loss(x, gate, up, kept=None):
        h = torch.zeros(rows, hidden, dtype=torch.float64, device="cuda")
        gated(kind, activation, x, gate, up, offsets, h, kept)
        return (h * c).sum().item()

    kept = torch.zeros(rows, 2 * hidden, dtype=torch.float64, device="cuda")
    loss(x, gate, up, kept)
    dx, dgate, dup = torch.zeros_like(x), torch.zeros_like(gate), torch.zeros_like(up)
    gated_backward(kind, activation, c, x, gate, up, offsets, kept, kept, dx, dgate, dup)
    step = 1e-5
    size = float((c.abs()).sum())
    for of in range(3):
        at = [x, gate, up]
        direction = torch.from_numpy(rng.standard_normal(tuple(at[of].shape))).cuda()
        direction /= direction.norm()
        ends = []
        for sign in (1, -1):
            moved = list(at)
            moved[of] = at[of] + sign * step * direction
            ends.append(loss(*moved))
        slope = ((dx, dgate, dup)[of] * direction).sum().item()
        # (relu's kink is passed by few of 800 values, by a distance of at most the step)
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 1e-8 * size + (1e-3 if activation == cb.RELU else 0)


@ALL
@pytest.mark.parametrize("activation", ACTIVATIONS, ids=ACTIVATIONS.get)
def test_activations_of_any_size(kind, activation):
    """One input, so that the gate is the source: activations and slopes from very small to infinite."""
    values = np.array([0.0, -0.0, 1e-30, -1e-30, 1e-3, -1e-3, 0.5, -0.5, 1, -1, 3, -3, 9, -9, 20, -20, 60, -60, 100, -100, 3e4, -3e4, np.inf, -np.inf])
    rows = len(values)
    x = padded(values[:, None], kind)
    ones = torch.ones(1, 1, 1, dtype=TYPES[kind], device="cuda")
    small = torch.zeros(1, 1, 1, dtype=TYPES[kind], device="cuda")
    # up values of 1: the weights of a second input that is 1
    x = torch.cat([x, torch.ones_like(x)], 1)
    gate, up = torch.cat([ones, small], 2), torch.cat([small, ones], 2)
    kept = torch.zeros(rows, 2, dtype=held_in(kind), device="cuda")
    h, d = torch.zeros(rows, 1, dtype=TYPES[kind], device="cuda"), torch.ones(rows, 1, dtype=TYPES[kind], device="cuda")
    gated(kind, activation, x, gate, up, 0, h, kept)
    finite = np.isfinite(exactly(x)[:, 0])
    g = exactly(x)[finite, 0]
    a, slope = act(ACTIVATIONS[activation], g)
    within(exactly(h)[finite, 0], a, 16 * u(kind) * np.minimum(np.abs(g), 1 + np.abs(a)) + 1e-37, kind)
    # infinite times 0 is NaN in the product; the gate itself is what a caller's kept values say
    kept[:, 0], kept[:, 1] = x[:, 0], 1
    pre = torch.zeros(rows, 2, dtype=TYPES[kind], device="cuda")
    gated_backward(kind, activation, d, x, gate, up, 0, kept, pre, None, None, None)
    P = exactly(pre)
    within(P[finite, 1], a, 16 * u(kind) * np.minimum(np.abs(g), 1 + np.abs(a)) + 1e-37, kind)
    within(P[finite, 0], slope, 24 * u(kind) * (1 + np.minimum(g * g, 200)) + 1e-37, kind)
    assert P[-2, 0] == 1 and P[-2, 1] == np.inf and P[-1, 0] == 0 and P[-1, 1] == 0
    kept[:, 0] = float("nan")
    gated_backward(kind, activation, d, x, gate, up, 0, kept, pre, None, None, None)
    assert torch.isnan(pre).all()


@ALL
def test_no_rows_no_inputs_no_outputs(kind):
    stream = torch.cuda.current_stream().cuda_stream
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    dw = torch.full((3, 4, 6), SENTINEL, dtype=TYPES[kind], device="cuda")
    cb.multiply_rows_backward(kind, 0, 6, 4, 3, offsets.data_ptr(), 0, 4, 0, 6, 0, 24, 0, 6, dw.data_ptr(), 24, stream)
    assert torch.all(dw == 0)
    du = torch.full_like(dw, SENTINEL)
    dw.fill_(SENTINEL)
    cb.gated_rows_backward(kind, cb.SILU, 0, 6, 4, 3, offsets.data_ptr(), 0, 4, 0, 6, 0, 0, 24, 0, 0, 0, 6, dw.data_ptr(), du.data_ptr(), 24, stream)
    assert torch.all(dw == 0) and torch.all(du == 0)
    # a product over no inputs is 0
    offsets = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    y = torch.full((6, 4), SENTINEL, dtype=TYPES[kind], device="cuda")
    cb.multiply_rows(kind, 6, 0, 4, 3, offsets.data_ptr(), 0, 0, 0, 0, y.data_ptr(), 4, stream)
    assert torch.all(y[:5] == 0) and torch.all(y[5] == SENTINEL)
    y.fill_(SENTINEL)
    cb.gated_rows(kind, cb.GELU, 6, 0, 4, 3, offsets.data_ptr(), 0, 0, 0, 0, 0, y.data_ptr(), 4, 0, stream)
    assert torch.all(y[:5] == 0) and torch.all(y[5] == SENTINEL)
    dx = torch.full((6, 4), SENTINEL, dtype=TYPES[kind], device="cuda")
    cb.multiply_rows_backward(kind, 6, 4, 0, 3, offsets.data_ptr(), 0, 0, 0, 4, 0, 0, dx.data_ptr(), 4, 0, 0, stream)
    assert torch.all(dx[:5] == 0) and torch.all(dx[5] == SENTINEL)


@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 2, 2, 100], [9, 9, 9, 9], [3, 3, 3, 3], [0, 0, 0, 0], [2, 4, 6, 8], [7, -1, 20, -5]], ids=str)
def test_offsets_of_any_value(offsets):
    """What they say inside [0, rows] holds; nothing else is read or written."""
    kind, rows, width, outputs = cb.FLOAT32, 9, 20, 12
    rng = np.random.default_rng(5)
    x, w = padded(rng.standard_normal((rows, width)), kind), weights_of(rng, kind, 3, outputs, width)
    y = torch.full((rows, outputs), SENTINEL, dtype=torch.float32, device="cuda")
    multiply(kind, x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda").data_ptr(), y)
    bounds = np.clip(offsets, 0, rows)
    X, W, Y = exactly(x), exactly(w), exactly(y)
    owners = [[e for e in range(3) if bounds[e] <= r < bounds[e + 1]] for r in range(rows)]
    for r, of in enumerate(owners):
        if not of:
            assert np.all(Y[r] == SENTINEL)
        elif len(of) == 1:
            within(Y[r:r + 1], X[r:r + 1] @ W[of[0]].T, product_bound(X[r:r + 1], W[of[0]], kind), kind)


@ALL
def test_infinities_stay_in_their_rows(kind):
    """What lies behind a row's end, in other rows, other experts and between weights does not reach a result."""
    rng = np.random.default_rng(11)
    rows, width, outputs, experts = 45, 37, 21, 3
    routes = Rows(rng, rows, experts, 4, 0)
    x = padded(rng.standard_normal((rows, width)), kind, 9, float("nan"))
    w = weights_of(rng, kind, experts, outputs, width, 3)
    d = padded(rng.standard_normal((rows, outputs)), kind, 7, float("inf"))
    x[routes.bounds[-1]:], d[routes.bounds[-1]:] = float("nan"), float("inf")
    w[1, 4, 0] = float("inf")
    first, second = routes.of(0), routes.of(1)
    y, dx = padded(np.zeros((rows, outputs)), kind), padded(np.zeros((rows, width)), kind)
    dw = torch.zeros_like(w.contiguous())
    multiply(kind, x, w, routes.offsets.data_ptr(), y)
    cb.multiply_rows_backward(kind, rows, width, outputs, experts, routes.offsets.data_ptr(), d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0),
                              w.data_ptr(), w.stride(0), dx.data_ptr(), dx.stride(0), dw.data_ptr(), dw.stride(0), torch.cuda.current_stream().cuda_stream)
    bad = ~torch.isfinite(y)
    assert not bad[first].any() and bad[second, 4].all() and bad.sum() == second.stop - second.start
    bad = ~torch.isfinite(dx)
    assert not bad[first].any() and bad[second, 0].all() and bad.sum() == second.stop - second.start
    assert torch.isfinite(dw).all()


def far(rows, width, stride, kind, fill):
    """Rows of random values `stride` apart, in memory that is not touched between them."""
    whole = torch.empty((rows - 1) * stride + width, dtype=TYPES[kind], device="cuda")
    t = whole.as_strided((rows, width), (stride, 1))
    t.copy_(fill)
    return t


@pytest.mark.parametrize("stride", [(1 << 22) - 8, (1 << 22) + 3], ids=["copied", "loaded"])
def test_offsets_past_32_bits(stride):
    """1100 rows that far apart: the last ones are 2^32 values and more behind the first."""
    kind, rows, width, outputs, experts = cb.BFLOAT16, 1100, 72, 64, 3
    rng = np.random.default_rng(2)
    routes = Rows(rng, rows, experts, 3, 0)
    x = far(rows, width, stride, kind, torch.from_numpy(rng.standard_normal((rows, width))))
    d = far(rows, outputs, stride, kind, torch.from_numpy(rng.standard_normal((rows, outputs))))
    w = weights_of(rng, kind, experts, outputs, width)
    y, dx = far(rows, outputs, stride, kind, torch.full((rows, outputs), SENTINEL)), far(rows, width, stride, kind, torch.full((rows, width), SENTINEL))
    dw = torch.full_like(w, SENTINEL)
    multiply(kind, x, w, routes.offsets.data_ptr(), y)
    cb.multiply_rows_backward(kind, rows, width, outputs, experts, routes.offsets.data_ptr(), d.data_ptr(), stride, x.data_ptr(), stride, w.data_ptr(),
                              w.stride(0), dx.data_ptr(), stride, dw.data_ptr(), dw.stride(0), torch.cuda.current_stream().cuda_stream)
    X, W, D, Y, DX, DW = (exactly(t) for t in (x, w, d, y, dx, dw))
    for e in range(experts):
        part = routes.of(e)
        within(Y[part], X[part] @ W[e].T, product_bound(X[part], W[e], kind), kind)
        within(DX[part], D[part] @ W[e], product_bound(D[part], W[e].T, kind), kind)
        within(DW[e], D[part].T @ X[part], product_bound(D[part].T, X[part].T, kind), kind)
    assert np.all(Y[routes.bounds[-1]:] == SENTINEL) and np.all(DX[routes.bounds[-1]:] == SENTINEL)


@pytest.mark.parametrize("kind", [cb.FLOAT32, cb.BFLOAT16], ids=NAMES.get)
def test_experts_far_apart(kind):
    """Weights whose experts are 2^31 values apart."""
    rng = np.random.default_rng(4)
    rows, width, outputs, apart = 300, 64, 72, 1 << 31
    routes = Rows(rng, rows, 3, 0, 0)
    values = torch.from_numpy(rng.standard_normal((3, outputs, width))).to(TYPES[kind])
    w, dw = (torch.empty(2 * apart + outputs * width, dtype=TYPES[kind], device="cuda").as_strided((3, outputs, width), (apart, width, 1)) for _ in range(2))
    w.copy_(values)
    x, d = padded(rng.standard_normal((rows, width)), kind), padded(rng.standard_normal((rows, outputs)), kind)
    y = torch.zeros(rows, outputs, dtype=TYPES[kind], device="cuda")
    multiply(kind, x, w, routes.offsets.data_ptr(), y)
    cb.multiply_rows_backward(kind, rows, width, outputs, 3, routes.offsets.data_ptr(), d.data_ptr(), outputs, x.data_ptr(), width, w.data_ptr(), apart, 0, 0,
                              dw.data_ptr(), apart, torch.cuda.current_stream().cuda_stream)
    X, W, D, Y, DW = (exactly(t) for t in (x, w, d, y, dw))
    for e in range(3):
        part = routes.of(e)
        within(Y[part], X[part] @ W[e].T, product_bound(X[part], W[e], kind), kind)
        within(DW[e], D[part].T @ X[part], product_bound(D[part].T, X[part].T, kind), kind)


# rows, width, outputs, experts: each of the kernels for many rows or few tiles
LARGER = [(3000, 136, 512, 2), (4200, 256, 2048, 4), (600, 520, 264, 3), (40, 2080, 512, 4), (14, 1000, 2056, 6), (33, 300, 5000, 2), (2500, 64, 16, 3), (9000, 72, 72, 1),
          (9000, 1032, 64, 2), (300, 1032, 1096, 16)]


@pytest.mark.parametrize("kind", [cb.FLOAT32, cb.FLOAT16, cb.BFLOAT16], ids=NAMES.get)
@pytest.mark.parametrize("shape", LARGER, ids=str)
def test_larger_sizes(kind, shape):
    rows, width, hidden, experts = shape
    rng = np.random.default_rng(rows)
    routes = Rows(rng, rows, experts, 0, 0)
    x, d = padded(rng.standard_normal((rows, width)), kind), padded(rng.standard_normal((rows, hidden)), kind)
    gate, up = (weights_of(rng, kind, experts, hidden, width).mul_(width ** -0.5) for _ in range(2))
    h, y = torch.zeros(rows, hidden, dtype=TYPES[kind], device="cuda"), torch.zeros(rows, hidden, dtype=TYPES[kind], device="cuda")
    kept, pre = torch.zeros(rows, 2 * hidden, dtype=torch.float32, device="cuda"), torch.zeros(rows, 2 * hidden, dtype=TYPES[kind], device="cuda")
    dx, dgate, dup = torch.zeros_like(x), torch.zeros_like(gate), torch.zeros_like(up)
    offsets = routes.offsets.data_ptr()
    multiply(kind, x, gate, offsets, y)
    gated(kind, cb.RELU, x, gate, up, offsets, h, kept)
    gated_backward(kind, cb.RELU, d, x, gate, up, offsets, kept, pre, dx, dgate, dup)
    X, G, U, H, Y, K, P, DX, DG, DU = (exactly(t) for t in (x, gate, up, h, y, kept, pre, dx, dgate, dup))
    for e in range(experts):
        part = routes.of(e)
        g, v = X[part] @ G[e].T, X[part] @ U[e].T
        g_off, v_off = product_bound(X[part], G[e], kind), product_bound(X[part], U[e], kind)
        within(Y[part], g, g_off, kind)
        within(K[part, :hidden], g, g_off, cb.FLOAT32)
        within(K[part, hidden:], v, v_off, cb.FLOAT32)
        a = np.maximum(g, 0)
        within(H[part], a * v, g_off * (np.abs(v) + v_off) + a * v_off + 2 * u(kind) * np.abs(a * v), kind)
        dg, du = P[part, :hidden], P[part, hidden:]
        both = np.concatenate([dg, du], 1)
        within(DX[part], dg @ G[e] + du @ U[e], product_bound(both, np.concatenate([G[e], U[e]]).T, kind, 64), kind)
        within(DG[e], dg.T @ X[part], product_bound(dg.T, X[part].T, kind), kind)
        within(DU[e], du.T @ X[part], product_bound(du.T, X[part].T, kind), kind)


class Block:
    """A step of a routed block, from rows to drawn classes and back to the gradients of what its experts learn."""

    def __init__(self, rows=300, width=128, hidden=192, experts=8, per_row=2, classes=5000, kind=cb.BFLOAT16):
        g = torch.Generator(device="cuda").manual_seed(5)
        t = TYPES[kind]
        self.sizes = rows, width, hidden, experts, per_row, classes, kind

        def randn(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.x, self.router = randn(rows, width).to(t), (randn(1, experts, width) * 0.2).to(t)
        self.gate, self.up = ((randn(experts, hidden, width) * width ** -0.5).to(t) for _ in range(2))
        self.down, self.head = (randn(experts, width, hidden) * hidden ** -0.5).to(t), (randn(1, classes, width) * 0.3).to(t)
        self.uniform, self.dout = torch.rand(rows, generator=g, device="cuda"), randn(rows, width).to(t)
        slots = rows * per_row
        empty = lambda *shape, dtype=t: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
        self.gates, self.ids, self.weights = empty(rows, experts), empty(rows, per_row, dtype=torch.int32), empty(rows, per_row, dtype=torch.float32)
        self.places, self.offsets = empty(slots, dtype=torch.int32), empty(experts + 1, dtype=torch.int32)
        self.work = empty(cb.sort_by_expert_bytes(slots, experts), dtype=torch.uint8)
        self.sorted, self.h, self.y = empty(slots, width), empty(slots, hidden), empty(slots, width)
        self.kept, self.pre = empty(slots, 2 * hidden, dtype=torch.float32), empty(slots, 2 * hidden)
        self.out, self.scores, self.classes, self.shares = empty(rows, width), empty(rows, classes), empty(rows, dtype=torch.int32), empty(rows, dtype=torch.float32)
        self.dy, self.dh, self.dsorted, self.dx = empty(slots, width), empty(slots, hidden), empty(slots, width), empty(rows, width)
        self.ddown, self.dgate, self.dup, self.dweights = (torch.zeros_like(v) for v in (self.down, self.gate, self.up, self.weights))

    def __call__(self):
        rows, width, hidden, experts, per_row, classes, kind = self.sizes
        s, slots, p = torch.cuda.current_stream().cuda_stream, rows * per_row, lambda t: t.data_ptr()  # noqa: E731
        cb.multiply_rows(kind, rows, width, experts, 1, 0, p(self.x), width, p(self.router), 0, p(self.gates), experts, s)
        cb.select_top(kind, rows, experts, p(self.gates), experts, per_row, True, p(self.ids), p(self.weights), s)
        cb.sort_by_expert(slots, experts, p(self.ids), p(self.places), p(self.offsets), p(self.work), self.work.numel(), s)
        cb.dispatch_rows(kind, rows, width, per_row, p(self.x), width, p(self.places), p(self.sorted), slots, width, s)
        cb.gated_rows(kind, cb.SILU, slots, width, hidden, experts, p(self.offsets), p(self.sorted), width, p(self.gate), p(self.up), hidden * width, p(self.h),
                      hidden, p(self.kept), s)
        cb.multiply_rows(kind, slots, hidden, width, experts, p(self.offsets), p(self.h), hidden, p(self.down), hidden * width, p(self.y), width, s)
        cb.combine_rows(kind, rows, width, per_row, p(self.y), slots, width, p(self.places), p(self.weights), p(self.out), width, s)
        cb.multiply_rows(kind, rows, width, classes, 1, 0, p(self.out), width, p(self.head), 0, p(self.scores), classes, s)
        cb.sample_classes(kind, rows, classes, p(self.scores), classes, cb.sampling(), p(self.uniform), p(self.classes), p(self.shares), 0, 0, s)
        # and back
        cb.combine_rows_backward(kind, rows, width, per_row, p(self.dout), width, p(self.y), slots, width, p(self.places), p(self.weights), p(self.dy), width,
                                 p(self.dweights), s)
        cb.multiply_rows_backward(kind, slots, hidden, width, experts, p(self.offsets), p(self.dy), width, p(self.h), hidden, p(self.down), hidden * width,
                                  p(self.dh), hidden, p(self.ddown), hidden * width, s)
        cb.gated_rows_backward(kind, cb.SILU, slots, width, hidden, experts, p(self.offsets), p(self.dh), hidden, p(self.sorted), width, p(self.gate), p(self.up),
                               hidden * width, p(self.kept), p(self.pre), p(self.dsorted), width, p(self.dgate), p(self.dup), hidden * width, s)
        cb.combine_rows(kind, rows, width, per_row, p(self.dsorted), slots, width, p(self.places), 0, p(self.dx), width, s)

    def results(self):
        return [self.out, self.scores, self.classes, self.shares, self.dx, self.dgate, self.dup, self.ddown, self.dweights]


def test_a_block_forward_and_back():
    """All of them as they are used together, against one expression in 64 bits and its derivatives."""
    b = Block()
    b()
    rows, width, hidden, experts, per_row, classes, kind = b.sizes
    x = b.x.double().requires_grad_()
    gate, up, down, weights = (t.double().requires_grad_() for t in (b.gate, b.up, b.down, b.weights))
    out = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    for k in range(per_row):
        for e in range(experts):
            at = torch.nonzero(b.ids[:, k] == e)[:, 0]
            h = torch.nn.functional.silu(x[at] @ gate[e].T) * (x[at] @ up[e].T)
            out = out.index_add(0, at, (h @ down[e].T) * weights[at, k, None])
    gradients = torch.autograd.grad(out, [x, gate, up, down, weights], b.dout.double())
    # In the norm, every rounding to bf16 on the way adds at most half a step, 2^-8, of what it rounds: rows have 3 (h, y, the sum), gradients of
    # rows 5 (dy, dh, the values' gradients, their product, the sum) and of weights up to 4
    for got, want, roundings in [(b.out, out, 3), (b.dx, gradients[0], 5), (b.dgate, gradients[1], 4), (b.dup, gradients[2], 4), (b.ddown, gradients[3], 3),
                                 (b.dweights, gradients[4], 2)]:
        assert (got.double() - want).norm() <= roundings * 2.0 ** -8 * want.norm()
    scores = b.out.double() @ b.head[0].double().T
    assert (b.scores.double() - scores).abs().max() <= 2.0 ** -8 * scores.abs().max() * 1.01
    p = torch.softmax(b.scores.double(), 1)
    drawn = torch.gather(p, 1, b.classes[:, None].long())[:, 0]
    assert torch.allclose(b.shares.double(), drawn, rtol=1e-6, atol=0)
    best_first = torch.sort(b.scores.double(), dim=1, descending=True, stable=True).indices
    sums = torch.cumsum(torch.gather(p, 1, best_first), 1)
    rank = (best_first == b.classes[:, None]).long().argmax(1)
    upto = torch.gather(sums, 1, rank[:, None])[:, 0]
    assert torch.all(upto > b.uniform.double() - 1e-9) and torch.all(upto - drawn <= b.uniform.double() + 1e-9)


def test_a_block_in_a_graph():
    """Captured, and replayed on other values with other work between, it gives what the eager calls give."""
    b = Block(rows=130)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b()
    for step in range(3):
        b.x.mul_(-0.9)
        b.uniform.copy_(torch.rand(130, device="cuda"))
        b()
        expected = [t.clone() for t in b.results()]
        for t in b.results():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(b.results(), expected))


def test_two_blocks_on_streams_of_their_own():
    blocks, streams = [Block(rows=200), Block(rows=400)], [torch.cuda.Stream() for _ in range(2)]
    expected = []
    for b in blocks:
        b()
        torch.cuda.synchronize()
        expected.append([t.clone() for t in b.results()])
        for t in b.results():
            t.zero_()
    torch.cuda.synchronize()
    for b, s in zip(blocks * 3, streams * 3):
        with torch.cuda.stream(s):
            b()
    torch.cuda.synchronize()
    for b, e in zip(blocks, expected):
        assert all(torch.equal(x, y) for x, y in zip(b.results(), e))


def test_more_experts_than_a_wave_has_lanes():
    rng = np.random.default_rng(8)
    kind, rows, width, outputs, experts = cb.BFLOAT16, 5000, 32, 24, 1024
    routes = Rows(rng, rows, experts, 9, 0.5)
    x, w = padded(rng.standard_normal((rows, width)), kind), weights_of(rng, kind, experts, outputs, width)
    y = torch.full((rows, outputs), SENTINEL, dtype=torch.bfloat16, device="cuda")
    multiply(kind, x, w, routes.offsets.data_ptr(), y)
    X, W, Y = exactly(x), exactly(w), exactly(y)
    of = np.searchsorted(routes.bounds[1:], np.arange(rows - 9), side="right")
    expected, bound = np.zeros((rows - 9, outputs)), np.zeros((rows - 9, outputs))
    for r, e in enumerate(of):
        expected[r], bound[r] = W[e] @ X[r], (width + 1) * 2.0 ** -24 * 1.01 * (np.abs(W[e]) @ np.abs(X[r]))
    within(Y[:rows - 9], expected, bound, kind)
    assert np.all(Y[rows - 9:] == SENTINEL)
