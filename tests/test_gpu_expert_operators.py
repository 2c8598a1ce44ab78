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
