"""The experts' products and their gradients at sizes that take the kernels for many tiles, against torch's in 64 bits. Needs an MI355X.

Tolerances count roundings of half a step: U is half a step of what sums are held in (2^-24, 2^-53 for 64-bit values). A sum of K
products, each and each addition rounded, is off by at most (K + 1) U times the sum of the products' sizes; for 64-bit values the
sum that it is compared with is off by as much."""
import numpy as np
import pytest
import torch

import catboost_amd as cb

pytestmark = pytest.mark.gpu

TYPES = {cb.FLOAT64: torch.float64, cb.FLOAT32: torch.float32, cb.FLOAT16: torch.float16, cb.BFLOAT16: torch.bfloat16}
NAMES = {cb.FLOAT64: "f64", cb.FLOAT32: "f32", cb.FLOAT16: "f16", cb.BFLOAT16: "bf16"}
HALF = {cb.FLOAT64: 2.0 ** -53, cb.FLOAT32: 2.0 ** -24, cb.FLOAT16: 2.0 ** -11, cb.BFLOAT16: 2.0 ** -8}
TINY = {cb.FLOAT64: 0.0, cb.FLOAT32: 2.0 ** -150, cb.FLOAT16: 2.0 ** -25, cb.BFLOAT16: 2.0 ** -134}
KEPT = {cb.FLOAT64: cb.FLOAT64, cb.FLOAT32: cb.FLOAT32, cb.FLOAT16: cb.FLOAT32, cb.BFLOAT16: cb.FLOAT32}
SENTINEL = 7.0


def u(kind):
    return 2.0 ** -53 if kind == cb.FLOAT64 else 2.0 ** -24


def table(shape, kind, pad=0, values=None):
    """Values as the first columns of a wider table of sentinels, and the whole table."""
    wide = torch.full(shape[:-1] + (shape[-1] + pad,), SENTINEL, dtype=TYPES[kind], device="cuda")
    t = wide[..., :shape[-1]]
    if values is not None:
        t.copy_(values)
    return t, wide


def weights(experts, outputs, width, kind, pad, values=None):
    """Experts' weights with `pad` sentinels behind each."""
    t, wide = table((experts, outputs * width), kind, pad, None if values is None else values.reshape(experts, -1))
    return t.as_strided((experts, outputs, width), (outputs * width + pad, width, 1)), wide


def outside(wide, width, rows):
    """What no call may write: behind the rows' ends, and the rows from `rows` on."""
    return torch.cat([wide[:, width:].flatten(), wide[rows:].flatten()])


def within(got, expected, bound, kind):
    """|got - expected| <= bound + one rounding to the type."""
    assert got.shape == expected.shape
    if got.numel():
        allowed = bound + HALF[kind] * (expected.abs() + bound) + TINY[kind]
        over = (got.to(torch.float64) - expected).abs() - allowed
        assert not torch.any(over > 0) and not torch.any(torch.isnan(over)), "off by %g more than allowed" % over.max().item()


def product(a, b, kind, extra=0):
    """a [m, k] times b [n, k] in 64 bits, and what a sum in the type's accumulator may be off by."""
    terms = (a.shape[1] + 1 + extra) * (2 if kind == cb.FLOAT64 else 1)
    return a @ b.T, terms * u(kind) * 1.01 * (a.abs() @ b.abs().T)


def act(activation, x):
    """act(x) and its derivative."""
    if activation == cb.SILU:
        y = torch.sigmoid(x)
        return x * y, y * (1 + x * (1 - y))
    if activation == cb.GELU:
        y = torch.erfc(-x * 0.5 ** 0.5) / 2
        return x * y, y + x * torch.exp(-x * x / 2) / (2 * np.pi) ** 0.5
    if activation == cb.GELU_TANH:
        c = (2 / np.pi) ** 0.5
        t = torch.tanh(c * (x + 0.044715 * x ** 3))
        return x * (1 + t) / 2, (1 + t) / 2 + x * (1 - t * t) / 2 * c * (1 + 3 * 0.044715 * x * x)
    return torch.relu(x), (x > 0).to(x.dtype)


class Case:
    def __init__(self, kind, rows, width, hidden, experts, pad, behind, alone=None):
        g = torch.Generator(device="cuda").manual_seed(rows + width)
        self.kind, self.sizes = kind, (rows, width, hidden, experts)
        counts = torch.zeros(experts, dtype=torch.int64)
        if alone is not None:  # a few experts have all rows
            counts[alone] = (rows - behind) // len(alone)
        else:
            counts += (rows - behind) // experts
            counts[:-1] += torch.arange(experts - 1) % 5 * 3 - 6 if rows > 40 * experts else 0
        counts[alone[-1] if alone is not None else -1] += rows - behind - counts.sum()
        self.bounds = [0] + torch.cumsum(counts, 0).tolist()
        self.offsets = torch.tensor(self.bounds, dtype=torch.int32, device="cuda")
        self.last, self.pad = self.bounds[-1], pad

        def randn(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.x, _ = table((rows, width), kind, pad, randn(rows, width))
        self.d, _ = table((rows, hidden), kind, pad, randn(rows, hidden))
        # what belongs to no expert must not show anywhere
        self.x[self.last:], self.d[self.last:] = float("nan"), float("inf")
        self.gate, _ = weights(experts, hidden, width, kind, pad, randn(experts, hidden, width) * width ** -0.5)
        self.up, _ = weights(experts, hidden, width, kind, pad, randn(experts, hidden, width) * width ** -0.5)

    def parts(self):
        return [(e, slice(self.bounds[e], self.bounds[e + 1])) for e in range(self.sizes[3]) if self.bounds[e] < self.bounds[e + 1]]

    def check_plain(self):
        kind, (rows, width, hidden, experts), pad = self.kind, self.sizes, self.pad
        s, offsets = torch.cuda.current_stream().cuda_stream, self.offsets.data_ptr()
        runs = []
        for _ in range(2):
            (y, wide_y), (dx, wide_x), (dw, wide_w) = table((rows, hidden), kind, pad), table((rows, width), kind, pad), weights(experts, hidden, width, kind, pad)
            cb.multiply_rows(kind, rows, width, hidden, experts, offsets, self.x.data_ptr(), width + pad, self.gate.data_ptr(), self.gate.stride(0), y.data_ptr(),
                             hidden + pad, s)
            cb.multiply_rows_backward(kind, rows, width, hidden, experts, offsets, self.d.data_ptr(), hidden + pad, self.x.data_ptr(), width + pad,
                                      self.gate.data_ptr(), self.gate.stride(0), dx.data_ptr(), width + pad, dw.data_ptr(), dw.stride(0), s)
            assert torch.all(outside(wide_y, hidden, self.last) == SENTINEL) and torch.all(outside(wide_x, width, self.last) == SENTINEL)
            assert torch.all(wide_w[:, hidden * width:] == SENTINEL)
            runs.append((wide_y, wide_x, wide_w))
        assert all(torch.equal(a, b) for a, b in zip(*runs))
        there = set()
        for e, part in self.parts():
            x, d, w = self.x[part].double(), self.d[part].double(), self.gate[e].double()
            within(y[part], *product(x, w, kind), kind)
            within(dx[part], *product(d, w.T, kind), kind)
            within(dw[e], *product(d.T, x.T, kind), kind)
            there.add(e)
        assert all(torch.all(dw[e] == 0) for e in range(experts) if e not in there)

    def check_gated(self, activation):
        kind, (rows, width, hidden, experts), pad = self.kind, self.sizes, self.pad
        s, offsets, step = torch.cuda.current_stream().cuda_stream, self.offsets.data_ptr(), u(kind)
        weight_args = self.gate.data_ptr(), self.up.data_ptr(), self.gate.stride(0)
        runs = []
        for _ in range(2):
            h, wide_h = table((rows, hidden), kind, pad)
            alone, wide_alone = table((rows, hidden), kind, pad)
            kept, pre = table((rows, 2 * hidden), KEPT[kind])[0], table((rows, 2 * hidden), kind)[0]
            dx, wide_x = table((rows, width), kind, pad)
            (dgate, wide_gate), (dup, wide_up) = (weights(experts, hidden, width, kind, pad) for _ in range(2))
            for result, keep in ((h, kept.data_ptr()), (alone, 0)):
                cb.gated_rows(kind, activation, rows, width, hidden, experts, offsets, self.x.data_ptr(), width + pad, *weight_args, result.data_ptr(), hidden + pad,
                              keep, s)
            cb.gated_rows_backward(kind, activation, rows, width, hidden, experts, offsets, self.d.data_ptr(), hidden + pad, self.x.data_ptr(), width + pad,
                                   *weight_args, kept.data_ptr(), pre.data_ptr(), dx.data_ptr(), width + pad, dgate.data_ptr(), dup.data_ptr(), dgate.stride(0), s)
            assert torch.equal(wide_h, wide_alone)
            assert torch.all(outside(wide_h, hidden, self.last) == SENTINEL) and torch.all(outside(wide_x, width, self.last) == SENTINEL)
            assert torch.all(kept[self.last:] == SENTINEL) and torch.all(pre[self.last:] == SENTINEL)
            assert torch.all(wide_gate[:, hidden * width:] == SENTINEL) and torch.all(wide_up[:, hidden * width:] == SENTINEL)
            runs.append((wide_h, kept, pre, wide_x, wide_gate, wide_up))
        assert all(torch.equal(a, b) for a, b in zip(*runs))
        there = set()
        for e, part in self.parts():
            x, d, gate, up = self.x[part].double(), self.d[part].double(), self.gate[e].double(), self.up[e].double()
            (g, g_off), (v, v_off) = product(x, gate, kind), product(x, up, kind)
            within(kept[part, :hidden], g, g_off, KEPT[kind])
            within(kept[part, hidden:], v, v_off, KEPT[kind])
            # no activation's slope is over 1.13; its own value is off by the exponential's and erfc's few steps: 16, of a value of at most |g|
            # (and for 64 bits by as many of what it is compared with)
            few = 2 if kind == cb.FLOAT64 else 1
            a, _ = act(activation, g)
            a_off = 1.13 * g_off + 16 * few * step * g.abs()
            within(h[part], a * v, a_off * (v.abs() + v_off) + a.abs() * v_off + 2 * few * step * (a * v).abs(), kind)
            # the gradients, step by step from what the step before left; a slope's terms are under 1 + |g| and 2 g^2, each a few steps off
            g, v = kept[part, :hidden].double(), kept[part, hidden:].double()
            a, slope = act(activation, g)
            slope_off = 24 * few * step * (1 + g.abs() + g * g)
            within(pre[part, :hidden], d * v * slope, (d * v).abs() * (slope_off + 2 * few * step * slope.abs()), kind)
            within(pre[part, hidden:], d * a, d.abs() * (16 * few * step * g.abs() + few * step * a.abs()), kind)
            dg, du = pre[part, :hidden].double(), pre[part, hidden:].double()
            within(dx[part], *product(torch.cat([dg, du], 1), torch.cat([gate, up]).T, kind, 64), kind)
            within(dgate[e], *product(dg.T, x.T, kind), kind)
            within(dup[e], *product(du.T, x.T, kind), kind)
            there.add(e)
        assert all(torch.all(dgate[e] == 0) and torch.all(dup[e] == 0) for e in range(experts) if e not in there)


# rows, width, outputs, experts of 16-bit products at multiples of 16 bytes: tiles of 256 x 256 with ends of rows, columns and k inside a tile; inputs'
# gradients by 128 x 256 and by 128 x 128; weights' gradients by 128 x 256 and by 128 x 128; forward by 64 x 128
COPIED = [(4400, 72, 13064, 4), (2100, 136, 36872, 1), (1400, 5512, 72, 3), (1400, 1400, 136, 3), (700, 1800, 2056, 4), (900, 704, 1096, 4), (60, 200, 40008, 2)]
# the same for any type at any address: tiles of 128 x 128 of each form, of 64 x 64, and shared ones
LOADED = [(1500, 71, 4231, 3), (1500, 4231, 67, 3), (600, 1303, 1001, 5), (400, 803, 901, 3), (63, 97, 6151, 1), (50, 2001, 75, 2)]


@pytest.mark.parametrize("kind", [cb.FLOAT16, cb.BFLOAT16], ids=NAMES.get)
@pytest.mark.parametrize("shape", COPIED, ids=str)
@pytest.mark.parametrize("pad", [0, 8])
def test_products_of_many_tiles(kind, shape, pad):
    case = Case(kind, *shape, pad, 5)
    case.check_plain()
    if shape[2] < 20000:
        case.check_gated(shape[0] // 100 % 4)


@pytest.mark.parametrize("kind", [cb.FLOAT16, cb.BFLOAT16], ids=NAMES.get)
@pytest.mark.parametrize("activation", [cb.SILU, cb.GELU_TANH], ids=["silu", "gelu_tanh"])
def test_gated_rows_by_the_largest_tiles(kind, activation):
    """From 2048 inputs on: 86 of 128 columns times 6 of 256 rows for each of two experts."""
    Case(kind, 2600, 2056, 10952, 2, 8, 11).check_gated(activation)


@pytest.mark.parametrize("kind", list(TYPES), ids=NAMES.get)
@pytest.mark.parametrize("shape", LOADED, ids=str)
@pytest.mark.parametrize("pad", [0, 3])
def test_products_of_many_tiles_at_any_address(kind, shape, pad):
    case = Case(kind, *shape, pad, 4)
    case.check_plain()
    case.check_gated(shape[0] // 50 % 4)


@pytest.mark.parametrize("kind", list(TYPES), ids=NAMES.get)
@pytest.mark.parametrize("rows,experts,alone", [(2048, 128, [3, 60, 61, 127]), (3000, 1000, [999]), (5000, 7, [2])], ids=str)
def test_few_experts_have_all_rows(kind, rows, experts, alone):
    """Kernels are chosen by what an expert has on average, and right for any share of them."""
    for width, hidden, pad in ((264, 136, 0), (75, 41, 1)):
        case = Case(kind, rows, width, hidden, experts, pad, 9, alone)
        case.check_plain()
        case.check_gated(cb.GELU)
