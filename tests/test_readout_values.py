"""Group norm and dense layers where values are extreme: arguments of activations far out, infinities, outliers, and gradients of few rows in 16 bits.

Tolerances.  Where nothing is said, 64 * 2^-24 of the magnitudes that go into a result, as for the other tests of these operators, and half a unit in the last place
of a 16-bit type.
"""
import math

import pytest
import torch

EPS = 64 * 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
pytestmark = pytest.mark.gpu

# the activations' derivatives are 0 below and 1 above, to the last bit of float32
FAR = [-3e38, -1e37, -1e30, -1.9e28, -1e20, -1e18, -1e14, -2e13, -1e12, -1e9, -1e4, -200.0, 200.0, 1e4, 1e9, 1e12, 2e13, 1e14, 1e18, 1e20, 1e30, 1e37, 3e38]


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 23, 230])
def test_layer_gradients_far_out(rows, dtype, act):
    """x w = x for k = 1 and w = 1, in rows that hold every value in turn; eight columns, so gx = 8 act'."""
    import gelib_b200 as G
    for at in range(0, len(FAR), min(rows, len(FAR))):
        values = [FAR[(at + i) % len(FAR)] for i in range(rows)]
        x = torch.tensor(values, device="cuda").to(dtype).view(rows, 1).requires_grad_()
        w = torch.ones(1, 8, dtype=dtype, device="cuda")
        bias = torch.zeros(8, dtype=dtype, device="cuda", requires_grad=True)
        y = G.linear(x, w, bias, activation=act)
        gx, gb = torch.autograd.grad(y, (x, bias), torch.ones_like(y))
        slope = (x.detach() > 0).double()
        assert torch.equal(gx.double(), 8 * slope), gx[gx.double() != 8 * slope]
        assert torch.equal(gb.double(), slope.sum().to(dtype).double().expand(8))


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,s", [(6, 1), (5, 4), (9, 37), (2, 3000)])
def test_norm_gradients_far_out(b, s, dtype, act):
    """The bias puts each channel far out, so the gradient is that of no activation for gy with the channels below zero left out."""
    import gelib_b200 as G
    n = 4 * len(FAR)
    gen = torch.Generator(device="cuda").manual_seed(b + s)
    x, gy = (torch.randn(b, s, n, generator=gen, device="cuda").to(dtype) for _ in range(2))
    x.requires_grad_()
    bias = torch.tensor(FAR * 4, device="cuda").to(dtype).requires_grad_()
    gx, gb = torch.autograd.grad(G.group_norm(x, 4, None, bias, activation=act), (x, bias), gy)
    none = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    masked = torch.where(bias.detach() > 0, gy, torch.zeros_like(gy))
    want, wb = torch.autograd.grad(G.group_norm(x, 4, None, none), (x, none), masked)
    half = HALF[dtype] or EPS
    assert ((gx - want).double().abs() <= 2 * half * want.double().abs() + EPS * gy.double().abs().max() * 8).all()
    assert torch.equal(gb, wb)


def classes(t):
    return torch.isnan(t), torch.isposinf(t), torch.isneginf(t)


@pytest.mark.parametrize("m", [3, 40, 300])
@pytest.mark.parametrize("wt", [False, True])
def test_infinities_of_float32_layers(m, wt):
    """An infinity times a number is an infinity of their signs, times 0 it is no number; what it does not meet stays."""
    import gelib_b200 as G
    inf, k, n = math.inf, 70, 48
    gen = torch.Generator(device="cuda").manual_seed(m)
    x, w, gy = (torch.randn(*shape, generator=gen, device="cuda") for shape in ((m, k), (k, n), (m, n)))
    w[:, :8] = 1.0            # numbers of few bits
    w[:, 8:12] = -0.375
    w[5, 12] = 0.0
    w[5, 13:16] = torch.tensor([1.5e-33, -1e-33, 2.0 ** -109], device="cuda")
    w[5, 16:19] = torch.tensor([1e37, -1e37, 2.0 ** 120], device="cuda")
    x[1, 5], x[2, 5], x[2, 6], x[0, 9] = inf, -inf, 2.0, 0.0
    w[9, 20] = inf            # times x[0, 9] = 0
    w[5, 21] = inf            # times both infinities
    gy[0, 3] = -inf
    # kept away from the infinities: rounding of huge sums
    x[x[:, 5].isfinite(), 5] = 1e-3
    w = (w.t().contiguous().t() if wt else w).requires_grad_()
    x.requires_grad_()
    y = G.linear(x, w)
    want = x.detach().double() @ w.detach().double()
    for got, ref in zip(classes(y), classes(want.float())):
        assert torch.equal(got, ref), (got != ref).nonzero()[:8].tolist()
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    for g, ref in ((gx, gy.double() @ w.detach().double().t()), (gw, x.detach().double().t() @ gy.double())):
        for got, r in zip(classes(g), classes(ref.float())):
            assert torch.equal(got, r), (got != r).nonzero()[:8].tolist()
    fine = torch.isfinite(want.float())
    size = x.detach().double().abs() @ w.detach().double().abs()
    assert ((y.double() - want).abs()[fine] <= EPS * size[fine]).all()


@pytest.mark.parametrize("outlier", [100.0, 1000.0, -30000.0])
def test_an_outlier_in_the_first_row_costs_no_digits(outlier):
    """A thread sums 4000 rows of one channel, which is a group of its own."""
    import gelib_b200 as G
    b, s, n = 300, 4000, 257
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(b, s, n, generator=gen, device="cuda")
    x[:, 0] += outlier
    y = G.group_norm(x, n)
    for i in (0, b // 2, b - 1):
        d = x[i].double()
        mean, spread = d.mean(0), d.std(0, unbiased=False)
        rstd = (spread ** 2 + 1e-5).rsqrt()
        want, size = (d - mean) * rstd, (d.abs() + d.abs().mean(0)) * rstd
        off = (y[i].double() - want).abs() / (EPS * (size + want.abs()))
        assert (off <= 1).all(), off.max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 24), (2, 33, 65), (5, 256, 520), (8, 70, 1030)])
def test_gradients_of_few_rows_are_rounded_once(m, k, n, act, wt, dtype):
    """At most eight rows are multiplied in float32: gx and gw are off by their own rounding alone, given x w + bias as it is kept."""
    import gelib_b200 as G
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, gy = (torch.randn(m, q, generator=gen, device="cuda").to(dtype) for q in (k, n))
    w = (torch.randn(k, n, generator=gen, device="cuda") * k ** -0.5).to(dtype)
    w = w.t().contiguous().t() if wt else w
    kept = G.linear(x, w)     # x w, rounded as it is for the backward call
    x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(G.linear(x, w, activation=act), (x, w), gy)
    z = kept.double().requires_grad_()
    f = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act](z)
    gz, = torch.autograd.grad(f, z, gy.double())
    slope = gy.double().abs() * 1.2 * (1 + z.detach().abs())   # what an error of a few units in float32 of the derivative's terms does
    x64, w64 = x.detach().double(), w.detach().double()
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    for got, want, size in ((gx, gz @ w64.t(), slope @ w64.abs().t()), (gw, x64.t() @ gz, x64.abs().t() @ slope)):
        off, allowed = (got.double() - want).abs(), EPS * size + HALF[dtype] * (want.abs() + EPS * size) + tiny
        assert (off <= allowed).all(), (off / allowed).max().item()


@pytest.mark.parametrize("m", [5, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_an_empty_sum(m, dtype):
    """k = 0: y = act(bias) + residual, and the bias's gradient is a sum over the rows."""
    import gelib_b200 as G
    n = 12
    gen = torch.Generator(device="cuda").manual_seed(m)
    x, w = torch.zeros(m, 0, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(0, n, dtype=dtype, device="cuda", requires_grad=True)
    bias, gy = (torch.randn(*shape, generator=gen, device="cuda").to(dtype) for shape in ((n,), (m, n)))
    bias.requires_grad_()
    y = G.linear(x, w, bias, activation="silu")
    gx, gw, gb = torch.autograd.grad(y, (x, w, bias), gy)
    z = bias.detach().double().requires_grad_()
    f = torch.nn.functional.silu(z)
    slope, = torch.autograd.grad(f.sum(), z)
    assert ((y.double() - f.detach()).abs() <= (EPS + HALF[dtype]) * f.detach().abs() + EPS).all()
    want, size = slope * gy.double().sum(0), gy.double().abs().sum(0) * 1.2 * (1 + z.detach().abs())
    assert ((gb.double() - want).abs() <= EPS * size + HALF[dtype] * want.abs()).all()
    assert gx.shape == (m, 0) and gw.shape == (0, n)
