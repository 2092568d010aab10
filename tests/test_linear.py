"""The dense layer and its gradients against float64, over sizes that do not fill a tile, single rows, long sums, layouts, alignments and types.

Tolerances.  A sum of products is off by its roundings, which mostly cancel, and in float32 by 2^-22 of each product, whose
factors are split in three: 64 * 2^-24 of the sum of magnitudes covers both, with the few units in the last place of an activation.  A 16-bit result is
rounded by half a unit in its last place; so are, on the way back, x w + bias where it was kept, and gz before its products.
"""
import math

import pytest
import torch

EPS = 64 * 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
SIZES = [(1, 1, 1), (1, 1280, 1280), (2, 7168, 33), (3, 16, 8), (7, 33, 65), (16, 256, 512), (33, 7, 1), (64, 64, 64), (130, 100, 257), (257, 129, 129),
         (777, 204, 131), (128, 4096, 24), (300, 64, 2000), (1000, 1280, 512), (5000, 112, 112), (70000, 6, 5), (512, 512, 512)]


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def reference(x, w, bias, residual, act, gy):
    """(result, allowed error) of y, gx, gw, gb in float64."""
    half, tiny = HALF[x.dtype], TINY[x.dtype]
    x, w, gy = x.double(), w.double(), gy.double()
    z = x @ w + (0 if bias is None else bias.double())
    off_z = EPS * (x.abs() @ w.abs() + (0 if bias is None else bias.double().abs()) + z.abs())
    z.requires_grad_()
    y = act64(z, act)
    gz, = torch.autograd.grad(y, z, gy)
    z, y = z.detach(), y.detach()
    off_y = 1.2 * off_z
    if residual is not None:
        y = y + residual.double()
        off_y = off_y + EPS * residual.double().abs()

    def stored(v, off):
        return v, off + half * (v.abs() + off) + tiny

    # slopes of the activations are at most 1.2, and change by at most 1.2 per unit of z
    off_gz = EPS * gy.abs()
    if act is not None:
        off_gz = off_gz + gy.abs() * 1.2 * (off_z + half * z.abs() + tiny)
        off_gz = off_gz + half * (gz.abs() + off_gz) + tiny
    size = gz.abs() + off_gz
    return (stored(y, off_y), stored(gz @ w.t(), off_gz @ w.abs().t() + EPS * (size @ w.abs().t())),
            stored(x.t() @ gz, x.abs().t() @ off_gz + EPS * (x.abs().t() @ size)), stored(gz.sum(0), off_gz.sum(0) + EPS * size.sum(0)))


def near(got, want, what):
    value, allowed = want
    off = (got.double() - value).abs()
    assert got.shape == value.shape and (off <= allowed).all(), (what, (off / allowed).max().item())


def make(m, k, n, dtype, wt=False, offset=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)

    def one(r, c, scale=1.0, extra=0):
        flat = (torch.randn(r * (c + extra) + offset, generator=gen, device="cuda") * scale).to(dtype)
        return flat[offset:].view(r, c + extra)[:, :c]

    w = one(n, k, k ** -0.5, pad).t() if wt else one(k, n, k ** -0.5, pad)
    return one(m, k, extra=pad), w, one(1, n, 0.5)[0], one(m, n), one(m, n)


def run(G, x, w, bias, residual, act, gy):
    leaves = [t.detach().requires_grad_() for t in (x, w, bias, residual) if t is not None]
    it = iter(leaves)
    x, w, bias, residual = (next(it) if t is not None else None for t in (x, w, bias, residual))
    y = G.linear(x, w, bias, residual, act)
    grads = iter(torch.autograd.grad(y, leaves, gy))
    gx, gw = next(grads), next(grads)
    gb = next(grads) if bias is not None else None
    if residual is not None:
        assert torch.equal(next(grads), gy)
    return y, gx, gw, gb


def away_from_the_kink(x, w, bias, act, gy):
    if act != "relu":
        return gy
    z = x.double() @ w.double() + bias.double()
    return torch.where(z.abs() < 1e-2, 0.0, gy.double()).to(gy.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["plain", "transposed", "odd", "odd transposed"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_against_float64(m, k, n, layout, dtype):
    """odd: one element off their alignment, rows three elements longer than the matrix."""
    import gelib_b200 as G
    odd = "odd" in layout
    x, w, bias, residual, gy = make(m, k, n, dtype, "transposed" in layout, offset=1 if odd else 0, pad=3 if odd else 0)
    acts = [None, "relu", "silu", "gelu_tanh"]
    for act in acts if m * k * n < 300000 else [acts[(m + k + n + odd) % 4]]:
        g = away_from_the_kink(x, w, bias, act, gy)
        got = run(G, x, w, bias, residual, act, g)
        for t, want, what in zip(got, reference(x, w, bias, residual, act, g), ("y", "gx", "gw", "gb")):
            assert t.dtype == dtype
            near(t, want, (what, act))


@pytest.mark.gpu
@pytest.mark.parametrize("has_bias", [False, True])
@pytest.mark.parametrize("has_residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(1, 100, 72), (9, 100, 72), (200, 100, 72), (200, 2048, 72)])
def test_without_bias_or_residual(m, k, n, dtype, has_residual, has_bias):
    import gelib_b200 as G
    x, w, bias, residual, gy = make(m, k, n, dtype)
    bias, residual = bias if has_bias else None, residual if has_residual else None
    for act in (None, "silu"):
        got = run(G, x, w, bias, residual, act, gy)
        for t, want, what in zip(got, reference(x, w, bias, residual, act, gy), ("y", "gx", "gw", "gb")):
            if t is not None:
                near(t, want, what)


@pytest.mark.gpu
@pytest.mark.parametrize("m", list(range(1, 20)) + [31, 32, 33, 63, 65, 127, 128, 129])
def test_every_small_number_of_rows(m):
    import gelib_b200 as G
    for dtype in (torch.float32, torch.bfloat16):
        for wt in (False, True):
            x, w, bias, residual, _ = make(m, 264, 136, dtype, wt)
            with torch.no_grad():
                y = G.linear(x, w, bias, residual, "silu")
            near(y, reference(x, w, bias, residual, "silu", torch.zeros_like(y))[0], (dtype, wt))


@pytest.mark.gpu
def test_float32_keeps_its_precision_and_range():
    """Exact results where every product and sum is one of float32's, over factors of all sizes."""
    import gelib_b200 as G
    gen = torch.Generator().manual_seed(0)
    for e in (-60, -20, 0, 20, 60):
        x = torch.zeros(200, 128)
        x[torch.arange(200), torch.randint(128, (200,), generator=gen)] = torch.randn(200, generator=gen) * 2.0 ** e   # one term a row
        w = 2.0 ** torch.randint(-3, 3, (128, 130), generator=gen).float()
        y = G.linear(x.cuda(), w.cuda())
        assert torch.equal(y.cpu(), (x.double() @ w.double()).float()), e
    x = torch.full((130, 64), 3.0e38 / 64).cuda()
    assert torch.isfinite(G.linear(x, torch.ones(64, 8, device="cuda"))).all()
    big = torch.zeros(130, 64).cuda()
    big[:, 0] = 3.4028234e38
    assert torch.equal(G.linear(big, torch.eye(64, 8, device="cuda")), big[:, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_that_are_no_numbers_stay_in_their_rows_and_columns(dtype):
    import gelib_b200 as G
    for m in (3, 200):
        x, w, bias, residual, gy = make(m, 96, 80, dtype)
        clean = run(G, x, w, bias, residual, "silu", gy)
        for bad in (float("nan"), float("inf")):
            x2, gy2 = x.clone(), gy.clone()
            x2[1, 5] = bad
            got = run(G, x2, w, bias, residual, "silu", gy2)
            rows = torch.arange(m, device="cuda") != 1
            assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows])
            assert not torch.isfinite(got[0][1]).all()
            gy2[2, 7] = bad
            got = run(G, x, w, bias, residual, "silu", gy2)
            cols = torch.arange(80, device="cuda") != 7
            assert torch.equal(got[2][:, cols], clean[2][:, cols]) and torch.equal(got[3][cols], clean[3][cols])
            assert not torch.isfinite(got[2][:, 7]).any()


@pytest.mark.gpu
def test_large_sums_before_an_activation_have_finite_gradients():
    """float16: x w beyond that type's range, on the flat side of the activation."""
    import gelib_b200 as G
    for act in ("relu", "silu", "gelu_tanh"):
        x = torch.full((2, 64), 100.0, device="cuda", dtype=torch.float16)
        w = torch.full((64, 8), -100.0, device="cuda", dtype=torch.float16)
        y, gx, gw, _ = run(G, x, w, None, None, act, torch.ones(2, 8, device="cuda", dtype=torch.float16))
        for t in (y, gx, gw):
            assert (t == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(2, 5, 3), (40, 24, 17)])
def test_gradients_against_differences(m, k, n):
    """Differences of the operator itself, in float32: a step of 2^-6 leaves its square, and 2^-24 / 2^-6 of the sums."""
    import gelib_b200 as G
    x, w, bias, residual, gy = make(m, k, n, torch.float32)
    _, gx, gw, gb = run(G, x, w, bias, residual, "gelu_tanh", gy)
    step = 2.0 ** -6
    for i, grad in enumerate((gx, gw, gb)):
        d = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        d = d / d.abs().max()
        sides = []
        for sign in (1, -1):
            a = [x, w, bias]
            a[i] = a[i] + sign * step * d
            sides.append((G.linear(a[0], a[1], a[2], residual, "gelu_tanh").double() * gy.double()).sum())
        slope, want = (sides[0] - sides[1]) / (2 * step), (grad.double() * d.double()).sum()
        size = gy.abs().double().sum() * (1 if i == 2 else k * d.abs().double().mean())
        assert abs(slope - want) <= 20 * step ** 2 * size + 64 * 2.0 ** -24 / step * size


@pytest.mark.gpu
def test_shapes_strides_streams_and_repeats():
    import gelib_b200 as G
    x, w, bias, residual, gy = make(60, 48, 40, torch.float32)
    want = G.linear(x, w, bias, residual, "silu")
    assert torch.equal(G.linear(x.view(3, 4, 5, 48), w, bias, residual.view(3, 4, 5, 40), "silu"), want.view(3, 4, 5, 40))
    assert torch.equal(G.linear(x[7], w, bias), G.linear(x[7:8], w, bias)[0])
    assert torch.equal(G.linear(x.t().contiguous().t(), w, bias, residual, "silu"), want)
    assert torch.equal(G.linear(x, w.t().contiguous().t(), bias, residual.t().contiguous().t(), "silu"), want)
    assert torch.equal(G.linear(torch.view_as_complex(torch.stack([x, x], -1)).real, w, bias, residual, "silu"), want)
    assert torch.equal(G.linear(x[:1].expand(60, 48), w, bias), G.linear(x[:1].expand(60, 48).contiguous(), w, bias))
    assert torch.equal(G.linear(x, w[:, :1].expand(48, 40), bias), G.linear(x, w[:, :1].expand(48, 40).contiguous(), bias))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = G.linear(x, w, bias, residual, "silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    for m, k, n in ((3000, 200, 100), (20000, 40, 24), (4, 2000, 300)):
        for dtype in (torch.float32, torch.bfloat16):
            args = make(m, k, n, dtype)
            first, second = (run(G, *args[:4], "silu", args[4]) for _ in range(2))
            assert all(torch.equal(p, q) for p, q in zip(first, second))


@pytest.mark.gpu
def test_only_some_gradients_and_broadcast_parameters():
    import gelib_b200 as G
    x, w, bias, residual, gy = make(70, 48, 40, torch.float32)
    all_of = run(G, x, w, bias, residual, "silu", gy)[1:]
    for i, want in enumerate(all_of):
        a = [x.clone(), w.clone(), bias.clone()]
        a[i].requires_grad_()
        G.linear(a[0], a[1], a[2], residual, "silu").backward(gy)
        assert torch.equal(a[i].grad, want)
    r = residual.clone().requires_grad_()
    G.linear(x, w, bias, r, "silu").backward(gy)
    assert torch.equal(r.grad, gy)
    one = torch.tensor(0.5, device="cuda", requires_grad=True)
    G.linear(x, w, one.expand(40), residual[:1].expand(70, 40), "silu").backward(gy)
    want = run(G, x, w, torch.full((40,), 0.5, device="cuda"), residual[:1].expand(70, 40).contiguous(), "silu", gy)[3].sum()
    assert torch.allclose(one.grad, want, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_empty_sizes():
    import gelib_b200 as G
    for m, k, n in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (0, 0, 0)):
        x, w, b = (torch.ones(s, device="cuda", requires_grad=True) for s in ((m, k), (k, n), (n,)))
        y = G.linear(x, w, b, activation="silu")
        assert y.shape == (m, n) and torch.allclose(y, torch.nn.functional.silu(torch.ones(m, n, device="cuda")) if k == 0 else y)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert gx.shape == x.shape and gw.shape == w.shape and gb.shape == b.shape
        if m == 0 or n == 0:
            assert (gx == 0).all() and (gw == 0).all() and (gb == 0).all()


@pytest.mark.gpu
def test_module():
    import gelib_b200 as G
    layer = G.Linear(24, 24, activation="silu", device="cuda")
    x = torch.randn(5, 24, device="cuda")
    y = layer(x, x)
    y.sum().backward()
    assert layer.weight.grad is not None and layer.bias.grad is not None
    with torch.no_grad():
        assert torch.equal(layer(x, x), y)


def test_cpu_tensors_are_refused(cabi):
    import gelib_b200 as G
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        G.linear(torch.zeros(2, 8), torch.zeros(8, 4))


REFUSALS = {
    "sizes": ("n_in", dict(x=torch.zeros(2, 7))),
    "w of three dimensions": ("n_in", dict(w=torch.zeros(1, 8, 4))),
    "bias": (r"bias must have shape \(4,\)", dict(bias=torch.zeros(8))),
    "residual": (r"residual must have shape \(2, 4\)", dict(residual=torch.zeros(1, 4))),
    "type of w": ("w must be of x's type", dict(w=torch.zeros(8, 4, dtype=torch.bfloat16))),
    "double": ("float32, bfloat16 or float16", dict(x=torch.zeros(2, 8, dtype=torch.float64))),
    "complex": ("float32, bfloat16 or float16", dict(x=torch.zeros(2, 8, dtype=torch.complex64))),
    "activation": ("activation is one of", dict(activation="gelu")),
}


@pytest.mark.gpu
@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    import gelib_b200 as G
    match, change = REFUSALS[what]
    a = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in {**dict(x=torch.zeros(2, 8), w=torch.zeros(8, 4)), **change}.items()}
    with pytest.raises((RuntimeError, ValueError), match=match):
        G.linear(a.pop("x"), a.pop("w"), **a)


@pytest.mark.gpu
def test_a_device_is_asked_of_all(cabi):
    import gelib_b200 as G
    with pytest.raises(RuntimeError, match="bias must be of x's type on x's device"):
        G.linear(torch.zeros(2, 8, device="cuda"), torch.zeros(8, 4, device="cuda"), torch.zeros(4))


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported():
    """The tensor-core product gives up when a test makes its first waits run out (no fault is involved), and the next call says so."""
    import gelib_b200 as G
    x, w, _, _, _ = make(512, 512, 512, torch.bfloat16)
    good = G.linear(x, w)
    G._lib.set_option("inject_timeout", "1")
    try:
        G.linear(x, w)
        torch.cuda.synchronize()
    finally:
        G._lib.set_option("inject_timeout", "0")
    with pytest.raises(RuntimeError, match="gemm_tc_kernel"):
        G.linear(x, w)
    assert torch.equal(G.linear(x, w), good)
    torch.cuda.synchronize()
    G._lib.async_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sums_and_many_tiles(dtype):
    """Sums of 20000 products, split and whole; more tiles than SMs; one tile of one column."""
    import gelib_b200 as G
    for m, k, n in ((300, 20000, 40), (5000, 64, 1100), (129, 20000, 1), (40000, 20, 9)):
        x, w, bias, residual, gy = make(m, k, n, dtype)
        got = run(G, x, w, bias, residual, "silu", gy)
        for t, want, what in zip(got, reference(x, w, bias, residual, "silu", gy), ("y", "gx", "gw", "gb")):
            near(t, want, (what, m, k, n))


@pytest.mark.gpu
def test_without_the_native_host_side(monkeypatch):
    import gelib_b200 as G
    for m, k, n, dtype, wt in ((5, 12, 9, torch.float32, False), (5, 12, 9, torch.float32, True), (300, 200, 100, torch.bfloat16, True), (300, 200, 100, torch.float32, False)):
        x, w, bias, residual, gy = make(m, k, n, dtype, wt)
        want = run(G, x, w, bias, residual, "silu", gy)
        with monkeypatch.context() as patch:
            patch.setattr(G._lib, "_native", G._lib._Declines())
            got = run(G, x, w, bias, residual, "silu", gy)
            plain = G.linear(x.view(1, m, k), w, bias, residual.view(1, m, n), "silu")
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(plain[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_a_second_derivative_is_refused(native, monkeypatch):
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(G.linear(x, torch.randn(8, 4, device="cuda"), activation="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
