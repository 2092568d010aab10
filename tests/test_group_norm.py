"""Group norm with an activation and its gradients against float64, over the ways that the kernels hold a sample (registers, shared
memory, two passes), odd sizes, alignments and types.

Tolerances.  Each result is a handful of float32 operations on the inputs, a mean and a variance; a mean's sums are chains of some hundred
additions whose roundings mostly cancel, the exponential and the quotients have a few units in the last place.  64 * 2^-24 of the magnitudes that go
into a result covers them; a 16-bit result is rounded once more, by half a unit in its last place.
"""
import math

import pytest
import torch

EPS = 64 * 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a unit in the last of 8 and of 11 bits
SIZES = [(1, 1, 1, 1), (3, 1, 24, 8), (64, 1, 192, 8), (5, 1, 7168, 32), (2, 1, 4096, 1), (700, 2, 10, 5), (37, 19, 204, 12), (2, 300, 33, 3),
         (3, 5000, 112, 7), (1, 70000, 6, 2), (2, 3000, 520, 8), (1, 4096, 2048, 16), (3, 1, 16384, 4), (1, 3, 16384, 1), (9, 1, 45, 15), (600, 1, 36, 1)]


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def reference(x, groups, w, b, eps, act, gy):
    """Results in float64 and the magnitudes that go into each."""
    x, gy = x.double(), gy.double()
    n = x.size(-1)
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()

    def by_group(t):   # (b, s, n) -> the mean over a group, spread over its elements
        g = t.view(t.size(0), t.size(1), groups, -1).mean((1, 3), keepdim=True)
        return g.expand(-1, t.size(1), -1, n // groups).reshape(t.shape)

    d = x - by_group(x)
    rstd = (by_group(d * d) + eps).rsqrt()
    h = d * rstd
    z = (h * w + b).requires_grad_()
    y = act64(z, act)
    gz, = torch.autograd.grad(y, z, gy)
    z, y = z.detach(), y.detach()
    size_h = (x.abs() + by_group(x.abs())) * rstd     # what the differences are made of
    slope = 1.2                                       # of any of the activations
    gh = gz * w
    gx = rstd * (gh - by_group(gh) - h * by_group(gh * h))
    more = gy.abs() * slope * (1 + size_h * w.abs() + z.abs())       # what an error of z does to gz
    size_g = more * w.abs()
    size_gx = rstd * (size_g + by_group(size_g) + size_h * by_group(size_g * (h.abs() + size_h)))
    return ((y, slope * (size_h * w.abs() + b.abs() + z.abs())), (gx, size_gx), ((gz * h).sum((0, 1)), (more * (h.abs() + size_h)).sum((0, 1))),
            (gz.sum((0, 1)), more.sum((0, 1))))


def near(got, want, size, what):
    half = HALF[got.dtype]
    off = (got.double() - want).abs()
    allowed = EPS * size + half * (want.abs() + EPS * size) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    assert (off <= allowed).all(), (what, (off / allowed).max().item())


def make(b, s, n, dtype, offset=0, mean=0.5):
    gen = torch.Generator(device="cuda").manual_seed(b + s + n)

    def one(*shape, scale=1.0, shift=0.0):
        k = math.prod(shape)
        flat = (torch.randn(k + offset, generator=gen, device="cuda") * scale + shift).to(dtype)
        return flat[offset:].view(shape)

    return one(b, s, n, shift=mean), one(n, scale=0.3, shift=1.0), one(n, scale=0.3), one(b, s, n)


def run(G, x, groups, w, b, act, gy, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    x, w, b = (next(it) if t is not None else None for t in (x, w, b))
    y = G.group_norm(x, groups, w, b, eps=eps, activation=act)
    grads = iter(torch.autograd.grad(y, leaves, gy))
    return y, next(grads), next(grads) if w is not None else None, next(grads) if b is not None else None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("b,s,n,groups", SIZES)
def test_against_float64(b, s, n, groups, offset, dtype):
    import gelib_b200 as G
    acts = [None, "relu", "silu", "gelu_tanh"]
    x, w, bias, gy = make(b, s, n, dtype, offset)
    for act in acts if b * s * n < 200000 else [acts[(b + s) % 4]]:
        if act == "relu":   # away from the kink, whose side depends on the last bit of z
            z = reference(x, groups, w, bias, 1e-5, None, gy)[0][0]
            gy = torch.where(z.abs() < 1e-3, 0.0, gy.double()).to(dtype).view(b, s, n)
        got = run(G, x, groups, w, bias, act, gy)
        for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, act, gy), ("y", "gx", "gw", "gb")):
            assert g.dtype == dtype
            near(g, want, size, (what, act))


@pytest.mark.gpu
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("b,s,n,groups", [(5, 1, 48, 4), (5, 7, 48, 4), (2, 9000, 48, 4)])
def test_without_weight_or_bias(b, s, n, groups, has_w, has_b):
    import gelib_b200 as G
    x, w, bias, gy = make(b, s, n, torch.float32)
    w, bias = w if has_w else None, bias if has_b else None
    got = run(G, x, groups, w, bias, "silu", gy)
    for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, "silu", gy), ("y", "gx", "gw", "gb")):
        if g is not None:
            near(g, want, size, what)


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,n,groups", [(4, 1, 512, 4), (4, 33, 60, 5), (2, 20000, 24, 3)])
def test_a_large_mean_costs_no_digits_of_the_spread(b, s, n, groups):
    import gelib_b200 as G
    x, w, bias, gy = make(b, s, n, torch.float32, mean=3000.0)
    got = run(G, x, groups, w, bias, None, gy)
    for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, None, gy), ("y", "gx", "gw", "gb")):
        near(g, want, size, what)
    # the variance in particular: its relative error is that of a sum of squares, not 2^-24 * mean^2
    h = G.group_norm(x, groups).double().view(b, s, groups, -1)
    assert (h.square().mean((1, 3)) - 1).abs().max() < 1e-5 + 2 * EPS


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,n,groups", [(2, 1, 6, 2), (2, 3, 4, 2), (1, 9000, 4, 2)])
def test_gradients_against_differences(b, s, n, groups):
    """Differences of the operator itself, in float32: a step of 2^-6 leaves a relative error of its square and of 2^-24 / 2^-6 of the sums."""
    import gelib_b200 as G
    x, w, bias, gy = make(b, s, n, torch.float32)
    _, gx, gw, gb = run(G, x, groups, w, bias, "silu", gy)
    step = 2.0 ** -6
    for t, grad, k in ((x, gx, 0), (w, gw, 1), (bias, gb, 2)):
        gen = torch.Generator(device="cuda").manual_seed(k)
        d = torch.randn(t.shape, generator=gen, device="cuda")
        d = d / (d.abs().max() if k == 0 else 1)
        sides = []
        for sign in (1, -1):
            args = [x, w, bias]
            args[k] = t + sign * step * d
            sides.append((G.group_norm(args[0], groups, args[1], args[2], activation="silu").double() * gy.double()).sum())
        slope = (sides[0] - sides[1]) / (2 * step)
        want = (grad.double() * d.double()).sum()
        size = (grad.abs().double() * d.abs().double()).sum() + gy.abs().double().sum() * 2.0 ** -10
        assert abs(slope - want) <= 20 * step ** 2 * size + 2.0 ** -24 / step * gy.abs().double().sum()


@pytest.mark.gpu
def test_shapes_strides_streams_and_repeats():
    import gelib_b200 as G
    x, w, bias, _ = make(6, 20, 48, torch.float32)
    want = G.group_norm(x, 4, w, bias, activation="silu")
    assert torch.equal(G.group_norm(x.view(6, 4, 5, 48), 4, w, bias, activation="silu"), want.view(6, 4, 5, 48))
    assert torch.equal(G.group_norm(x[:, 0], 4, w, bias), G.group_norm(x[:, :1].contiguous(), 4, w, bias).view(6, 48))
    z = torch.view_as_complex(torch.stack([x, x], -1))
    assert torch.equal(G.group_norm(z.real, 4, w, bias, activation="silu"), want)                      # channel stride 2
    assert torch.equal(G.group_norm(x.transpose(0, 1).contiguous().transpose(0, 1), 4, w, bias, activation="silu"), want)
    assert torch.equal(G.group_norm(x[:1].expand(6, 20, 48), 4, w, bias, activation="silu")[5], want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = G.group_norm(x, 4, w, bias, activation="silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    for b, sp, n, groups in ((3000, 1, 192, 8), (300, 19, 204, 12), (3, 30000, 48, 4)):
        x, w, bias, gy = make(b, sp, n, torch.bfloat16)
        first, second = (run(G, x, groups, w, bias, "silu", gy) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(first, second))


@pytest.mark.gpu
def test_broadcast_parameters_and_only_some_gradients():
    import gelib_b200 as G
    x, w, bias, gy = make(4, 9, 24, torch.float32)
    one = torch.tensor(1.5, device="cuda", requires_grad=True)
    G.group_norm(x, 3, one.expand(24), bias, activation="silu").backward(gy)
    _, _, gw, _ = run(G, x, 3, torch.full((24,), 1.5, device="cuda"), bias, "silu", gy)
    assert torch.allclose(one.grad, gw.sum(), rtol=1e-5)
    _, gx, gw, gb = run(G, x, 3, w, bias, "silu", gy)
    for i, want in enumerate((gx, gw, gb)):
        a = [x.clone(), w.clone(), bias.clone()]
        a[i].requires_grad_()
        G.group_norm(a[0], 3, a[1], a[2], activation="silu").backward(gy)
        assert torch.equal(a[i].grad, want)


@pytest.mark.gpu
def test_values_that_are_no_numbers_stay_in_their_sample_and_group():
    import gelib_b200 as G
    for b, s, n, groups in ((4, 1, 48, 4), (4, 9, 48, 4), (2, 9000, 48, 4)):
        x, w, bias, _ = make(b, s, n, torch.float32)
        clean = G.group_norm(x, groups, w, bias, activation="silu")
        for bad in (float("nan"), float("inf")):
            y = x.clone()
            y[1, s // 2, 17] = bad
            got = G.group_norm(y, groups, w, bias, activation="silu")
            spoilt = torch.zeros_like(x, dtype=torch.bool).view(b, s, groups, -1)
            spoilt[1, :, 1] = True
            spoilt = spoilt.view(b, s, n)
            assert torch.isnan(got[spoilt]).all()
            assert torch.equal(got[~spoilt], clean[~spoilt])


@pytest.mark.gpu
def test_empty_and_constant_inputs():
    import gelib_b200 as G
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    for shape in ((0, 8), (3, 0, 8), (0, 5, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = G.group_norm(x, 2, w, b)
        assert y.shape == x.shape
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()
    y = G.group_norm(torch.full((2, 8), 7.0, device="cuda"), 8, w, b + 0.25)     # one element a group
    assert (y == 0.25).all()


@pytest.mark.gpu
def test_module_and_no_grad():
    import gelib_b200 as G
    m = G.GroupNorm(4, 24, activation="silu", device="cuda")
    x = torch.randn(5, 24, device="cuda")
    y = m(x)
    y.sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
    with torch.no_grad():
        assert torch.equal(m(x), y)


def test_cpu_tensors_are_refused(cabi):
    import gelib_b200 as G
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        G.group_norm(torch.zeros(2, 8), 2)


REFUSALS = {
    "groups": ("do not divide", dict(groups=3)),
    "no groups": ("do not divide", dict(groups=0)),
    "shape of the weight": (r"weight must have shape \(8,\)", dict(weight=torch.zeros(7))),
    "type of the bias": ("bias must be of x's type", dict(bias=torch.zeros(8, dtype=torch.bfloat16))),
    "double": ("float32, bfloat16 or float16", dict(x=torch.zeros(2, 8, dtype=torch.float64))),
    "complex": ("float32, bfloat16 or float16", dict(x=torch.zeros(2, 8, dtype=torch.complex64))),
    "one dimension": ("at least 2 dimensions", dict(x=torch.zeros(8))),
    "activation": ("activation is one of", dict(activation="tanh")),
    "eps": ("eps is negative", dict(eps=-1.0)),
    "channels": ("GELIB_NORM_MAX_CHANNELS", dict(x=torch.zeros(1, 16386))),
}


@pytest.mark.gpu
@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    import gelib_b200 as G
    match, change = REFUSALS[what]
    a = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in {**dict(x=torch.zeros(2, 8), groups=2), **change}.items()}
    with pytest.raises((RuntimeError, ValueError), match=match):
        G.group_norm(a.pop("x"), a.pop("groups"), **a)


@pytest.mark.gpu
def test_without_the_native_host_side(monkeypatch):
    import gelib_b200 as G
    for b, s, n, groups in ((5, 1, 24, 3), (5, 7, 24, 3), (2, 9000, 24, 3)):
        x, w, bias, gy = make(b, s, n, torch.bfloat16)
        want = run(G, x, groups, w, bias, "silu", gy)
        with monkeypatch.context() as patch:
            patch.setattr(G._lib, "_native", G._lib._Declines())
            got = run(G, x, groups, w, bias, "silu", gy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_a_second_derivative_is_refused(native, monkeypatch):
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(G.group_norm(x, 2, activation="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,n,groups,dtype,offset", [(2, 90000, 112, 7, torch.float32, 0), (1, 90000, 111, 3, torch.float32, 1), (1, 170000, 112, 7, torch.bfloat16, 0)])
def test_samples_larger_than_the_shared_memory_of_all_sms(b, s, n, groups, dtype, offset):
    import gelib_b200 as G
    x, w, bias, gy = make(b, s, n, dtype, offset)
    got = run(G, x, groups, w, bias, "silu", gy)
    for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, "silu", gy), ("y", "gx", "gw", "gb")):
        near(g, want, size, what)
    again = run(G, x, groups, w, bias, "silu", gy)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,n,groups", [(1, 9001, 64, 4), (3, 4003, 112, 7), (7, 2500, 200, 8), (40, 700, 333, 3), (150, 600, 256, 8), (2, 65536, 60, 5), (1, 37, 16384, 2), (5, 60, 12000, 3)])
def test_samples_larger_than_the_shared_memory_of_one_sm(b, s, n, groups):
    """Few and many of them, rows that do not divide among the blocks."""
    import gelib_b200 as G
    for dtype, offset in ((torch.float32, 0), (torch.bfloat16, 0), (torch.float32, 1)):
        x, w, bias, gy = make(b, s, n, dtype, offset)
        got = run(G, x, groups, w, bias, "gelu_tanh", gy)
        for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, "gelu_tanh", gy), ("y", "gx", "gw", "gb")):
            near(g, want, size, (what, dtype, offset))
        only_w = w.detach().requires_grad_()
        G.group_norm(x, groups, only_w, bias, activation="gelu_tanh").backward(gy)
        assert torch.equal(only_w.grad, got[2])


@pytest.mark.gpu
@pytest.mark.parametrize("b,s,n,groups", [(50, 8, 512, 32), (9, 2, 64, 8), (300, 3, 32, 2), (41, 16, 64, 2), (5, 100, 24, 6), (17, 7, 128, 4), (3, 5, 4, 4), (70, 4, 1024, 4), (11, 64, 16, 2),
                                          (6, 128, 8, 1), (5, 31, 96, 3)])
def test_small_samples_of_several_rows(b, s, n, groups):
    import gelib_b200 as G
    for dtype, offset in ((torch.float32, 0), (torch.bfloat16, 0), (torch.float16, 1)):
        x, w, bias, gy = make(b, s, n, dtype, offset)
        got = run(G, x, groups, w, bias, "silu", gy)
        for g, (want, size), what in zip(got, reference(x, groups, w, bias, 1e-5, "silu", gy), ("y", "gx", "gw", "gb")):
            near(g, want, size, (what, dtype, offset))
        again = run(G, x, groups, w, bias, "silu", gy)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
