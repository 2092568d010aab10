"""The AdamW step against the formula in float64: 32-bit states within the rounding of their operations, 8-bit states by the rule that
rounds them, over odd sizes, alignments, types and more tensors than one launch takes.

Tolerances.  A new moment is two products and a sum of float32 (and two rounded coefficients): 5 roundings of 2^-24 of the sum of the magnitudes.
The step adds a root, two products, a sum and a quotient with their coefficients: fewer than 16 in all, so 16 * 2^-24 of the magnitudes that go in.
"""
import math

import pytest
import torch

EPS = 2.0 ** -24
HYPER = dict(step=7, lr=3e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _bits(seed, n):
    """The hash that rounds 8-bit states, in arithmetic modulo 2^32."""
    low = (1 << 32) - 1
    i = torch.arange(n)
    h = (i & low) * 0x9E3779B1 + (i >> 32) * 0x7FEB352D + (seed & low) * 0x6A09E667 + (seed >> 32) * 0x3C6EF373 & low
    h = (h ^ h >> 15) * 0x2C1B3C6D & low
    h = (h ^ h >> 12) * 0x297A2D39 & low
    return h ^ h >> 15


def _step64(p, g, m, v, step, lr, betas, eps, weight_decay, scale=1.0):
    """New values, and the magnitudes that went into each."""
    b1, b2 = betas
    g = g * scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    size_m = b1 * m.abs() + (1 - b1) * g.abs()
    rate = lr / (1 - b1 ** step) / ((v1 / (1 - b2 ** step)).sqrt() + eps)
    return (p * (1 - lr * weight_decay) - rate * m1, p.abs() + rate * size_m), (m1, size_m), (v1, v1)


def _near(got, want, size, what):
    off = (got.double().cpu() - want).abs()
    worst = (off / (size + 1e-30)).max().item() if off.numel() else 0.0
    assert worst <= 16 * EPS, (what, worst / EPS)


def _blocks(x):
    pad = -x.numel() % 256
    return torch.nn.functional.pad(x, (0, pad)).view(-1, 256)


def _codes(x):
    b = _blocks(x.float())
    scale = torch.exp2((torch.floor(torch.log2(b.abs().amax(1))) - 7).clamp(min=-100))
    return (b / scale[:, None]).reshape(-1)[:x.numel()].to(torch.float8_e4m3fn), scale


def _of_codes(codes, scale):
    return codes.double() * scale.double().repeat_interleave(256)[:codes.numel()]


def _network(sizes, dtype, offset=0):
    """Parameters, gradients and moments (float64) of a list of sizes; offset: elements by which the tensors are off their alignment."""
    gen = torch.Generator().manual_seed(sum(sizes) + offset)
    made = []
    for n in sizes:
        def one(scale=1.0, dt=torch.float32):
            flat = torch.randn(n + offset, generator=gen) * scale
            return flat.to(dt).cuda()[offset:]
        if dtype == torch.complex64:
            p, g = (torch.view_as_complex((torch.randn(n, 2, generator=gen)).cuda()) for _ in range(2))
        else:
            p, g = one(dt=dtype), one(0.1, dtype)
        k = 2 * n if dtype == torch.complex64 else n
        size = torch.exp(2 * torch.randn(k, generator=gen)) * 0.05
        made.append((p, g, torch.randn(k, generator=gen) * size, torch.rand(k, generator=gen) * size * size))
    return made


def _flat(t):
    t = t.detach()
    return (torch.view_as_real(t) if t.is_complex() else t).reshape(-1)


SIZES = [[1], [2, 3, 255, 256, 257], [0, 5, 2047, 2048, 2049, 70001], [7] * 800]


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SIZES, ids=["one", "blocks", "pieces", "many"])
@pytest.mark.parametrize("bits", [32, 8])
def test_step(bits, sizes, dtype, offset, native, monkeypatch):
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    made = _network(sizes, dtype, offset)
    scale = torch.tensor([0.5], device="cuda")
    low = dtype in (torch.bfloat16, torch.float16)
    params, grads = [x[0] for x in made], [x[1] for x in made]
    before = [_flat(p).double().cpu() for p in params]
    master = None
    if low:
        gen = torch.Generator().manual_seed(1)
        before = [b + torch.randn(b.shape, generator=gen).double() * 1e-4 for b in before]
        before = [b.float().double() for b in before]
        master = [torch.cat([torch.zeros(offset), b.float()]).cuda()[offset:] for b in before]
    more = {}
    if bits == 32:
        m, v = ([torch.cat([torch.zeros(offset), x[k]]).cuda()[offset:] for x in made] for k in (2, 3))
        m64, v64 = ([t.double().cpu() for t in s] for s in (m, v))
    else:
        cm, cv = [_codes(x[2]) for x in made], [_codes(x[3].sqrt()) for x in made]
        m64, v64 = [_of_codes(*c) for c in cm], [_of_codes(*c) ** 2 for c in cv]

        def moved(codes):
            return torch.cat([torch.zeros(offset, dtype=torch.uint8), codes.view(torch.uint8)]).cuda()[offset:].view(torch.float8_e4m3fn)

        m, v = [moved(c) for c, _ in cm], [moved(c) for c, _ in cv]
        more = dict(exp_avg_scale=[s.cuda() for _, s in cm], exp_avg_sq_scale=[s.cuda() for _, s in cv], seed=(5 << 32) + 9)
    n0 = G.backend.kernel_launch_count()
    G.adamw_step(params, grads, m, v, master=master, grad_scale=scale, **HYPER, **more)
    torch.cuda.synchronize()
    assert G.backend.kernel_launch_count() - n0 == -(-sum(1 for n in sizes if n) // 350)
    at = 0
    for i, n in enumerate(sizes):
        g64 = _flat(grads[i]).double().cpu()
        new_p, new_m, new_v = _step64(before[i], g64, m64[i], v64[i], scale=0.5, **HYPER)
        _near(_flat(params[i]) if not low else master[i], *new_p, "p")
        if low:
            assert torch.equal(params[i], master[i].to(dtype))
        if bits == 32:
            _near(m[i], *new_m, "m")
            _near(v[i], *new_v, "v")
            continue
        k = g64.numel()
        u = _bits(more["seed"], at + k)[at:]
        at += -(-k // 256) * 256
        for codes, s, x, w, least in ((m[i], more["exp_avg_scale"][i], new_m[0], u & 0xffff, False),
                                      (v[i], more["exp_avg_sq_scale"][i], new_v[0].sqrt(), u >> 16, True)):
            if not k:
                continue
            top = _blocks(x).abs().amax(1)
            assert torch.equal(s.cpu().double(), torch.exp2((torch.floor(torch.log2(top)) - 7).clamp(min=-100)))
            q = x.abs() / s.cpu().double().repeat_interleave(256)[:k]
            grid = torch.exp2((torch.floor(torch.log2(q)) - 3).clamp(min=-9))
            want = torch.floor(q / grid + (w.double() * 16 + 8) / 2 ** 20) * grid
            if least:
                want = torch.where((q > 0) & (want == 0), 2.0 ** -9, want)
            got = codes.float().cpu().double().abs()
            # one of the two neighbours always; the one that the hash takes unless the rounding of the value itself turns it
            assert ((got - q).abs() <= grid * (1 + 1e-4)).all()
            differ = (got != want)
            near = ((q / grid + (w.double() * 16 + 8) / 2 ** 20) % 1)
            assert (torch.minimum(near, 1 - near)[differ] < 1e-3).all() and differ.double().mean() <= 1e-2
            assert torch.equal(torch.signbit(codes.float().cpu())[got > 0], torch.signbit(x)[got > 0])


@pytest.mark.gpu
def test_values_that_are_no_numbers_spoil_their_own_element_alone():
    import gelib_b200 as G
    n = 700
    p, g = torch.ones(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    g[3], g[300] = float("nan"), float("inf")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = torch.ones(3, device="cuda"), torch.ones(3, device="cuda")
    G.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, exp_avg_scale=[ms], exp_avg_sq_scale=[vs])
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[3, 300]] = True
    for t in (p, G.block8_values(m, ms), G.block8_values(v, vs)):
        assert torch.equal(~torch.isfinite(t.float()).cpu(), bad)


@pytest.mark.gpu
def test_blocks_of_zeros_tiny_and_huge_values():
    import gelib_b200 as G
    g = torch.zeros(1024, device="cuda")
    g[256:512], g[512:768], g[768:] = 1e-30, 1e18, 1e-12
    p = torch.zeros(1024, device="cuda")
    m, v = (torch.zeros(1024, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    G.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, betas=(0.9, 0.99), eps=0.0 + 1e-8, weight_decay=0, exp_avg_scale=[ms], exp_avg_sq_scale=[vs])
    assert torch.isfinite(p).all() and (p[:256] == 0).all()
    a, r = G.block8_values(m, ms).double(), G.block8_values(v, vs).double()
    assert (a[:256] == 0).all() and (r[:256] == 0).all()
    for k in (2, 3):
        assert ((a[256 * k:256 * k + 256] / (0.1 * g[256 * k:256 * k + 256].double()) - 1).abs() <= 0.125 + 1e-4).all()
        assert ((r[256 * k:256 * k + 256] / (0.1 * g[256 * k:256 * k + 256].double()) - 1).abs() <= 0.125 + 1e-4).all()


@pytest.mark.gpu
def test_rounding_is_unbiased_and_a_small_change_moves_a_moment():
    """4096 seeds' worth of roundings of one value: their mean is within five standard errors of it."""
    import gelib_b200 as G
    n, x = 256 * 4096, 0.7177
    g = torch.full((n,), x * 10, device="cuda")   # m = 0.1 g
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.ones(n // 256, device="cuda") for _ in range(2))
    G.adamw_step([torch.zeros(n, device="cuda")], [g], [m], [v], step=1, lr=0.0, exp_avg_scale=[ms], exp_avg_sq_scale=[vs], seed=3)
    for t, want in ((G.block8_values(m, ms), x), (G.block8_values(v, vs), math.sqrt(0.001) * x * 10)):
        t = t.double()
        step = 2.0 ** (math.floor(math.log2(want)) - 3)
        assert t.unique().numel() == 2
        assert abs(t.mean().item() - want) <= 5 * 0.5 * step / math.sqrt(n) + step * 2 ** -15


@pytest.mark.gpu
def test_a_call_repeats_bit_for_bit_and_goes_by_its_stream():
    import gelib_b200 as G
    results = []
    for _ in range(2):
        made = _network([5000, 33], torch.float32)
        codes = [_codes(x[2]) for x in made]
        m, ms = [c.cuda() for c, _ in codes], [s.cuda() for _, s in codes]
        v, vs = [c.clone().view(torch.uint8).bitwise_and(0x7f).view(torch.float8_e4m3fn) for c in m], [s.clone() for s in ms]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            G.adamw_step([x[0] for x in made], [x[1] for x in made], m, v, exp_avg_scale=ms, exp_avg_sq_scale=vs, seed=4, **HYPER)
        torch.cuda.current_stream().wait_stream(stream)
        results.append([x[0] for x in made] + [c.view(torch.uint8) for c in m + v] + ms + vs)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_trains_and_its_state_comes_back(bits):
    """Complex, float32 and bfloat16 weights of a least-squares fit; the second half of the run goes on from a state dict.  What is left of the
    loss is what torch.optim.AdamW leaves of it in the same number of steps, to a quarter (the rounding to 8 bits is noise in the steps'
    lengths; a weight moves by at most the rate a step, so neither has arrived)."""
    import gelib_b200 as G

    def problem():
        gen = torch.Generator().manual_seed(0)
        a = torch.randn(512, 24, generator=gen).cuda()
        w = [torch.nn.Parameter(torch.zeros(24, 8, dtype=d, device="cuda")) for d in (torch.float32, torch.complex64, torch.bfloat16)]
        goal = torch.randn(24, 8, generator=gen).cuda()

        def loss():
            r = a @ (w[0] - goal)
            c = a.to(torch.complex64) @ (w[1] - goal * (1 + 2j))
            q = a.to(torch.bfloat16) @ (w[2] - goal.to(torch.bfloat16))
            return r.square().mean() + c.abs().square().mean() + q.float().square().mean()
        return w, loss

    w, loss = problem()
    opt = G.AdamW([dict(params=w[:1]), dict(params=w[1:], lr=3e-2)], lr=3e-2, weight_decay=0.0, state_bits=bits)
    first = loss().item()
    for _ in range(60):
        opt.zero_grad()
        loss().backward()
        opt.step()
    saved = opt.state_dict()
    w2, loss2 = problem()
    opt2 = G.AdamW([dict(params=w2[:1]), dict(params=w2[1:])], lr=1.0, state_bits=bits)
    opt2.load_state_dict(saved)
    with torch.no_grad():
        for a, b in zip(w2, w):
            a.copy_(b)
    for o, f in ((opt, loss), (opt2, loss2)):
        for _ in range(60):
            o.zero_grad()
            f().backward()
            o.step()
    assert all(torch.equal(a, b) for a, b in zip(w, w2))
    w3, loss3 = problem()
    opt3 = torch.optim.AdamW(w3, lr=3e-2, weight_decay=0.0)
    for _ in range(120):
        opt3.zero_grad()
        loss3().backward()
        opt3.step()
    assert loss3().item() < 0.1 * first
    assert abs(loss().item() / loss3().item() - 1) < 0.25


@pytest.mark.gpu
def test_lazily_conjugated_and_strided_gradients():
    import gelib_b200 as G
    p = torch.zeros(6, 4, dtype=torch.complex64, device="cuda")
    q = p.clone()
    g = torch.view_as_complex(torch.randn(4, 6, 2, device="cuda"))
    state = [[torch.zeros(48, device="cuda")] for _ in range(4)]
    G.adamw_step([p], [g.t().conj()], *state[:2], **HYPER)
    G.adamw_step([q], [g.t().conj().resolve_conj().contiguous()], *state[2:], **HYPER)
    assert torch.equal(p, q) and p.abs().min() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-8, 0.0])
def test_codes_are_those_of_moments_rounded_operation_by_operation(eps):
    """A last place of a moment decides an eighth of its code once in 2^20 elements.  With each operation rounded to nearest by itself no code of 2^24
    differs: the root's last step is off by 2^-43 of it at most, which would show once in 2^19 * 2^20 elements."""
    import gelib_b200 as G
    n, b1, b2, seed = 1 << 24, 0.9, 0.999, 29
    gen = torch.Generator(device="cuda").manual_seed(3)
    size = torch.exp(torch.randn(n // 256, generator=gen, device="cuda")).repeat_interleave(256) * 1e-2
    g = torch.randn(n, generator=gen, device="cuda") * size
    old = [torch.randn(n, generator=gen, device="cuda") * size, (0.3 + torch.rand(n, generator=gen, device="cuda")) * size]
    old[1][::1001] = 0
    g[::1001] = 0
    codes, scales = zip(*(_codes(x) for x in old))
    m, r = (c.float() * k.repeat_interleave(256) for c, k in zip(codes, scales))
    want = [m * b1 + g * (1 - b1), torch.sqrt(r * r * b2 + g * (1 - b2) * g)]
    want[1][::1001] = 0
    G.adamw_step([torch.zeros(n, device="cuda")], [g], [codes[0]], [codes[1]], step=1000, lr=1e-3, betas=(b1, b2), eps=eps, weight_decay=0.0,
                 exp_avg_scale=[scales[0]], exp_avg_sq_scale=[scales[1]], seed=seed)
    bits = _bits(seed, n).cuda()
    for x, u, got, scale in ((want[0], bits & 0xffff, codes[0], scales[0]), (want[1], bits >> 16, codes[1], scales[1])):
        b = x.view(-1, 256).double()
        power = torch.exp2(torch.floor(torch.log2(b.abs().amax(1))) - 7)
        assert torch.equal(power, scale.double())
        y = (b / power[:, None]).abs().view(-1)
        step = torch.exp2((torch.floor(torch.log2(y)) - 3).clamp(min=-9))
        q = torch.floor(y / step + (u.double() * 16 + 8) / 2 ** 20) * step
        if got is codes[1]:
            q = torch.where((y > 0) & (q == 0), 2.0 ** -9, q)
        assert torch.equal(got.double().abs(), q), (got.double().abs() != q).sum().item()


@pytest.mark.gpu
def test_saved_tensors_are_told_of_the_step():
    import gelib_b200 as G
    w = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
    y = (w * w).sum()
    G.adamw_step([w], [torch.ones_like(w)], [torch.zeros(16, device="cuda")], [torch.zeros(16, device="cuda")], **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def _refused(match, device, **change):
    import gelib_b200 as G
    one = lambda n=8, d=torch.float32: torch.zeros(n, device=device).to(d)  # noqa: E731
    a = dict(params=[one()], grads=[one()], exp_avg=[one()], exp_avg_sq=[one()], **HYPER)
    a.update({k: f(one) if callable(f) else f for k, f in change.items()})
    with pytest.raises((RuntimeError, TypeError), match=match):
        G.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avg"), a.pop("exp_avg_sq"), **a)


def test_cpu_tensors_are_refused(cabi):
    _refused("CUDA tensors only", "cpu")


REFUSALS = {
    "lengths": ("params and 0 grads", dict(grads=[])),
    "shape": ("shape", dict(grads=lambda o: [o(9)])),
    "type of a gradient": ("contiguous tensor of float32", dict(grads=lambda o: [o(8, torch.bfloat16)])),
    "double": ("contiguous tensor", dict(params=lambda o: [o(8, torch.float64)])),
    "strided": ("contiguous", dict(params=lambda o: [o(16)[::2]])),
    "size of a moment": ("7 numbers where 8", dict(exp_avg=lambda o: [o(7)])),
    "type of a moment": ("float32 or complex64", dict(exp_avg_sq=lambda o: [o(8, torch.bfloat16)])),
    "one scale": ("exp_avg_scale and exp_avg_sq_scale", dict(exp_avg_scale=lambda o: [o(1)])),
    "codes": ("float8_e4m3fn", dict(exp_avg_scale=lambda o: [o(1)], exp_avg_sq_scale=lambda o: [o(1)])),
    "master": ("master copy", dict(params=lambda o: [o(8, torch.float16)], grads=lambda o: [o(8, torch.float16)])),
    "master of float32": ("master copy", dict(master=lambda o: [o()])),
    "step": ("counted from 1", dict(step=0)),
    "betas": ("betas", dict(betas=(0.9, 1.0))),
    "eps": ("negative", dict(eps=-1.0)),
    "device": ("on cuda", dict(grads=[torch.zeros(8)])),
    "lr": ("on the host", dict(lr=torch.tensor(1e-3))),
}


@pytest.mark.gpu
@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    match, change = REFUSALS[what]
    _refused(match, "cuda", **change)


@pytest.mark.gpu
def test_a_capture_is_refused():
    import gelib_b200 as G
    one = torch.zeros(8, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="captured graph"):
                G.adamw_step([one], [one], [one], [one], **HYPER)
        finally:
            one.add_(0)
            graph.capture_end()
