"""Group norm, dense layers and the AdamW step beyond 2^31 elements, and sums of a million products: what is checked are the last rows, which an offset of 32
bits would have put elsewhere.  Tolerances: half a unit in the last place of the type, and what test_linear.py and test_group_norm.py allow for float sums.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _room(gigabytes):
    if torch.cuda.get_device_properties(0).total_memory < gigabytes * 2 ** 30:
        pytest.skip("needs %d GB of device memory" % gigabytes)


@pytest.mark.parametrize("b,s,n,groups", [(600000, 1, 4096, 32), (75000, 8, 4096, 64), (3, 200000, 4096, 8)])
def test_group_norm(b, s, n, groups):
    import gelib_b200 as G
    _room(64)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(b, s, n, dtype=torch.bfloat16, device="cuda").normal_(generator=gen).requires_grad_()
    y = G.group_norm(x, groups, activation="relu")
    gx, = torch.autograd.grad(y, x, x.detach())
    assert x.numel() > 2 ** 31
    for at in (0, b - 1):
        one = x[at:at + 1].detach().clone().requires_grad_()
        want = G.group_norm(one, groups, activation="relu")
        gone, = torch.autograd.grad(want, one, one.detach())
        for got, ref in ((y[at:at + 1], want), (gx[at:at + 1], gone)):   # the same kernel or one that adds in another order
            assert torch.allclose(got.float(), ref.float(), rtol=2.0 ** -7, atol=1e-4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(dtype):
    import gelib_b200 as G
    _room(100)
    m, k, n = 600000, 16, 4096
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(m, k, dtype=dtype, device="cuda").normal_(generator=gen)
    w = torch.empty(k, n, dtype=dtype, device="cuda").normal_(generator=gen)
    y = G.linear(x, w)
    assert y.numel() > 2 ** 31
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for at in (0, m // 2, m - 200):
        a, b = x[at:at + 200].double(), w.double()
        want, size = a @ b, a.abs() @ b.abs()
        assert ((y[at:at + 200].double() - want).abs() <= 64 * 2.0 ** -24 * size + half * want.abs()).all()
    g = torch.autograd.grad(G.linear(x, w.requires_grad_()), w, y)[0]   # sums of 600000 products
    part = sum((x[i:i + 50000].double().t() @ y[i:i + 50000].double() for i in range(0, m, 50000)))
    # cuts of 2e-8 of a sum after every 16 products of at most 131072
    assert ((g.double() - part).abs() <= (half + 4e-4) * part.abs() + 1e-5 * part.abs().max()).all()


@pytest.mark.parametrize("m", [300000, 1000000])
def test_long_sums_of_float16(m):
    """Products all of one sign, the worst of cuts: 8192 of them at 2^-24 are half of float16's own rounding."""
    import gelib_b200 as G
    x = torch.rand(m, 64, device="cuda").half() * 1e-2
    gy = torch.rand(m, 48, device="cuda").half() * 1e-2
    w = torch.zeros(64, 48, device="cuda", dtype=torch.float16, requires_grad=True)
    g, = torch.autograd.grad(G.linear(x, w), w, gy)
    want = x.double().t() @ gy.double()
    assert ((g.double() - want).abs() / want).max() <= 2.0 ** -11 + 8192 * 2.0 ** -24


def test_adamw_in_8_bits():
    import gelib_b200 as G
    _room(64)
    n, tail = 2 ** 31 + 3000, 2000
    gen = torch.Generator(device="cuda").manual_seed(3)
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    master = torch.zeros(n, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.ones(-(-n // 256), device="cuda") for _ in range(2))
    g[-tail:].normal_(generator=gen)
    G.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, weight_decay=0.0, exp_avg_scale=[ms], exp_avg_sq_scale=[vs], master=[master])
    want = -1e-2 * g[-tail:].double() / (g[-tail:].double().abs() + 1e-8)   # the first step
    assert ((master[-tail:].double() - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all()
    assert (master[:-tail].view(-1)[::4096] == 0).all() and torch.equal(p[-tail:], master[-tail:].bfloat16())
    values = G.block8_values(m, ms)
    assert ((values[-tail:].double() - 0.1 * g[-tail:].double()).abs() <= 0.125 * 0.1 * g[-tail:].double().abs() + 2.0 ** -9 * ms[-9:].max()).all()
    assert (values[:-tail][::4096] == 0).all()
