"""The gradient of an embedding table whose numbers are sorted in one, two and three passes, by one cluster and by the whole machine; every row is compared."""
import pytest
import torch

from test_embedding import HALF, near, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("v", [1 << 9, (1 << 10) - 1, 1 << 10, (1 << 20) - 1, 1 << 20, (1 << 20) + 5, (1 << 21) + 3])
@pytest.mark.parametrize("n", [900, 5001, 65536, 65537, 200000])
def test_numbers_that_repeat_in_large_tables(n, v, dtype):
    """Up to a few hundred different numbers, spread over the table with its first and last rows; each is met from once to thousands of times."""
    import gelib_b200 as G
    gen = torch.Generator(device="cuda").manual_seed(n + v)
    some = torch.randint(v, (400,), generator=gen, device="cuda")
    some[0], some[1], some[2] = 0, v - 1, v // 2
    ids = some[(torch.rand(n, generator=gen, device="cuda") ** 3 * 400).long().clamp(max=399)]
    ids[::50] = torch.randint(v, ids[::50].shape, generator=gen, device="cuda")
    d = 8
    weight = torch.randn(v, d, generator=gen, device="cuda").to(dtype).requires_grad_()
    gy = torch.randn(n, d, generator=gen, device="cuda").to(dtype)
    y = G.embedding(ids, weight, 0.5, padding_idx=int(some[5]))
    gw, = torch.autograd.grad(y, weight, gy)
    wants = reference(ids, weight.detach(), gy, 0.5, int(some[5]))
    near(y.detach(), wants[0])
    near(gw, wants[1])
    met = torch.zeros(v, dtype=torch.bool, device="cuda")
    met[ids] = True
    assert (gw[~met] == 0).all()
