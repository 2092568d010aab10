"""Long sums of 16-bit products: their errors over the number of channels, and z that both passes and all pieces of the classes have alike."""
import pytest
import torch

from test_losses import call, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [1024, 1216, 1280, 1344, 1408, 1920, 1984, 2048, 4096, 16384])
def test_losses_are_off_by_a_millionth_on_average(k, dtype):
    """z leaves the tensor cores' accumulators before what they cut off comes to 2^-20 of a loss, the mean over rows; a tenth of that for the mean's own spread."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    off = []
    for _ in range(4):
        x = torch.randn(1000, k, generator=gen, device="cuda").to(dtype)
        w = (torch.randn(k, 300, generator=gen, device="cuda") * 2 * k ** -0.5).to(dtype)
        target = torch.randint(300, (1000,), generator=gen, device="cuda")
        with torch.no_grad():
            got = call(x, w, None, target, None, reduction="none").double()
        want = torch.nn.functional.cross_entropy(x.double() @ w.double(), target, reduction="none")
        off.append((got - want) / want.clamp(min=0.5))
    assert abs(torch.cat(off).mean()) <= 1.1 * 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wt", [False, True])
def test_a_sure_class_of_any_piece_has_no_gradient(wt, dtype):
    """dz is made in pieces of the classes, whose last is narrow; the log-sum comes of all of them at once."""
    m, k, n = 40000, 200, 2500 if dtype == torch.float32 else 4500
    x, w, _, _, _ = make(m, k, n, dtype, wt=wt)
    x.abs_()
    for sure in (7, n - 3):
        v = w.clone()
        v[:, sure] = 8.0   # z is near 6.4 k there, and within some tens elsewhere: the others' shares are zero
        got = run(x, v, None, torch.full((m,), sure, device="cuda"), None, torch.tensor(1.0, device="cuda"), reduction="sum")
        assert all((t == 0).all() for t in got)
