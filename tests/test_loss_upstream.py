"""What comes from above to rows of a loss of their own: rows without a loss, and rows with an infinity there, change no other row's gradients.

float16 holds dz relative to the largest upstream gradient, so that number may be taken from finite ones of rows that have a loss alone.
"""
import math

import pytest
import torch

from test_losses import DTYPES, check, make, run

pytestmark = pytest.mark.gpu


def upstream(m, size, rows):
    """Around `size`, the largest in row 0; nothing in rows without a loss."""
    gy = size * (0.5 + 0.5 * torch.rand(m, generator=torch.Generator(device="cuda").manual_seed(m), device="cuda"))
    gy[0] = 2 * size
    return torch.where(rows, 0.0, gy)


def some_rows(m, dtype, top):
    """Arguments of a call, and which rows have no loss: never the first, at least one."""
    x, w, bias, target, logits = make(m, 64, 90, dtype, top=top)
    target[0] = 3
    target[m - 1] = -100
    rows = (target < 0).all(1) if top else target < 0
    return (x, w, bias, target, logits), rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("size", [8.0, 1e-6])
@pytest.mark.parametrize("m", [2, 150])
def test_gradients_that_come_to_rows_without_a_loss(m, size, top, dtype):
    args, rows = some_rows(m, dtype, top)
    gy = upstream(m, size, rows)
    clean = check(args, "none", gy=gy)
    for bad in (math.inf, -math.inf, math.nan, 1e30, -1e30, 1e-30):
        got = run(*args, torch.where(rows, bad, gy), reduction="none")
        assert all(torch.equal(a, b) for a, b in zip(got, clean)), bad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("size", [8.0, 1e-6])
def test_an_infinite_gradient_stays_in_its_row(size, top, dtype):
    args, rows = some_rows(150, dtype, top)
    one = int((~rows).nonzero()[5])
    gy = upstream(150, size, rows)
    clean = run(*args, gy, reduction="none")
    others = torch.arange(150, device="cuda") != one
    for bad in (math.inf, -math.inf, math.nan):
        there = gy.clone()
        there[one] = bad
        got = run(*args, there, reduction="none")
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1][others], clean[1][others]), bad
        assert not torch.isfinite(got[1][one]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_but_infinities(dtype):
    """No finite gradient, or none in a row with a loss: every number of theirs is none, and rows without a loss stay zero."""
    args, rows = some_rows(40, dtype, 0)
    got = run(*args, torch.full((40,), math.inf, device="cuda"), reduction="none")
    assert not torch.isfinite(got[1][~rows]).any() and (got[1][rows] == 0).all()
    for t in run(*args, torch.where(rows, 5.0, 0.0), reduction="none")[1:]:
        assert (t == 0).all()
