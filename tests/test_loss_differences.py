"""Gradients of the losses against differences along the gradient itself, where the slope is the gradient's norm and many times what is allowed.

With f(t) the sum of the losses along a direction, (f(h) - f(-h)) / 2h is off by at most h^2 / 6 times the largest third derivative.  z moves by t v, so
that derivative is the sum over rows of T^2 / T^3 times the third central moment of v's entries under p, at most (largest - least)^3 / (6 sqrt 3).  Beside that
there are the errors of both losses over 2h, half a unit in the last place of the operand that is moved, and the gradient's own error.
"""
import math

import pytest
import torch

from test_losses import call, make, reference, run

T = 2.0
STEP = 2.0 ** -3
SIZES = [(40, 24, 17), (3, 24, 17), (150, 40, 33)]


def moved(args, i, by):
    return tuple(a + by if k == i else a for k, a in enumerate(args))


def allowance(args, target, logits, i, d, grad, off_grad):
    """What (f(h) - f(-h)) / 2h may differ by from the gradient's product with d."""
    x, w, bias = (a.double() for a in args)
    v = (lambda: d.double() @ w, lambda: x @ d.double(), lambda: d.double().expand(x.size(0), -1))[i]()
    third = ((v.amax(1) - v.amin(1)) ** 3).sum() / (6 * math.sqrt(3)) / (T if logits is not None else 1.0)
    ones = torch.ones(x.size(0), device=x.device)
    off = sum(reference(*moved(args, i, s * STEP * d), target, logits, T, ones, "none")[0][1].sum() for s in (1, -1))
    rounded = 2.0 ** -24 * ((args[i].abs().double() + STEP) * grad.double().abs()).sum()   # of the operand that was moved
    return float(STEP ** 2 / 6 * third + (off + 2 * rounded) / (2 * STEP) + (off_grad * d.double().abs()).sum())


def directions(grad, seed):
    fixed = torch.randn(grad.shape, generator=torch.Generator(device=grad.device).manual_seed(seed), device=grad.device)
    return grad / grad.norm(), fixed / fixed.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gradients_against_differences_along_them(m, k, n, top):
    x, w, bias, target, logits = make(m, k, n, torch.float32, top=top)
    gy = torch.ones(m, device="cuda")
    grads = run(x, w, bias, target, logits, gy, temperature=T, reduction="none")[1:]
    wants = reference(x, w, bias, target, logits, T, gy, "none")[1:]
    for i, (grad, (_, off)) in enumerate(zip(grads, wants)):
        for along, d in enumerate(directions(grad, i)):
            sides = [call(*moved((x, w, bias), i, s * STEP * d), target, logits, T, "none").double().sum() for s in (1, -1)]
            slope, want = float((sides[0] - sides[1]) / (2 * STEP)), float((grad.double() * d.double()).sum())
            allowed = allowance((x, w, bias), target, logits, i, d, grad, off)
            assert along == 1 or abs(want) >= 10 * allowed
            assert abs(slope - want) <= allowed, (i, along, slope, want, allowed)


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_what_is_allowed_would_show_a_gradient_of_zero(m, k, n, top):
    """The same in float64 on the host: the differences agree with the formula, and a gradient that is missing or has the wrong sign is ten times the allowance off."""
    x, w, bias, target, logits = make(m, k, n, torch.float32, top=top, dev="cpu")
    wants = reference(x, w, bias, target, logits, T, torch.ones(m), "none")[1:]
    for i, (grad, off) in enumerate(wants):
        d = directions(grad, i)[0].float()
        d = d / d.norm()
        args = tuple(a.double() for a in (x, w, bias))
        sides = [in_double(moved(args, i, s * STEP * d.double()), target, logits) for s in (1, -1)]
        slope, want = float((sides[0] - sides[1]) / (2 * STEP)), float((grad * d.double()).sum())
        allowed = allowance((x, w, bias), target, logits, i, d, grad, off)
        assert abs(slope - want) <= allowed and abs(want) >= 10 * allowed, (i, slope, want, allowed)


def in_double(args, target, logits):
    """The sum of the losses in float64."""
    x, w, bias = args
    z = x @ w + bias
    if logits is None:
        return torch.nn.functional.cross_entropy(z, target, reduction="sum")
    entry = target >= 0
    live = entry.any(1)
    s = torch.where(entry, logits.double() / T, -math.inf)[live]
    log_q = torch.log_softmax(s, 1)
    log_p = torch.log_softmax(z[live] / T, 1).gather(1, target[live].clamp(min=0))
    return T * T * torch.where(entry[live], log_q.exp() * (log_q - log_p), 0.0).sum()
