"""The gradient of the whole example against differences along itself, weight by weight, where the slope is its norm.

(f(h) - f(-h)) / 2h = slope + c h^2 + ..., so the same with 2h differs from it by 3 c h^2: three times its error, which is allowed.  Beside that the losses, of
some five and less, are off by some 2^-20 of themselves through products, norm and layers, eight times which is allowed.  Both together may come to a tenth
of the slope at the most, so that a gradient of zero or of the wrong sign is seen.
"""
import pytest
import torch

from test_species_example import _example

pytestmark = pytest.mark.gpu


def test_gradient_of_the_whole_against_differences_along_it():
    example = _example()
    torch.manual_seed(0)
    network = example.Network(species=12, channels=4, hidden=16)
    generator = torch.Generator(device="cuda").manual_seed(1)
    points, of, hidden = example.atoms(40, 6, 12, generator)

    def loss():
        return network.head.cross_entropy(network(points, of), hidden)

    weights = list(network.named_parameters())
    grads = torch.autograd.grad(loss(), [w for _, w in weights])
    for (name, w), g in zip(weights, grads):
        norm = g.abs().square().sum().sqrt()
        d, start = g / norm, w.detach().clone()
        step = 2.0 ** -6

        def slope(h):
            with torch.no_grad():
                sides = []
                for sign in (1, -1):
                    w.copy_(start + sign * h * d)
                    sides.append(loss().double())
                w.copy_(start)
            return float(sides[0] - sides[1]) / (2 * h)

        near, far = slope(step), slope(2 * step)
        allowed = abs(far - near) + 8 * 2.0 ** -20 * float(loss().detach()) / step
        assert allowed <= 0.1 * float(norm), (name, allowed, float(norm))
        assert abs(near - float(norm)) <= allowed, (name, near, float(norm), allowed)
