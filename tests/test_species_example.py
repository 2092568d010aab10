"""The example that runs the table, the products, the readout, both losses and the optimizer step together: that it runs, and its gradients."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("train_species", os.path.join(ROOT, "examples", "train_species.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_runs_and_every_weight_is_reached():
    example = _example()
    large, small, losses = example.train(steps=3, batch=64)
    assert torch.isfinite(losses).all()
    generator = torch.Generator(device="cuda").manual_seed(1)
    points, of, hidden = example.atoms(64, 12, 100, generator)
    for network in (large, small):
        network.zero_grad()
        network.head.cross_entropy(network(points, of), hidden).backward()
        for name, p in network.named_parameters():
            assert p.grad is not None and torch.isfinite(torch.view_as_real(p.grad) if p.is_complex() else p.grad).all() and p.grad.abs().sum() > 0, name


def test_gradient_of_the_whole_against_differences():
    """Along a direction in all weights, in float32: the loss is off by some 2^-20 of itself, a step of 2^-8 leaves the square of it."""
    example = _example()
    torch.manual_seed(0)
    network = example.Network(species=12, channels=4, hidden=16)
    generator = torch.Generator(device="cuda").manual_seed(1)
    points, of, hidden = example.atoms(40, 6, 12, generator)

    def loss():
        return network.head.cross_entropy(network(points, of), hidden)

    weights = list(network.parameters())
    grads = torch.autograd.grad(loss(), weights)
    step = 2.0 ** -8
    for w, g in zip(weights, grads):
        d = torch.randn(w.shape, generator=generator, device="cuda", dtype=w.dtype)
        d = d / d.abs().square().sum().sqrt()
        with torch.no_grad():
            sides = []
            for sign in (1, -2, 1):
                w += sign * step * d
                sides.append(loss().double())
        slope = (sides[0] - sides[1]) / (2 * step)
        want = (g.conj() * d).real.sum().double()
        # the error of the two losses over their distance, and the third derivative's share, which a norm of 40 atoms keeps below some hundreds
        assert abs(slope - want) <= 2.0 ** -20 * 8 / step + 200 * step ** 2, (w.shape, slope, want)


def test_a_turned_cloud_has_the_same_loss():
    """A rotation changes the harmonics by their rounding, some 1e-5 of the loss through a norm that may enlarge it."""
    example = _example()
    torch.manual_seed(0)
    network = example.Network()
    generator = torch.Generator(device="cuda").manual_seed(2)
    points, of, hidden = example.atoms(200, 12, 100, generator)
    q, r = torch.linalg.qr(torch.randn(3, 3, generator=generator, device="cuda"))
    q = q * torch.sign(torch.diagonal(r))
    q[:, 0] *= torch.det(q)
    with torch.no_grad():
        a, b = (network.head.cross_entropy(network(p, of), hidden) for p in (points, (q @ points).contiguous()))
    assert abs(a - b) < 1e-3 * abs(a)
