"""The example that runs the products, the readout and the optimizer step together."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("train_readout", os.path.join(ROOT, "examples", "train_readout.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_network_learns_and_does_not_see_rotations():
    """The variance of what is to be learned is what a constant answer leaves; half of it is a low bar.  A rotation changes the answer by the
    rounding of the harmonics and of sums, some 1e-5 of it, through a norm that may enlarge it."""
    example = _example()
    network, losses = example.train(steps=150)
    generator = torch.Generator(device="cuda").manual_seed(5)
    x, want = example.clouds(512, 32, generator)
    assert torch.isfinite(losses).all()
    with torch.no_grad():
        got = network(x)
        q, r = torch.linalg.qr(torch.randn(3, 3, generator=generator, device="cuda"))
        q = q * torch.sign(torch.diagonal(r))
        q[:, 0] *= torch.det(q)
        turned = network(q @ x)
    assert (got - want).square().mean() < 0.5 * want.var()
    assert (turned - got).abs().max() < 1e-2 * want.std()


def test_a_captured_forward_and_backward_repeats():
    """After a first call of each size, forward and backward can be captured: nothing in them waits for the host."""
    import gelib_b200 as G
    dev = "cuda"
    x = torch.randn(300, 96, device=dev, dtype=torch.bfloat16)
    norm = G.GroupNorm(8, 96, activation="silu", device=dev, dtype=torch.bfloat16)
    layer = G.Linear(96, 160, activation="silu", device=dev, dtype=torch.bfloat16)
    params = list(norm.parameters()) + list(layer.parameters())

    def step():
        y = layer(norm(x))
        return [y, *torch.autograd.grad(y, params, torch.ones_like(y))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, [t.clone() for t in step()]))
