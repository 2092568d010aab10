"""Trains a small rotation-invariant network on synthetic point clouds.

    PYTHONPATH=. python examples/train_readout.py [steps]

Every cloud is a few points in space; what is learned is the logarithm of the determinant of its second moments, its volume so to speak.
The harmonics of the points are summed over the cloud, mixed by learned weights and multiplied with themselves (Clebsch-Gordan products); the
l=0 parts that come out do not change when the cloud is rotated.  They are normalised and go through dense layers to the answer.
All weights, complex and real, take an AdamW step whose moments are held in 8 bits.
"""
import sys

import torch

import gelib_b200 as gelib


class Network(torch.nn.Module):

    def __init__(self, maxl=2, channels=8, hidden=64, device="cuda"):
        super().__init__()
        self.maxl = maxl
        self.mix = gelib.SO3linear({l: 2 for l in range(maxl + 1)}, {l: channels for l in range(maxl + 1)}, device=device)
        invariants = 2 * (maxl + 1) * channels * channels   # real and imaginary parts of every pair of channels at every l
        self.norm = gelib.GroupNorm(maxl + 1, invariants, activation="silu", device=device)
        self.first = gelib.Linear(invariants, hidden, activation="silu", device=device)
        self.second = gelib.Linear(hidden, hidden, activation="silu", device=device)
        self.last = gelib.Linear(hidden, 1, device=device)

    def forward(self, points):
        """points (b, 3, n): n points of each cloud."""
        b, _, n = points.shape
        radius = points.norm(dim=1)
        with torch.no_grad():
            parts = []
            for l in range(self.maxl + 1):
                y = gelib.SO3part.spharm(l, points.contiguous()).as_subclass(torch.Tensor)               # (b, 2l+1, n)
                parts.append(torch.stack([(y * f[:, None]).mean(2) for f in (radius, radius * radius)], 2))   # two radial weights
        v = gelib.SO3vec(*parts) * self.mix.W
        z = gelib.CGproduct(v, v, maxl=0).parts[0].as_subclass(torch.Tensor)                               # (b, 1, invariants / 2)
        x = self.norm(torch.view_as_real(z).reshape(b, -1))
        x = self.first(x)
        x = self.second(x, residual=x)
        return self.last(x)[:, 0]


def clouds(batch, points, generator, device="cuda"):
    """Clouds stretched by random amounts, and what is to be learned of them."""
    stretch = 0.5 + torch.rand(batch, 3, 1, generator=generator, device=device)
    x = torch.randn(batch, 3, points, generator=generator, device=device) * stretch
    moments = x @ x.transpose(1, 2) / points
    return x, torch.logdet(moments)


def train(steps=200, batch=256, points=32, seed=0, report=None):
    torch.manual_seed(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    network = Network()
    optimizer = gelib.AdamW(network.parameters(), lr=3e-3, state_bits=8, seed=seed)
    losses = []
    for step in range(steps):
        x, want = clouds(batch, points, generator)
        loss = (network(x) - want).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report and step % report == 0:
            print("step %d: loss %.4f" % (step, losses[-1].item()))
    return network, torch.stack(losses).cpu()


if __name__ == "__main__":
    steps = int(sys.argv[1]) if len(sys.argv) > 1 else 200
    network, losses = train(steps, report=max(1, steps // 10))
    print("mean loss of the first ten steps %.3f, of the last ten %.3f" % (losses[:10].mean(), losses[-10:].mean()))
