"""Trains a small rotation-invariant network to tell the species of a hidden atom from its neighbours, then a smaller one to follow it.

    PYTHONPATH=. python examples/train_species.py [steps]

Every neighbour's species is looked up in a complex table, whose rows are the channels of an l=0 part, and multiplied with the harmonics of
where the neighbour lies; the sums over the neighbours are mixed by learned weights and multiplied with themselves (Clebsch-Gordan
products).  The l=0 parts go through a norm and a dense layer to a vector that is scored against all species.  The scores themselves are
never written: the loss, and the divergence that the smaller network is trained by, come from the vectors and the matrix of species.
"""
import sys

import torch

import gelib_b200 as gelib


class Network(torch.nn.Module):

    def __init__(self, species=100, maxl=2, channels=8, hidden=64, device="cuda"):
        super().__init__()
        self.maxl = maxl
        self.table = gelib.Embedding(species, channels, device=device, dtype=torch.complex64)
        self.mix = gelib.SO3linear({l: channels for l in range(maxl + 1)}, {l: channels for l in range(maxl + 1)}, device=device)
        invariants = 2 * (maxl + 1) * channels * channels   # real and imaginary parts of every pair of channels at every l
        self.norm = gelib.GroupNorm(maxl + 1, invariants, activation="silu", device=device)
        self.layer = gelib.Linear(invariants, hidden, activation="silu", device=device)
        self.head = gelib.Classifier(hidden, species, device=device)

    def forward(self, points, species):
        """points (b, 3, n) around the hidden atom, species (b, n): a vector for each of the b atoms."""
        b = points.size(0)
        e = self.table(species)                                                                          # (b, n, channels)
        near = torch.exp(-points.square().sum(1))
        parts = []
        for l in range(self.maxl + 1):
            with torch.no_grad():
                y = gelib.SO3part.spharm(l, points).as_subclass(torch.Tensor) * near[:, None]            # (b, 2l+1, n)
            parts.append(y @ e)
        v = gelib.SO3vec(*parts) * self.mix.W
        z = gelib.CGproduct(v, v, maxl=0).parts[0].as_subclass(torch.Tensor)                             # (b, 1, invariants / 2)
        return self.layer(self.norm(torch.view_as_real(z).reshape(b, -1)))


def atoms(batch, neighbours, species, generator, device="cuda"):
    """Neighbours and the hidden atom's species: that of the nearest one; some atoms are not asked for."""
    points = torch.randn(batch, 3, neighbours, generator=generator, device=device)
    of = torch.randint(species, (batch, neighbours), generator=generator, device=device)
    hidden = of.gather(1, points.square().sum(1).argmin(1, keepdim=True))[:, 0]
    return points, of, torch.where(torch.rand(batch, generator=generator, device=device) < 0.1, -100, hidden)


def train(steps=200, batch=512, neighbours=12, species=100, top=8, seed=0, report=None):
    """The network, the smaller one, and the losses of both."""
    torch.manual_seed(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    large, small = Network(species, hidden=64), Network(species, maxl=1, channels=4, hidden=32)
    optimizers = [gelib.AdamW(n.parameters(), lr=3e-3, seed=seed) for n in (large, small)]
    losses = []
    for step in range(steps):
        points, of, hidden = atoms(batch, neighbours, species, generator)
        h = large(points, of)
        loss = large.head.cross_entropy(h, hidden)
        with torch.no_grad():
            logits, ids = large.head(h).topk(top)
        follow = small.head.distillation(small(points, of), ids, logits, temperature=2.0)
        for optimizer, value in zip(optimizers, (loss, follow)):
            optimizer.zero_grad()
            value.backward()
            optimizer.step()
        losses.append(torch.stack([loss.detach(), follow.detach()]))
        if report and step % report == 0:
            print("step %d: loss %.4f, divergence of the smaller one %.4f" % (step, *losses[-1].tolist()))
    return large, small, torch.stack(losses).cpu()


if __name__ == "__main__":
    steps = int(sys.argv[1]) if len(sys.argv) > 1 else 200
    _, _, losses = train(steps, report=max(1, steps // 10))
    print("mean losses of the first ten steps %.3f and %.3f, of the last ten %.3f and %.3f" % (*losses[:10].mean(0), *losses[-10:].mean(0)))
