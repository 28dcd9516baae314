"""A model of one attention layer over built neighbour lists, trained on a batch of structures.

    python examples/structure_energies.py [--structures 32] [--atoms 64] [--steps 30] [--float32]

Each step of a model that is called on what the graph build returns, with the operators that go
with it:

  radius_graph_pbc_cuda   the batch's edges, structure after structure
  neighbor_plan           their lists by target and by source, and each edge's distance bucket
  grouped_linear          q, k and v of each structure's atoms, by weights mixed for the structure
                          out of a few experts' (rows by structure: ``natoms``)
  neighbor_attention      every atom over its neighbours, with a learned bias by distance
  grouped_linear          the atoms' energies, by the structure's own read-out

The energies to learn are a sum over pairs of a Lennard-Jones-like well, so that they depend on
what the layer can see: the distances' buckets and the atoms' species.
"""
from __future__ import annotations

import argparse
import os
import sys
import time
import types

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from dynamis_amd import dynamis_state  # noqa: E402

RADIUS, SPECIES, BUCKETS, EXPERTS = 6.0, 3, 32, 4


def make_batch(structures, atoms, seed=0, device="cuda"):
    """Jittered cubic lattices at 0.1 atoms per cubic Angstrom, of `atoms` / 2 to `atoms` atoms each."""
    g = torch.Generator().manual_seed(seed)
    natoms = torch.randint(max(2, atoms // 2), atoms + 1, (structures,), generator=g)
    pos, cells = [], []
    for n in natoms.tolist():
        side = next(s for s in range(1, n + 1) if s ** 3 >= n)
        a = (10.0 * n) ** (1 / 3) / side
        at = torch.randperm(side ** 3, generator=g)[:n]
        grid = torch.stack([at // (side * side), at // side % side, at % side], 1)
        pos.append((grid + 0.5 * torch.rand(n, 3, generator=g)) * a)
        cells.append(torch.eye(3) * a * side)
    species = torch.randint(0, SPECIES, (int(natoms.sum()),), generator=g)
    return types.SimpleNamespace(pos=torch.cat(pos).to(device), cell=torch.stack(cells).to(device),
                                 natoms=natoms.to(device), pbc=torch.tensor([True, True, True]),
                                 species=species.to(device))


def make_graph(batch):
    """The batch's plan, and its energies per atom."""
    edges, offsets, per_structure = dynamis_state.radius_graph_pbc_cuda(batch, RADIUS, 0)
    cell = torch.repeat_interleave(batch.cell, per_structure, 0)
    source, target = edges
    vectors = batch.pos[source] - batch.pos[target] + (offsets.unsqueeze(-1) * cell).sum(1)
    distances = vectors.norm(dim=1)
    boundaries = torch.linspace(0.0, RADIUS, BUCKETS + 1, device=edges.device)[1:-1]
    plan = dynamis_state.neighbor_plan(edges, batch.pos.size(0), distances=distances, boundaries=boundaries)
    x = (2.2 / distances.clamp(min=2.0)) ** 6
    depth = 1.0 + 0.5 * (batch.species[source] == batch.species[target])
    structure = torch.repeat_interleave(torch.arange(batch.natoms.numel(), device=edges.device), batch.natoms)
    energies = torch.zeros(batch.natoms.numel(), device=edges.device)
    energies.index_add_(0, structure[target], depth * (x * x - x))
    return plan, structure, energies / batch.natoms


class Layer(torch.nn.Module):
    """Attention of each atom over its neighbours, its linear maps mixed for every structure."""

    def __init__(self, structures, channels=64, heads=4, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.heads, self.dim, self.dtype = heads, channels // heads, dtype
        new = lambda *s: torch.nn.Parameter(torch.randn(*s, device=device))  # noqa: E731
        self.embed = new(SPECIES, channels)
        self.mix = torch.nn.Parameter(torch.zeros(structures, EXPERTS, device=device))
        self.qkv = torch.nn.Parameter(torch.randn(EXPERTS, 3 * channels, channels, device=device) * channels ** -0.5)
        self.bias = torch.nn.Parameter(torch.zeros(BUCKETS, heads, device=device))
        self.out = torch.nn.Parameter(torch.randn(EXPERTS, 1, channels, device=device) * channels ** -0.5)
        self.shift = torch.nn.Parameter(torch.zeros(structures, 1, device=device))

    def forward(self, batch, plan, structure):
        share = torch.softmax(self.mix, 1)
        mixed = lambda w: (share @ w.flatten(1)).unflatten(1, w.shape[1:]).to(self.dtype)  # noqa: E731
        x = self.embed[batch.species].to(self.dtype)
        qkv = dynamis_state.grouped_linear(x, mixed(self.qkv), batch.natoms)
        # (views of one product: whole rows, read in place)
        q, k, v = (t.unflatten(1, (self.heads, self.dim)) for t in qkv.chunk(3, 1))
        y = dynamis_state.neighbor_attention(q, k, v, plan, self.bias).flatten(1)
        y = torch.nn.functional.silu(x + y)
        atoms = dynamis_state.grouped_linear(y, mixed(self.out), batch.natoms, self.shift.to(self.dtype))
        sums = torch.zeros(batch.natoms.numel(), device=atoms.device)
        return sums.index_add_(0, structure, atoms[:, 0].float()) / batch.natoms


def train(structures=32, atoms=64, steps=30, dtype=torch.bfloat16, seed=0, rate=3e-2, report=None):
    """The losses of `steps` steps of training on one batch."""
    torch.manual_seed(seed)
    batch = make_batch(structures, atoms, seed)
    plan, structure, energies = make_graph(batch)
    layer = Layer(structures, dtype=dtype)
    optimizer = torch.optim.Adam(layer.parameters(), lr=rate)
    losses = []
    for step in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = ((layer(batch, plan, structure) - energies) ** 2).mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report is not None and step % 10 == 0:
            report(f"step {step}: loss {float(losses[-1]):.5f}")
    return torch.stack(losses).cpu()


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--structures", type=int, default=32)
    parser.add_argument("--atoms", type=int, default=64)
    parser.add_argument("--steps", type=int, default=30)
    parser.add_argument("--float32", action="store_true")
    args = parser.parse_args()
    began = time.perf_counter()
    losses = train(args.structures, args.atoms, args.steps, torch.float32 if args.float32 else torch.bfloat16,
                   report=print)
    print(f"{args.structures} structures, {args.steps} steps in {time.perf_counter() - began:.2f} s: "
          f"loss {losses[0]:.5f} -> {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
