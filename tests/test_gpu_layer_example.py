"""The example that trains one layer on a built batch (examples/structure_energies.py): the graph
build and the operators that read its result, together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    path = os.path.join(ROOT, "examples", "structure_energies.py")
    spec = importlib.util.spec_from_file_location("structure_energies", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_layer_learns(cuda, example, dtype):
    """One fixed batch can be learnt by heart: the loss falls by half and more."""
    losses = example.train(structures=6, atoms=40, steps=40, dtype=dtype)
    assert torch.isfinite(losses).all()
    assert losses[-5:].mean() < 0.5 * losses[0]


@pytest.mark.parametrize("structures,atoms", [(1, 30), (9, 40)])
def test_the_layers_output(cuda, example, structures, atoms):
    """The layer's energies and gradients in float32 against the same layer of plain 64-bit
    products.  (A chain of sums of up to a few hundred terms: 1e-4 of the largest is 800 roundings.)"""
    torch.manual_seed(1)
    batch = example.make_batch(structures, atoms, seed=1)
    plan, structure, energies = example.make_graph(batch)
    layer = example.Layer(structures, dtype=torch.float32)
    with torch.no_grad():
        layer.mix.normal_(), layer.bias.normal_(), layer.shift.normal_()
    got = layer(batch, plan, structure)
    names, params = zip(*layer.named_parameters())
    grads = torch.autograd.grad(((got - energies) ** 2).sum(), params)

    edges, offsets, per_structure = example.dynamis_state.radius_graph_pbc_cuda(batch, example.RADIUS, 0)
    cell = torch.repeat_interleave(batch.cell, per_structure, 0)
    d = (batch.pos[edges[0]] - batch.pos[edges[1]] + (offsets.unsqueeze(-1) * cell).sum(1)).norm(dim=1).cpu()
    bucket = torch.bucketize(d, torch.linspace(0.0, example.RADIUS, example.BUCKETS + 1)[1:-1], right=True)
    src, dst = edges.cpu()
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in zip(names, params)}
    share = torch.softmax(p["mix"], 1)[structure.cpu()]
    x = p["embed"][batch.species.cpu()]
    qkv = sum(share[:, e:e + 1] * (x @ p["qkv"][e].T) for e in range(example.EXPERTS))
    q, k, v = (t.unflatten(1, (layer.heads, layer.dim)) for t in qkv.chunk(3, 1))
    logits = (q[dst] * k[src]).sum(-1) * layer.dim ** -0.5 + p["bias"][bucket]
    w = torch.exp(logits)
    total = torch.zeros(q.shape[:2], dtype=torch.float64).index_add(0, dst, w)
    y = torch.zeros_like(q).index_add(0, dst, (w / total[dst])[..., None] * v[src]).flatten(1)
    y = torch.nn.functional.silu(x + y)
    atom = sum(share[:, e:e + 1] * (y @ p["out"][e].T) for e in range(example.EXPERTS)) + p["shift"][structure.cpu()]
    want = torch.zeros(structures, dtype=torch.float64).index_add(0, structure.cpu(), atom[:, 0]) / batch.natoms.cpu()
    wants = torch.autograd.grad(((want - energies.double().cpu()) ** 2).sum(), list(p.values()))
    for name, a, b in zip(("energies", *names), (got, *grads), (want, *wants)):
        err = (a.detach().double().cpu() - b.detach()).abs().max()
        assert err <= 1e-4 * b.detach().abs().max(), (name, float(err))
