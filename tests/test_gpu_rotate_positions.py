"""rotate_heads' gradient of float64 positions: it is summed in 64 bits, as its type says.

Tolerance, U = 2^-53 of the sum of the terms' magnitudes: a head's mean square has dim terms (dim U, half of it in
its root) and with root, quotient and products 8; an angle theta errs by 2 |theta| U here and |theta| U in the
definition, with the sines' own 6; a sum over heads, a lane's channels and the lanes of an atom has heads + 16 additions;
products with the frequencies and the rest 8: (dim + heads + 40 + 4 |theta|) U."""
import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


def _inputs(targets, nodes, heads, kv, dim, sections, dtype, far, seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)
    at = far * torch.rand(nodes, len(sections), generator=g, dtype=torch.float64)
    freq = 3.0 * torch.rand(sum(sections), generator=g)
    return q, k, at, freq, 1 + 0.2 * rand(dim), 1 + 0.2 * rand(dim), rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("targets,nodes,heads,kv,dim,sections", [(1, 1, 1, 1, 8, (4,)), (30, 41, 8, 8, 32, (5, 5, 5)), (50, 50, 5, 2, 24, (0, 7)),
                                                                 (20, 33, 16, 4, 64, (8, 8, 8)), (9, 17, 3, 1, 256, (128,)),
                                                                 (3000, 5000, 4, 4, 40, (1, 2, 3, 1, 1, 2, 3, 2)), (0, 7, 2, 2, 16, (3, 3))])
def test_in_64_bits(cuda, targets, nodes, heads, kv, dim, sections, norm, interleaved, dtype):
    for far in (10.0, 1e4):
        print(f"\n[case] positions {targets} {nodes} {heads} {kv} {dim} {sections} {norm} {interleaved} {dtype} {far}", flush=True)
        q, k, at, freq, qw, kw, gq, gk = _inputs(targets, nodes, heads, kv, dim, sections, dtype, far, dim + targets)
        eps = 2.0 ** -20
        weights = (qw, kw) if norm else (None, None)
        want, mag = np.zeros(at.shape), np.zeros(at.shape)
        for x, w, g in ((q, weights[0], gq), (k, weights[1], gk)):
            r, m = oracle.rotate_heads(x.double().numpy(), at.numpy(), freq.double().numpy(), sections,
                                       None if w is None else w.double().numpy(), eps, norm, interleaved, g.double().numpy())
            want += r["dpositions"]
            mag += m["dpositions"]
        atd = at.cuda().requires_grad_(True)
        wd = [None if w is None else w.cuda() for w in weights]

        def step(positions):
            a, b = ds.rotate_heads(q.cuda(), k.cuda(), positions, freq.cuda(), sections, *wd, eps=eps, norm=norm, interleaved=interleaved)
            return torch.autograd.grad([a, b], positions, [gq.cuda(), gk.cuda()])[0]

        got = step(atd)
        assert got.dtype == torch.float64 and torch.equal(got, step(atd))
        tol = (dim + heads + 40 + 4 * far * 3) * U * mag + 1e-300
        bad = ~(np.abs(got.cpu().numpy() - want) <= tol)
        assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {(np.abs(got.cpu().numpy() - want) / tol).max():.3g} of the tolerance"


@pytest.mark.parametrize("interleaved", [False, True])
def test_other_gradients_are_the_same_bits(cuda, interleaved):
    """With and without the positions' gradient; an angle that is not finite stays in its atom."""
    q, k, at, freq, qw, kw, gq, gk = (t.cuda() for t in _inputs(40, 60, 4, 2, 32, (5, 5, 5), torch.bfloat16, 10.0, 3))
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]

    def step(positions, *more):
        a, b = ds.rotate_heads(q, k, positions, freq, None, qw, kw, interleaved=interleaved)
        return torch.autograd.grad([a, b], [*leaves, *more], [gq, gk])

    want = step(at)
    atd = at.clone().requires_grad_(True)
    got = step(atd, atd)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    at2 = at.clone()
    at2[7, 1] = float("nan")
    at2.requires_grad_(True)
    d = step(at2, at2)[-1]
    keep = torch.arange(60) != 7
    assert torch.equal(d[keep], got[-1][keep]) and d[7].isnan().any()


def test_other_gradients_of_many_atoms(cuda):
    """More atoms than workgroups at once: the heads' gradients have the same bits; the weights' are summed in another order,
    each of 30,000 atoms and 4 heads' terms once, 2^-24 of their magnitudes for a term's place in a chain of some 200."""
    q, k, at, freq, qw, kw, gq, gk = (t.cuda() for t in _inputs(30000, 30000, 4, 4, 32, (5, 5, 5), torch.float32, 10.0, 6))
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    atd = at.clone().requires_grad_(True)
    out = []
    for positions in (at, atd):
        y = ds.rotate_heads(q, k, positions, freq, None, qw, kw)
        out.append(torch.autograd.grad(y, leaves + ([positions] if positions is atd else []), [gq, gk]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    for x, g, a, b in ((q, gq, out[0][2], out[1][2]), (k, gk, out[0][3], out[1][3])):
        # (a turned gradient is at most |g_a| + |g_b|, a normalised channel at most sqrt(32) times its mean size)
        hat = x.detach() / x.detach().pow(2).mean(-1, keepdim=True).sqrt()
        mag = (hat.abs() * 2 * g.abs().amax(-1, keepdim=True)).sum((0, 1))
        assert ((a - b).abs() <= 400 * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_images_of_a_periodic_cell(cuda, interleaved):
    """Fractional coordinates and whole waves: an atom's images have its angles, and a query and a key the same product
    wherever the cell's boundary lies between them.  A frequency is off by half a step, 2^-24 of itself, a turn of it by 2 pi m
    2^-24 for a wave number m; three turns of 4 waves, and 8 roundings of 2^-24 of the results' own."""
    print(f"\n[case] images {interleaved}", flush=True)
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(30, 4, 32, generator=g).cuda(), torch.randn(30, 4, 32, generator=g).cuda()
    frac = torch.rand(30, 3, generator=g, dtype=torch.float64).cuda()
    freq = (2 * np.pi * torch.arange(5, dtype=torch.float64).repeat(3)).float().cuda()
    shift = torch.randint(-3, 4, (30, 3), generator=g).cuda()
    a, b = ds.rotate_heads(q, k, frac, freq, norm=False, interleaved=interleaved)
    c, d = ds.rotate_heads(q, k, frac + shift, freq, norm=False, interleaved=interleaved)
    tol = (3 * 2 * np.pi * 4 + 8) * 2.0 ** -24
    for x, y, z in ((a, c, q), (b, d, k)):
        pair = z.abs().amax(-1, keepdim=True) * 2
        assert ((x - y).abs() <= tol * pair).all()


def test_steps_from_graphs(cuda):
    """Captured steps with float64 positions, replayed with eager work between, against eager steps."""
    q, k, at, freq, qw, kw, gq, gk = (t.cuda() for t in _inputs(300, 400, 4, 2, 32, (5, 5, 5), torch.bfloat16, 10.0, 4))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, at, qw, kw)]
        out = ds.rotate_heads(*leaves[:3], freq, None, *leaves[3:])
        return torch.autograd.grad(out, leaves, [gq, gk])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        at.add_(0.37)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
