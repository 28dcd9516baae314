"""Gradients of grouped_linear with an activation in bfloat16: they are as near to 64 bits as their own rounding,
the activation's gradient on the way to them included.

Tolerances, EPS = 2^-24, as in test_gpu_grouped_apply.py but for dz: it is held as two bfloat16, each off by
at most half a step, 2^-8 of what it stands for, so that dz is off by 2^-16 of itself.  The products then sum twice the
terms."""
import math

import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
ACTS = pytest.mark.parametrize("act", ["silu", "gelu"])


def _f(act, z):
    """(f', the relative error's growth with z)."""
    if act == "silu":
        s, t = np.exp(-np.logaddexp(0, -z)), np.exp(-np.logaddexp(0, z))
        return s * (1 + z * t), 2 * np.abs(z)
    share = 0.5 * np.vectorize(math.erfc)(-z / math.sqrt(2))
    return share + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi), 2 * z * z


def _make(sizes, k, n, seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    rows = sum(sizes)
    return rand(rows, k), (2 * rand(len(sizes), n, k) / math.sqrt(k)), rand(len(sizes), n), rand(rows, n)


def _grads(x, w, b, sizes, act, grad):
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = ds.grouped_linear(leaves[0], leaves[1], torch.tensor(sizes).cuda(), leaves[2], activation=act)
    return torch.autograd.grad(y, leaves, grad.cuda())


@ACTS
@pytest.mark.parametrize("sizes,k,n", [([5, 0, 130, 1, 64], 64, 128), ([5, 0, 130, 1, 64], 33, 65), ([1], 8, 8), ([300, 41], 256, 512),
                                       ([300, 41], 520, 136), ([255, 257], 100, 164), ([250] * 128, 64, 64), ([9000] * 4, 72, 96),
                                       ([20000], 24, 200), ([700, 0, 900], 50, 130)],
                         ids=lambda v: v if isinstance(v, int) else f"{len(v)}_{sum(v)}")
def test_as_near_as_their_rounding(cuda, sizes, k, n, act):
    print(f"\n[case] gradients {sizes[:4]} {k} {n} {act}", flush=True)
    x, w, b, grad = _make(sizes, k, n, k + n)
    got = _grads(x, w, b, sizes, act, grad)
    x64, w64, b64, g64 = (t.double().numpy() for t in (x, w, b, grad))
    r, m = oracle.grouped_linear(x64, w64, sizes, b64)
    z, z_err = r["y"], (k + 3) * EPS * m["y"]
    slope, growth = _f(act, z)
    dz = g64 * slope
    d_err = np.abs(g64) * (0.8 * z_err + (8 + growth) * EPS * (np.abs(slope) + 1)) + 2.0 ** -16 * np.abs(dz)
    r, m = oracle.grouped_linear(x64, w64, sizes, b64, dz)
    _, e = oracle.grouped_linear(x64, w64, sizes, None, d_err)
    for name, t, terms in zip(("dx", "dweight", "dbias"), got, (n, max(sizes), max(sizes))):
        t = t.double().cpu().numpy()
        tol = (2 * terms + 2) * EPS * (m[name] + e[name]) + e[name] + 2.0 ** -8 * np.abs(r[name]) + 1e-37
        bad = ~(np.abs(t - r[name]) <= tol)
        assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, worst {np.abs(t - r[name])[bad].max():.3g} at {np.argwhere(bad)[0]}"
    assert all(torch.equal(p, q) for p, q in zip(got, _grads(x, w, b, sizes, act, grad)))


@ACTS
@pytest.mark.parametrize("k,n", [(40, 104), (41, 101)])
def test_what_is_not_finite_shows_as_such(cuda, k, n, act):
    """An infinite gradient, and one that rounds to infinity, is one in its row, its columns' weights and bias: no NaN."""
    print(f"\n[case] infinite {k} {n} {act}", flush=True)
    x, w, b, grad = _make([30, 40], k, n, 3)
    x, w, b = x.abs() + 0.25, w.abs() + 0.25, b.abs() + 4  # (slopes near 1, nothing of another sign)
    want = _grads(x, w, b, [30, 40], act, grad)
    for value in (float("inf"), torch.finfo(torch.bfloat16).max):
        grad2 = grad.clone()
        grad2[50, 7] = value
        dx, dw, db = _grads(x, w * 3 if value < float("inf") else w, b, [30, 40], act, grad2)
        assert not dx.isnan().any() and not dw.isnan().any() and not db.isnan().any()
        if value == float("inf"):
            keep = torch.arange(70) != 50
            assert (dx[50] == value).all() and torch.equal(dx[keep], want[0][keep])
            assert (dw[1, 7] == value).all() and db[1, 7] == value and torch.equal(dw[0], want[1][0])
            assert torch.equal(db[0], want[2][0])


@ACTS
@pytest.mark.parametrize("k,n", [(64, 96), (50, 70)])
def test_only_what_is_asked(cuda, k, n, act):
    """Each gradient alone has the bits that it has among the others (without the weight's the workspace is smaller)."""
    x, w, b, grad = (t.cuda() for t in _make([33, 100, 0, 300], k, n, 4))
    sizes = torch.tensor([33, 100, 0, 300]).cuda()
    want = _grads(x, w, b, [33, 100, 0, 300], act, grad)
    for i in range(3):
        leaves = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(ds.grouped_linear(*leaves[:2], sizes, leaves[2], activation=act), leaves[i], grad)
        assert torch.equal(got, want[i])


def test_steps_from_graphs_and_streams(cuda):
    """Two captured training steps replayed in turn and on two streams, with eager work between, against eager steps."""
    sizes = [60, 0, 130, 7]
    n_rows = torch.tensor(sizes).cuda()
    sets = [[t.cuda() for t in _make(sizes, 64, 96, seed)] for seed in (1, 2)]

    def step(x, w, b, grad):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ds.grouped_linear(leaves[0], leaves[1], n_rows, leaves[2], activation="gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for s in sets:
            s[0].copy_(torch.randn(197, 64, device="cuda"))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, step(*s))), i
