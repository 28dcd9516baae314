"""rotate_heads on the GPU against its definition in 64 bits (oracle/layers.py), forward and backward:
head widths, odd numbers of pairs, axes, both layouts of the pairs, ghosts, strides, far positions,
what is not finite, streams, graphs, and bit-equal repeats.

Tolerances, in units of EPS = 2^-24 of a result's magnitude (the sum of its terms').  1 / rms: the sum
of `dim` squares errs by dim EPS, half of it after the root, with 3 for the rest; a sine or cosine:
2 EPS from the angle (half a turn rounded to 24 bits: 2 pi 2^-26) and 4 from the function; products and
sums of a pair 4.  So a value: dim / 2 + 16.  dx has a mean of `dim` products on top: 2 dim + 40.
Sums over rows and heads: one more for each term.  bfloat16 results are rounded once, 2^-8 of themselves."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
LAYOUTS = pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])


def _near(name, got, want, mag, n, rounded):
    got = got.detach().double().cpu().numpy()
    tol = n * EPS * mag + (2.0 ** -8 * np.abs(want) if rounded else 0)
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    assert got.shape == want.shape and not bad.any(), \
        f"{name}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want)[bad]):.3g} at {np.argwhere(bad)[0]}"


def _make(targets, nodes, heads, kv, dim, sections, dtype, weights, pos=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)
    at = (20 * torch.rand(nodes, len(sections), generator=g, dtype=torch.float64)).to(pos)
    f = torch.exp(-2 * torch.rand(sum(sections), generator=g))
    qw = (1 + 0.3 * rand(dim)).to(weights) if weights else None
    kw = (1 + 0.3 * rand(dim)).to(weights) if weights else None
    return q, k, at, f, qw, kw, rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)


def _check(targets, nodes, heads, kv, dim, sections, dtype, interleaved=False, norm=True, weights="own", pos=torch.float32,
           eps=1e-6, seed=0):
    print(f"\n[case] rotate {targets}/{nodes} {heads}/{kv}x{dim} {sections} {dtype} {interleaved} {norm} {weights} {pos}", flush=True)
    wtype = {None: None, "own": dtype, "float": torch.float32}[weights if norm else None]
    q, k, at, f, qw, kw, gq, gk = _make(targets, nodes, heads, kv, dim, sections, dtype, wtype, pos, seed)
    leaves = [t.cuda() for t in (q, k)]
    w = [t.cuda() if t is not None else None for t in (qw, kw)]
    at_d, f_d = at.cuda(), f.cuda()
    wanted = leaves + [t for t in w if t is not None] + ([at_d] if pos.is_floating_point else [])
    for t in wanted:
        t.requires_grad_(True)

    def step():
        y = ds.rotate_heads(leaves[0], leaves[1], at_d, f_d, sections, w[0], w[1], eps=eps, norm=norm, interleaved=interleaved)
        return [*y, *torch.autograd.grad(y, wanted, [gq.cuda(), gk.cuda()])]

    got = step()
    np64 = lambda t: None if t is None else t.double().numpy()  # noqa: E731
    r = [oracle.rotate_heads(np64(x), np64(at), np64(f), sections, np64(wt), eps, norm, interleaved, np64(g))
         for x, wt, g in ((q, qw, gq), (k, kw, gk))]
    names, rounded, value, back = ["q", "k"], dtype == torch.bfloat16, dim / 2 + 16, 2 * dim + 40
    for i in range(2):
        _near(names[i], got[i], r[i][0]["y"], r[i][1]["y"], value, rounded)
        _near("d" + names[i], got[2 + i], r[i][0]["dx"], r[i][1]["dx"], back, rounded)
    more = got[4:]
    if wtype:
        for i, (n, t) in enumerate(zip((targets * heads, nodes * kv), more[:2])):
            _near("dweight", t, r[i][0]["dweight"], r[i][1]["dweight"], n + back, wtype == torch.bfloat16)
        more = more[2:]
    if pos.is_floating_point:
        want, mag = (r[0][j]["dpositions"] + r[1][j]["dpositions"] for j in range(2))
        _near("dpositions", more[0], want, mag, heads + kv + sum(sections) + back, False)
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
    with torch.no_grad():
        y = ds.rotate_heads(leaves[0], leaves[1], at_d, f_d, sections, w[0], w[1], eps=eps, norm=norm, interleaved=interleaved)
    assert torch.equal(y[0], got[0]) and torch.equal(y[1], got[1])


@TYPES
@LAYOUTS
@pytest.mark.parametrize("dim,sections", [(8, (1,)), (8, (4,)), (16, (3, 2)), (24, (12,)), (24, (2, 2, 3)), (32, (5, 5, 5)),
                                          (32, (16,)), (48, (0, 7, 17)), (64, (31,)), (64, (32,)), (96, (16, 16, 16)),
                                          (128, (21, 21, 21)), (128, (64,)), (200, (1, 99)), (256, (128,)),
                                          (256, (9, 10, 11, 12, 13, 14, 15, 16))])
def test_widths_and_sections(cuda, dim, sections, dtype, interleaved):
    _check(37, 37, 4, 2, dim, sections, dtype, interleaved, seed=dim)


@TYPES
@LAYOUTS
@pytest.mark.parametrize("targets,nodes,heads,kv", [(1, 1, 1, 1), (1, 1, 8, 8), (3, 1000, 5, 3), (0, 9, 4, 4), (300, 301, 1, 1),
                                                    (63, 65, 32, 1), (128, 128, 3, 24), (2100, 2100, 8, 8)])
def test_rows_and_heads(cuda, targets, nodes, heads, kv, dtype, interleaved):
    _check(targets, nodes, heads, kv, 40, (6, 7), dtype, interleaved, seed=nodes)


@TYPES
@LAYOUTS
@pytest.mark.parametrize("norm,weights", [(True, None), (True, "float"), (False, None)])
@pytest.mark.parametrize("pos", [torch.float32, torch.float64, torch.int64], ids=["p32", "p64", "pint"])
def test_norms_weights_positions(cuda, norm, weights, pos, dtype, interleaved):
    _check(70, 90, 6, 2, 32, (5, 6), dtype, interleaved, norm, weights, pos, eps=1e-3, seed=3)


def test_many_rows_a_wave(cuda):
    """More atoms than the backward pass has workgroups."""
    _check(20000, 20000, 2, 1, 8, (3,), torch.float32, seed=4)
    _check(9000, 9001, 8, 8, 64, (10, 10, 10), torch.bfloat16, seed=5)


@TYPES
@LAYOUTS
def test_far_positions(cuda, dtype, interleaved):
    """Angles of 10^8 radians: their 64-bit error is 10^8 2^-51, the rest is that of near ones."""
    print(f"\n[case] far {dtype} {interleaved}", flush=True)
    q, k, at, f, *_ = _make(50, 50, 2, 2, 32, (16,), dtype, None, torch.int64)
    at = at * 10 ** 7 + torch.arange(50)[:, None]
    for pos in (at, at.double(), -at):
        got = ds.rotate_heads(q.cuda(), k.cuda(), pos.cuda(), f.cuda(), norm=False, interleaved=interleaved)
        for x, t in zip((q, k), got):
            r, m = oracle.rotate_heads(x.double().numpy(), pos.double().numpy(), f.double().numpy(), (16,), norm=False,
                                       interleaved=interleaved)
            _near("far", t, r["y"], m["y"], 16 + 2e8 * 2.0 ** -51 / EPS, dtype == torch.bfloat16)


@TYPES
def test_strides(cuda, dtype):
    """Views of one product, transposed heads, broadcast rows, odd alignment: the same bits."""
    print(f"\n[case] strides {dtype}", flush=True)
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(50, 3 * 4 * 24, generator=g).to(dtype).cuda()
    at, f = torch.rand(50, 3, generator=g).cuda(), torch.rand(9, generator=g).cuda()
    q, k, _ = (t.unflatten(1, (4, 24)) for t in qkv.chunk(3, 1))
    want = ds.rotate_heads(q.contiguous(), k.contiguous(), at, f)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    for p, o in ((q, k), (odd(q), odd(k)), (q.transpose(0, 1).contiguous().transpose(0, 1), k.permute(2, 0, 1).contiguous().permute(1, 2, 0))):
        got = ds.rotate_heads(p, o, at, f)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = ds.rotate_heads(q, k, at.t().contiguous().t(), torch.stack([f, f], 1)[:, 0])
    assert torch.equal(got[0], want[0])
    one = q[:1].expand(50, 4, 24)
    assert torch.equal(ds.rotate_heads(one, k, at, f)[0], ds.rotate_heads(one.contiguous(), k, at, f)[0])
    # a gradient that is broadcast, and one of a single result
    p, o = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    y = ds.rotate_heads(p, o, at, f)
    a = torch.autograd.grad(y[0].sum() + y[1].sum(), (p, o))
    b = torch.autograd.grad(ds.rotate_heads(p, o, at, f), (p, o), [torch.ones_like(p), torch.ones_like(o)])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert not torch.autograd.grad(ds.rotate_heads(p, o, at, f)[0].sum(), o)[0].any()


@TYPES
@LAYOUTS
def test_what_is_not_finite_stays_in_its_head(cuda, dtype, interleaved):
    print(f"\n[case] not finite {dtype} {interleaved}", flush=True)
    q, k, at, f, qw, kw, gq, gk = (t.cuda() for t in _make(20, 30, 3, 5, 32, (4, 5), dtype, dtype))
    want = ds.rotate_heads(q, k, at, f, (4, 5), qw, kw, interleaved=interleaved)
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[7, 1, 3] = bad
        got = ds.rotate_heads(q2, k, at, f, (4, 5), qw, kw, interleaved=interleaved)
        keep = torch.ones(20, 3, dtype=torch.bool)
        keep[7, 1] = False
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1], want[1]) and got[0][7, 1].isnan().any()
    # a position of a ghost: k's row, and neither q's weight nor another atom's anything
    at2 = at.clone()
    at2[25, 0] = float("nan")
    leaves = [t.requires_grad_(True) for t in (q, k, at, at2, qw, kw)]
    run = lambda p: ds.rotate_heads(leaves[0], leaves[1], p, f, (4, 5), qw, kw, interleaved=interleaved)  # noqa: E731
    got = run(at2)
    rows = torch.arange(30) != 25
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][rows], want[1][rows]) and got[1][25].isnan().any()
    a = torch.autograd.grad(got, [q, k, at2, qw], [gq, gk])
    b = torch.autograd.grad(run(at), [q, k, at, qw], [gq, gk])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1][rows], b[1][rows]) and torch.equal(a[2][rows], b[2][rows])
    assert torch.equal(a[3], b[3])
    # rows of zeros: zeros (eps is not), and no NaN in the gradients
    z = torch.zeros_like(q).requires_grad_(True)
    y = ds.rotate_heads(z, k, at, f, (4, 5), qw, kw, interleaved=interleaved)
    assert not y[0].any()
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad(y, [z, k, qw, kw], [gq, gk]))


def test_eps_of_zero_leaves_idle_lanes_out(cuda):
    """Five heads on eight places: the places without a head add no NaN to the weights' gradients."""
    q, k, at, f, qw, kw, gq, gk = (t.cuda() for t in _make(9, 11, 5, 3, 24, (7,), torch.float32, torch.float32))
    w = [qw.requires_grad_(True), kw.requires_grad_(True)]
    got = torch.autograd.grad(ds.rotate_heads(q, k, at, f, None, *w, eps=0.0), w, [gq, gk])
    for t, x, wt, g in zip(got, (q, k), w, (gq, gk)):
        c = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
        r, m = oracle.rotate_heads(c(x), c(at), c(f), (7,), c(wt), 0.0, grad=c(g))
        _near("dweight", t, r["dweight"], m["dweight"], 11 * 5 + 88, False)


@LAYOUTS
def test_gradients_against_differences(cuda, interleaved):
    q, k, at, f, qw, kw, gq, gk = _make(6, 7, 3, 2, 16, (3, 4), torch.float32, torch.float32, torch.float64, 8)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, at, qw, kw)]
    y = ds.rotate_heads(leaves[0], leaves[1], leaves[2], f.cuda(), (3, 4), leaves[3], leaves[4], interleaved=interleaved)
    grads = torch.autograd.grad(y, leaves, [gq.cuda(), gk.cuda()])
    p = [t.double().numpy() for t in (q, k, at, qw, kw)]
    rng = np.random.default_rng(9)

    def loss(v):
        a, b = (oracle.rotate_heads(v[i], v[2], f.numpy(), (3, 4), v[3 + i], interleaved=interleaved)[0]["y"] for i in range(2))
        return (a * gq.double().numpy()).sum() + (b * gk.double().numpy()).sum()

    for i, g in enumerate(grads):
        d, h = rng.standard_normal(p[i].shape), 1e-5
        up, down = ([*p[:i], p[i] + e * h * d, *p[i + 1:]] for e in (1, -1))
        diff, g = (loss(up) - loss(down)) / (2 * h), g.double().cpu().numpy()
        assert abs(diff - (g * d).sum()) < 1e-5 * (1 + np.abs(g * d).sum()), i


def test_streams_and_graphs(cuda):
    """On a side stream, and replayed from a graph with eager work in between: the same bits."""
    print("\n[case] streams and graphs", flush=True)
    q, k, at, f, qw, kw, gq, gk = (t.cuda() for t in _make(500, 600, 8, 2, 64, (10, 10, 10), torch.bfloat16, torch.bfloat16))
    leaves = [t.requires_grad_(True) for t in (q, k, at, qw, kw)]
    step = lambda: (y := ds.rotate_heads(q, k, at, f, None, qw, kw),  # noqa: E731
                    torch.autograd.grad(y, leaves, [gq, gk]))
    flat = lambda r: [*r[0], *r[1]]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = flat(step())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, flat(step())))
    fixed = [t.detach() for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        out = ds.rotate_heads(fixed[0], fixed[1], fixed[2], f, None, fixed[3], fixed[4])
    for i in range(4):
        fresh = torch.randn(500, 8, 64, device="cuda").bfloat16()
        with torch.no_grad():
            fixed[0].copy_(fresh)
            graph.replay()
            eager = ds.rotate_heads(fresh, fixed[1], fixed[2], f, None, fixed[3], fixed[4])
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), i


def test_no_rows(cuda):
    q, k = torch.empty(0, 4, 32, device="cuda"), torch.empty(0, 2, 32, device="cuda")
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = ds.rotate_heads(q, k, torch.empty(0, 3, device="cuda"), torch.ones(6, device="cuda"), None, w, w)
    assert y[0].shape == q.shape and y[1].shape == k.shape
    assert not torch.autograd.grad(y, w, [q, k])[0].any()


def test_a_row_is_the_same_alone(cuda):
    """One new atom (or token) at a time gives the bits of the whole."""
    q, k, at, f, qw, kw, *_ = (t.cuda() for t in _make(40, 40, 4, 2, 64, (32,), torch.bfloat16, torch.float32))
    whole = ds.rotate_heads(q, k, at, f, None, qw, kw)
    for i in (0, 17, 39):
        one = ds.rotate_heads(q[i:i + 1], k[i:i + 1], at[i:i + 1], f, None, qw, kw)
        assert torch.equal(one[0][0], whole[0][i]) and torch.equal(one[1][0], whole[1][i])


def test_refusals(cuda):
    q, k = torch.zeros(8, 4, 32, device="cuda"), torch.zeros(10, 2, 32, device="cuda")
    at, f, w = torch.zeros(10, 2, device="cuda"), torch.ones(6, device="cuda"), torch.ones(32, device="cuda")
    bad = lambda match, *a, **kw: pytest.raises(RuntimeError, ds.rotate_heads, *a, **kw).match(match)  # noqa: E731
    bad("CUDA tensor", q.cpu(), k, at, f)
    bad("CUDA tensor", None, k, at, f)
    bad("must have shape", q[0], k, at, f)
    bad("float32 or bfloat16", q.half(), k.half(), at, f)
    bad("one dtype", q, k.bfloat16(), at, f)
    bad("one head width", q, k[..., :16], at, f)
    bad("multiple of 8", q[..., :12], k[..., :12], at, f)
    bad("at most k's", torch.cat([q, q]), k, at, f)
    bad("positions must have shape", q, k, at[:8], f)
    bad("positions must be float32", q, k, at.int(), f)
    bad("axes", q, k, at.repeat(1, 5), f)
    bad("positions must be a tensor", q, k, at.cpu(), f)
    bad("1 to 16 pairs", q, k, at, torch.ones(17, device="cuda"))
    bad("frequencies must be float32", q, k, at, f.double())
    bad("frequencies have no gradient", q, k, at, f.clone().requires_grad_(True))
    bad("equal sections", q, k, at, f[:5])
    bad("add up to 6", q, k, at, f, (3, 4))
    bad("add up to 6", q, k, at, f, (7, -1))
    bad("comes with norm", q, k, at, f, None, w, w, norm=False)
    bad("q_weight must be", q, k, at, f, None, w[:8], w)
    bad("k_weight must be", q, k, at, f, None, w, w.double())
    bad("one dtype", q.bfloat16(), k.bfloat16(), at, f, None, w, w.bfloat16())
    bad("eps", q, k, at, f, eps=-1.0)
    bad("eps", q, k, at, f, eps=float("nan"))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        bad("forward-mode", dual, k, at, f)


@LAYOUTS
def test_offsets_past_32_bits(cuda, interleaved):
    """Atoms whose heads lie past 2^31 elements, and past 2^32 where rows lie apart: the bits that the same atoms get by
    themselves (a head's sums are its own lanes', however many atoms there are)."""
    print("\n[case] far atoms", flush=True)
    n, last, freq = (1 << 22) + 37, 50, torch.linspace(0.1, 1.0, 32, device="cuda")
    g = torch.Generator("cuda").manual_seed(3)
    piece = torch.randn(1 << 12, 8, 64, device="cuda", generator=g).bfloat16()
    q = piece.repeat(n // (1 << 12) + 1, 1, 1)[:n].requires_grad_(True)
    k, at, w = q.detach()[:, 3:4].clone(), torch.rand(n, 1, device="cuda", generator=g), torch.rand(64, device="cuda", generator=g)
    assert q.numel() > 2 ** 31
    y, z = ds.rotate_heads(q, k, at, freq, None, w, w, interleaved=interleaved)
    few = q.detach()[-last:].clone().requires_grad_(True)
    want, want_z = ds.rotate_heads(few, k[-last:], at[-last:], freq, None, w, w, interleaved=interleaved)
    assert torch.equal(y[-last:], want) and torch.equal(z[-last:], want_z)
    dq, = torch.autograd.grad(y, q, y.detach())
    assert torch.equal(dq[-last:], torch.autograd.grad(want, few, want.detach())[0])
    del q, y, z, dq
    apart = torch.empty(1 << 12, (1 << 20) + 8, dtype=torch.bfloat16, device="cuda")[:, :512].unflatten(1, (8, 64))
    apart.copy_(piece)
    at = at[:1 << 12]
    got, got_k = ds.rotate_heads(apart, apart[:, 2:4], at, freq, interleaved=interleaved)
    want, want_k = ds.rotate_heads(piece, piece[:, 2:4], at, freq, interleaved=interleaved)
    assert torch.equal(got, want) and torch.equal(got_k, want_k)
