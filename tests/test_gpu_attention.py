"""neighbor_plan and neighbor_attention on the GPU against the definitions in 64 bits
(oracle/operators.py), forward and backward: head layouts, widths, row lengths around the
kernels' tiles and parts, masks that leave rows empty, table entries of -inf, NaN and infinity
in masked places, strides, and bit-equal repeats.

Tolerances.  A logit of D terms errs by at most (D + 8) eps times the sum S of its terms'
magnitudes (the scale's, the table's and the base-2 factor's roundings among the 8), so a
probability errs by that relative amount; a row's sum of n terms adds n eps, the last steps a
few eps.  Relative to the sum of a result's magnitudes: c eps, c = (D + 8) S + n + 64.  With
bfloat16 tensors a probability and its gradient enter the matrix units as two bfloat16 parts
(2^-16), and the result is rounded once (2^-8 of itself)."""
import numpy as np
import pytest
import torch

from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def _graph(kind, rng):
    """(src, dst, num_nodes, num_targets), grouped by target."""
    if kind == "ragged":  # rows of 0 .. 70, and around the tiles of 16 and 32
        deg = np.concatenate([rng.integers(0, 71, 60), [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0]])
        n, t = 97, len(deg)
    elif kind == "long":  # rows around the limit of 512 and its parts of 128
        deg = np.array([3, 511, 512, 513, 0, 640, 641, 1500, 1])
        n, t = 150, len(deg)
    elif kind == "one":
        deg, n, t = np.array([1]), 2, 1
    elif kind == "symmetric":
        n = t = 83
        a, b = rng.integers(0, n, 900), rng.integers(0, n, 900)
        src, dst = np.concatenate([a, b]), np.concatenate([b, a])
        order = np.argsort(rng.permutation(n)[dst], kind="stable")
        return src[order], dst[order], n, t
    elif kind == "hub":  # one source of every target: long rows by source
        n, t = 700, 690
        dst = np.repeat(np.arange(t), 2)
        src = np.stack([np.full(t, 5), rng.integers(0, n, t)], 1).reshape(-1)
        return src, dst, n, t
    run = rng.permutation(t)  # targets in an order of their own
    dst = np.repeat(run, deg[:t])
    return rng.integers(0, n, len(dst)), dst, n, t


def _dev(x, dtype=None):
    return torch.as_tensor(x).to("cuda", dtype)


def _make(kind, heads, kv, dim, dtype, buckets, seed):
    rng = np.random.default_rng(seed)
    src, dst, n, t = _graph(kind, rng)
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    c = {"q": rand(t, heads, dim), "k": rand(n, kv, dim), "v": rand(n, kv, dim), "grad": rand(t, heads, dim),
         "src": src, "dst": dst, "n": n, "t": t, "table": None, "bucket": None, "bounds": None, "dist": None}
    if buckets:
        c["dist"] = rng.uniform(0, 6, len(src)).astype(np.float32)
        if kind == "symmetric":  # (i, j) as far as (j, i)
            c["dist"] = ((src + 1) * (dst + 1) % 97 / 97 * 6).astype(np.float32)
        c["bounds"] = np.linspace(0, 6, buckets + 1)[1:-1].astype(np.float32)
        c["bucket"] = (c["bounds"][None] <= c["dist"][:, None]).sum(1)
        c["table"] = torch.randn(buckets, heads, generator=g)
    return c


def _plan(c, mask=None, **kw):
    dist = None if c["dist"] is None else _dev(c["dist"])
    return ds.neighbor_plan(_dev(np.stack([c["src"], c["dst"]])), c["n"], c["t"], distances=dist,
                            boundaries=None if c["bounds"] is None else _dev(c["bounds"]), edge_mask=mask, **kw)


def _np(t):
    return None if t is None else t.double().numpy()


def _near(name, got, want, mag, c, dtype):
    got = got.double().cpu().numpy()
    tol = c * EPS * mag
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -16 * mag
        if name != "dtable":
            tol = tol + 2.0 ** -8 * np.abs(want)
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want)[bad]):.3g}"


def _check(c, mask=None, plan=None, strides=False):
    dtype = c["q"].dtype
    keep = np.ones(len(c["src"]), bool) if mask is None else mask
    src, dst = c["src"][keep], c["dst"][keep]
    bucket = None if c["bucket"] is None else c["bucket"][keep]
    plan = plan or _plan(c, None if mask is None else _dev(mask))
    q, k, v, grad = (_dev(c[x]) for x in ("q", "k", "v", "grad"))
    if strides:  # parts of wider rows, 16 bytes aligned
        w = torch.cat([k.flatten(1), v.flatten(1)], 1)
        k, v = (x.unflatten(1, c["k"].shape[1:]) for x in w.split(w.shape[1] // 2, 1))
        assert not k.is_contiguous()
    table = None if c["table"] is None else _dev(c["table"])
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)] + ([table.requires_grad_(True)] if table is not None else [])
    out, lse = ds.neighbor_attention(*leaves[:3], plan, table, return_lse=True)
    grads = torch.autograd.grad(out, leaves, grad)
    with torch.no_grad():
        again = ds.neighbor_attention(*leaves[:3], plan, table)
    same = torch.equal(again, out)
    assert same, "inference and training differ"
    args = (_np(c["q"]), _np(c["k"]), _np(c["v"]), src, dst)
    f = oracle.attention(*args, bucket, _np(c["table"]))
    g, m = oracle.attention_grads(*args, _np(c["grad"]), bucket, _np(c["table"]))
    S = f["logit_mag"].max(initial=0)
    rows = np.bincount(dst, minlength=1).max(initial=1), np.bincount(src, minlength=1).max(initial=1)
    const = (c["q"].shape[2] + 8) * S + 64
    _near("out", out.detach(), f["out"], f["out_mag"], const + rows[0], dtype)
    empty = f["lse"] == -np.inf
    got = lse.cpu().numpy()
    assert np.array_equal(got == -np.inf, empty)
    got, want = got[~empty], f["lse"][~empty]
    assert (np.abs(got - want) <= (const + rows[0]) * EPS * (1 + np.abs(want))).all()
    for name, x in zip(("dq", "dk", "dv", "dtable"), grads):
        n = {"dq": rows[0], "dk": rows[1] * 8, "dv": rows[1] * 8, "dtable": len(src)}[name]
        _near(name, x, g[name], m[name], 2 * const + rows[0] + n, dtype)
    return out.detach(), grads


LAYOUTS = [(4, 4, 32), (8, 8, 16), (8, 2, 32), (6, 3, 24), (1, 1, 8), (16, 4, 64), (3, 1, 40), (5, 5, 128), (2, 2, 256),
           (12, 12, 48), (20, 20, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_layouts(cuda, layout, dtype):
    print(f"\n[case] layout {layout} {dtype}", flush=True)
    _check(_make("ragged", *layout, dtype, 20, seed=1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["one", "long", "symmetric", "hub"])
@pytest.mark.parametrize("buckets", [0, 1, 32])
def test_graphs(cuda, kind, buckets, dtype):
    print(f"\n[case] graph {kind} {buckets} {dtype}", flush=True)
    c = _make(kind, 8, 4, 32, dtype, buckets, seed=2)
    _check(c)
    assert _plan(c).symmetric == (kind == "symmetric")


@pytest.mark.parametrize("buckets,heads,dim", [(128, 8, 8), (128, 1, 8), (64, 16, 16), (128, 32, 16)])
def test_large_tables(cuda, buckets, heads, dim):
    for dtype in (torch.float32, torch.bfloat16):
        print(f"\n[case] table {buckets} {heads} {dim} {dtype}", flush=True)
        _check(_make("ragged", heads, heads, dim, dtype, buckets, seed=3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_masks_and_what_they_hide(cuda, dtype):
    """Masked edges, rows left empty, and NaN and infinity in every row that only masked edges read."""
    c = _make("ragged", 8, 4, 32, dtype, 20, seed=4)
    rng = np.random.default_rng(5)
    mask = rng.random(len(c["src"])) < 0.6
    mask[np.isin(c["dst"], [3, 7, 8])] = False  # whole rows
    hidden = rng.choice(c["n"], 20, replace=False)
    mask[np.isin(c["src"], hidden)] = False
    print(f"\n[case] masked {dtype}", flush=True)
    want, wgrads = _check(c, mask)
    for x in ("k", "v"):
        c[x][hidden[:7]], c[x][hidden[7:14]], c[x][hidden[14:]] = float("nan"), float("inf"), -float("inf")
    plan = _plan(c, _dev(mask))
    leaves = [_dev(c[x]).requires_grad_(True) for x in ("q", "k", "v", "table")]
    out = ds.neighbor_attention(*leaves[:3], plan, leaves[3])
    grads = torch.autograd.grad(out, leaves, _dev(c["grad"]))
    assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(grads, wgrads))
    assert not out[torch.tensor([3, 7, 8])].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_table_entries_of_minus_infinity(cuda, dtype):
    """They take edges out for a head, the other heads keep them; a whole column leaves a head
    empty; what k and v hold there does not show.  The type's lowest value is an ordinary one."""
    c = _make("ragged", 8, 8, 16, dtype, 12, seed=6)
    c["table"][3, :] = -float("inf")
    c["table"][5, 2] = -float("inf")
    c["table"][:, 4] = -float("inf")
    c["table"][:, 6] = torch.finfo(torch.float32).min
    print(f"\n[case] -inf {dtype}", flush=True)
    # head 6: every logit is the lowest value, so its weights are equal (and its magnitudes, which
    # the bounds scale with, vast): checked by itself below
    plan = _plan(c)
    leaves = [_dev(c[x]).requires_grad_(True) for x in ("q", "k", "v", "table")]
    out = ds.neighbor_attention(*leaves[:3], plan, leaves[3])
    grads = torch.autograd.grad(out, leaves, _dev(c["grad"]))
    assert all(torch.isfinite(x).all() for x in (out, *grads))
    # (bucket 3 is among them: its entry for head 6 is the lowest value too)
    mean = np.zeros((c["t"], 16))
    np.add.at(mean, c["dst"], c["v"].double().numpy()[c["src"], 6])
    mean /= np.maximum(np.bincount(c["dst"], minlength=c["t"]), 1)[:, None]
    others = torch.arange(8) != 6
    assert np.abs(out[:, 6].detach().double().cpu().numpy() - mean).max() < (0.02 if dtype == torch.bfloat16 else 1e-5)
    assert not out[:, 4].any() and not grads[0][:, 4].any() and not grads[3][3, others].any()
    c["table"][:, 6] = 0.25
    c["table"][3, :] = -float("inf")
    want, wgrads = _check(c)
    # a source that only edges of bucket 3 read may hold anything
    node = c["n"] - 1
    c["bucket"][c["src"] == node] = 3
    c["dist"][c["src"] == node] = 0.5 * (c["bounds"][2] + c["bounds"][3])
    want, wgrads = _check(c)
    for x in ("k", "v"):
        c[x][node] = float("nan")
    leaves = [_dev(c[x]).requires_grad_(True) for x in ("q", "k", "v", "table")]
    out = ds.neighbor_attention(*leaves[:3], _plan(c), leaves[3])
    grads = torch.autograd.grad(out, leaves, _dev(c["grad"]))
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, wgrads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_nan_stays_in_its_head(cuda, dtype):
    """A NaN (an infinity) in one head of a node shows in that head of the rows that read it only."""
    c = _make("ragged", 8, 8, 16, dtype, 12, seed=7)
    plan = _plan(c)
    q, k, v, table = (_dev(c[x]) for x in ("q", "k", "v", "table"))
    want = ds.neighbor_attention(q, k, v, plan, table)
    for name, x in (("k", k), ("v", v)):
        for value in (float("nan"), float("inf")):
            print(f"\n[case] {name} {value} {dtype}", flush=True)
            y = x.clone()
            y[11, 3] = value
            got = ds.neighbor_attention(q, y if name == "k" else k, y if name == "v" else v, plan, table)
            reads = torch.zeros(c["t"], dtype=torch.bool)
            reads[c["dst"][c["src"] == 11]] = True
            others = torch.arange(8) != 3
            assert torch.equal(got[:, others], want[:, others])
            assert torch.equal(got[~reads.cuda()], want[~reads.cuda()])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_streams_and_repeats(cuda, dtype):
    c = _make("ragged", 8, 4, 32, dtype, 20, seed=8)
    print(f"\n[case] strides {dtype}", flush=True)
    out, grads = _check(c, strides=True)
    out2, grads2 = _check(c)
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    plan = _plan(c)
    q, k, v, table = (_dev(c[x]) for x in ("q", "k", "v", "table"))
    # rows that do not start at 16 bytes, and a transposed layout: copied
    for t in (q, k):
        odd = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(t).copy_(t)
        swapped = t.transpose(0, 1).contiguous().transpose(0, 1)
        for x in (odd, swapped):
            args = (x, k, v) if t is q else (q, x, v)
            assert torch.equal(ds.neighbor_attention(*args, plan, table), out)
    # the same row for every target, as a broadcast, with its gradient
    one = q[:1].clone().requires_grad_(True)
    full = q[:1].repeat(c["t"], 1, 1).requires_grad_(True)
    a, b = (ds.neighbor_attention(x, k, v, plan, table) for x in (one.expand(c["t"], -1, -1), full))
    assert torch.equal(a, b)
    ga, = torch.autograd.grad(a.float().sum(), one)
    gb, = torch.autograd.grad(b.float().sum(), full)
    assert torch.allclose(ga.float(), gb.float().sum(0, keepdim=True), rtol=2 ** -6, atol=2 ** -6 * gb.float().abs().sum(0).max().item())
    # another stream than the plan's
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = ds.neighbor_attention(q, k, v, plan, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(x, out)


def test_gradients_against_differences(cuda):
    """The gradients along random directions against central differences of the definition."""
    c = _make("ragged", 4, 2, 16, torch.float32, 12, seed=9)
    _, grads = _check(c)
    rng = np.random.default_rng(10)
    names = ("q", "k", "v", "table")
    x = {n: _np(c[n]) for n in names}
    w = _np(c["grad"])

    def loss(y):
        return (oracle.attention(y["q"], y["k"], y["v"], c["src"], c["dst"], c["bucket"], y["table"])["out"] * w).sum()

    for name, g in zip(names, grads):
        d = rng.standard_normal(x[name].shape)
        h = 1e-5
        diff = (loss({**x, name: x[name] + h * d}) - loss({**x, name: x[name] - h * d})) / (2 * h)
        got = (g.double().cpu().numpy() * d).sum()
        # differences: h^2 and 1e-16 / h of a loss of some hundreds; the gradient: 32 bits
        assert abs(diff - got) < 1e-5 * (1 + np.abs(g.cpu().numpy() * d).sum()), name


@pytest.mark.parametrize("kind", ["ragged", "symmetric", "long", "hub"])
@pytest.mark.parametrize("masked", [False, True])
def test_plan_lists(cuda, kind, masked):
    c = _make(kind, 1, 1, 8, torch.float32, 16, seed=11)
    rng = np.random.default_rng(12)
    mask = rng.random(len(c["src"])) < 0.7 if masked else None
    print(f"\n[case] plan {kind} {masked}", flush=True)
    plan = _plan(c, None if mask is None else _dev(mask))
    want = oracle.neighbor_lists(c["src"], c["dst"], c["n"], mask, c["bucket"])
    for rows, lists in zip((plan.by_target, plan.by_source), want):
        order, ptr = rows.order.cpu().numpy(), rows.ptr.cpu().numpy()
        assert sorted(order.tolist()) == list(range(c["n"])) and ptr[0] == 0 and ptr[-1] == plan.num_edges
        idx, bucket = rows.idx.cpu().numpy(), rows.bucket.cpu().numpy()
        for slot, node in enumerate(order):
            at = slice(ptr[slot], ptr[slot + 1])
            assert sorted(zip(idx[at].tolist(), bucket[at].tolist())) == lists[int(node)], node


def test_plan_of_edges_in_any_order(cuda):
    c = _make("ragged", 4, 4, 32, torch.float32, 12, seed=13)
    p = np.random.default_rng(14).permutation(len(c["src"]))
    for x in ("src", "dst", "dist", "bucket"):
        c[x] = c[x][p]
    print("\n[case] shuffled", flush=True)
    mask = np.random.default_rng(15).random(len(p)) < 0.8
    _check(c, mask)


def test_plan_of_float64_distances_at_the_boundaries(cuda):
    """A distance equal to a boundary lies above it; a NaN counts no boundary."""
    b = torch.tensor([1.0, 2.0, 3.0], dtype=torch.float64, device="cuda")
    d = torch.tensor([0.0, 1.0, np.nextafter(1.0, 0), 2.5, 3.0, 9.0, float("nan")], dtype=torch.float64, device="cuda")
    ei = torch.stack([torch.arange(7), torch.zeros(7, dtype=torch.long)]).cuda()
    plan = ds.neighbor_plan(ei, 7, 1, distances=d, boundaries=b)
    assert plan.by_target.bucket[:7].tolist() == [0, 1, 0, 2, 3, 3, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_nothing_to_do(cuda, dtype):
    for n, t in ((5, 5), (5, 0), (0, 0)):
        print(f"\n[case] empty {n} {t} {dtype}", flush=True)
        plan = ds.neighbor_plan(torch.empty(2, 0, dtype=torch.long, device="cuda"), n, t)
        q, k, v = (torch.randn(m, 4, 16, device="cuda", dtype=dtype, requires_grad=True) for m in (t, n, n))
        out, lse = ds.neighbor_attention(q, k, v, plan, return_lse=True)
        assert out.shape == q.shape and not out.any() and (lse == -torch.inf).all()
        for g in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)):
            assert not g.any()


def test_attention_on_a_built_graph_replays_in_a_graph(cuda):
    """The plan of a built radius graph; the attention, forward and backward, captured and
    replayed with eager work between the replays."""
    from dynamis_amd import configs
    from dynamis_amd.dynamis_state import dynamis_state_impl as impl

    box = configs.fcc(cells=3)
    pos = _dev(box.pos)
    ei, _, _, _, _, dist = impl.radius_graph_pbc_vectors(pos, torch.from_numpy(box.cell), torch.tensor(box.pbc), 5.0)
    n = len(box.pos)
    plan = ds.neighbor_plan(ei, n, distances=dist, boundaries=torch.linspace(2, 5, 15, dtype=dist.dtype, device="cuda"))
    assert plan.symmetric and plan.num_edges == ei.shape[1]
    q, k, v = (torch.randn(n, 4, 32, device="cuda").bfloat16().requires_grad_(True) for _ in range(3))
    table = torch.randn(16, 4, device="cuda", requires_grad=True)
    grad = torch.randn(n, 4, 32, device="cuda").bfloat16()

    def step():
        out = ds.neighbor_attention(q, k, v, plan, table)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v, table), grad)]

    print("\n[case] graph capture", flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(4):
        with torch.no_grad():
            q.mul_(1.1)
            table.add_(0.1)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_refusals(cuda):
    ei = torch.tensor([[0, 1, 2], [0, 0, 1]], device="cuda")
    bad = lambda match, f, *a, **k: pytest.raises(RuntimeError, f, *a, **k).match(match)  # noqa: E731
    plan = ds.neighbor_plan(ei, 4, 2, distances=torch.ones(3, device="cuda"), boundaries=torch.ones(2, device="cuda"))
    q, k = torch.zeros(2, 4, 16, device="cuda"), torch.zeros(4, 2, 16, device="cuda")
    bad("CUDA tensor", ds.neighbor_plan, ei.cpu(), 4)
    bad("shape", ds.neighbor_plan, ei[0], 4)
    bad("int64", ds.neighbor_plan, ei.int(), 4)
    bad("num_targets", ds.neighbor_plan, ei, 4, 5)
    bad("outside", ds.neighbor_plan, ei, 2)
    bad("outside", ds.neighbor_plan, ei, 4, 1)
    bad("outside", ds.neighbor_plan, ei - 1, 4)
    bad("boundaries", ds.neighbor_plan, ei, 4, distances=torch.ones(3, device="cuda"))
    bad("distances", ds.neighbor_plan, ei, 4, boundaries=torch.ones(3, device="cuda"))
    bad("distances", ds.neighbor_plan, ei, 4, distances=torch.ones(2, device="cuda"), boundaries=[1.0])
    bad("127", ds.neighbor_plan, ei, 4, distances=torch.ones(3, device="cuda"), boundaries=torch.arange(128.0))
    bad("edge_mask", ds.neighbor_plan, ei, 4, edge_mask=torch.ones(3, device="cuda"))
    at = ds.neighbor_attention
    bad("CUDA tensor", at, q.cpu(), k, k, plan)
    bad("float32 or bfloat16", at, q.half(), k.half(), k.half(), plan)
    bad("one dtype", at, q, k.bfloat16(), k, plan)
    bad("head width", at, q, k[..., :8], k, plan)
    bad("2 rows", at, k, k, k, plan)
    bad("4 rows", at, q, q, q, plan)
    bad("multiple of kv_heads", at, q[:, :3], k, k, plan)
    bad("multiple of 8", at, q[..., :12], k[..., :12], k[..., :12], plan)
    bad("bias_table", at, q, k, k, plan, torch.zeros(4, 4, device="cuda"))
    bad("plan with distances", at, q, k, k, ds.neighbor_plan(ei, 4, 2), torch.zeros(3, 4, device="cuda"))
    bad("scale", at, q, k, k, plan, scale=float("nan"))
    out = at(q.requires_grad_(True), k, k, ds.neighbor_plan(ei, 4, 2, backward=False))
    bad("backward=False", torch.autograd.grad, out.sum(), q)
