"""The operators on a built graph in the regimes that small inputs do not reach: waves that walk many
rows, rows of 100,000 entries, rows past 4 GiB and nodes past 2^24, every panel width of the grouped
products, groups by the ten thousand; and what hides or shows where values are not finite.

Bounds are those of test_gpu_attention and test_gpu_grouped where nothing else is said."""
import numpy as np
import pytest
import torch

import test_gpu_attention as attention
import test_gpu_grouped as grouped
from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])


def _case(src, dst, nodes, targets, heads, kv, dim, dtype, buckets, seed):
    """A case as test_gpu_attention makes them, of the given edges."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    c = {"q": rand(targets, heads, dim), "k": rand(nodes, kv, dim), "v": rand(nodes, kv, dim),
         "grad": rand(targets, heads, dim), "src": src, "dst": dst, "n": nodes, "t": targets, "table": None, "bucket": None,
         "bounds": None, "dist": None}
    if buckets:
        c["bucket"] = rng.integers(0, buckets, len(src))
        c["dist"], c["bounds"] = c["bucket"].astype(np.float32) + 0.5, np.arange(1, buckets).astype(np.float32)
        c["table"] = torch.randn(buckets, heads, generator=g)
    return c


# ---------------------------------------------------------------- many rows for each wave


@pytest.mark.parametrize("layout,dtype", [((8, 8, 16), BF16), ((4, 4, 16), BF16), ((8, 2, 32), BF16), ((4, 1, 128), BF16),
                                          ((8, 4, 16), F32), ((1, 1, 144), BF16)], ids=str)
def test_waves_that_walk_many_rows(cuda, layout, dtype):
    """13,000 rows and nodes, where the card holds 2,048 to 6,144 waves: a row's entries, bounds and
    operands come from what was fetched while the rows before were worked on.  Rows of none to eight
    edges, one in a hundred of up to a hundred, two in parts; masked edges, and rows left empty."""
    print(f"\n[case] many rows {layout} {dtype}", flush=True)
    rng = np.random.default_rng(1)
    n = t = 13_000
    deg = rng.integers(0, 7, t)
    deg[rng.choice(t, t // 100, replace=False)] = rng.integers(20, 100, t // 100)
    deg[[17, 9000]] = 700
    dst = np.repeat(rng.permutation(t), deg)
    src = rng.integers(0, n, len(dst))
    src[rng.choice(len(src), 600, replace=False)] = 77  # (a long row by source)
    mask = rng.random(len(src)) < 0.85
    mask[np.isin(dst, rng.choice(t, 300, replace=False))] = False
    attention._check(_case(src, dst, n, t, *layout, dtype, 20, seed=2), mask)


# ---------------------------------------------------------------- rows of many parts


@pytest.mark.parametrize("layout,dtype", [((2, 2, 8), BF16), ((2, 1, 16), BF16), ((2, 2, 8), F32), ((1, 1, 136), BF16)], ids=str)
@pytest.mark.parametrize("by", ["target", "source"])
def test_rows_of_100_000_entries(cuda, by, layout, dtype):
    """Three rows in several hundred parts of more than 128 entries, joined by workgroups of 64 strands:
    by target (forward, dq) and by source (dk, dv)."""
    print(f"\n[case] 100,000 entries by {by} {layout} {dtype}", flush=True)
    rng = np.random.default_rng(3)
    per = 100_000 if layout[2] <= 16 else 30_000
    n = per + 50
    many, few = np.concatenate([rng.permutation(n)[:per] for _ in range(3)]), np.repeat([2, 0, 1], per)
    if by == "target":
        c = _case(many, few, n, 3, *layout, dtype, 6, seed=4)
    else:
        order = np.argsort(many, kind="stable")
        c = _case(few[order], many[order], n, n, *layout, dtype, 6, seed=4)
    plan = attention._plan(c)
    rows = plan.by_target if by == "target" else plan.by_source
    assert rows.c.n_long == 3 and rows.c.n_items > 16 * rows.c.n_long
    attention._check(c, plan=plan)


# ---------------------------------------------------------------- far rows


def _step(q, k, v, plan, table, grad):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, table) if x is not None]
    out, lse = ds.neighbor_attention(*leaves[:3], plan, leaves[3] if table is not None else None, return_lse=True)
    return [out.detach(), lse, *torch.autograd.grad(out, leaves, grad)]


@TYPES
@pytest.mark.parametrize("buckets", [0, 20])
@pytest.mark.parametrize("layout", [(8, 8, 16), (4, 4, 16), (8, 2, 32), (4, 2, 8)], ids=str)
def test_rows_that_lie_past_4_gib(cuda, layout, buckets, dtype):
    """q, k, v and the gradient with rows 16 MiB and more apart, the last of them past 4 GiB: the bits of
    the same rows side by side."""
    print(f"\n[case] far rows {layout} {buckets} {dtype}", flush=True)
    heads, kv, dim = layout
    rng = np.random.default_rng(5)
    n = t = 280
    deg = rng.integers(0, 50, t)
    deg[40] = 600
    dst = np.repeat(rng.permutation(t), deg)
    src = rng.integers(0, n, len(dst))
    src[:600] = 279  # (a long row by source)
    c = _case(src, dst, n, t, *layout, dtype, buckets, seed=6)
    plan = attention._plan(c)
    near = [attention._dev(c[x]) for x in ("q", "k", "v", "grad")]
    table = None if c["table"] is None else attention._dev(c["table"])
    want = _step(*near[:3], plan, table, near[3])
    pitch = 2 ** 24 // near[0].element_size() + 64
    far = torch.empty(n, pitch, dtype=dtype, device="cuda")
    assert far.numel() * far.element_size() > 2 ** 32
    spread, at = [], 0
    for x in near:
        wide = x.shape[1] * x.shape[2]
        y = far[:, at:at + wide].unflatten(1, x.shape[1:])
        y.copy_(x)
        assert y.stride(0) == pitch
        spread.append(y)
        at += wide
    got = _step(*spread[:3], plan, table, spread[3])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@TYPES
@pytest.mark.parametrize("layout", [(1, 1, 8), (2, 1, 8)], ids=str)
def test_nodes_past_2_to_the_24(cuda, layout, dtype):
    """A few edges among the last of 2^24 + 100 nodes: the same edges among few nodes, bit for bit, and
    zeros for every other node."""
    print(f"\n[case] nodes past 2^24 {layout} {dtype}", flush=True)
    heads, kv, dim = layout
    rng = np.random.default_rng(7)
    few, n = 90, 2 ** 24 + 100
    dst = np.repeat(rng.permutation(few), rng.integers(1, 40, few))
    src = rng.integers(0, few, len(dst))
    c = _case(src, dst, few, few, *layout, dtype, 9, seed=8)
    near = [attention._dev(c[x]) for x in ("q", "k", "v", "grad")]
    table = attention._dev(c["table"])
    want = _step(*near[:3], attention._plan(c), table, near[3])
    wide = []
    for x in near:
        y = torch.zeros(n, *x.shape[1:], dtype=dtype, device="cuda")
        y[n - few:] = x
        wide.append(y)
    plan = attention._plan({**c, "src": src + n - few, "dst": dst + n - few, "n": n, "t": n})
    got = _step(*wide[:3], plan, table, wide[3])
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), got, want):
        assert torch.equal(a[n - few:], b), name
        rest = a[:n - few]
        assert (rest == -torch.inf).all() if name == "lse" else not rest.any(), name
    # (the table's sums follow the rows' order: a few hundred terms in another one)
    assert torch.allclose(got[5], want[5], rtol=0, atol=len(src) * EPS * want[5].abs().max().item() * 64)


# ---------------------------------------------------------------- scales


@TYPES
@pytest.mark.parametrize("scale", [0.3, -0.5, 0.0, 2])
def test_scales(cuda, scale, dtype):
    print(f"\n[case] scale {scale} {dtype}", flush=True)
    c = attention._make("ragged", 4, 2, 16, dtype, 12, seed=9)
    names = ("q", "k", "v", "table")
    leaves = [attention._dev(c[x]).requires_grad_(True) for x in names]
    out = ds.neighbor_attention(*leaves[:3], attention._plan(c), leaves[3], scale=scale)
    grads = torch.autograd.grad(out, leaves, attention._dev(c["grad"]))
    args = [*(attention._np(c[x]) for x in names[:3]), c["src"], c["dst"]]
    f = oracle.attention(*args, c["bucket"], attention._np(c["table"]), scale)
    g, m = oracle.attention_grads(*args, attention._np(c["grad"]), c["bucket"], attention._np(c["table"]), scale)
    const = 24 * f["logit_mag"].max() + 64
    attention._near("out", out.detach(), f["out"], f["out_mag"], const + 71, dtype)
    for name, x in zip(("dq", "dk", "dv", "dtable"), grads):
        attention._near(name, x, g[name], m[name], 2 * const + 71 + len(c["src"]), dtype)


# ---------------------------------------------------------------- how many bits a probability has


def _rests():
    """Biases whose probability beside a logit of zero leaves much when it is taken apart into two
    bfloat16 parts; and what is left, of the two probabilities' sum."""
    bias = np.linspace(-0.7, -0.01, 20001).astype(np.float32)
    p = np.exp(bias.astype(np.float64)).astype(np.float32)
    part = lambda x: torch.from_numpy(x).bfloat16().float().numpy()  # noqa: E731
    rest = p - part(p)
    rest = (rest - part(rest)) / (1 + p)
    best = np.argsort(rest)[-6:]
    return bias[best], rest[best]


@TYPES
def test_probabilities_keep_the_bits_of_a_float(cuda, dtype):
    """Rows of two edges with v = 1 and a gradient of 1: the weights add up to one, <g, out> is the head's
    width and every slope is zero.  What is not: the roundings of the sum of two weights, of the two
    products' sums, of the division and of the product with it, and of the slope's own difference, 2^-24
    each (the last step of one unit twice): at most 8 of them.  Weights of two bfloat16 parts would be
    off by several times that, all to one side."""
    print(f"\n[case] bits of a probability {dtype}", flush=True)
    for bias, rest in zip(*_rests()):
        assert rest > 3 * 8 * EPS
        t = 500
        ei = torch.stack([torch.arange(2 * t), torch.arange(t).repeat_interleave(2)]).cuda()
        plan = ds.neighbor_plan(ei, 2 * t, t, distances=torch.tensor([0.0, 1.0]).repeat(t).cuda(), boundaries=[0.5])
        one = lambda n: torch.ones(n, 4, 16, device="cuda", dtype=dtype)  # noqa: E731
        table = torch.tensor([[0.0] * 4, [float(bias)] * 4], device="cuda", requires_grad=True)
        out = ds.neighbor_attention(torch.zeros_like(one(t)), one(2 * t), one(2 * t), plan, table)
        assert ((out - 1).abs() <= 8 * EPS).all()
        d, = torch.autograd.grad(out, table, one(t))
        p = np.exp(float(bias)) / (1 + np.exp(float(bias)))
        for row, share in zip(d.double().cpu().numpy(), (1 - p, p)):
            assert np.abs(row).max() <= t * 16 * share * 8 * EPS, (float(bias), row)


# ---------------------------------------------------------------- what is not finite


@TYPES
@pytest.mark.parametrize("layout", [(8, 8, 16), (4, 4, 16), (8, 2, 32), (2, 2, 256)], ids=str)
@pytest.mark.parametrize("where", ["q", "k", "v", "grad"])
def test_a_nan_shows_in_its_head_and_in_no_other(cuda, where, layout, dtype):
    """Forward and backward: the head's results that read the value are NaN, all other bits are kept."""
    print(f"\n[case] NaN in {where} {layout} {dtype}", flush=True)
    heads, kv, dim = layout
    c = attention._make("ragged", *layout, dtype, 12, seed=10)
    plan = attention._plan(c)
    args = {x: attention._dev(c[x]) for x in ("q", "k", "v", "table", "grad")}
    want = _step(args["q"], args["k"], args["v"], plan, args["table"], args["grad"])
    per, c_head, node = heads // kv, 1, int(c["dst"][0])
    at = c_head if where in ("k", "v") else c_head * per  # (a head of k, or of q)
    args[where][node, at, 3] = float("nan")
    got = _step(args["q"], args["k"], args["v"], plan, args["table"], args["grad"])
    hit_q = torch.zeros(heads, dtype=torch.bool)
    hit_q[at if where in ("q", "grad") else slice(c_head * per, (c_head + 1) * per)] = True
    hit_kv = torch.arange(kv) == c_head
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv", "dtable"), got, want):
        others = ~(hit_kv if name in ("dk", "dv") else hit_q)
        assert torch.equal(a[:, others], b[:, others]), name
    reads = c["dst"][c["src"] == node] if where in ("k", "v") else np.array([node])
    read = torch.zeros(c["t"], dtype=torch.bool)
    read[reads] = True
    out, _, dq, dk, dv, dtable = got
    if where == "grad":
        assert torch.equal(out, want[0])
    else:
        shown = out[read][:, hit_q]
        assert torch.isnan(shown if where != "v" else shown[..., 3]).all()
        assert torch.equal(out[~read], want[0][~read])
    assert torch.isnan(dq[read][:, hit_q]).all() and torch.equal(dq[~read], want[2][~read])
    assert torch.isnan(dtable[:, hit_q]).any()
    sources = torch.as_tensor(np.unique(c["src"][np.isin(c["dst"], reads)]))
    assert torch.isnan(dk[sources][:, hit_kv]).all()
    if where != "v":
        shown = dv[sources][:, hit_kv]
        assert torch.isnan(shown if where != "grad" else shown[..., 3]).all()
    else:
        assert torch.equal(dv, want[4])


@TYPES
@pytest.mark.parametrize("kind", ["ragged", "long", "hub"])
@pytest.mark.parametrize("layout", [(4, 4, 16), (8, 2, 32), (8, 4, 16), (6, 2, 128), (8, 8, 16)], ids=str)
def test_what_the_table_hides_from_some_heads(cuda, layout, kind, dtype):
    """Entries of -inf for the heads of one head of k: what that head of k and v holds in sources that
    only such edges read, and what those heads of q and of the gradient hold in targets that have only
    such edges, does not show; the other heads see the edges.  Short rows, parts of long ones by target
    and by source, heads shared or not."""
    print(f"\n[case] hidden from some heads {layout} {kind} {dtype}", flush=True)
    heads, kv, dim = layout
    c = attention._make(kind, *layout, dtype, 6, seed=11)
    rng = np.random.default_rng(12)
    per = heads // kv
    mine = slice(per, 2 * per)  # the heads of q of k's head 1
    c["table"][3, mine] = -float("inf")
    sources = rng.choice(np.unique(c["src"]), 9, replace=False)
    targets = rng.choice(np.unique(c["dst"]), 3, replace=False)
    if kind == "hub":
        targets = np.unique(np.append(targets, c["dst"][c["src"] == 5][0]))
    hidden = np.isin(c["src"], sources) | np.isin(c["dst"], targets)
    c["bucket"][hidden] = 3
    c["dist"] = c["bucket"].astype(np.float32) + 0.5
    c["bounds"] = np.arange(1, 6).astype(np.float32)
    attention._check(c)
    bad = [float("nan"), float("inf"), -float("inf")]
    for i, s in enumerate(sources):
        c["k"][s, 1, i % dim], c["v"][s, 1, (i + 3) % dim] = bad[i % 3], bad[(i + 1) % 3]
    for i, t in enumerate(targets):
        c["q"][t, mine, i], c["grad"][t, mine, i + 1] = bad[i % 3], bad[(i + 1) % 3]
    with np.errstate(invalid="ignore"):
        attention._check(c)


# ---------------------------------------------------------------- grouped products


@pytest.mark.parametrize("rows,groups,k,n,dtype", [
    (3000, 5, 512, 128, BF16),    # forward: panels of 32 columns, rows of 1 KB; dx: of 32, four panels
    (30_000, 5, 128, 128, BF16),  # 123 tiles of 256 rows: panels of 64, forward and dx
    (60_000, 5, 128, 120, BF16),  # 240 tiles: panels of 128, the last one's columns not all there
    (40_000, 3, 512, 136, BF16),  # rows of 1 KB leave the panel 64 columns; dx panels of 128
    (30_000, 4, 256, 64, F32),    # the same in floats: 1 KB forward, 256 bytes for dx
    (70_000, 6, 40, 33, BF16),    # rows that are no multiple of 16 bytes, several tiles a workgroup
    (70_000, 6, 33, 40, F32),
    (40_000, 16, 512, 256, BF16),  # weight gradients in items, joined by eight workgroups a tile
    (40_000, 16, 512, 256, F32),
], ids=str)
def test_grouped_shapes(cuda, rows, groups, k, n, dtype):
    rng = np.random.default_rng(13)
    w = np.exp(0.5 * rng.standard_normal(groups))
    w[groups // 2] = 0
    grouped._check(rng.multinomial(rows, w / w.sum()).tolist(), k, n, dtype, seed=14)


@TYPES
def test_20_000_groups(cuda, dtype):
    sizes = np.random.default_rng(15).integers(0, 4, 20_000)
    sizes[5000:9000] = 0
    sizes[12_345] = 900
    grouped._check(sizes.tolist(), 24, 16, dtype, seed=16)
