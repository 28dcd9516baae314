"""The operators on a built graph at the ends of their ranges, on the GPU: lists without edges,
infinities, derivatives that they do not have, what two backward passes share."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from dynamis_amd import _lib
from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _leave_nans(sizes):
    """Freed memory of these many floats holds NaN, so that a result which is not written shows."""
    for n in sizes:
        del [torch.full((n,), float("nan"), device="cuda") for _ in range(16)][:]


# ---------------------------------------------------------------- no edges


@TYPES
@pytest.mark.parametrize("nodes,targets,edges", [(5, 5, 0), (5, 0, 0), (5, 5, 40)], ids=str)
def test_no_edges_with_a_table(cuda, nodes, targets, edges, dtype):
    """An edge list without edges, or one whose mask leaves none: zeros everywhere."""
    print(f"\n[case] no edges {nodes} {targets} {edges} {dtype}", flush=True)
    ei = torch.randint(0, max(targets, 1), (2, edges), device="cuda")
    plan = ds.neighbor_plan(ei, nodes, targets, distances=torch.rand(edges, device="cuda") * 4,
                            boundaries=[1.0, 2.0, 3.0], edge_mask=torch.zeros(edges, dtype=torch.bool, device="cuda"))
    assert plan.num_edges == 0 and plan.num_buckets == 4
    q, k, v = (torch.randn(m, 4, 16, device="cuda", dtype=dtype, requires_grad=True) for m in (targets, nodes, nodes))
    table = torch.randn(4, 4, device="cuda", requires_grad=True)
    out, lse = ds.neighbor_attention(q, k, v, plan, table, return_lse=True)
    assert out.shape == q.shape and not out.any() and (lse == -torch.inf).all()
    _leave_nans([16, 128, 512])
    for g, of in zip(torch.autograd.grad(out, (q, k, v, table), torch.ones_like(out)), (q, k, v, table)):
        assert g.shape == of.shape and not g.any()


@TYPES
def test_the_tables_gradient_of_no_nodes(cuda, dtype):
    print(f"\n[case] no nodes {dtype}", flush=True)
    plan = ds.neighbor_plan(torch.empty(2, 0, dtype=torch.long, device="cuda"), 0,
                            distances=torch.empty(0, device="cuda"), boundaries=[1.0, 2.0, 3.0])
    q, k, v = (torch.empty(0, 4, 16, device="cuda", dtype=dtype, requires_grad=True) for _ in range(3))
    table = torch.randn(4, 4, device="cuda", requires_grad=True)
    out = ds.neighbor_attention(q, k, v, plan, table)
    _leave_nans([16, 128])
    assert not torch.autograd.grad(out, table, torch.ones_like(out))[0].any()


# ---------------------------------------------------------------- derivatives that there are not


@pytest.mark.parametrize("of", ["q", "k", "v", "table"])
def test_attention_refuses_tangents(cuda, of):
    """Forward-mode derivatives are refused, not dropped."""
    print(f"\n[case] tangent of {of}", flush=True)
    ei = torch.tensor([[0, 1, 2], [0, 0, 1]], device="cuda")
    plan = ds.neighbor_plan(ei, 4, 2, distances=torch.ones(3, device="cuda"), boundaries=[1.0])
    t = {"q": torch.randn(2, 2, 8, device="cuda"), "k": torch.randn(4, 2, 8, device="cuda"),
         "v": torch.randn(4, 2, 8, device="cuda"), "table": torch.randn(2, 2, device="cuda")}
    want = ds.neighbor_attention(t["q"], t["k"], t["v"], plan, t["table"])
    with forward_ad.dual_level():
        # (tensors without a tangent may be used at a level)
        assert torch.equal(ds.neighbor_attention(t["q"], t["k"], t["v"], plan, t["table"]), want)
        t[of] = forward_ad.make_dual(t[of], torch.ones_like(t[of]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                ds.neighbor_attention(t["q"], t["k"], t["v"], plan, t["table"])


@pytest.mark.parametrize("of", ["x", "weight", "bias"])
def test_grouped_refuses_tangents(cuda, of):
    print(f"\n[case] tangent of {of}", flush=True)
    t = {"x": torch.randn(7, 8, device="cuda"), "weight": torch.randn(2, 4, 8, device="cuda"),
         "bias": torch.randn(2, 4, device="cuda")}
    want = ds.grouped_linear(t["x"], t["weight"], [3, 4], t["bias"])
    with forward_ad.dual_level():
        assert torch.equal(ds.grouped_linear(t["x"], t["weight"], [3, 4], t["bias"]), want)
        t[of] = forward_ad.make_dual(t[of], torch.ones_like(t[of]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                ds.grouped_linear(t["x"], t["weight"], [3, 4], t["bias"])


# ---------------------------------------------------------------- backward passes side by side


def test_backward_passes_share_no_descriptor(cuda, monkeypatch):
    """Two backward passes of a retained graph may run at the same time: what one hands to the
    library is not written by the other."""
    print("\n[case] descriptors", flush=True)
    plan = ds.neighbor_plan(torch.tensor([[0, 1, 2], [0, 0, 1]], device="cuda"), 4)
    q, k, v = (torch.randn(4, 2, 8, device="cuda", requires_grad=True) for _ in range(3))
    out = ds.neighbor_attention(q, k, v, plan)
    seen, lib = [], _lib.lib()

    class Spy:
        def __getattr__(self, name):
            return getattr(lib, name)

        def dg_attention_backward(self, desc, *args):
            seen.append((desc, desc.ld_g))
            return lib.dg_attention_backward(desc, *args)

    monkeypatch.setattr(_lib, "lib", lambda: Spy())
    wide = torch.randn(4, 64, device="cuda")
    for grad in (wide[:, :16].unflatten(1, (2, 8)), wide[:, :16].contiguous().unflatten(1, (2, 8))):
        torch.autograd.grad(out, (q, k, v), grad, retain_graph=True)
    assert [ld for _, ld in seen] == [64, 16]
    assert [d.ld_g for d, _ in seen] == [64, 16]


# ---------------------------------------------------------------- infinities that are there to see


def _infinite_case(heads, kv, dim, dtype, table, seed=0):
    """Rows of 1 to 70 edges whose sources are all different; returns also, for some rows, an edge
    in the row's middle and its last one."""
    rng = np.random.default_rng(seed)
    deg = np.concatenate([[1, 2, 31, 32, 33, 600, 5], rng.integers(1, 71, 30)])
    n = 700
    dst = np.repeat(rng.permutation(len(deg)), deg)
    src = np.concatenate([rng.permutation(n)[:d] for d in deg])
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    c = {"q": rand(len(deg), heads, dim), "k": rand(n, kv, dim), "v": rand(n, kv, dim), "grad": rand(len(deg), heads, dim),
         "table": None}
    bucket = rng.integers(0, 6, len(src))
    if table:
        c["table"] = torch.randn(8, heads, generator=g)
        if table == "unused":
            c["table"][7] = -float("inf")  # no edge is in it
        if table == "used":
            c["table"][5] = -float("inf")
    end = np.cumsum(deg)
    at = np.concatenate([end[[1, 2, 5, 8]] - 1, (end - deg // 2 - 1)[[3, 5, 9]]])
    return c, src, dst, bucket, at


def _infinite_plan(c, src, dst, bucket):
    """(buckets by distances)"""
    return ds.neighbor_plan(torch.as_tensor(np.stack([src, dst])).cuda(), len(c["k"]), len(c["q"]),
                            distances=torch.as_tensor(bucket + 0.5).cuda(), boundaries=np.arange(1.0, 8.0))


def _same_kind(name, got, want):
    """NaN where the definition has NaN, the same infinities, all else finite."""
    got = got.detach().double().cpu().numpy()
    for what, f in (("NaN", np.isnan), ("+inf", np.isposinf), ("-inf", np.isneginf)):
        a, b = f(got), f(want)
        assert (a == b).all(), f"{name}: {what} at {a.sum()} places, {b.sum()} are right, {(a & b).sum()} in both"


LAYOUTS = pytest.mark.parametrize("layout", [(8, 8, 16), (4, 4, 16), (8, 2, 32), (6, 3, 24), (8, 1, 128), (1, 1, 8), (2, 2, 256)],
                                  ids=str)
TABLES = pytest.mark.parametrize("table", [None, "plain", "unused", "used"])


def _infinite_v(layout, dtype, table):
    """Inputs with infinities and a NaN in v, and what the kernels and the definitions make of them."""
    c, src, dst, bucket, at = _infinite_case(*layout, dtype, table)
    for i, e in enumerate(at):
        c["v"][src[e], i % layout[1], i % layout[2]] = (1 if i % 2 else -1) * float("inf")
    c["v"][src[at[3]], 0, :] = float("nan")
    return c, src, dst, bucket, _run(c, src, dst, bucket)


def _run(c, src, dst, bucket):
    plan = _infinite_plan(c, src, dst, bucket)
    leaves = [c[x].cuda().requires_grad_(True) for x in ("q", "k", "v", "table") if c[x] is not None]
    out = ds.neighbor_attention(*leaves[:3], plan, leaves[3] if c["table"] is not None else None)
    got = [out.detach(), *torch.autograd.grad(out, leaves, c["grad"].cuda())]
    f = {x: None if c[x] is None else c[x].double().numpy() for x in c}
    args = (f["q"], f["k"], f["v"], src, dst)
    with np.errstate(invalid="ignore"):
        want = {"out": oracle.attention(*args, bucket, f["table"])["out"],
                **oracle.attention_grads(*args, f["grad"], bucket, f["table"])[0]}
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), got)), want


@TYPES
@LAYOUTS
@TABLES
def test_infinities_in_v_show_as_the_definition_has_them(cuda, layout, dtype, table):
    """An infinity times a probability above zero is an infinity, whichever edge of a row holds it and
    whatever the table's other entries are; two of opposite signs make a NaN."""
    print(f"\n[case] inf in v {layout} {dtype} {table}", flush=True)
    got, want = _infinite_v(layout, dtype, table)[-1]
    assert np.isinf(want["out"]).any() and np.isnan(want["out"]).any()
    _same_kind("out", got["out"], want["out"])
    finite = np.isfinite(want["out"])
    want, got = want["out"][finite], got["out"].double().cpu().numpy()[finite]
    # (a rounding to bfloat16, or those of some hundreds of terms of order one; the kind is what is tested)
    assert np.abs(got - want).max() < (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -14) * max(1, np.abs(want).max())


@TYPES
@LAYOUTS
@TABLES
def test_the_gradients_of_infinities_in_v(cuda, layout, dtype, table):
    """The gradients have their NaN and infinities where the formulas have them."""
    print(f"\n[case] gradients, inf in v {layout} {dtype} {table}", flush=True)
    got, want = _infinite_v(layout, dtype, table)[-1]
    assert np.isinf(want["dk"]).any() and np.isnan(want["dq"]).any()
    for name in ("dq", "dk", "dv", "dtable")[:len(got) - 1]:
        _same_kind(name, got[name], want[name])


@TYPES
@LAYOUTS
@TABLES
def test_infinities_in_the_gradient_show_as_the_formulas_have_them(cuda, layout, dtype, table):
    print(f"\n[case] inf in the gradient {layout} {dtype} {table}", flush=True)
    c, src, dst, bucket, at = _infinite_case(*layout, dtype, table, seed=1)
    for i, e in enumerate(at):
        c["grad"][dst[e], i % layout[0], i % layout[2]] = (1 if i % 2 else -1) * float("inf")
    got, want = _run(c, src, dst, bucket)
    assert np.isinf(want["dv"]).any()
    for name in ("dq", "dk", "dv", "dtable")[:len(got) - 1]:
        _same_kind(name, got[name], want[name])


# ---------------------------------------------------------------- as many workgroups as there may be


def test_weight_gradients_of_more_than_2_to_the_32_threads(cuda):
    """4,097 groups of 4,096 tiles of the weight's gradient, a workgroup each."""
    groups, k, sizes = 4097, 4096 * 128, {3: 2, 4000: 1, 4096: 2}
    print("\n[case] weights of 4.3 GB", flush=True)
    at = torch.zeros(groups, dtype=torch.long)
    for g, n in sizes.items():
        at[g] = n
    x = torch.randn(5, k, device="cuda").bfloat16()
    w = torch.zeros(1, device="cuda", dtype=torch.bfloat16).expand(groups, 1, k).contiguous().requires_grad_(True)
    b = torch.zeros(groups, 1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    grad = torch.tensor([[1.0], [2.0], [-1.0], [0.5], [4.0]], device="cuda").bfloat16()
    dw, db = torch.autograd.grad(ds.grouped_linear(x, w, at.cuda(), b), (w, b), grad)
    f = x.double()
    want = {3: f[0] + 2 * f[1], 4000: -f[2], 4096: 0.5 * f[3] + 4 * f[4]}
    for g, y in want.items():
        # (products by powers of two and one sum in 32 bits: the result's rounding to bfloat16, and what it moves)
        assert ((dw[g, 0].double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -22 * f.abs().max() * 4).all(), g
        dw[g] = 0
    assert db[:, 0].nonzero()[:, 0].tolist() == [3, 4000, 4096] and db[[3, 4000, 4096], 0].tolist() == [3.0, -1.0, 4.5]
    assert not any(part.any() for part in dw.split(512))


def test_joins_of_more_than_2_to_the_32_threads(cuda):
    """Lists that say 2^26 + 2 long rows, of which the last is there: a workgroup of 64 threads each."""
    print("\n[case] joins of 2^26 rows", flush=True)
    n, entries, said = 700, 600, 2 ** 26 + 2
    plan = ds.neighbor_plan(torch.stack([torch.arange(entries), torch.zeros(entries, dtype=torch.long)]).cuda(), n, 1)
    q, k, v = (torch.randn(m, 1, 8, device="cuda", requires_grad=True) for m in (1, n, n))
    grad = torch.randn(1, 1, 8, device="cuda")

    def step():
        out, lse = ds.neighbor_attention(q, k, v, plan, return_lse=True)
        return [out, lse, *torch.autograd.grad(out, (q, k, v), grad)]

    want = step()
    rows = plan.by_target
    assert rows.c.n_long == 1 and rows.c.n_items > 1
    slots = torch.full((said,), -1, dtype=torch.int32, device="cuda")
    slots[-1:] = rows.long_slot
    rows.c.long_slot, rows.c.n_long = slots.data_ptr(), said
    _leave_nans([1, 8])
    got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- lists near 2^31 entries


@pytest.mark.parametrize("chunk", [2048, 4096])
def test_parts_of_a_row_that_ends_near_2_to_the_31(cuda, chunk):
    """The parts of rows are made from the pointers alone: one row of two up to the last entry that a
    list may hold."""
    print(f"\n[case] parts near 2^31, {chunk}", flush=True)
    end, start = 2 ** 31 - 256, 1000
    ptr = torch.tensor([0, start, end], dtype=torch.int32, device="cuda")
    order = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    parts = [-(-n // chunk) for n in (start, end - start)]
    n_items = end // chunk + 2
    new = lambda *n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    first, items, slots = new(3), new(n_items, 4), new(2)
    lib = _lib.lib()
    size = lib.dg_neighbors_parts_workspace_size(2)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.check(lib.dg_neighbors_parts(_lib.ptr(order), _lib.ptr(ptr), 2, chunk, n_items, 2, _lib.ptr(first), _lib.ptr(items),
                                      _lib.ptr(slots), _lib.ptr(ws), size, _lib.stream_of(ptr.device)), "parts")
    assert first.tolist() == [0, parts[0], sum(parts)] and slots.tolist() == [0, 1]
    items = items.cpu().long()
    rest = items[sum(parts):]
    assert (rest[:, :2] == 0).all() and (rest[:, 2] == -1).all()
    items = items[:sum(parts)]
    at = torch.cat([torch.arange(0, start, chunk), torch.arange(start, end, chunk)])
    slot = torch.repeat_interleave(torch.arange(2), torch.tensor(parts))
    assert torch.equal(items[:, 0], at)
    assert torch.equal(items[:, 1], torch.minimum(at + chunk, torch.tensor([start, end])[slot]))
    assert torch.equal(items[:, 2], 1 - slot) and torch.equal(items[:, 3], slot)


# ---------------------------------------------------------------- arguments that are no tensors


def test_refusals_of_what_is_no_tensor(cuda):
    ei = torch.tensor([[0, 1, 2], [0, 0, 1]], device="cuda")
    one = torch.ones(3, device="cuda")
    bad = lambda match, f, *a, **k: pytest.raises(RuntimeError, f, *a, **k).match(match)  # noqa: E731
    bad("distances must be a tensor", ds.neighbor_plan, ei, 4, distances=[1.0, 1.0, 1.0], boundaries=[1.0])
    bad("edge_mask must be a tensor", ds.neighbor_plan, ei, 4, edge_mask=[True, True, False])
    plan = ds.neighbor_plan(ei, 4, distances=one, boundaries=[1.0])
    q = torch.zeros(4, 2, 8, device="cuda")
    bad("plan must be a NeighborPlan", ds.neighbor_attention, q, q, q, None)
    bad("plan must be a NeighborPlan", ds.neighbor_attention, q, q, q, ei)
    bad("bias_table must be a tensor", ds.neighbor_attention, q, q, q, plan, [[0.0, 0.0], [0.0, 0.0]])
    bad("k must be a CUDA tensor", ds.neighbor_attention, q, None, q, plan)
    x, w = torch.zeros(3, 8, device="cuda"), torch.zeros(1, 4, 8, device="cuda")
    bad("bias must be a tensor", ds.grouped_linear, x, w, [3], [[0.0] * 4])
    bad("weight must be on", ds.grouped_linear, x, None, [3])
