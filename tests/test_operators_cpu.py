"""The operators on a built graph, what needs no GPU: the C entry points' refusals (nothing is
launched), the Python calls', the shares of the workspace, and the 64-bit definitions that the GPU
tests check against, themselves checked against differences and against matrices of whole rows."""
import ctypes

import numpy as np
import pytest
import torch

from dynamis_amd import _lib as L
from dynamis_amd import dynamis_state as ds
from oracle import operators as oracle

P = ctypes.c_void_p(4096)  # an address that is never read: the refusals come first


def _error(lib):
    return lib.dg_last_error().decode()


def _lists(n=8, entries=16, items=0):
    c = L.NeighborLists()
    c.order = c.ptr = c.idx = 4096
    c.n_rows = n
    if items:
        c.n_items = items
    return c


def _attention(lib, desc, to=None, fro=None, **null):
    """Status of the forward and of the backward call, with some pointers NULL."""
    to = _lists() if to is None else to
    fro = to if fro is None else fro
    at = lambda name: None if name in null else P  # noqa: E731
    forward = lib.dg_attention_forward(desc, ctypes.byref(to), at("q"), at("k"), at("v"), at("table"), at("out"), None,
                                       None, None, None, 0, None)
    message = _error(lib)
    return forward, message


def _desc(**kw):
    d = dict(n_targets=8, n_nodes=8, ld_q=64, ld_k=64, ld_v=64, ld_g=64, heads=2, kv_heads=2, dim=32, n_buckets=0,
             dtype=L.DG_BF16, scale=1.0)
    d.update(kw)
    return L.AttentionDesc(*(d[name] for name, _ in L.AttentionDesc._fields_))


@pytest.mark.parametrize("change", [dict(heads=0), dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(heads=1025),
                                    dict(dim=0), dict(dim=12), dict(dim=264), dict(n_targets=-1), dict(n_targets=9),
                                    dict(dtype=7), dict(dtype=L.DG_F64), dict(n_buckets=-1), dict(n_buckets=4096),
                                    dict(ld_q=63), dict(ld_k=4), dict(scale=float("nan")), dict(scale=float("inf"))],
                         ids=lambda c: "_".join(f"{k}={v}" for k, v in c.items()))
def test_attention_refuses_a_bad_description(change):
    lib = L.lib()
    d = _desc(**change)
    status, message = _attention(lib, d)
    assert status == L.DG_ERR_INVALID and message
    assert lib.dg_attention_workspace_size(d, ctypes.byref(_lists()), None) == 0 or "ld_" in str(change)


@pytest.mark.parametrize("null", ["q", "k", "v", "out"])
def test_attention_refuses_null(null):
    status, message = _attention(L.lib(), _desc(), **{null: True})
    assert status == L.DG_ERR_INVALID and message


def test_attention_refuses_lists_of_another_size_and_a_small_workspace():
    lib = L.lib()
    status, message = _attention(lib, _desc(n_targets=8, n_nodes=9))
    assert status == L.DG_ERR_INVALID and message
    lists = _lists()
    d = _desc()
    need = lib.dg_attention_workspace_size(d, ctypes.byref(lists), ctypes.byref(lists))
    assert need > 0
    status = lib.dg_attention_backward(d, ctypes.byref(lists), ctypes.byref(lists), P, P, P, None, P, P, P, P, P, P,
                                       None, P, need - 1, None)
    assert status == L.DG_ERR_WORKSPACE


def test_grouped_refusals():
    lib = L.lib()
    good = dict(rows=10, groups=2, k=8, n=8, dtype=L.DG_F32, pad=0)
    for change in (dict(rows=-1), dict(groups=0), dict(k=0), dict(n=0), dict(dtype=9), dict(k=(1 << 20) + 1)):
        d = L.GroupedDesc(*{**good, **change}.values())
        assert lib.dg_grouped_forward(d, P, P, P, None, P, None) == L.DG_ERR_INVALID, change
        assert _error(lib)
    d = L.GroupedDesc(*good.values())
    for i in (0, 1, 2, 4):
        args = [P, P, P, None, P]
        args[i] = None
        assert lib.dg_grouped_forward(d, *args, None) == L.DG_ERR_INVALID, i
    need = lib.dg_grouped_workspace_size(d)
    assert need > 0
    assert lib.dg_grouped_backward(d, P, P, P, P, P, P, None, P, need - 1, None) == L.DG_ERR_WORKSPACE


def test_neighbor_list_refusals():
    lib = L.lib()
    for bad in ((-1, 8, 8, 0), (10, 8, 9, 0), (10, 8, 8, 128), (1 << 31, 8, 8, 0)):
        assert lib.dg_neighbors_workspace_size(L.NeighborDesc(*bad, L.DG_F32)) == 0, bad
        assert _error(lib)
    # (edges without nodes are found on the device, as any index out of range is)
    assert lib.dg_neighbors_workspace_size(L.NeighborDesc(10, 0, 0, 0, L.DG_F32)) > 0
    d = L.NeighborDesc(10, 8, 8, 0, L.DG_F32)
    need = lib.dg_neighbors_workspace_size(d)
    assert need > 0
    call = lambda src, size: lib.dg_neighbors_by_target(d, src, P, None, None, None, P, P, P, None, 1, P, size,  # noqa: E731
                                                        None)
    assert call(None, need) == L.DG_ERR_INVALID
    assert call(P, need - 1) == L.DG_ERR_WORKSPACE
    assert lib.dg_neighbors_parts(P, P, 8, 0, 1, 1, P, P, P, P, 1 << 20, None) == L.DG_ERR_INVALID
    assert lib.dg_neighbors_parts(P, P, 8, 128, 1, 0, P, P, P, P, 1 << 20, None) == L.DG_ERR_INVALID
    assert lib.dg_neighbors_parts(P, P, 8, 128, 1, 1, P, P, None, P, 1 << 20, None) == L.DG_ERR_INVALID
    assert lib.dg_neighbors_parts(P, P, 8, 128, 1, 1, P, P, P, P, 16, None) == L.DG_ERR_WORKSPACE


def test_python_calls_want_the_gpu():
    with pytest.raises(RuntimeError, match="edge_index must be a CUDA tensor"):
        ds.neighbor_plan(torch.zeros(2, 3, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        ds.grouped_linear(torch.zeros(3, 4), torch.zeros(1, 4, 4), [3])


# ---------------------------------------------------------------- the definitions


def _case(seed, heads=4, kv=2, dim=8, targets=5, nodes=7, edges=30, buckets=3):
    r = np.random.default_rng(seed)
    q, grad = r.standard_normal((2, targets, heads, dim))
    k, v = r.standard_normal((2, nodes, kv, dim))
    return q, k, v, r.integers(0, nodes, edges), r.integers(0, targets - 1, edges), grad, r.integers(0, buckets, edges), \
        r.standard_normal((buckets, heads))


def test_attention_definition_against_whole_rows():
    """Every pair once, as matrices: softmax(q k^T) v."""
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal((6, 2, 8)) for _ in range(3))
    src, dst = (x.reshape(-1) for x in np.meshgrid(np.arange(6), np.arange(6)))
    f = oracle.attention(q, k, v, src, dst)
    for h in range(2):
        w = np.exp(q[:, h] @ k[:, h].T / np.sqrt(8.0))
        assert np.allclose(f["out"][:, h], w / w.sum(1, keepdims=True) @ v[:, h], rtol=1e-13, atol=1e-13)
        assert np.allclose(f["lse"][:, h], np.log(w.sum(1)), rtol=1e-13)


def test_attention_definition_of_empty_rows():
    q, k, v, src, dst, _, bucket, table = _case(1)
    f = oracle.attention(q, k, v, src, dst, bucket, table)
    assert not f["out"][-1].any() and (f["lse"][-1] == -np.inf).all()
    f = oracle.attention(q, k, v, src, dst, bucket, np.full_like(table, -np.inf))
    assert not f["out"].any() and (f["lse"] == -np.inf).all()


@pytest.mark.parametrize("of", ["q", "k", "v", "table"])
def test_attention_gradients_against_differences(of):
    """Central differences of step h err by h^2 times a third derivative (of order one here) and by
    1e-16 / h: 1e-9 at h = 1e-5, with room for both constants 1e-7."""
    q, k, v, src, dst, grad, bucket, table = _case(2)
    g, _ = oracle.attention_grads(q, k, v, src, dst, grad, bucket, table)
    x = {"q": q, "k": k, "v": v, "table": table}[of]

    def loss():
        return float((oracle.attention(q, k, v, src, dst, bucket, table)["out"] * grad).sum())

    want = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + 1e-5
        up = loss()
        x[i] = keep - 1e-5
        want[i] = (up - loss()) / 2e-5
        x[i] = keep
    assert np.abs(g["d" + of] - want).max() < 1e-7


def test_grouped_definition_against_loops():
    r = np.random.default_rng(3)
    sizes = [3, 0, 5]
    x, grad = r.standard_normal((10, 4)), r.standard_normal((10, 6))
    w, b = r.standard_normal((3, 6, 4)), r.standard_normal((3, 6))
    got, _ = oracle.grouped_linear(x, w, sizes, b, grad)
    group = [0] * 3 + [2] * 5
    for i, gi in enumerate(group):
        assert np.allclose(got["y"][i], w[gi] @ x[i] + b[gi]) and np.allclose(got["dx"][i], w[gi].T @ grad[i])
    assert not got["y"][8:].any() and not got["dx"][8:].any()  # rows of no group
    for gi in range(3):
        rows = [i for i, other in enumerate(group) if other == gi]
        assert np.allclose(got["dweight"][gi], sum((np.outer(grad[i], x[i]) for i in rows), np.zeros((6, 4))))
        assert np.allclose(got["dbias"][gi], sum((grad[i] for i in rows), np.zeros(6)))


def test_neighbor_lists_definition():
    to, fro = oracle.neighbor_lists(np.array([1, 2, 0, 1]), np.array([0, 0, 1, 1]), 3,
                                    np.array([True, True, True, False]), np.array([0, 1, 2, 3]))
    assert to == {0: [(1, 0), (2, 1)], 1: [(0, 2)], 2: []}
    assert fro == {0: [(1, 2)], 1: [(0, 0)], 2: [(0, 1)]}
