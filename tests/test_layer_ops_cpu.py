"""The operators of a layer, what needs no GPU: the C entry points' refusals (nothing is launched), the Python
calls', and the 64-bit definitions that the GPU tests check against, themselves checked another way."""
import ctypes

import numpy as np
import pytest
import torch

from dynamis_amd import _lib as L
from dynamis_amd import dynamis_state as ds
from oracle import layers as oracle

P = ctypes.c_void_p(4096)  # an address that is never read: the refusals come first


def _error(lib):
    return lib.dg_last_error().decode()


def _rotate(**kw):
    d = dict(n_targets=8, n_nodes=8, ld_q=64, ld_k=64, ld_gq=64, ld_gk=64, heads=2, kv_heads=2, dim=32, axes=2,
             sections=(ctypes.c_int32 * 8)(4, 5), dtype=L.DG_BF16, weight_dtype=L.DG_F32, pos_dtype=L.DG_F64, norm=1,
             interleaved=0, eps=1e-6)
    d.update(kw)
    return L.RotateDesc(*(d[name] for name, _ in L.RotateDesc._fields_))


def _ints(*x):
    return (ctypes.c_int32 * 8)(*x)


@pytest.mark.parametrize("change", [dict(n_targets=9), dict(n_targets=-1), dict(n_nodes=-1), dict(n_nodes=1 << 41), dict(heads=0),
                                    dict(heads=1025), dict(kv_heads=0), dict(dim=0), dict(dim=12), dict(dim=264), dict(axes=0),
                                    dict(axes=9), dict(sections=_ints(8, 9)), dict(sections=_ints(-1, 4)), dict(sections=_ints(0, 0)),
                                    dict(sections=_ints(2 ** 31 - 1, 2 ** 31 - 1)), dict(dtype=7), dict(dtype=L.DG_F64),
                                    dict(weight_dtype=L.DG_F64), dict(dtype=L.DG_F32, weight_dtype=L.DG_BF16),
                                    dict(pos_dtype=L.DG_I32), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                    dict(ld_q=63), dict(ld_k=4), dict(ld_gq=-8), dict(ld_gk=1 << 60)],
                         ids=lambda c: "_".join(c))
def test_rotate_refuses_a_bad_description(change):
    lib, d = L.lib(), _rotate(**change)
    assert lib.dg_rotate_forward(d, P, P, P, P, P, P, P, P, None) == L.DG_ERR_INVALID and _error(lib)
    assert lib.dg_rotate_backward(d, P, P, P, P, P, P, P, P, P, P, P, P, P, P, 1 << 30, None) == L.DG_ERR_INVALID
    assert lib.dg_rotate_workspace_size(d) == 0


def test_rotate_refuses_pointers():
    lib, d = L.lib(), _rotate()
    for i in (0, 1, 2, 3, 6, 7):  # q, k, positions, frequencies, the results
        args = [P] * 8
        args[i] = None
        assert lib.dg_rotate_forward(d, *args, None) == L.DG_ERR_INVALID, i
    odd = ctypes.c_void_p(4104)
    for i in (0, 1, 6, 7):
        args = [P] * 8
        args[i] = odd
        assert lib.dg_rotate_forward(d, *args, None) == L.DG_ERR_INVALID and "16 bytes" in _error(lib), i
    assert lib.dg_rotate_forward(_rotate(norm=0), *[P] * 8, None) == L.DG_ERR_INVALID and "norm" in _error(lib)
    back = lambda d, *a, size=1 << 30: lib.dg_rotate_backward(d, *a, size, None)  # noqa: E731
    for i in (0, 1, 2, 3, 6, 7, 8, 9):
        args = [P] * 14
        args[i] = None
        assert back(d, *args) == L.DG_ERR_INVALID, i
    need = lib.dg_rotate_workspace_size(d)
    assert need > 0 and back(d, *[P] * 14, size=need - 1) == L.DG_ERR_WORKSPACE
    assert back(d, *[P] * 13, None) == L.DG_ERR_WORKSPACE
    args = [P] * 14
    args[4] = None  # a weight's gradient without the weight
    assert back(d, *args) == L.DG_ERR_INVALID
    assert back(_rotate(pos_dtype=L.DG_I64), *[P] * 14) == L.DG_ERR_INVALID and "whole" in _error(lib)


def _route(**kw):
    d = dict(n_rows=100, ld=16, n_experts=16, k=4, groups=1, top_groups=1, group_best=1, sigmoid=0, renormalize=1, dtype=L.DG_F32,
             scale=1.0, pad_=0)
    d.update(kw)
    return L.RouteDesc(*(d[name] for name, _ in L.RouteDesc._fields_))


@pytest.mark.parametrize("change", [dict(n_rows=-1), dict(n_rows=1 << 29), dict(n_rows=1 << 62), dict(n_experts=0), dict(n_experts=1025),
                                    dict(k=0), dict(k=17), dict(n_experts=128, k=65), dict(groups=0), dict(groups=3),
                                    dict(n_experts=1024, groups=128), dict(top_groups=0), dict(groups=4, top_groups=5),
                                    dict(group_best=0), dict(group_best=3), dict(dtype=L.DG_F64), dict(ld=-1), dict(ld=1 << 40),
                                    dict(scale=float("nan")), dict(scale=float("inf"))], ids=lambda c: "_".join(c))
def test_route_refuses_a_bad_description(change):
    lib, d = L.lib(), _route(**change)
    assert lib.dg_route_forward(d, P, P, P, P, P, P, P, 1 << 40, None) == L.DG_ERR_INVALID and _error(lib)
    assert lib.dg_route_backward(d, P, P, P, P, None) == L.DG_ERR_INVALID
    assert lib.dg_route_workspace_size(d) == 0


def test_route_refuses_pointers_and_a_small_workspace():
    lib, d = L.lib(), _route()
    need = lib.dg_route_workspace_size(d)
    assert need > 0
    for i in (0, 2, 3, 4, 5):  # logits, weights, experts, sizes, places
        args = [P] * 6
        args[i] = None
        assert lib.dg_route_forward(d, *args, P, need, None) == L.DG_ERR_INVALID, i
    assert lib.dg_route_forward(d, *[P] * 7, need - 1, None) == L.DG_ERR_WORKSPACE
    assert lib.dg_route_forward(d, *[P] * 6, None, need, None) == L.DG_ERR_WORKSPACE
    for i in range(4):
        args = [P] * 4
        args[i] = None
        assert lib.dg_route_backward(d, *args, None) == L.DG_ERR_INVALID, i
    assert lib.dg_route_backward(_route(n_rows=0), None, None, None, None, None) == L.DG_OK


def _exchange(**kw):
    d = dict(n_rows=100, ld=16, k=4, width=16, dtype=L.DG_F32, pad_=0)
    d.update(kw)
    return L.ExchangeDesc(*(d[name] for name, _ in L.ExchangeDesc._fields_))


def test_exchange_refusals():
    lib = L.lib()
    for change in (dict(n_rows=-1), dict(n_rows=1 << 29), dict(k=0), dict(k=65), dict(width=0), dict(width=(1 << 20) + 1),
                   dict(dtype=L.DG_I64), dict(ld=-1), dict(ld=1 << 40)):
        d = _exchange(**change)
        assert lib.dg_exchange_dispatch(d, P, P, P, None) == L.DG_ERR_INVALID and _error(lib), change
        assert lib.dg_exchange_combine(d, P, P, P, P, P, None) == L.DG_ERR_INVALID, change
        assert lib.dg_exchange_combine_backward(d, P, P, P, P, P, P, None) == L.DG_ERR_INVALID, change
    d = _exchange()
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert lib.dg_exchange_dispatch(d, *args, None) == L.DG_ERR_INVALID
    for args in ((None, P, P, P, P), (P, None, P, P, P), (P, P, P, P, None)):
        assert lib.dg_exchange_combine(d, *args, None) == L.DG_ERR_INVALID
    for args in ((None, P, P, P, P, P), (P, None, P, P, P, P), (P, P, None, P, P, P), (P, P, P, None, P, P)):
        assert lib.dg_exchange_combine_backward(d, *args, None) == L.DG_ERR_INVALID
    assert lib.dg_exchange_combine_backward(d, P, P, P, P, None, None, None) == L.DG_OK  # (nothing is asked for)
    empty = _exchange(n_rows=0)
    assert lib.dg_exchange_dispatch(empty, None, None, None, None) == L.DG_OK


def test_grouped_apply_refusals():
    lib = L.lib()
    good = dict(rows=10, groups=2, k=8, n=8, dtype=L.DG_F32, pad=0)
    for call in (lib.dg_grouped_apply, lib.dg_grouped_apply_backward):
        for change in (dict(rows=-1), dict(groups=0), dict(k=0), dict(n=0), dict(dtype=9), dict(k=(1 << 20) + 1)):
            assert call(L.GroupedDesc(*{**good, **change}.values()), L.DG_ACT_SILU, P, P, P, P, P, P, None) == L.DG_ERR_INVALID
        d = L.GroupedDesc(*good.values())
        for act in (-1, 3):
            assert call(d, act, P, P, P, P, P, P, None) == L.DG_ERR_INVALID and "activation" in _error(lib)
        for i in (0, 1, 2, 5):
            args = [P] * 6
            args[i] = None
            assert call(d, L.DG_ACT_GELU, *args, None) == L.DG_ERR_INVALID, i
    assert lib.dg_grouped_apply_backward(d, L.DG_ACT_GELU, P, P, P, P, None, P, None) == L.DG_ERR_INVALID


def test_python_calls_want_the_gpu():
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ds.rotate_heads(torch.zeros(3, 2, 8), torch.zeros(3, 2, 8), torch.zeros(3, 1), torch.ones(2))
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        ds.route_rows(x, 2)
    with pytest.raises(RuntimeError, match="routing must be a Routing"):
        ds.dispatch_rows(x, None)
    with pytest.raises(RuntimeError, match="routing must be a Routing"):
        ds.combine_rows(x, (x, x))
    with pytest.raises(RuntimeError, match="activation must be"):
        ds.grouped_linear(x, torch.zeros(1, 4, 8), [3], activation="tanh")


def test_a_routing_of_another_make_is_refused():
    """A Routing that was made, moved or changed by its user."""
    x, e, n = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    for places in (e, e.long(), e[0], None, torch.zeros(3, 65, dtype=torch.int32)):
        r = ds.Routing(4, torch.zeros(3, 2), e, n, places)
        with pytest.raises(RuntimeError, match="routing.places must be"):
            ds.dispatch_rows(x, r)
        with pytest.raises(RuntimeError, match="routing.places must be"):
            ds.combine_rows(torch.zeros(6, 8), r)


# ---------------------------------------------------------------- the definitions


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_definition_by_differentiation(norm, interleaved):
    """Against torch's gradients of the rotation as a complex product."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 16, generator=g, dtype=torch.float64, requires_grad=True)
    at = torch.randn(7, 2, generator=g, dtype=torch.float64, requires_grad=True)
    f = torch.rand(5, generator=g, dtype=torch.float64)
    w = torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True)
    grad = torch.randn(5, 3, 16, generator=g, dtype=torch.float64)
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-3) * w if norm else x
    theta = (at[:5, [0, 0, 1, 1, 1]] * f)[:, None]
    turn = torch.polar(torch.ones_like(theta), theta)
    if interleaved:
        t = torch.view_as_real(torch.view_as_complex(n[..., :10].unflatten(-1, (5, 2)).contiguous()) * turn).flatten(-2)
    else:
        t = torch.complex(n[..., :5], n[..., 5:10]) * turn
        t = torch.cat([t.real, t.imag], -1)
    y = torch.cat([t, n[..., 10:]], -1)
    grads = torch.autograd.grad(y, [x, at] + [w] * norm, grad)
    r, m = oracle.rotate_heads(x.detach().numpy(), at.detach().numpy(), f.numpy(), (2, 3), w.detach().numpy() if norm else None, 1e-3,
                               norm, interleaved, grad.numpy())
    near = lambda a, b: np.allclose(a, b.detach().numpy(), rtol=1e-12, atol=1e-12)  # noqa: E731
    assert near(r["y"], y) and near(r["dx"], grads[0]) and near(r["dpositions"], grads[1])
    assert not norm or near(r["dweight"], grads[2])
    assert all((np.abs(r[k]) <= m[k] * (1 + 1e-12)).all() for k in r)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_routing_definition_by_differentiation(scoring, renormalize):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 12, generator=g, dtype=torch.float64, requires_grad=True)
    bias = 0.3 * torch.randn(12, generator=g, dtype=torch.float64)
    grad = torch.randn(9, 3, generator=g, dtype=torch.float64)
    s = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    v = (s + bias).detach().reshape(9, 4, 3)
    worth = torch.topk(v, 2, 2).values.sum(2)
    kept = torch.topk(worth, 2, 1).indices
    v = torch.where(torch.zeros(9, 4, dtype=torch.bool).scatter(1, kept, True)[..., None], v, -torch.inf).flatten(1)
    chosen = torch.topk(v, 3, 1).indices
    w = torch.gather(s, 1, chosen)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    dx, = torch.autograd.grad(2.5 * w, x, grad)
    r = oracle.route_rows(x.detach().numpy(), 3, scoring, bias.numpy(), 4, 2, 2, renormalize, 2.5, grad.numpy())
    assert np.array_equal(r["experts"], chosen.numpy())
    assert np.allclose(r["weights"], 2.5 * w.detach().numpy(), rtol=1e-12)
    assert np.allclose(r["dlogits"], dx.numpy(), rtol=1e-11, atol=1e-13)
    assert (np.abs(r["dlogits"]) <= r["mag"] * (1 + 1e-12)).all()
    assert np.array_equal(r["sizes"], np.bincount(chosen.numpy().ravel(), minlength=12))


def test_routing_definition_of_ties_and_padding():
    x = np.array([[0.0, 1.0, 1.0, -np.inf], [-np.inf] * 4, [np.nan, 3.0, 0.0, 0.0], [-np.inf, 2.0, -np.inf, -np.inf]])
    r = oracle.route_rows(x, 2)
    assert r["experts"].tolist() == [[1, 2], [-1, -1], [0, 1], [1, -1]]
    assert np.allclose(r["weights"][[0, 1, 3]], [[0.5, 0.5], [0, 0], [1, 0]]) and np.isnan(r["weights"][2]).all()
    assert r["sizes"].tolist() == [1, 3, 1, 0]
    # by expert, then row: expert 0: row 2; expert 1: rows 0, 2, 3; expert 2: row 0; none: row 1 twice, row 3
    assert r["places"].tolist() == [[1, 4], [-6, -7], [0, 2], [3, -8]]


def test_exchange_definition_against_loops():
    r = np.random.default_rng(4)
    e = np.array([[1, 0], [-1, -1], [2, 1], [0, -1]])
    _, places = oracle.places_of(e, 3)
    x, go, w = r.standard_normal((4, 5)), r.standard_normal((8, 5)), r.standard_normal((4, 2))
    out, dx, _ = oracle.dispatch_rows(x, places, go)
    want = [x[0], x[3], x[0], x[2], x[2]]  # experts 0, 0, 1, 1, 2
    assert np.array_equal(out, np.array(want + [np.zeros(5)] * 3))
    assert np.allclose(dx, [go[2] + go[0], np.zeros(5), go[4] + go[3], go[1]])
    y, g = r.standard_normal((8, 5)), r.standard_normal((4, 5))
    c, _ = oracle.combine_rows(y, places, w, x, g)
    assert np.allclose(c["out"], [x[0] + w[0, 0] * y[2] + w[0, 1] * y[0], x[1], x[2] + w[2, 0] * y[4] + w[2, 1] * y[3],
                                  x[3] + w[3, 0] * y[1]])
    assert np.allclose(c["dy"][[0, 1, 2, 3, 4]], [w[0, 1] * g[0], w[3, 0] * g[3], w[0, 0] * g[0], w[2, 1] * g[2], w[2, 0] * g[2]])
    assert not c["dy"][5:].any()
    assert np.allclose(c["dweights"], [[g[0] @ y[2], g[0] @ y[0]], [0, 0], [g[2] @ y[4], g[2] @ y[3]], [g[3] @ y[1], 0]])
