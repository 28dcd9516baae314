"""dg_grouped_apply_gradients, what needs no GPU: refusals (nothing is launched) and the workspace."""
import ctypes

import pytest

from dynamis_amd import _lib as L

P = ctypes.c_void_p(4096)  # an address that is never read: the refusals come first


def _desc(rows=300, groups=3, k=24, n=40, dtype=L.DG_BF16):
    return L.GroupedDesc(rows, groups, k, n, dtype, 0)


def _call(d, act=L.DG_ACT_SILU, size=1 << 40, **null):
    args = {name: P for name in ("x", "weight", "sizes", "bias", "grad", "dx", "dw", "db", "ws")}
    args.update(null)
    return L.lib().dg_grouped_apply_gradients(d, act, *args.values(), size, None)


def test_refusals():
    for bad in (dict(dtype=L.DG_F64), dict(rows=-1), dict(groups=0), dict(k=0), dict(n=(1 << 20) + 1)):
        assert _call(_desc(**bad)) == L.DG_ERR_INVALID, bad
        assert L.lib().dg_grouped_apply_workspace_size(_desc(**bad)) == 0
    assert _call(None) == L.DG_ERR_INVALID
    for act in (-1, 3):
        assert _call(_desc(), act) == L.DG_ERR_INVALID
    for name in ("x", "weight", "sizes", "grad", "dw"):  # (a bias' gradient comes with the weight's)
        assert _call(_desc(), **{name: None}) == L.DG_ERR_INVALID, name
        assert _call(_desc(), L.DG_ACT_NONE, **{name: None}) == L.DG_ERR_INVALID, name
    assert _call(_desc(), ws=None) == L.DG_ERR_WORKSPACE


@pytest.mark.parametrize("dtype,size", [(L.DG_BF16, 2), (L.DG_F32, 4)])
def test_workspace(dtype, size):
    """The activation's gradient in 32 bits beside what the sums of the weights' need."""
    lib, d = L.lib(), _desc(dtype=dtype)
    need = lib.dg_grouped_apply_workspace_size(d)
    assert need >= lib.dg_grouped_workspace_size(d) + 300 * 40 * 4
    assert _call(d, size=need - 1) == L.DG_ERR_WORKSPACE
    only_x = need - lib.dg_grouped_workspace_size(d)
    assert _call(d, size=only_x - 1, dw=None, db=None) == L.DG_ERR_WORKSPACE
    far = _desc(rows=1 << 40, n=1 << 20, k=8, dtype=dtype)
    assert lib.dg_grouped_apply_workspace_size(far) >= (1 << 62)
