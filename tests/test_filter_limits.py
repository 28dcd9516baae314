"""dg_filter_edges_to_radius refuses more edges than it can launch threads for (no GPU; no call here
has a workspace, so none goes as far as a launch)."""
import ctypes

import pytest

from dynamis_amd import _lib as L


@pytest.mark.parametrize("edges,status", [(2 ** 32 - 256, L.DG_ERR_WORKSPACE), (2 ** 32 - 255, L.DG_ERR_INVALID),
                                          (2 ** 32 + 777, L.DG_ERR_INVALID), (2 ** 40, L.DG_ERR_INVALID)])
def test_edges_of_the_index_filter(edges, status):
    lib = L.lib()
    p = ctypes.c_void_p(4096)  # never read
    cell = (ctypes.c_double * 9)(10, 0, 0, 0, 10, 0, 0, 0, 10)
    assert lib.dg_filter_edges_to_radius(p, L.DG_F32, 2, cell, 2.0, p, p, p, L.DG_I32, edges, p, p, p, 0, None) == status
    assert lib.dg_last_error()
