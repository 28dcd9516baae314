"""The magnitudes that the operators' 64-bit definitions give beside their results (no GPU)."""
import numpy as np
import pytest

from oracle import operators as oracle


@pytest.mark.parametrize("scale", [0.7, -0.7])
def test_magnitudes_bound_the_results_at_any_scale(scale):
    r = np.random.default_rng(0)
    q, grad = r.standard_normal((2, 5, 4, 8))
    k, v = r.standard_normal((2, 7, 2, 8))
    src, dst = r.integers(0, 7, 30), r.integers(0, 5, 30)
    f = oracle.attention(q, k, v, src, dst, scale=scale)
    assert (np.abs(f["out"]) <= f["out_mag"] * (1 + 1e-12)).all() and (f["logit_mag"] >= 0).all()
    g, m = oracle.attention_grads(q, k, v, src, dst, grad, scale=scale)
    for name in g:
        assert (np.abs(g[name]) <= m[name] * (1 + 1e-12)).all(), name
