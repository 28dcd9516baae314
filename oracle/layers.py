"""The steps of a layer around attention and grouped products from their definitions, in 64 bits on
the CPU -- TEST INFRASTRUCTURE ONLY (the product never imports it).

Results come with the sum of the magnitudes of their terms, what a rounding error of the
kernels' 32-bit arithmetic scales with.
"""
from __future__ import annotations

import numpy as np


def _where(pairs, interleaved):
    j = np.arange(pairs)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)


def rotate_heads(x, positions, frequencies, sections, weight=None, eps=1e-6, norm=True, interleaved=False, grad=None):
    """One of q and k: dict of y and, with grad, dx, dweight, dpositions; dict of their magnitudes."""
    x, positions, f = (np.asarray(t, np.float64) for t in (x, positions, frequencies))
    dim, pairs = x.shape[2], len(f)
    axis = np.repeat(np.arange(len(sections)), sections)
    theta = (positions[:len(x), axis] * f)[:, None]
    cos, sin = np.cos(theta), np.sin(theta)
    a, b = _where(pairs, interleaved)
    with np.errstate(all="ignore"):
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if norm else np.ones(x.shape[:2] + (1,))
        hat = x * r
    w = np.ones(dim) if weight is None else np.asarray(weight, np.float64)
    n = hat * w
    y, mag = n.copy(), np.abs(n)
    y[..., a], y[..., b] = n[..., a] * cos - n[..., b] * sin, n[..., a] * sin + n[..., b] * cos
    both = np.abs(n[..., a]) + np.abs(n[..., b])
    mag[..., a] = mag[..., b] = both
    out, m = {"y": y}, {"y": mag}
    if grad is None:
        return out, m
    g = np.asarray(grad, np.float64)
    back, bm = g.copy(), np.abs(g)
    back[..., a], back[..., b] = g[..., a] * cos + g[..., b] * sin, g[..., b] * cos - g[..., a] * sin
    bm[..., a] = bm[..., b] = np.abs(g[..., a]) + np.abs(g[..., b])
    t, tm = back * w, bm * np.abs(w)
    out["dx"], m["dx"] = t, tm
    if norm:
        out["dx"] = r * (t - hat * (t * hat).mean(-1, keepdims=True))
        m["dx"] = r * (tm + np.abs(hat) * (tm * np.abs(hat)).mean(-1, keepdims=True))
        out["dweight"], m["dweight"] = (back * hat).sum((0, 1)), (bm * np.abs(hat)).sum((0, 1))
    dtheta = (n[..., a] * back[..., b] - n[..., b] * back[..., a]).sum(1)
    dm = (np.abs(n[..., a]) * bm[..., b] + np.abs(n[..., b]) * bm[..., a]).sum(1)
    out["dpositions"], m["dpositions"] = np.zeros(positions.shape), np.zeros(positions.shape)
    for j in range(pairs):
        out["dpositions"][:len(x), axis[j]] += f[j] * dtheta[:, j]
        m["dpositions"][:len(x), axis[j]] += np.abs(f[j]) * dm[:, j]
    return out, m
