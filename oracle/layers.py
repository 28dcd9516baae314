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


def _first_largest(v, k):
    """Indices of the k largest in falling order: NaN above all, the first of equals, -1 for -inf."""
    key = [(0 if np.isnan(x) else 1, 0.0 if np.isnan(x) else -x, i) for i, x in enumerate(v) if x != -np.inf]
    picks = [i for _, _, i in sorted(key)[:k]]
    return picks + [-1] * (k - len(picks))


def route_rows(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0,
               grad=None):
    """dict of weights, experts, sizes, places and, with grad, dlogits (mag: of dlogits' terms)."""
    x = np.asarray(logits, np.float64)
    rows, n = x.shape
    b = None if bias is None else np.asarray(bias, np.float64)
    weights, experts = np.zeros((rows, k)), np.full((rows, k), -1)
    dlogits, mag = np.zeros((rows, n)), np.zeros((rows, n))
    with np.errstate(all="ignore"):
        for i in range(rows):
            out = x[i] == -np.inf
            top = 0.0 if out.all() else np.nanmax(x[i])
            if scoring == "softmax":
                e = np.exp(x[i] - top)
                s = e / e.sum()
            else:
                s = np.where(x[i] < 0, np.exp(x[i]) / (1 + np.exp(x[i])), 1 / (1 + np.exp(-x[i])))
            v = x[i].copy()
            if b is not None or (groups > 1 and group_best == 2):
                v = s + (0 if b is None else b)
                out = out | (False if b is None else b == -np.inf)
            v[out] = -np.inf
            if groups > 1:
                per = n // groups
                worth = []
                for g in range(groups):
                    mine = v[g * per:(g + 1) * per]
                    best = [mine[j] for j in _first_largest(mine, group_best) if j >= 0]
                    worth.append(sum(best) if best else -np.inf)
                kept = _first_largest(np.array(worth), top_groups)
                for g in range(groups):
                    if g not in kept:
                        v[g * per:(g + 1) * per] = -np.inf
            e = np.array(_first_largest(v, k))
            experts[i] = e
            taken = e[e >= 0]
            if not len(taken):
                continue
            if renormalize:
                # (as exp of differences of log s: nothing vanishes)
                c = x[i, taken]
                ls = c if scoring == "softmax" else -np.logaddexp(0, -c)
                u = np.exp(ls - (np.nanmax(ls) if not np.isinf(np.nanmax(ls)) else 0))
                if np.isnan(ls).any() or np.isposinf(ls).any():
                    u = np.full(len(taken), np.nan)
                u = u / u.sum()
                if scoring == "softmax" and np.isnan(s).any():
                    u = np.full(len(taken), np.nan)
            else:
                u = s[taken]
            weights[i, :len(taken)] = scale * u
            if grad is not None:
                g = np.asarray(grad[i, :len(taken)], np.float64) * scale
                slope = 1 - s[taken] if scoring == "sigmoid" else np.ones(len(taken))
                if scoring == "sigmoid":
                    slope = np.where(x[i, taken] > 0, np.exp(-x[i, taken]) / (1 + np.exp(-x[i, taken])), slope)
                if renormalize:
                    dlogits[i, taken] = u * (g - (g * u).sum()) * slope
                    mag[i, taken] = u * (np.abs(g) + np.abs(g * u).sum()) * slope
                else:
                    dlogits[i, taken], mag[i, taken] = u * g * slope, u * np.abs(g) * slope
                    if scoring == "softmax":
                        dlogits[i] -= s * (g * u).sum()
                        mag[i] += s * np.abs(g * u).sum()
    sizes, places = places_of(experts, n)
    return {"weights": weights, "experts": experts, "sizes": sizes, "places": places, "dlogits": dlogits, "mag": mag}


def places_of(experts, n):
    """(sizes, places) of the order by expert, then row."""
    flat = np.where(experts < 0, n, experts).ravel()
    order = np.argsort(flat, kind="stable")
    place = np.empty(flat.size, np.int64)
    place[order] = np.arange(flat.size)
    return (np.bincount(flat, minlength=n + 1)[:n],
            np.where(flat == n, -1 - place, place).reshape(experts.shape))


def dispatch_rows(x, places, grad=None):
    """(rows in the experts' order, dx, the magnitudes of its terms)."""
    x = np.asarray(x, np.float64)
    rows, k = places.shape
    out, dx, mag = np.zeros((rows * k, x.shape[1])), np.zeros_like(x), np.zeros_like(x)
    for j in range(k):
        there = places[:, j] >= 0
        out[places[there, j]] = x[there]
        if grad is not None:
            dx[there] += np.asarray(grad, np.float64)[places[there, j]]
            mag[there] += np.abs(np.asarray(grad, np.float64)[places[there, j]])
    return out, dx, mag


def combine_rows(y, places, weights, residual=None, grad=None):
    """dict of out and, with grad, dy, dweights; dict of the magnitudes."""
    y, w = np.asarray(y, np.float64), np.asarray(weights, np.float64)
    rows, k = places.shape
    out = np.zeros((rows, y.shape[1])) if residual is None else np.asarray(residual, np.float64).copy()
    r, m = {"out": out, "dy": np.zeros_like(y), "dweights": np.zeros((rows, k))}, {"out": np.abs(out), "dweights": np.zeros((rows, k))}
    for j in range(k):
        there = places[:, j] >= 0
        at = places[there, j]
        out[there] += w[there, j, None] * y[at]
        m["out"][there] += np.abs(w[there, j, None] * y[at])
        if grad is not None:
            g = np.asarray(grad, np.float64)[there]
            r["dy"][at] = w[there, j, None] * g
            r["dweights"][there, j] = (g * y[at]).sum(1)
            m["dweights"][there, j] = np.abs(g * y[at]).sum(1)
    return r, m
