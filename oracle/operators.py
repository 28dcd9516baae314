"""The operators on a built graph from their definitions, in 64 bits on the CPU -- TEST
INFRASTRUCTURE ONLY (the product never imports it).

Every function also returns, for each result, the sum of the magnitudes of its terms: what
a rounding error of the kernels' 32-bit arithmetic scales with.
"""
from __future__ import annotations

import numpy as np


def _rows_sum(n, at, x):
    out = np.zeros((n,) + x.shape[1:])
    np.add.at(out, at, x)
    return out


def attention(q, k, v, src, dst, bucket=None, table=None, scale=None):
    """dict of out, lse, p (per edge and head) and the magnitudes ``out_mag`` and ``logit_mag``."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    T, H, D = q.shape
    r = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    ke, ve = np.repeat(k[src], r, 1), np.repeat(v[src], r, 1)
    terms = q[dst] * ke * scale
    logit, mag = terms.sum(-1), np.abs(terms).sum(-1)
    there = np.ones(logit.shape, bool)
    if table is not None:
        b = np.asarray(table, np.float64)[bucket]
        there = b != -np.inf
        logit, mag = logit + b, mag + np.where(there, np.abs(b), 0)
    logit = np.where(there, logit, -np.inf)
    top = np.full((T, H), -np.inf)
    np.maximum.at(top, dst, logit)
    base = np.where(top == -np.inf, 0, top)
    w = np.where(there, np.exp(logit - base[dst]), 0)
    total = _rows_sum(T, dst, w)
    p = w / np.where(total == 0, 1, total)[dst]
    pv = np.where(there[..., None], p[..., None] * ve, 0)
    with np.errstate(divide="ignore"):
        lse = base + np.log(total)
    return {"out": _rows_sum(T, dst, pv), "lse": lse, "p": p, "there": there,
            "out_mag": _rows_sum(T, dst, np.abs(pv)), "logit_mag": np.where(there, mag, 0)}


def attention_grads(q, k, v, src, dst, grad, bucket=None, table=None, scale=None):
    """(dict of dq, dk, dv, dtable, dict of their magnitudes)."""
    f = attention(q, k, v, src, dst, bucket, table, scale)
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    T, H, D = q.shape
    N, KV = k.shape[:2]
    r = H // KV
    scale = D ** -0.5 if scale is None else scale
    ke, ve = np.repeat(k[src], r, 1), np.repeat(v[src], r, 1)
    gv = grad[dst] * ve
    delta = (grad * f["out"]).sum(-1)
    there = f["there"]
    ds = np.where(there, f["p"] * (gv.sum(-1) - delta[dst]), 0)
    mag = np.where(there, f["p"] * (np.abs(gv).sum(-1) + (np.abs(grad) * f["out_mag"]).sum(-1)[dst]), 0)

    def by_kv(x):
        return x.reshape(len(src), KV, r, D).sum(2)

    def terms(s, x):
        return np.where(there[..., None], s[..., None] * x, 0)

    g, m = {}, {}
    g["dq"], m["dq"] = (_rows_sum(T, dst, terms(s, x)) * f for s, x, f in ((ds, ke, scale), (mag, np.abs(ke), abs(scale))))
    g["dk"], m["dk"] = (_rows_sum(N, src, by_kv(terms(s, x))) * f
                        for s, x, f in ((ds, q[dst], scale), (mag, np.abs(q[dst]), abs(scale))))
    g["dv"], m["dv"] = (_rows_sum(N, src, by_kv(terms(f["p"], x))) for x in (grad[dst], np.abs(grad[dst])))
    if table is not None:
        g["dtable"], m["dtable"] = (_rows_sum(len(table), bucket, s) for s in (ds, mag))
    return g, m


def neighbor_lists(src, dst, n_nodes, mask=None, bucket=None):
    """What ``neighbor_plan`` lists, as {node: sorted [(other node, bucket)]}, by target and by source."""
    keep = np.ones(len(src), bool) if mask is None else mask
    b = np.zeros(len(src), int) if bucket is None else bucket
    to, fro = {i: [] for i in range(n_nodes)}, {i: [] for i in range(n_nodes)}
    for s, d, c, m in zip(src.tolist(), dst.tolist(), b.tolist(), keep.tolist()):
        if m:
            to[d].append((s, c))
            fro[s].append((d, c))
    return {i: sorted(x) for i, x in to.items()}, {i: sorted(x) for i, x in fro.items()}


def grouped_linear(x, weight, sizes, bias=None, grad=None):
    """dict of y and, with grad, dx, dweight, dbias; dict of their magnitudes."""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    G, N, K = weight.shape
    y, y_mag = np.zeros((len(x), N)), np.zeros((len(x), N))
    r = {"y": y}
    m = {"y": y_mag}
    if grad is not None:
        grad = np.asarray(grad, np.float64)
        r |= {"dx": np.zeros_like(x), "dweight": np.zeros_like(weight), "dbias": np.zeros((G, N))}
        m |= {k: np.zeros_like(r[k]) for k in ("dx", "dweight", "dbias")}
    at = 0
    for g, size in enumerate(sizes):
        s = slice(at, at + int(size))
        at += int(size)
        y[s], y_mag[s] = x[s] @ weight[g].T, np.abs(x[s]) @ np.abs(weight[g]).T
        if bias is not None:
            y[s] += np.asarray(bias[g], np.float64)
            y_mag[s] += np.abs(np.asarray(bias[g], np.float64))
        if grad is not None:
            d = grad[s]
            r["dx"][s], m["dx"][s] = d @ weight[g], np.abs(d) @ np.abs(weight[g])
            r["dweight"][g], m["dweight"][g] = d.T @ x[s], np.abs(d).T @ np.abs(x[s])
            r["dbias"][g], m["dbias"][g] = d.sum(0), np.abs(d).sum(0)
    return r, m
