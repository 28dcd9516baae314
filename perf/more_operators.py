"""Cases of the operators of a transformer layer around ``neighbor_attention`` and
``grouped_linear``, over the sizes they are called at, with the operators' plain forms.

Each kind of call alone and, with ``_train``, with its gradients:

  rotate    ``rotate_heads``: queries and keys normalised head by head and rotated by angles that
            go with the atoms' positions along several axes (in training the positions' gradient,
            which forces need, and the norms' weights' are among the results)
  route     ``route_rows``: the experts of each row, their weights, how many rows each expert
            takes and where they lie in the experts' order
  dispatch  ``dispatch_rows``: rows into the experts' order
  combine   ``combine_rows``: the experts' results back, weighted and added to a residual
  linear    ``grouped_linear`` with an activation and a residual: a layer of the experts

``listed`` gives cases of each kind from the smallest crystal up; ``draw`` gives others of the
same ranges.
"""
from __future__ import annotations

import math
import types

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float64": torch.float64, "int64": torch.int64}


def listed():
    return [
        # q and k of one layer on the smallest crystal: launches and host instructions show
        {"name": "rotate_crystal_864", "kind": "rotate", "targets": 864, "ghosts": 0, "heads": 8, "kv_heads": 8,
         "dim": 32, "pairs": 15, "axes": 3, "positions": "float64", "interleaved": False, "norm": True,
         "fused": True, "dtype": "bfloat16"},
        # the largest box of the benchmark, one rank's; q, k and v are views of one product
        {"name": "rotate_1m", "kind": "rotate", "targets": 1_000_000, "ghosts": 0, "heads": 8, "kv_heads": 8,
         "dim": 32, "pairs": 16, "axes": 1, "positions": "float32", "interleaved": True, "norm": True,
         "fused": True, "dtype": "bfloat16"},
        # a training step on a batch of 128 small structures, wider heads, keys shared by four
        {"name": "rotate_train_batch_128", "kind": "rotate_train", "targets": 32_000, "ghosts": 0, "heads": 16,
         "kv_heads": 4, "dim": 64, "pairs": 24, "axes": 3, "positions": "float32", "interleaved": False,
         "norm": True, "fused": True, "dtype": "bfloat16"},
        # the atoms of the smallest crystal over a few experts: launches and host instructions show
        {"name": "route_crystal_864", "kind": "route", "rows": 864, "experts": 8, "k": 2, "scoring": "softmax",
         "biased": False, "groups": 1, "top_groups": 1, "group_best": 1, "renormalize": True, "padded": 0.0,
         "dtype": "bfloat16"},
        # a large box over many experts in groups, chosen with a bias that keeps them balanced
        {"name": "route_300k_groups", "kind": "route", "rows": 300_007, "experts": 64, "k": 6,
         "scoring": "sigmoid", "biased": True, "groups": 8, "top_groups": 4, "group_best": 2,
         "renormalize": True, "padded": 0.0, "dtype": "float32"},
        # a training step on a padded batch
        {"name": "route_train_batch_128", "kind": "route_train", "rows": 32_000, "experts": 128, "k": 8,
         "scoring": "softmax", "biased": False, "groups": 1, "top_groups": 1, "group_best": 1,
         "renormalize": False, "padded": 0.1, "dtype": "bfloat16"},
        # a slab of odd size in single precision, rows of an odd width
        {"name": "dispatch_slab_9973_f32", "kind": "dispatch", "rows": 9973, "experts": 8, "k": 2, "width": 100,
         "padded": 0.0, "dtype": "float32"},
        # a training step's rows to their experts
        {"name": "dispatch_train_100k", "kind": "dispatch_train", "rows": 100_000, "experts": 16, "k": 2,
         "width": 256, "padded": 0.05, "dtype": "bfloat16"},
        # the experts' results of a large box back to its atoms
        {"name": "combine_300k", "kind": "combine", "rows": 300_007, "experts": 64, "k": 6, "width": 128,
         "residual": True, "padded": 0.0, "dtype": "bfloat16"},
        # a training step on a batch in single precision, some of its rows padding
        {"name": "combine_train_batch_128_f32", "kind": "combine_train", "rows": 32_000, "experts": 8, "k": 2,
         "width": 256, "residual": True, "padded": 0.1, "dtype": "float32"},
        # the first layer of the experts of a large box
        {"name": "linear_200k", "kind": "linear", "rows": 200_003, "groups": 16, "width": 256, "out": 512,
         "bias": True, "activation": "silu", "residual": False, "skew": 0.3, "dtype": "bfloat16"},
        # a training step of a layer with a residual on a batch by structure
        {"name": "linear_train_batch_128", "kind": "linear_train", "rows": 32_000, "groups": 128, "width": 256,
         "out": 256, "bias": True, "activation": "gelu", "residual": True, "skew": 0.3, "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate_train", "route", "route_train", "dispatch", "dispatch_train", "combine",
                       "combine_train", "linear", "linear_train"])
    case = {"kind": kind, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    size = 4 if case["dtype"] == "float32" else 2
    train = kind.endswith("_train")
    if kind.startswith("rotate"):
        heads, kv = rng.choice([(4, 4), (8, 8), (16, 4), (8, 2), (6, 3), (8, 1)])
        dim = rng.choice([16, 24, 32, 48, 64, 128, 256])
        axes = rng.choice([1, 2, 3, 3])
        per = rng.randint(1, dim // 2 // axes)
        # the listed ones' bytes
        most = 1_000_000 * 16 * 32 * 2 if not train else 4 * 32_000 * 20 * 64 * 2
        n = _log_int(rng, 1 if rng.random() < 0.2 else 100, most // ((heads + kv) * dim * size))
        ghosts = n // 10 if rng.random() < 0.3 else 0
        norm = rng.random() < 0.8
        return case | {"targets": n - ghosts, "ghosts": ghosts, "heads": heads, "kv_heads": kv, "dim": dim,
                       "pairs": rng.choice([per * axes, dim // 2 // axes * axes]), "axes": axes,
                       # (gradients of positions are worked out in 32 bits)
                       "positions": rng.choice(["float32", "int64"] if train else ["float32", "float64", "int64"]),
                       "interleaved": rng.random() < 0.5, "norm": norm, "fused": rng.random() < 0.7}
    if kind.startswith("linear"):
        k, n = rng.choice([64, 96, 100, 128, 256, 512]), rng.choice([64, 100, 128, 164, 256, 512])
        most = 32_000 * 256 * 256 if train else 200_003 * 256 * 512 // 2
        residual = rng.random() < 0.5
        return case | {"rows": _log_int(rng, 1 if rng.random() < 0.2 else 200, most // (k * n) // (size // 2) // 2),
                       "groups": _log_int(rng, 1, 128), "width": k, "out": n, "bias": rng.random() < 0.7,
                       "activation": rng.choice(["silu", "gelu", "none"] if residual else ["silu", "gelu"]),
                       "residual": residual, "skew": round(rng.uniform(0, 0.8), 2)}
    experts = rng.choice([4, 8, 16, 24, 60, 64, 100, 128, 256])
    k = rng.randint(1, min(8, experts))
    case |= {"experts": experts, "k": k, "padded": rng.choice([0.0, 0.0, 0.1, 0.3])}
    least = 1 if rng.random() < 0.2 else 100
    if kind.startswith("route"):
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
        top = rng.randint(1, groups)
        while top * (experts // groups) < k:
            top += 1
        # a softmax's row is chosen from in 32 bits times the experts, a grouped one in more passes
        most = 32_000 * 128 if train else 300_007 * 64
        return case | {"rows": _log_int(rng, least, most // (experts * size // 2)),
                       "scoring": rng.choice(["softmax", "sigmoid"]), "biased": rng.random() < 0.5,
                       "groups": groups, "top_groups": top, "group_best": rng.choice([1, 2]) if groups > 1 else 1,
                       # (one weight, renormalised, is one: it has no gradient)
                       "renormalize": rng.random() < 0.5 and not (train and k == 1)}
    width = rng.choice([32, 64, 100, 128, 130, 256, 333, 512])
    most = {"dispatch": 9973 * 100 * 4 * 3, "dispatch_train": 100_000 * 256 * 2 * 3, "combine": 300_007 * 128 * 2 * 8,
            "combine_train": 32_000 * 256 * 4 * 4}[kind]
    case |= {"width": width, "rows": _log_int(rng, least, most // ((k + 2) * width * size))}
    if kind.startswith("combine"):
        case["residual"] = rng.random() < 0.7
    return case


# ---------------------------------------------------------------- inputs


def _rotate_inputs(case, rand, g):
    s = types.SimpleNamespace(q_weight=None, k_weight=None)
    dtype, targets, nodes = _TYPES[case["dtype"]], case["targets"], case["targets"] + case["ghosts"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:  # q, k and v are parts of the rows of one product
        rows = rand(nodes, (heads + 2 * kv) * dim).to(dtype)
        q, k, _ = rows.split([heads * dim, kv * dim, kv * dim], 1)
        s.q, s.k = q[:targets].unflatten(1, (heads, dim)), k.unflatten(1, (kv, dim))
    else:
        s.q, s.k = rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)
    # atoms of a box at 0.1 per cubic Angstrom, or the sites of a lattice by number
    side = (10.0 * nodes) ** (1 / 3)
    at = torch.rand(nodes, case["axes"], generator=g, device="cuda", dtype=torch.float64) * side
    s.positions = at.to(_TYPES[case["positions"]])
    # wavelengths from two Angstrom up to twice the box, the same for each axis
    s.sections = (case["pairs"] // case["axes"],) * case["axes"]
    j = torch.arange(s.sections[0], device="cuda", dtype=torch.float64) / max(1, s.sections[0])
    s.frequencies = (math.pi * (1 / (2 + side)) ** j).float().repeat(case["axes"])
    if case["norm"]:
        s.q_weight, s.k_weight = (1 + 0.2 * rand(dim)).to(dtype), (1 + 0.2 * rand(dim)).to(dtype)
    if case["kind"] == "rotate_train":
        s.grads = [rand(targets, heads, dim).to(dtype), rand(nodes, kv, dim).to(dtype)]
        s.leaves = [s.q, s.k]
        if case["norm"]:
            s.leaves += [s.q_weight, s.k_weight]
        if s.positions.is_floating_point():
            s.leaves.append(s.positions)
    return s


def _logits(case, rand, dtype):
    """A router's logits; rows of padding are -inf, which no expert takes."""
    rows, experts = case["rows"], case["experts"]
    logits = 1.5 * rand(rows, experts) + 0.5 * rand(experts)
    if case["padded"]:
        logits[rows - int(case["padded"] * rows):] = -torch.inf
    return logits.to(dtype)


def _route_inputs(case, rand):
    s = types.SimpleNamespace(bias=None)
    s.logits = _logits(case, rand, _TYPES[case["dtype"]])
    if case["biased"]:
        s.bias = 0.1 * rand(case["experts"])
    if case["kind"] == "route_train":
        s.grads = [rand(case["rows"], case["k"])]
        s.leaves = [s.logits]
    return s


def _exchange_inputs(case, rand):
    s = types.SimpleNamespace(residual=None)
    dtype, rows, k, width = _TYPES[case["dtype"]], case["rows"], case["k"], case["width"]
    s.logits = _logits(case, rand, torch.float32)
    if case["kind"].startswith("dispatch"):
        s.x = rand(rows, width).to(dtype)
        if case["kind"] == "dispatch_train":
            s.grads = [rand(rows * k, width).to(dtype)]
            s.leaves = [s.x]
        return s
    s.y = rand(rows * k, width).to(dtype)
    if case["residual"]:
        s.residual = rand(rows, width).to(dtype)
    if case["kind"] == "combine_train":
        s.grads = [rand(rows, width).to(dtype)]
    return s


def _linear_inputs(case, rand, g):
    s = types.SimpleNamespace(bias=None, residual=None)
    dtype, rows, groups, k, n = _TYPES[case["dtype"]], case["rows"], case["groups"], case["width"], case["out"]
    share = torch.exp(case["skew"] * torch.randn(groups, generator=g, device="cuda", dtype=torch.float64))
    ends = torch.round(torch.cumsum(share, 0) / share.sum() * rows).long()
    ends[-1] = rows
    s.sizes = torch.diff(ends, prepend=ends.new_zeros(1))
    s.most = int(s.sizes.max())
    s.x, s.weight = rand(rows, k).to(dtype), (rand(groups, n, k) / math.sqrt(k)).to(dtype)
    if case["bias"]:
        s.bias = rand(groups, n).to(dtype)
    if case["residual"]:
        s.residual = rand(rows, n).to(dtype)
    s.activation = None if case["activation"] == "none" else case["activation"]
    if case["kind"] == "linear_train":
        s.grads = [rand(rows, n).to(dtype)]
        s.leaves = [t for t in (s.x, s.weight, s.bias, s.residual) if t is not None]
    return s


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    what = case["kind"].split("_")[0]
    if what == "rotate":
        s = _rotate_inputs(case, rand, g)
    elif what == "route":
        s = _route_inputs(case, rand)
    elif what == "linear":
        s = _linear_inputs(case, rand, g)
    else:
        s = _exchange_inputs(case, rand)
    s.case, s.kind, s.train = case, what, case["kind"].endswith("_train")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from dynamis_amd import dynamis_state

        s.ops = dynamis_state
        if s.train:
            for t in s.leaves if s.kind != "combine" else ():
                t.requires_grad_(True)
        if s.kind in ("dispatch", "combine"):  # the routing that the layer's router has made
            s.logits.requires_grad_(s.kind == "combine" and s.train)
            s.routing = dynamis_state.route_rows(s.logits, case["k"])
            if s.kind == "combine" and s.train:
                s.leaves = [t for t in (s.y, s.residual) if t is not None]
                for t in s.leaves:
                    t.requires_grad_(True)
                s.leaves.insert(1, s.routing.weights)
    elif s.kind in ("dispatch", "combine"):
        s.weights, s.experts, _, s.places = _route(s.logits, case["k"])
    return s


# ---------------------------------------------------------------- the operators' plain forms


def _angles(s):
    """cos and sin [nodes, 1, pairs]; the angles of far positions need 64 bits."""
    axis = torch.repeat_interleave(torch.arange(len(s.sections), device="cuda"),
                                   torch.tensor(s.sections, device="cuda"), output_size=s.frequencies.numel())
    theta = s.positions.double()[:, axis] * s.frequencies.double()
    return torch.cos(theta).float()[:, None], torch.sin(theta).float()[:, None], axis


def _pairs(x, pairs, interleaved):
    if interleaved:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], x[..., 2 * pairs:]
    return x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]


def _unpair(a, b, rest, interleaved):
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _rotate_one(x, weight, cos, sin, c):
    """(y, normalised x, n, 1 / rms) in 32 bits."""
    x = x.float()
    rstd, hat = None, x
    if c["norm"]:
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        hat = x * rstd
    n = hat if weight is None else hat * weight.float()
    a, b, rest = _pairs(n, c["pairs"], c["interleaved"])
    return _unpair(a * cos - b * sin, a * sin + b * cos, rest, c["interleaved"]), hat, n, rstd


def _rotate_one_grads(g, weight, hat, n, rstd, cos, sin, c):
    """(dx, dweight, dtheta): in 32 bits, the sum over all heads and axes that dtheta enters in 64."""
    a, b, rest = _pairs(g.float(), c["pairs"], c["interleaved"])
    ga, gb = a * cos + b * sin, b * cos - a * sin
    na, nb, _ = _pairs(n, c["pairs"], c["interleaved"])
    dtheta = (na.double() * gb - nb.double() * ga).sum(1)
    back = _unpair(ga, gb, rest, c["interleaved"])
    if not c["norm"]:
        return back, None, dtheta
    dweight = (back * hat).sum((0, 1))
    t = back * weight.float()
    return rstd * (t - hat * (t * hat).mean(-1, keepdim=True)), dweight, dtheta


def _rotate(s):
    c, (cos, sin, axis), targets = s.case, _angles(s), s.q.shape[0]
    q = _rotate_one(s.q, s.q_weight, cos[:targets], sin[:targets], c)
    k = _rotate_one(s.k, s.k_weight, cos, sin, c)
    out = [q[0].to(s.q.dtype), k[0].to(s.k.dtype)]
    if not s.train:
        return out
    dq, dqw, tq = _rotate_one_grads(s.grads[0], s.q_weight, *q[1:], cos[:targets], sin[:targets], c)
    dk, dkw, tk = _rotate_one_grads(s.grads[1], s.k_weight, *k[1:], cos, sin, c)
    out += [dq.to(s.q.dtype), dk.to(s.k.dtype)]
    if c["norm"]:
        out += [dqw.to(s.q.dtype), dkw.to(s.k.dtype)]
    if s.positions.is_floating_point():
        tk[:targets] += tq
        dpos = torch.zeros_like(s.positions, dtype=torch.float64).index_add(1, axis, tk * s.frequencies)
        out.append(dpos.to(s.positions.dtype))
    return out


def _places(experts, count):
    """(sizes, places) of the stable order by expert; choices of none come last."""
    key = torch.where(experts < 0, count, experts).flatten().long()
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(key.numel(), device="cuda")
    place = place.reshape(experts.shape)
    sizes = torch.zeros(count + 1, dtype=torch.long, device="cuda").index_add(0, key, torch.ones_like(key))[:count]
    return sizes, torch.where(experts < 0, -1 - place, place).int()


def _route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True):
    """(weights, experts, sizes, places); what is chosen by is exact or in 64 bits, as neighbours
    may lie next to each other."""
    x = logits.float()
    rows, experts = x.shape
    out = x == -torch.inf
    none = out.all(1, keepdim=True)
    if scoring == "softmax":
        top = x.amax(1, keepdim=True).masked_fill(none, 0.0)
        e = torch.exp(x - top)
        scores = e / e.sum(1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-x))
    if bias is None and group_best == 1:
        v = x.double()
    else:
        d = x.double()
        if scoring == "softmax":
            e = torch.exp(d - top.double())
            v = e / e.sum(1, keepdim=True)
        else:
            v = 1 / (1 + torch.exp(-d))
        if bias is not None:
            v = v + bias.double()
            out = out | (bias == -torch.inf)
        v = v.masked_fill(out, -torch.inf)
    if groups > 1:
        best = torch.sort(v.reshape(rows, groups, -1), dim=2, descending=True).values[..., :group_best]
        worth = best.masked_fill(best == -torch.inf, 0.0).sum(2).masked_fill(best[..., 0] == -torch.inf, -torch.inf)
        kept = torch.sort(worth, dim=1, descending=True, stable=True).indices[:, :top_groups]
        there = torch.zeros(rows, groups, dtype=torch.bool, device="cuda").scatter(1, kept, True)
        v = v.masked_fill(~there.repeat_interleave(experts // groups, 1), -torch.inf)
    v, chosen = torch.sort(v, dim=1, descending=True, stable=True)
    there = v[:, :k] != -torch.inf
    chosen = chosen[:, :k]
    weights = torch.gather(scores, 1, chosen).masked_fill(~there, 0.0)
    if renormalize:
        weights = weights / weights.sum(1, keepdim=True).masked_fill(~there[:, :1], 1.0)
    chosen = torch.where(there, chosen, -1).int()
    return weights, chosen, *_places(chosen, experts)


def _route_grads(s, weights, chosen):
    c, x = s.case, s.logits.float()
    there, at = chosen >= 0, chosen.long().clamp(min=0)
    g = s.grads[0].masked_fill(~there, 0.0)
    if c["renormalize"]:
        d = weights * (g - (g * weights).sum(1, keepdim=True))
    else:
        d = weights * g
    if c["scoring"] == "sigmoid":
        d = d / (1 + torch.exp(torch.gather(x, 1, at)))
    grad = torch.zeros_like(x).scatter_add(1, at, d.masked_fill(~there, 0.0))
    if c["scoring"] == "softmax" and not c["renormalize"]:
        e = torch.exp(x - x.amax(1, keepdim=True).masked_fill(~there[:, :1], 0.0))
        p = e / e.sum(1, keepdim=True).masked_fill(~there[:, :1], 1.0)
        grad = grad - p * d.masked_fill(~there, 0.0).sum(1, keepdim=True)
    return grad.to(s.logits.dtype)


def _route_case(s):
    c = s.case
    out = _route(s.logits, c["k"], c["scoring"], s.bias, c["groups"], c["top_groups"], c["group_best"], c["renormalize"])
    return [*out, _route_grads(s, out[0], out[1])] if s.train else list(out)


def _slots(places):
    return torch.where(places < 0, -1 - places, places).long(), (places >= 0)[..., None]


def _dispatch(s):
    at, there = _slots(s.places)
    rows = torch.empty(at.numel(), s.x.shape[1], dtype=s.x.dtype, device="cuda")
    rows[at] = torch.where(there, s.x[:, None], 0)
    if not s.train:
        return rows
    return [rows, (s.grads[0][at].float() * there).sum(1).to(s.x.dtype)]


def _combine(s):
    at, there = _slots(s.places)
    y = torch.where(there, s.y[at].float(), 0.0)
    out = (s.weights[..., None] * y).sum(1)
    if s.residual is not None:
        out = out + s.residual.float()
    if not s.train:
        return out.to(s.y.dtype)
    g = s.grads[0].float()[:, None]
    dy = torch.empty_like(s.y)
    dy[at] = torch.where(there, s.weights[..., None] * g, 0.0).to(s.y.dtype)
    grads = [dy, (g * y).sum(2)] + ([s.grads[0].clone()] if s.residual is not None else [])
    return [out.to(s.y.dtype), *grads]


def _linear(s):
    rows, groups = s.x.shape[0], s.weight.shape[0]
    group = torch.repeat_interleave(torch.arange(groups, device="cuda"), s.sizes, output_size=rows)
    place = torch.arange(rows, device="cuda") - (torch.cumsum(s.sizes, 0) - s.sizes)[group]
    x = torch.zeros(groups, s.most, s.x.shape[1], device="cuda")
    x[group, place] = s.x.float()
    z = torch.bmm(x, s.weight.float().transpose(1, 2).contiguous())[group, place]
    if s.bias is not None:
        z = z + s.bias.float()[group]
    y, slope = z, None
    if s.activation == "silu":
        share = 1 / (1 + torch.exp(-z))
        y, slope = z * share, share * (1 + z * (1 - share))
    elif s.activation == "gelu":
        share = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        y, slope = z * share, share + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if s.residual is not None:
        y = y + s.residual.float()
    y = y.to(s.x.dtype)
    if not s.train:
        return y
    g = torch.zeros(groups, s.most, s.weight.shape[1], device="cuda")
    g[group, place] = s.grads[0].float() if slope is None else s.grads[0].float() * slope
    grads = [torch.bmm(g, s.weight.float())[group, place].to(s.x.dtype),
             torch.bmm(g.transpose(1, 2).contiguous(), x).to(s.weight.dtype)]
    if s.bias is not None:
        grads.append(g.sum(1).to(s.bias.dtype))
    if s.residual is not None:
        grads.append(s.grads[0].clone())
    return [y, *grads]


_PLAIN = {"rotate": _rotate, "route": _route_case, "dispatch": _dispatch, "combine": _combine, "linear": _linear}


def _own(s):
    c = s.case
    if s.kind == "rotate":
        return s.ops.rotate_heads(s.q, s.k, s.positions, s.frequencies, s.sections, s.q_weight, s.k_weight,
                                  norm=c["norm"], interleaved=c["interleaved"])
    if s.kind == "dispatch":
        return s.ops.dispatch_rows(s.x, s.routing)
    if s.kind == "combine":
        return s.ops.combine_rows(s.y, s.routing, s.residual)
    if s.kind == "linear":
        return s.ops.grouped_linear(s.x, s.weight, s.sizes, s.bias, activation=s.activation, residual=s.residual)
    r = s.ops.route_rows(s.logits, c["k"], scoring=c["scoring"], bias=s.bias, groups=c["groups"],
                         top_groups=c["top_groups"], group_best=c["group_best"], renormalize=c["renormalize"])
    return r.weights, r.experts, r.sizes, r.places


def run(s):
    if not own:
        return _PLAIN[s.kind](s)
    out = _own(s)
    if not s.train:
        return out
    out = [out] if isinstance(out, torch.Tensor) else list(out)
    grads = torch.autograd.grad(out[:len(s.grads)], s.leaves, s.grads)
    return [*(t.detach() for t in out), *grads]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    what, train = case["kind"].split("_")[0], case["kind"].endswith("_train")
    if what == "rotate":
        nodes = case["targets"] + case["ghosts"]
        values = (case["targets"] * case["heads"] + nodes * case["kv_heads"]) * case["dim"]
        at = nodes * case["axes"] * (4 if case["positions"] == "float32" else 8)
        if train and case["positions"] != "int64":
            at *= 2
        return {"bytes": (4 if train else 2) * size * values + at, "flops": (20 if train else 7) * values}
    if what == "route":
        rows, experts, k = case["rows"], case["experts"], case["k"]
        return {"bytes": rows * ((experts * size + k * 4) * (2 if train else 1) + k * 8) + experts * 8,
                "flops": rows * experts * (9 if train else 5)}
    if what in ("dispatch", "combine"):
        rows, k = case["rows"], case["k"]
        there = rows - int(case["padded"] * rows)
        wide = rows + rows * k if what == "dispatch" else rows + there * k + (rows if case["residual"] else 0)
        if what == "dispatch":
            back = there * k + rows
        else:  # the results again are not counted: each input is read once
            back = rows + rows * k + (rows if case["residual"] else 0)
        moved = (wide + (back if train else 0)) * case["width"] * size
        index = rows * k * (4 if what == "dispatch" else 12 if train else 8)
        return {"bytes": moved + index,
                "flops": there * k * case["width"] * ((2 if what == "combine" else 0) + (0 if not train else 3 if what == "combine" else 1))}
    rows, groups, k, n = case["rows"], case["groups"], case["width"], case["out"]
    moved = rows * (k + n * (2 if case["residual"] else 1)) + groups * n * (k + (1 if case["bias"] else 0))
    return {"bytes": size * moved * (2 if train else 1), "flops": (6 if train else 2) * rows * k * n}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _rotate_exact(case, s):
    """Pairs as complex numbers, norms by division, gradients by differentiation."""
    leaves = [t.detach().double().requires_grad_(s.train) for t in (s.q, s.k)]
    weights = [None, None]
    if case["norm"]:
        weights = [t.detach().double().requires_grad_(s.train) for t in (s.q_weight, s.k_weight)]
        leaves += weights
    at = s.positions.detach().double()
    if s.positions.is_floating_point():
        leaves.append(at.requires_grad_(s.train))
    theta = torch.cat([at[:, i:i + 1] * f for i, f in enumerate(s.frequencies.double().split(list(s.sections)))], 1)
    p = case["pairs"]
    out = []
    for x, w in zip(leaves, weights):
        turn = torch.polar(torch.ones_like(theta), theta)[:x.shape[0], None]
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        if case["interleaved"]:
            t = torch.view_as_real(torch.view_as_complex(x[..., :2 * p].unflatten(-1, (p, 2)).contiguous()) * turn)
            t = t.flatten(-2)
        else:
            t = torch.complex(x[..., :p], x[..., p:2 * p]) * turn
            t = torch.cat([t.real, t.imag], -1)
        out.append(torch.cat([t, x[..., 2 * p:]], -1))
    if not s.train:
        return out
    grads = torch.autograd.grad(out, leaves, [g.double() for g in s.grads])
    return [t.detach() for t in out] + list(grads)


def _choose(v, k):
    """The k largest, one after the other, the first of equals; -1 where nothing is left."""
    v, picks = v.clone(), []
    for _ in range(k):
        top, at = v.max(1).values, v.argmax(1)
        picks.append(torch.where(top == -torch.inf, -1, at))
        v.scatter_(1, at[:, None], -torch.inf)
    return torch.stack(picks, 1)


def _route_exact(case, s):
    rows, experts, k = case["rows"], case["experts"], case["k"]
    x = s.logits.detach().double()
    there = x != -torch.inf
    real = there.any(1)
    safe = torch.where(real[:, None], x, 0.0)
    safe = safe.detach().requires_grad_(s.train)
    scores = torch.softmax(safe, 1) if case["scoring"] == "softmax" else torch.sigmoid(safe)
    v = x
    if s.bias is not None or case["group_best"] > 1:
        v = scores.detach() + (0 if s.bias is None else s.bias.double())
        v = v.masked_fill(~there, -torch.inf)
    if case["groups"] > 1:
        per = v.reshape(rows, case["groups"], -1)
        first = per.max(2)
        worth = first.values
        if case["group_best"] == 2:
            second = per.scatter(2, per.argmax(2, keepdim=True), -torch.inf).max(2).values
            worth = torch.where(second == -torch.inf, worth, worth + second)
        kept = _choose(worth, case["top_groups"])
        mine = torch.arange(experts, device="cuda") // (experts // case["groups"])
        v = v.masked_fill(~(mine[None, None] == kept[..., None]).any(1), -torch.inf)
    chosen = _choose(v, k)
    taken = chosen >= 0
    w = torch.gather(scores, 1, chosen.clamp(min=0)) * taken
    if case["renormalize"]:
        w = w / torch.where(taken[:, :1], w.sum(1, keepdim=True), 1.0)
    # an entry's place: those of smaller experts, and the same expert's in rows before
    flat = torch.where(taken, chosen, experts).flatten()
    sizes = torch.bincount(flat, minlength=experts + 1)
    order = torch.argsort(flat * flat.numel() + torch.arange(flat.numel(), device="cuda"))
    places = torch.argsort(order).reshape(rows, k)
    out = [w.detach(), chosen, sizes[:experts], torch.where(taken, places, -1 - places)]
    if s.train:
        grad, = torch.autograd.grad(w, safe, s.grads[0].double())
        out.append(torch.where(real[:, None], grad, 0.0))
    return out


def _exchange_exact(case, s):
    """The exchange as sums over (row, choice) pairs sorted by expert."""
    rows, k, experts = case["rows"], case["k"], case["experts"]
    x = s.logits.detach().double()
    chosen = _choose(x, k)
    taken = chosen >= 0
    top = torch.gather(x, 1, chosen.clamp(min=0))
    w = torch.softmax(torch.where(taken, top, -1e300), 1) * taken
    flat = torch.where(taken, chosen, experts).flatten()
    order = torch.argsort(flat * flat.numel() + torch.arange(flat.numel(), device="cuda"))
    row, real = order // k, flat[order] < experts
    if s.kind == "dispatch":
        out = torch.where(real[:, None], s.x.detach()[row].double(), 0.0)
        if not s.train:
            return out
        g = torch.where(real[:, None], s.grads[0].double(), 0.0)
        return [out, torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda").index_add(0, row, g)]
    share = w.flatten()[order]
    y = torch.where(real[:, None], s.y.detach().double(), 0.0)
    out = torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda")
    if s.residual is not None:
        out += s.residual.detach().double()
    out.index_add_(0, row, share[:, None] * y)
    if not s.train:
        return out
    g = s.grads[0].double()
    dw = torch.zeros(rows * k, dtype=torch.float64, device="cuda")
    dw[order] = (g[row] * y).sum(1)
    return [out, share[:, None] * g[row], dw.reshape(rows, k)] + ([g] if s.residual is not None else [])


def _linear_exact(case, s):
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, None: lambda z: z}[s.activation]
    x, w = s.x.detach().double(), s.weight.detach().double()
    y = torch.empty(case["rows"], case["out"], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.zeros_like(w), torch.zeros(w.shape[:2], dtype=torch.float64, device="cuda")
    a = 0
    for i, size in enumerate(s.sizes.tolist()):
        b = a + size
        z = x[a:b] @ w[i].T
        if s.bias is not None:
            z = z + s.bias[i].detach().double()
        z = z.detach().requires_grad_(s.train)
        f = act(z)
        y[a:b] = f.detach()
        if s.train:
            g, = torch.autograd.grad(f, z, s.grads[0][a:b].double())
            dx[a:b], dw[i], db[i] = g @ w[i], g.T @ x[a:b], g.sum(0)
        a = b
    if s.residual is not None:
        y += s.residual.detach().double()
    if not s.train:
        return y
    return ([y, dx, dw] + ([db] if s.bias is not None else [])
            + ([s.grads[0].double()] if s.residual is not None else []))


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotate": _rotate_exact, "route": _route_exact, "dispatch": _exchange_exact, "combine": _exchange_exact,
            "linear": _linear_exact}[s.kind](case, s)
