"""Cases of the operators that a model runs on a built neighbour list, over the sizes they are
called at, with the operators' plain forms.

Four kinds of call:

  attend        ``neighbor_attention``: every target attends to the sources of its edges, the
                logits biased by a learned table over distance buckets (inference)
  attend_train  the same with the gradients of q, k, v and the table
  group         ``grouped_linear``: rows times the weight of their group (a structure, a
                species, an expert), ragged sizes
  group_train   the same with the gradients of the rows, the weights and the bias

The lists are those of periodic boxes: jittered lattices with vacancies, targets in blocks of
space, atoms numbered at random as a caller's are.  ``listed`` gives cases of each kind from
the smallest crystal up; ``draw`` gives others of the same ranges.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one force call on a small crystal (the 864 atoms of the smallest configuration):
        # launches and host instructions show
        {"name": "attend_crystal_864", "kind": "attend", "n": 864, "boxes": 1, "radius": 5.9,
         "heads": 8, "kv_heads": 8, "dim": 32, "buckets": 32, "masked": 0.0, "vapour": False,
         "dtype": "bfloat16"},
        # a slab under vapour (lone atoms, empty rows) in single precision, an odd number of
        # atoms, an edge list with a skin whose outer edges are masked
        {"name": "attend_slab_9973_f32", "kind": "attend", "n": 9973, "boxes": 1, "radius": 5.0,
         "heads": 4, "kv_heads": 4, "dim": 32, "buckets": 20, "masked": 0.2, "vapour": True,
         "dtype": "float32"},
        # a condensed-phase box of the size of the vector benchmark, heads of 16
        {"name": "attend_300k", "kind": "attend", "n": 300_007, "boxes": 1, "radius": 6.0,
         "heads": 8, "kv_heads": 8, "dim": 16, "buckets": 32, "masked": 0.0, "vapour": False,
         "dtype": "bfloat16"},
        # four read-out tokens, each over every atom of a large box: few rows, long lists
        {"name": "attend_readout_4", "kind": "attend", "n": 100_000, "boxes": 1, "tokens": 4,
         "heads": 8, "kv_heads": 8, "dim": 32, "buckets": 0, "masked": 0.0, "vapour": False,
         "dtype": "bfloat16"},
        # a training step on a small crystal in single precision
        {"name": "attend_train_864_f32", "kind": "attend_train", "n": 864, "boxes": 1, "radius": 5.9,
         "heads": 4, "kv_heads": 4, "dim": 32, "buckets": 32, "masked": 0.0, "vapour": False,
         "dtype": "float32"},
        # a training batch of 128 small structures
        {"name": "attend_train_batch_128", "kind": "attend_train", "n": 32_000, "boxes": 128,
         "radius": 6.0, "heads": 8, "kv_heads": 8, "dim": 32, "buckets": 32, "masked": 0.0,
         "vapour": False, "dtype": "bfloat16"},
        # a training step on the ordinary box, keys and values shared by four heads each
        {"name": "attend_train_100k_shared", "kind": "attend_train", "n": 100_000, "boxes": 1,
         "radius": 6.0, "heads": 8, "kv_heads": 2, "dim": 32, "buckets": 32, "masked": 0.1,
         "vapour": False, "dtype": "bfloat16"},
        # the atoms of a small crystal by species
        {"name": "group_species_864", "kind": "group", "rows": 864, "groups": 4, "k": 128, "n": 128,
         "skew": 0.5, "empty": 0, "bias": True, "dtype": "bfloat16"},
        # the edges of a training batch by structure, the weights mixed per structure
        {"name": "group_edges_2m", "kind": "group", "rows": 2_200_003, "groups": 128, "k": 128, "n": 128,
         "skew": 0.3, "empty": 0, "bias": False, "dtype": "bfloat16"},
        # a large box by species in single precision, one species absent
        {"name": "group_species_100k_f32", "kind": "group", "rows": 100_000, "groups": 5, "k": 256,
         "n": 256, "skew": 0.7, "empty": 1, "bias": True, "dtype": "float32"},
        # a training step on the atoms of a batch by structure
        {"name": "group_train_batch_128", "kind": "group_train", "rows": 32_000, "groups": 128, "k": 256,
         "n": 512, "skew": 0.3, "empty": 0, "bias": True, "dtype": "bfloat16"},
        # a training step of odd widths in single precision, few groups, some of them empty
        {"name": "group_train_odd_f32", "kind": "group_train", "rows": 9973, "groups": 7, "k": 100,
         "n": 164, "skew": 0.8, "empty": 2, "bias": True, "dtype": "float32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend_train", "attend_train", "group", "group_train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind.startswith("attend"):
        heads, kv = rng.choice([(4, 4), (8, 8), (16, 16), (8, 2), (16, 4), (6, 3)])
        dim = rng.choice([16, 24, 32, 48, 64, 128])
        case = {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "dtype": dtype}
        if kind == "attend" and rng.random() < 0.2:
            case |= {"n": _log_int(rng, 500, 100_000), "boxes": 1, "tokens": rng.randint(1, 8),
                     "buckets": 0, "masked": 0.0, "vapour": False}
            # tokens times atoms times channels within the listed read-out's
            while case["n"] * case["tokens"] * heads * dim > 100_000 * 4 * 256:
                case["n"] = case["n"] // 2 + 1
            return case
        case |= {"radius": round(rng.uniform(2.5, 6.0), 2), "buckets": rng.choice([0, 16, 20, 32, 64]),
                 "masked": rng.choice([0.0, 0.0, 0.2]), "vapour": rng.random() < 0.3}
        case["boxes"] = rng.choice([1, 1, rng.randint(2, 128)])
        # edges times channels within the largest listed case of the kind
        most = 300_007 * 90 * 128 if kind == "attend" else 100_000 * 81 * 256
        per_atom = 0.1 * 4.19 * case["radius"] ** 3 * heads * dim
        case["n"] = _log_int(rng, max(64, 40 * case["boxes"]), max(min(300_000, int(most / per_atom)), 64 * case["boxes"]))
        return case
    most = 2_200_003 * 128 * 128 if kind == "group" else 32_000 * 256 * 512
    if dtype == "float32":
        most = 100_000 * 256 * 256 if kind == "group" else 9973 * 100 * 164 * 4
    k, n = rng.choice([64, 96, 100, 128, 192, 256, 384, 512]), rng.choice([64, 100, 128, 164, 256, 512])
    groups = _log_int(rng, 1, 256)
    rows = _log_int(rng, 200, max(400, most // (k * n)))
    return {"kind": kind, "rows": rows, "groups": groups, "k": k, "n": n, "skew": round(rng.uniform(0, 0.8), 2),
            "empty": rng.randint(0, max(0, groups // 4)), "bias": rng.random() < 0.5, "dtype": dtype}


# ---------------------------------------------------------------- inputs


def _lattice(case, g):
    """Edges (source, target, distance) of jittered lattices with vacancies: ``boxes`` periodic
    cubes at 0.1 atoms per cubic Angstrom, the targets in blocks of 4^3 sites, the atoms numbered
    at random within their box."""
    dev, n, boxes, radius = "cuda", case["n"], case["boxes"], case["radius"]
    # four sites of five are taken; under `vapour` so in the lower half, hardly any in the upper
    share = 0.42 if case["vapour"] else 0.8
    side = max(2, math.ceil((n / boxes / share) ** (1 / 3)))
    sites = side ** 3
    a = (10.0 * n / (boxes * sites) * (2 if case["vapour"] else 1)) ** (1 / 3)
    x = torch.arange(side, device=dev)
    grid = torch.stack(torch.meshgrid(x, x, x, indexing="ij"), -1).reshape(-1, 3)
    nb = -(-side // 4)
    block, inner = grid // 4, grid % 4
    order = torch.argsort((((block[:, 0] * nb + block[:, 1]) * nb + block[:, 2]) * 64
                           + (inner[:, 0] * 4 + inner[:, 1]) * 4 + inner[:, 2]))
    grid = grid[order]
    rank = torch.empty(sites, dtype=torch.long, device=dev)  # of a site in the blocks' order
    rank[order] = torch.arange(sites, device=dev)
    # how likely a site is taken; boxes of a batch are unlike
    fill = torch.rand(boxes, 1, generator=g, device=dev) * 0.5 + 0.5 if boxes > 1 else torch.ones(1, 1, device=dev)
    weight = fill.expand(boxes, sites).clone()
    if case["vapour"]:
        weight[:, grid[:, 2] * 2 >= side] *= 0.03
    score = torch.rand(boxes, sites, generator=g, device=dev) / weight
    taken = torch.zeros(boxes * sites, dtype=torch.bool, device=dev)
    taken[torch.topk(score.reshape(-1), n, largest=False).indices] = True
    site = torch.nonzero(taken).reshape(-1)  # atoms in the order of space
    box, at = site // sites, site % sites
    jitter = (torch.rand(n, 3, generator=g, device=dev) - 0.5) * (0.5 * a)
    # a caller's numbers: random within the box
    key = box.double() + torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    number = torch.empty(n, dtype=torch.long, device=dev)
    number[torch.argsort(key)] = torch.arange(n, device=dev)
    atom = torch.full((boxes * sites,), -1, dtype=torch.long, device=dev)
    atom[site] = torch.arange(n, device=dev)
    r = math.ceil(radius / a + 0.9)
    o = torch.arange(-r, r + 1, device=dev)
    o = torch.stack(torch.meshgrid(o, o, o, indexing="ij"), -1).reshape(-1, 3)
    o = o[(o * o).sum(1).float().sqrt() * a <= radius + 0.87 * a]
    near = (grid[at][:, None, :] + o[None]) % side
    near = rank[(near[..., 0] * side + near[..., 1]) * side + near[..., 2]]
    near = atom[box[:, None] * sites + near]
    d = o[None].float() * a + jitter[near.clamp(min=0)] - jitter[:, None, :]
    d2 = (d * d).sum(-1)
    t, c = torch.nonzero((near >= 0) & (d2 <= radius * radius) & (d2 > 1e-8), as_tuple=True)
    return number[near[t, c]], number[t], d2[t, c].sqrt()


def _attend_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = types.SimpleNamespace(kind=case["kind"], mask=None, table=None, distances=None, boundaries=None)
    if "tokens" in case:  # the tokens come first, then the atoms; a token's list is every atom
        s.targets, s.nodes = case["tokens"], case["tokens"] + case["n"]
        target = torch.arange(s.targets, device="cuda").repeat_interleave(case["n"])
        source = (torch.arange(case["n"], device="cuda") + s.targets).repeat(s.targets)
    else:
        s.targets = s.nodes = case["n"]
        source, target, s.distances = _lattice(case, g)
        if case["masked"]:
            s.mask = s.distances <= case["radius"] * (1 - case["masked"]) ** (1 / 3)
    s.edge_index = torch.stack([source, target])
    dtype, h, kv, d = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s.q, s.k, s.v = rand(s.targets, h, d).to(dtype), rand(s.nodes, kv, d).to(dtype), rand(s.nodes, kv, d).to(dtype)
    if case["buckets"]:
        s.boundaries = torch.linspace(0.0, case["radius"], case["buckets"] + 1, device="cuda")[1:-1].contiguous()
        s.table = rand(case["buckets"], h) * 0.5
    else:
        s.distances = None
    if case["kind"] == "attend_train":
        s.grad = rand(s.targets, h, d).to(dtype)
    return s


def _sizes(case, seed):
    rng = np.random.default_rng(seed)
    w = np.exp(case["skew"] * rng.standard_normal(case["groups"]))
    w[rng.permutation(case["groups"])[:case["empty"]]] = 0.0
    return rng.multinomial(case["rows"], w / w.sum())


def _group_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes = _sizes(case, seed)
    s = types.SimpleNamespace(kind=case["kind"], bias=None, most=int(sizes.max()))
    s.sizes = torch.from_numpy(sizes).cuda()
    dtype, groups, k, n = _TYPES[case["dtype"]], case["groups"], case["k"], case["n"]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s.x, s.weight = rand(case["rows"], k).to(dtype), (rand(groups, n, k) / math.sqrt(k)).to(dtype)
    if case["bias"]:
        s.bias = rand(groups, n).to(dtype)
    if case["kind"] == "group_train":
        s.grad = rand(case["rows"], n).to(dtype)
    return s


def prepare(case, seed):
    attend = case["kind"].startswith("attend")
    s = (_attend_inputs if attend else _group_inputs)(case, seed)
    if s.kind == "attend_train":
        s.leaves = [t for t in (s.q, s.k, s.v, s.table) if t is not None]
    elif s.kind == "group_train":
        s.leaves = [t for t in (s.x, s.weight, s.bias) if t is not None]
    if own:
        from dynamis_amd import dynamis_state

        s.ops = dynamis_state
        for t in getattr(s, "leaves", ()):
            t.requires_grad_(True)
        if attend:  # made once for a list, read by every layer
            s.plan = dynamis_state.neighbor_plan(s.edge_index, s.nodes, s.targets, distances=s.distances,
                                                 boundaries=s.boundaries, edge_mask=s.mask)
    elif attend:
        # the same for the plain form: the edges that are not masked, and their buckets
        kept = s.edge_index if s.mask is None else s.edge_index[:, s.mask]
        s.source, s.target = kept[0].contiguous(), kept[1].contiguous()
        if s.table is not None:
            d = s.distances if s.mask is None else s.distances[s.mask]
            s.bucket = torch.bucketize(d, s.boundaries, right=True)
    return s


# ---------------------------------------------------------------- the operators


def _attend(s):
    """(out, probabilities and what they are made of) in 32 bits."""
    targets, heads, dim = s.q.shape
    per = heads // s.k.shape[1]
    q, k, v = s.q.float(), s.k.float(), s.v.float()
    logits = (q[s.target].unflatten(1, (-1, per)) * k[s.source].unsqueeze(2)).sum(-1).flatten(1) / math.sqrt(dim)
    if s.table is not None:
        logits = logits + s.table[s.bucket]
    rows = s.target[:, None].expand(-1, heads)
    top = torch.full((targets, heads), -torch.inf, device="cuda").scatter_reduce(0, rows, logits, "amax")
    p = torch.exp(logits - top[s.target])
    total = torch.zeros(targets, heads, device="cuda").index_add(0, s.target, p)
    p = p / total[s.target]
    out = torch.zeros(targets, heads, dim, device="cuda")
    out = out.index_add(0, s.target, (p.unflatten(1, (-1, per)).unsqueeze(-1) * v[s.source].unsqueeze(2)).flatten(1, 2))
    return out, p


def _attend_grads(s, out, p):
    targets, heads, dim = s.q.shape
    per = heads // s.k.shape[1]
    q, k, v, grad = s.q.float(), s.k.float(), s.v.float(), s.grad.float()
    delta = (grad * out).sum(-1)
    g = grad[s.target].unflatten(1, (-1, per))  # [edges, kv heads, heads of each, dim]
    ds = p * ((g * v[s.source].unsqueeze(2)).sum(-1).flatten(1) - delta[s.target])
    dv = torch.zeros_like(v).index_add(0, s.source, (p.unflatten(1, (-1, per)).unsqueeze(-1) * g).sum(2))
    del g
    dsg = (ds / math.sqrt(dim)).unflatten(1, (-1, per)).unsqueeze(-1)
    dq = torch.zeros_like(q).index_add(0, s.target, (dsg * k[s.source].unsqueeze(2)).flatten(1, 2))
    dk = torch.zeros_like(k).index_add(0, s.source, (dsg * q[s.target].unflatten(1, (-1, per))).sum(2))
    grads = [dq.to(s.q.dtype), dk.to(s.k.dtype), dv.to(s.v.dtype)]
    if s.table is not None:
        grads.append(torch.zeros_like(s.table).index_add(0, s.bucket, ds))
    return grads


def _group(s):
    """(y, the padded rows, each row's group and place in it) in 32 bits."""
    rows, k = s.x.shape
    groups = s.weight.shape[0]
    group = torch.repeat_interleave(torch.arange(groups, device="cuda"), s.sizes, output_size=rows)
    place = torch.arange(rows, device="cuda") - (torch.cumsum(s.sizes, 0) - s.sizes)[group]
    x = torch.zeros(groups, s.most, k, device="cuda")
    x[group, place] = s.x.float()
    y = torch.bmm(x, s.weight.float().transpose(1, 2).contiguous())[group, place]
    if s.bias is not None:
        y = y + s.bias.float()[group]
    return y, x, group, place


def _group_grads(s, x, group, place):
    g = torch.zeros(s.weight.shape[0], s.most, s.weight.shape[1], device="cuda")
    g[group, place] = s.grad.float()
    grads = [torch.bmm(g, s.weight.float())[group, place].to(s.x.dtype),
             torch.bmm(g.transpose(1, 2).contiguous(), x).to(s.weight.dtype)]
    if s.bias is not None:
        grads.append(g.sum(1).to(s.bias.dtype))
    return grads


def run(s):
    if own:
        if s.kind.startswith("attend"):
            out = s.ops.neighbor_attention(s.q, s.k, s.v, s.plan, s.table)
        else:
            out = s.ops.grouped_linear(s.x, s.weight, s.sizes, s.bias)
        if not s.kind.endswith("train"):
            return out
        return [out.detach(), *torch.autograd.grad(out, s.leaves, s.grad)]
    if s.kind.startswith("attend"):
        out, p = _attend(s)
        if s.kind == "attend":
            return out.to(s.q.dtype)
        return [out.to(s.q.dtype), *_attend_grads(s, out, p)]
    y, x, group, place = _group(s)
    if s.kind == "group":
        return y.to(s.x.dtype)
    return [y.to(s.x.dtype), *_group_grads(s, x, group, place)]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    train = case["kind"].endswith("train")
    if case["kind"].startswith("attend"):
        if "tokens" in case:
            targets, nodes, edges = case["tokens"], case["tokens"] + case["n"], case["tokens"] * case["n"]
        else:
            targets = nodes = case["n"]
            edges = case["n"] * 0.1 * 4 / 3 * math.pi * case["radius"] ** 3 * (1 - case["masked"])
            if case["vapour"]:  # all but a few atoms in half of the box
                edges *= 1.6
        wide, narrow = targets * case["heads"] * case["dim"], nodes * case["kv_heads"] * case["dim"]
        # q and out, k and v, the source and the bucket of each edge; in training the
        # gradient that comes in and those that go out
        moved = size * 2 * (wide + narrow) * (2 if train else 1) + edges * (5 if case["buckets"] else 4)
        return {"bytes": moved, "flops": (14 if train else 4) * edges * case["heads"] * case["dim"]}
    rows, groups, k, n = case["rows"], case["groups"], case["k"], case["n"]
    return {"bytes": size * (rows * (k + n) + groups * k * n) * (2 if train else 1),
            "flops": (6 if train else 2) * rows * k * n}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _attend_exact(case, s):
    """Each target's edges in a padded row, softmax over the row, gradients by differentiation."""
    train = case["kind"] == "attend_train"
    keep = torch.ones_like(s.edge_index[0], dtype=torch.bool) if s.mask is None else s.mask
    source, target = s.edge_index[0][keep], s.edge_index[1][keep]
    order = torch.argsort(target, stable=True)
    source, target = source[order], target[order]
    degree = torch.bincount(target, minlength=s.targets)
    start = torch.cumsum(degree, 0) - degree
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    bucket = None
    if s.table is not None:
        bucket = (s.distances[keep][order][:, None] >= s.boundaries[None]).sum(1)
    q, k, v = s.q.double(), s.k.double(), s.v.double()
    table = None if s.table is None else s.table.double()
    leaves = [t for t in (q, k, v, table) if t is not None]
    sums = [torch.zeros_like(t) for t in leaves] if train else []
    out = torch.zeros(s.targets, heads, dim, dtype=torch.float64, device="cuda")
    widest = max(1, int(degree.max()))
    step = max(1, int(1.5e8 / (widest * heads * dim)))
    for a in range(0, s.targets, step):
        b = min(s.targets, a + step)
        width = max(1, int(degree[a:b].max()))
        slot = start[a:b, None] + torch.arange(width, device="cuda")[None]
        real = torch.arange(width, device="cuda")[None] < degree[a:b, None]
        slot = slot.clamp(max=max(0, source.numel() - 1))
        with torch.set_grad_enabled(train):
            mine = [t.detach().requires_grad_(train) for t in leaves]
            qq, kk, vv = mine[0][a:b], mine[1], mine[2]
            idx = source[slot].reshape(-1)
            keys = torch.index_select(kk, 0, idx).reshape(b - a, width, kv, dim).repeat_interleave(heads // kv, 2)
            values = torch.index_select(vv, 0, idx).reshape(b - a, width, kv, dim).repeat_interleave(heads // kv, 2)
            logits = (keys * qq[:, None]).sum(-1) / math.sqrt(dim)
            if table is not None:
                logits = logits + mine[3][bucket[slot]]
            logits = logits.masked_fill(~real[..., None], -1e300)
            p = torch.softmax(logits, 1).masked_fill(~real[..., None], 0.0)
            o = (p[..., None] * values).sum(1)
            out[a:b] = o.detach()
            if train:
                for total, grad in zip(sums, torch.autograd.grad(o, mine, s.grad[a:b].double())):
                    total += grad
    return [out, *sums] if train else out


def _group_exact(case, s, sizes):
    train = case["kind"] == "group_train"
    x, w = s.x.double(), s.weight.double()
    y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.zeros_like(w), torch.zeros(w.shape[:2], dtype=torch.float64, device="cuda")
    a = 0
    for i, size in enumerate(sizes.tolist()):
        b = a + size
        y[a:b] = x[a:b] @ w[i].T
        if s.bias is not None:
            y[a:b] += s.bias[i].double()
        if train:
            g = s.grad[a:b].double()
            dx[a:b], dw[i], db[i] = g @ w[i], g.T @ x[a:b], g.sum(0)
        a = b
    if not train:
        return y
    return [y, dx, dw] + ([db] if s.bias is not None else [])


def exact(case, seed):
    if case["kind"].startswith("attend"):
        return _attend_exact(case, _attend_inputs(case, seed))
    return _group_exact(case, _group_inputs(case, seed), _sizes(case, seed))
