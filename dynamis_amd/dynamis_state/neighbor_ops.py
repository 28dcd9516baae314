"""What a model runs on a built neighbour list: attention of every atom over its neighbours
with a learned bias by distance, and linear maps whose weights go by group.

    ei, _, nn, _, vec, dist = impl.radius_graph_pbc_vectors(pos, cell, pbc, 6.0)
    plan = neighbor_plan(ei, num_nodes=len(pos), distances=dist, boundaries=edges)
    y = grouped_linear(x, weight, sizes)                  # rows by structure, species, expert
    out = neighbor_attention(q, k, v, plan, bias_table)   # differentiable in q, k, v, bias_table

No counterpart in the reference, whose force models bring their own layers.  The kernels are
those of libdynamis_graph.so (dg_neighbors_*, dg_attention_*, dg_grouped_*); there is no CPU
path.  Everything runs on the current stream; tensors follow torch's rules for streams, and a
plan made on one stream may be read on another once the caller has ordered the two.

Distances enter by their buckets alone, so positions get no gradient through these operators: forces
as the derivative of an energy need a term that depends on them smoothly beside it.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from .. import _lib as L
from .dynamis_state_impl import _check, _shape, sfc_order

_DTYPES = {torch.float32: L.DG_F32, torch.bfloat16: L.DG_BF16}


class _Rows:
    """One direction's index lists, as the kernels take them."""

    def __init__(self, order, ptr, idx, bucket):
        self.order, self.ptr, self.idx, self.bucket = order, ptr, idx, bucket
        self.items = self.item_first = self.long_slot = None
        c = self.c = L.NeighborLists()
        c.n_rows = order.numel()
        c.order, c.ptr, c.idx = order.data_ptr(), ptr.data_ptr(), idx.data_ptr()
        c.bucket = bucket.data_ptr() if bucket is not None else None
        self.byref = ctypes.byref(c)

    def split(self, long_rows, long_entries, stream):
        """Rows above DG_NEIGHBOR_SPLIT entries in parts: as many as the card holds waves for two
        groups of heads (4 rows of 100,000: 62 us with 768 parts to 4096, the join of them 7 us and
        more the more there are), at least 128 entries (a part's result costs as much as some)."""
        if not long_rows:
            return
        lib, dev, c = L.lib(), self.ptr.device, self.c
        chunk = min(2048, max(128, (-(-long_entries // 1536) + 31) // 32 * 32))
        c.n_items, c.n_long = long_entries // chunk + long_rows, long_rows
        new = lambda *n: torch.empty(n, dtype=torch.int32, device=dev)  # noqa: E731
        self.items, self.item_first, self.long_slot = new(c.n_items, 4), new(c.n_rows + 1), new(long_rows)
        c.items, c.item_first = self.items.data_ptr(), self.item_first.data_ptr()
        c.long_slot = self.long_slot.data_ptr()
        wsb = lib.dg_neighbors_parts_workspace_size(c.n_rows)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        L.check(lib.dg_neighbors_parts(L.ptr(self.order), L.ptr(self.ptr), c.n_rows, chunk, c.n_items, long_rows,
                                       L.ptr(self.item_first), L.ptr(self.items), L.ptr(self.long_slot), L.ptr(ws), wsb,
                                       stream), "neighbor_plan")

    def tensors(self):
        lists = self.order, self.ptr, self.idx, self.bucket, self.items, self.item_first, self.long_slot
        return [t for t in lists if t is not None]


class NeighborPlan:
    """Index lists of a graph for ``neighbor_attention`` (see ``neighbor_plan``).

    num_nodes, num_targets, num_edges (those kept), num_buckets (0: made without distances),
    symmetric (the lists by source are those by target)."""

    def __init__(self, device, num_nodes, num_targets, num_edges, num_buckets, by_target, by_source, symmetric):
        self.device = device
        self.num_nodes, self.num_targets = num_nodes, num_targets
        self.num_edges, self.num_buckets = num_edges, num_buckets
        self.by_target, self.by_source, self.symmetric = by_target, by_source, symmetric
        self._stream = L.raw_stream(device)

    def _use(self, stream):
        """Keeps the lists' memory from being handed out again while another stream reads it."""
        if stream != self._stream:
            self.record_stream(torch.cuda.current_stream(self.device))

    def record_stream(self, stream):
        for rows in {id(r): r for r in (self.by_target, self.by_source) if r is not None}.values():
            for t in rows.tensors():
                t.record_stream(stream)


def neighbor_plan(edge_index, num_nodes, num_targets=None, distances=None, boundaries=None, edge_mask=None,
                  backward=True):
    """Index lists of an edge list, made once and read by every layer.

    edge_index [2, E] int64 (sources, targets) as the builders here return it.  Nodes are
    [0, num_nodes), targets [0, num_targets) (default: all nodes; a rank's own atoms come first,
    then its ghosts).  Edges of a target need not be together, but then they are sorted first.
    distances [E] with boundaries [B - 1], ascending and of the same type, put an edge into
    bucket #{boundaries <= distance} of B <= 128.  edge_mask [E] bool leaves edges out (a list
    with a skin, cut to the radius).  backward=False leaves out the lists that only gradients
    need.  E <= 2^31 - 256.

    A plan costs as much as several calls and more (864 atoms, 74,000 edges: 115 us; 300,000 atoms, 26.5M
    edges: 0.47 ms, and 2.2 ms with lists by source that are not those by target).  It synchronises the
    host once; once more where the lists by source have to be sorted, which a mask or boundaries that
    part an edge from its opposite bring about; and once more where the edges have to be sorted.
    """
    _check(isinstance(edge_index, torch.Tensor) and edge_index.is_cuda, "edge_index must be a CUDA tensor")
    _check(edge_index.dim() == 2 and edge_index.size(0) == 2,
           f"edge_index must have shape [2, E], got {_shape(edge_index)}")
    _check(edge_index.dtype == torch.int64, f"edge_index must be int64, got {edge_index.dtype}")
    dev, E = edge_index.device, edge_index.size(1)
    num_nodes = int(num_nodes)
    num_targets = num_nodes if num_targets is None else int(num_targets)
    _check(0 <= num_targets <= num_nodes, f"num_targets must be in [0, num_nodes], got {num_targets}")
    n_bounds = 0
    if distances is not None:
        _check(isinstance(distances, torch.Tensor), "distances must be a tensor")
        _check(distances.device == dev and distances.dim() == 1 and distances.size(0) == E,
               f"distances must have shape [{E}] on {dev}, got {_shape(distances)} on {distances.device}")
        _check(distances.dtype in (torch.float32, torch.float64),
               f"distances must be float32 or float64, got {distances.dtype}")
        _check(boundaries is not None, "distances come with boundaries")
        boundaries = torch.as_tensor(boundaries, dtype=distances.dtype, device=dev).contiguous()
        _check(boundaries.dim() == 1, f"boundaries must be 1-D, got {_shape(boundaries)}")
        n_bounds = boundaries.numel()
        _check(n_bounds <= 127, f"at most 127 boundaries (128 buckets), got {n_bounds}")
        distances = distances.detach().contiguous()
    else:
        _check(boundaries is None, "boundaries come with distances")
    if edge_mask is not None:
        _check(isinstance(edge_mask, torch.Tensor), "edge_mask must be a tensor")
        _check(edge_mask.device == dev and edge_mask.dtype == torch.bool and edge_mask.dim() == 1
               and edge_mask.size(0) == E, f"edge_mask must be bool [{E}] on {dev}")
        edge_mask = edge_mask.contiguous()
    lib = L.lib()
    edge_index = edge_index.contiguous()
    d = L.NeighborDesc(E, num_nodes, num_targets, n_bounds,
                       L.DG_F64 if distances is not None and distances.dtype == torch.float64 else L.DG_F32)
    wsb = lib.dg_neighbors_workspace_size(d)
    if wsb == 0:
        raise RuntimeError(f"neighbor_plan: {lib.dg_last_error().decode()}")
    with torch.cuda.device(dev):
        s = L.stream_of(dev)
        pad = L.DG_NEIGHBOR_PAD
        new = lambda n, t=torch.int32: torch.empty(n, dtype=t, device=dev)  # noqa: E731
        ws, order, ptr, idx = new(wsb, torch.uint8), new(num_nodes), new(num_nodes + 1), new(E + pad)
        bucket = new(E + pad, torch.uint8) if distances is not None else None
        base = edge_index.data_ptr()
        L.check(lib.dg_neighbors_by_target(d, ctypes.c_void_p(base), ctypes.c_void_p(base + 8 * E), L.ptr(edge_mask),
                                           L.ptr(distances), L.ptr(boundaries), L.ptr(order), L.ptr(ptr), L.ptr(idx),
                                           L.ptr(bucket), int(backward), L.ptr(ws), wsb, s), "neighbor_plan")
        t = L.NeighborTotals()
        L.check(lib.dg_neighbors_read_totals(d, L.ptr(ws), t, s), "neighbor_plan")
        if not t.grouped:
            perm = sfc_order(edge_index[1].contiguous())
            return neighbor_plan(edge_index[:, perm], num_nodes, num_targets,
                                 None if distances is None else distances[perm], boundaries,
                                 None if edge_mask is None else edge_mask[perm], backward)
        by_target = _Rows(order, ptr, idx, bucket)
        by_target.split(t.long_rows, t.long_entries, s)
        by_source, n = None, t.n_entries
        symmetric = bool(backward and t.symmetric)
        if symmetric:
            by_source = by_target
        elif backward:
            sptr, sidx = new(num_nodes + 1), new(n + pad)
            sbucket = new(n + pad, torch.uint8) if bucket is not None else None
            sort_bytes = lib.dg_neighbors_sort_workspace_size(n)
            sort_ws = new(sort_bytes, torch.uint8)
            L.check(lib.dg_neighbors_by_source(d, n, L.ptr(idx), L.ptr(bucket), L.ptr(sptr), L.ptr(sidx),
                                               L.ptr(sbucket), L.ptr(ws), wsb, L.ptr(sort_ws), sort_bytes, s),
                    "neighbor_plan")
            L.check(lib.dg_neighbors_read_totals(d, L.ptr(ws), t, s), "neighbor_plan")
            by_source = _Rows(order, sptr, sidx, sbucket)
            by_source.split(t.long_rows, t.long_entries, s)
        return NeighborPlan(dev, num_nodes, num_targets, n, n_bounds + 1 if bucket is not None else 0, by_target,
                            by_source, symmetric)


def _rows_16(t):
    """t [n, heads, dim] as it is if its rows are whole, start at 16 bytes and lie a multiple of
    16 bytes apart; else a copy."""
    row, head, one = t.stride()
    step = 16 // t.element_size()
    if one == 1 and (t.size(1) == 1 or head == t.size(2)) and row % step == 0 and row >= 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _new_like(t):
    """A contiguous tensor like t."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _workspace(lib, d, to, fro, dev):
    wsb = lib.dg_attention_workspace_size(d, to, fro)
    if wsb == 0:
        raise RuntimeError(f"neighbor_attention: {lib.dg_last_error().decode()}")
    return torch.empty(wsb, dtype=torch.uint8, device=dev), wsb


def _forward(q, k, v, table, plan, scale, want_lse, ctx=None):
    lib, dev = L.lib(), plan.device
    q, k, v = _rows_16(q), _rows_16(k), _rows_16(v)
    if table is not None:
        table = table.contiguous()
    targets, heads, dim = q.shape
    dtype = q.dtype
    d = L.AttentionDesc(targets, plan.num_nodes, q.stride(0), k.stride(0), v.stride(0), 0, heads, k.size(1), dim,
                        0 if table is None else table.size(0), _DTYPES[dtype], scale)
    rows = plan.by_target
    with L.on_device(dev):
        stream = L.raw_stream(dev)
        plan._use(stream)
        out = torch.empty((targets, heads, dim), dtype=dtype, device=dev)
        out32 = norm = lse = ws = None
        wsb = 0
        if ctx is not None:
            norm = torch.empty((targets, heads, 2), dtype=torch.float32, device=dev)
            if dtype != torch.float32:
                out32 = torch.empty((targets, heads, dim), dtype=torch.float32, device=dev)
        if want_lse:
            lse = torch.empty((targets, heads), dtype=torch.float32, device=dev)
        if rows.c.n_items:  # (partial results of long rows are all that the forward pass keeps there)
            ws, wsb = _workspace(lib, d, rows.byref, None, dev)
        addr = L.addr
        status = lib.dg_attention_forward(d, rows.byref, q.data_ptr(), k.data_ptr(), v.data_ptr(), addr(table),
                                          out.data_ptr(), addr(out32), addr(norm), addr(lse), addr(ws), wsb, stream)
        if status:
            L.check(status, "neighbor_attention")
    if ctx is not None:
        # (the backward pass runs on a thread of its own, where each host instruction costs twice:
        # it takes over what is worked out here)
        ctx.save_for_backward(q, k, v, table, out if out32 is None else out32, norm)
        ctx.desc, ctx.plan = d, plan
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, plan, scale, want_lse):
        out, lse = _forward(q, k, v, table, plan, scale, want_lse, ctx)
        if lse is not None:
            ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _grad_lse):
        q, k, v, table, out32, norm = ctx.saved_tensors
        plan, lib = ctx.plan, L.lib()
        dev = plan.device
        if plan.by_source is None:
            raise RuntimeError("neighbor_attention: the plan was made with backward=False")
        grad = _rows_16(grad)
        # (its own: another backward pass of the same graph may be under way with another stride)
        d = L.AttentionDesc.from_buffer_copy(ctx.desc)
        d.ld_g = grad.stride(0)
        to, fro = plan.by_target.byref, plan.by_source.byref
        with L.on_device(dev):
            stream = L.raw_stream(dev)
            plan._use(stream)
            dq, dk, dv = _new_like(q), _new_like(k), _new_like(v)
            dtable = torch.empty_like(table) if table is not None else None
            ws, wsb = _workspace(lib, d, to, fro, dev)
            addr = L.addr
            status = lib.dg_attention_backward(d, to, fro, q.data_ptr(), k.data_ptr(), v.data_ptr(), addr(table),
                                               out32.data_ptr(), norm.data_ptr(), grad.data_ptr(), dq.data_ptr(),
                                               dk.data_ptr(), dv.data_ptr(), addr(dtable), ws.data_ptr(), wsb, stream)
            if status:
                L.check(status, "neighbor_attention")
        return dq, dk, dv, dtable, None, None, None


def _refuse_tangents(name, *tensors):
    """Called at a level of forward-mode differentiation, where a tensor may carry a tangent without
    requiring a gradient: a result without one would be a derivative of zero."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


def _check_attention(q, k, v, plan, bias_table):
    """The refusals of neighbor_attention, with their messages."""
    _check(isinstance(plan, NeighborPlan), "plan must be a NeighborPlan")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
        _check(t.dim() == 3, f"{name} must have shape [nodes, heads, dim], got {_shape(t)}")
        _check(t.device == plan.device, f"{name} must be on the plan's device {plan.device}, got {t.device}")
        _check(t.dtype in _DTYPES, f"{name} must be float32 or bfloat16, got {t.dtype}")
        _check(t.dtype == q.dtype, f"q, k and v must have one dtype, got {q.dtype} and {t.dtype}")
        _check(t.size(2) == q.size(2), f"q, k and v must have one head width, got {q.size(2)} and {t.size(2)}")
    _check(q.size(0) == plan.num_targets, f"q must have {plan.num_targets} rows, got {q.size(0)}")
    _check(k.size(0) == plan.num_nodes and v.shape == k.shape,
           f"k and v must have {plan.num_nodes} rows and one shape, got {_shape(k)} and {_shape(v)}")
    heads, kv, dim = q.size(1), k.size(1), q.size(2)
    _check(heads >= 1 and kv >= 1 and heads % kv == 0, f"heads ({heads}) must be a multiple of kv_heads ({kv})")
    _check(heads <= 1024, f"at most 1024 heads, got {heads}")
    _check(8 <= dim <= 256 and dim % 8 == 0, f"the head width must be a multiple of 8, 8 to 256, got {dim}")
    if bias_table is not None:
        _check(isinstance(bias_table, torch.Tensor), "bias_table must be a tensor")
        _check(plan.num_buckets > 0, "bias_table needs a plan with distances")
        _check(bias_table.device == plan.device and bias_table.is_floating_point()
               and tuple(bias_table.shape) == (plan.num_buckets, heads),
               f"bias_table must be floating [{plan.num_buckets}, {heads}] on {plan.device}, got {_shape(bias_table)}")
        _check(bias_table.numel() <= 4096, f"bias_table must hold at most 4096 entries, got {bias_table.numel()}")


def _attention_is_fine(q, k, v, plan, bias_table):
    """Whether _check_attention would pass, without its messages' host time."""
    if not (type(q) in _TENSORS and type(k) in _TENSORS and type(v) in _TENSORS and q.dim() == 3 and k.dim() == 3
            and type(plan) is NeighborPlan and (bias_table is None or type(bias_table) in _TENSORS)):
        return False
    (targets, heads, dim), (nodes, kv, kdim) = q.shape, k.shape
    dtype, dev = q.dtype, plan.device
    return (targets == plan.num_targets and nodes == plan.num_nodes and dim == kdim and v.shape == k.shape
            and dtype in _DTYPES and k.dtype == dtype and v.dtype == dtype
            and q.device == dev and k.device == dev and v.device == dev
            and 1 <= heads <= 1024 and kv >= 1 and heads % kv == 0 and 8 <= dim <= 256 and dim % 8 == 0
            and (bias_table is None
                 or bias_table.dtype == torch.float32 and bias_table.device == dev and plan.num_buckets > 0
                 and bias_table.shape == (plan.num_buckets, heads) and plan.num_buckets * heads <= 4096))


_TENSORS = (torch.Tensor, torch.nn.Parameter)


def neighbor_attention(q, k, v, plan, bias_table=None, scale=None, return_lse=False):
    """Attention of every target over the sources of its edges.

      logit[e, h] = scale <q[t, h], k[s, h // (heads // kv_heads)]> + bias_table[bucket(e), h]
      out[t, h]   = sum_e softmax_e(logit)[e, h] v[s, h // (heads // kv_heads)]

    q [num_targets, heads, dim], k and v [num_nodes, kv_heads, dim], float32 or bfloat16; heads a
    multiple of kv_heads, dim a multiple of 8 up to 256; any strides (rows that are whole and
    start at 16 bytes are read in place).  bias_table [plan.num_buckets, heads], at most 4096
    entries, used in float32; an entry of -inf takes its edges out for that head, whatever q, k
    and v hold there.  scale defaults to dim ** -0.5.  A target without edges gives zeros (and a
    log-sum of -inf).  Returns out like q, and with return_lse also the natural log-sums
    [num_targets, heads] in float32 (not differentiable).

    What is not finite shows in the head that reads it and in no other, as the formulas have it.

    Differentiable in q, k, v and bias_table (once, in reverse: a tensor with a forward-mode tangent
    is refused); all four gradients are formed, whichever are asked for.  All sums are float32, in a fixed order:
    results repeat bit for bit.
    """
    if forward_ad._current_level >= 0:  # (unpack_dual itself takes half a microsecond a tensor)
        _refuse_tangents("neighbor_attention", q, k, v, bias_table)
    if not _attention_is_fine(q, k, v, plan, bias_table):
        _check_attention(q, k, v, plan, bias_table)
        if bias_table is not None:
            bias_table = bias_table.float()
    if scale is None:
        scale = q.size(2) ** -0.5
    elif not math.isfinite(scale):
        raise RuntimeError(f"scale must be finite, got {scale}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or bias_table is not None and bias_table.requires_grad):
        out, lse = _Attention.apply(q, k, v, bias_table, plan, float(scale), return_lse)
    else:
        out, lse = _forward(q, k, v, bias_table, plan, float(scale), return_lse)
    return (out, lse) if return_lse else out


def _grouped_desc(x, weight):
    return L.GroupedDesc(x.size(0), weight.size(0), weight.size(2), weight.size(1), _DTYPES[x.dtype], 0)


def _grouped_forward(x, weight, sizes, bias):
    dev = x.device
    with L.on_device(dev):
        y = torch.empty((x.size(0), weight.size(1)), dtype=x.dtype, device=dev)
        status = L.lib().dg_grouped_forward(_grouped_desc(x, weight), x.data_ptr(), weight.data_ptr(), sizes.data_ptr(),
                                            L.addr(bias), y.data_ptr(), L.raw_stream(dev))
        if status:
            L.check(status, "grouped_linear")
    return y


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, sizes, bias):
        ctx.save_for_backward(x, weight, sizes)
        ctx.desc = _grouped_desc(x, weight)
        return _grouped_forward(x, weight, sizes, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, sizes = ctx.saved_tensors
        need_x, need_w, _, need_b = ctx.needs_input_grad
        lib, dev, grad = L.lib(), x.device, grad.contiguous()
        d = ctx.desc
        with L.on_device(dev):
            dx = torch.empty_like(x) if need_x else None
            dw = torch.empty_like(weight) if need_w or need_b else None
            db = torch.empty(weight.shape[:2], dtype=x.dtype, device=dev) if need_b else None
            wsb = lib.dg_grouped_workspace_size(d) if dw is not None else 0
            ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
            addr = L.addr
            status = lib.dg_grouped_backward(d, x.data_ptr(), weight.data_ptr(), sizes.data_ptr(), grad.data_ptr(),
                                             addr(dx), addr(dw), addr(db), addr(ws), wsb, L.raw_stream(dev))
            if status:
                L.check(status, "grouped_linear")
        return dx, dw if need_w else None, None, db


def _check_grouped(x, weight, sizes, bias):
    """The refusals of grouped_linear, with their messages."""
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a CUDA tensor")
    _check(x.dim() == 2, f"x must have shape [rows, k], got {_shape(x)}")
    _check(x.dtype in _DTYPES, f"x must be float32 or bfloat16, got {x.dtype}")
    _check(isinstance(weight, torch.Tensor) and weight.device == x.device, f"weight must be on {x.device}")
    _check(weight.dim() == 3 and weight.size(2) == x.size(1),
           f"weight must have shape [groups, n, {x.size(1)}], got {_shape(weight)}")
    _check(weight.dtype == x.dtype, f"weight must be {x.dtype}, got {weight.dtype}")
    groups = weight.size(0)
    _check(1 <= groups <= 1 << 20, f"weight must hold 1 to 2^20 groups, got {groups}")
    _check(1 <= x.size(1) <= 1 << 20 and 1 <= weight.size(1) <= 1 << 20, "the widths must be 1 to 2^20")
    _check(sizes.dim() == 1 and sizes.size(0) == groups and sizes.dtype == torch.int64,
           f"sizes must be int64 [{groups}], got {sizes.dtype} {_shape(sizes)}")
    if sizes.is_cuda:
        _check(sizes.device == x.device, f"sizes must be on {x.device}")
    else:
        _check(bool((sizes >= 0).all()) and int(sizes.sum()) == x.size(0),
               f"sizes must be non-negative and add up to {x.size(0)} rows")
    if bias is not None:
        _check(isinstance(bias, torch.Tensor), "bias must be a tensor")
        _check(bias.device == x.device and bias.dtype == x.dtype and tuple(bias.shape) == tuple(weight.shape[:2]),
               f"bias must be {x.dtype} [{groups}, {weight.size(1)}] on {x.device}, got {bias.dtype} {_shape(bias)}")


def _grouped_is_fine(x, weight, sizes, bias):
    """Whether _check_grouped would pass for tensors on one device, without its messages' host time."""
    if not (type(x) in _TENSORS and type(weight) in _TENSORS and x.dim() == 2 and weight.dim() == 3 and x.is_cuda
            and (bias is None or type(bias) in _TENSORS)):
        return False
    groups, n, k = weight.shape
    dev, dtype = x.device, x.dtype
    return (x.size(1) == k and 1 <= groups <= 1 << 20 and 1 <= k <= 1 << 20 and 1 <= n <= 1 << 20
            and dtype in _DTYPES and weight.dtype == dtype and weight.device == dev
            and sizes.device == dev and sizes.dtype == torch.int64 and sizes.shape == (groups,)
            and (bias is None or bias.dtype == dtype and bias.device == dev and bias.shape == (groups, n)))


def grouped_linear(x, weight, sizes, bias=None):
    """Linear maps by group over ragged rows: y[i] = weight[g(i)] @ x[i] + bias[g(i)].

    x [rows, k], weight [groups, n, k] (torch.nn.Linear's layout for each group), bias
    [groups, n]; float32 or bfloat16, one type.  sizes [groups] int64: the first sizes[0] rows are
    group 0's, the next sizes[1] group 1's and so on -- ``num_neighbors_image`` for rows per edge
    of a batch, its ``natoms`` for rows per atom.  On the device (no synchronisation) rows behind
    the last group give zeros and sizes are not checked otherwise; on the host, or as a list, they
    have to be non-negative and to add up to the rows.  Groups may be empty.  The weight's gradient reads
    all sizes once for each group and 128 x 128 of its weight: its time grows with the square of
    the groups (of one such tile: 4,096 groups 0.26 ms, 65,536 groups 45 ms).

    Differentiable in x, weight and bias (once, in reverse: a tensor with a forward-mode tangent is
    refused).  Sums are float32, in a fixed order: results
    repeat bit for bit.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents("grouped_linear", x, weight, bias)
    if not isinstance(sizes, torch.Tensor):
        sizes = torch.as_tensor(sizes)
    if not _grouped_is_fine(x, weight, sizes, bias):
        _check_grouped(x, weight, sizes, bias)
        sizes = sizes.to(x.device)
    x, weight, sizes = x.contiguous(), weight.contiguous(), sizes.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias is not None and bias.requires_grad):
        return _Grouped.apply(x, weight, sizes, bias)
    return _grouped_forward(x, weight, sizes, bias)
