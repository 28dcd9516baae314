"""The steps of a transformer layer around ``neighbor_attention`` and ``grouped_linear``: heads
normalised and rotated by the atoms' positions, rows routed to experts, taken into their order and
back.

    q, k = rotate_heads(q, k, positions, frequencies)     # before neighbor_attention

No counterpart in the reference.  The kernels are those of libdynamis_graph.so (dg_rotate_*); there
is no CPU path.  Everything runs on the current stream without synchronising the host and can be
captured in a HIP graph; tensors follow torch's rules for streams.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from .. import _lib as L
from .dynamis_state_impl import _check, _shape
from .neighbor_ops import _DTYPES, _TENSORS, _new_like, _refuse_tangents, _rows_16

_POSITIONS = {torch.float32: L.DG_F32, torch.float64: L.DG_F64, torch.int64: L.DG_I64}


@functools.lru_cache(maxsize=64)
def _sections(sections):
    return (ctypes.c_int32 * 8)(*sections)


def _rotate_desc(q, k, axes, sections, weight, norm, eps, interleaved, pos_dtype):
    dtype = _DTYPES[q.dtype]
    return L.RotateDesc(q.size(0), k.size(0), q.stride(0), k.stride(0), 0, 0, q.size(1), k.size(1), q.size(2), axes,
                        _sections(sections), dtype, dtype if weight is None else _DTYPES[weight.dtype],
                        _POSITIONS[pos_dtype], norm, interleaved, eps)


def _rotate_forward(q, k, positions, frequencies, q_weight, k_weight, sections, eps, norm, interleaved):
    q, k, dev = _rows_16(q), _rows_16(k), q.device
    d = _rotate_desc(q, k, positions.size(1), sections, q_weight if k_weight is None else k_weight, norm, eps, interleaved,
                     positions.dtype)
    with L.on_device(dev):
        q_out, k_out = _new_like(q), _new_like(k)
        status = L.lib().dg_rotate_forward(d, q.data_ptr(), k.data_ptr(), positions.data_ptr(), frequencies.data_ptr(),
                                           L.addr(q_weight), L.addr(k_weight), q_out.data_ptr(), k_out.data_ptr(),
                                           L.raw_stream(dev))
        if status:
            L.check(status, "rotate_heads")
    return q, k, d, q_out, k_out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, q_weight, k_weight, *how):
        q, k, ctx.desc, q_out, k_out = _rotate_forward(q, k, positions, frequencies, q_weight, k_weight, *how)
        ctx.save_for_backward(q, k, positions, frequencies, q_weight, k_weight)
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, positions, frequencies, q_weight, k_weight = ctx.saved_tensors
        _, _, need_positions, _, need_qw, need_kw = ctx.needs_input_grad[:6]
        lib, dev = L.lib(), q.device
        grad_q, grad_k = _rows_16(grad_q), _rows_16(grad_k)
        # (its own: another backward pass of the same graph may be under way with other strides)
        d = L.RotateDesc.from_buffer_copy(ctx.desc)
        d.ld_gq, d.ld_gk = grad_q.stride(0), grad_k.stride(0)
        with L.on_device(dev):
            dq, dk = _new_like(q), _new_like(k)
            dpos = torch.empty_like(positions) if need_positions else None
            dqw = torch.empty_like(q_weight) if need_qw else None
            dkw = torch.empty_like(k_weight) if need_kw else None
            wsb = lib.dg_rotate_workspace_size(d) if need_qw or need_kw else 0
            ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
            addr = L.addr
            status = lib.dg_rotate_backward(d, q.data_ptr(), k.data_ptr(), positions.data_ptr(), frequencies.data_ptr(),
                                            addr(q_weight), addr(k_weight), grad_q.data_ptr(), grad_k.data_ptr(),
                                            dq.data_ptr(), dk.data_ptr(), addr(dpos), addr(dqw), addr(dkw), addr(ws), wsb,
                                            L.raw_stream(dev))
            if status:
                L.check(status, "rotate_heads")
        return dq, dk, dpos, None, dqw, dkw, None, None, None, None


def _check_rotate(q, k, positions, frequencies, q_weight, k_weight, norm):
    """The refusals of rotate_heads, with their messages."""
    for name, t in (("q", q), ("k", k)):
        _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
        _check(t.dim() == 3, f"{name} must have shape [nodes, heads, dim], got {_shape(t)}")
        _check(t.device == q.device, f"{name} must be on {q.device}, got {t.device}")
        _check(t.dtype in _DTYPES, f"{name} must be float32 or bfloat16, got {t.dtype}")
        _check(t.dtype == q.dtype, f"q and k must have one dtype, got {q.dtype} and {t.dtype}")
        _check(t.size(2) == q.size(2), f"q and k must have one head width, got {q.size(2)} and {t.size(2)}")
        _check(1 <= t.size(1) <= 1024, f"{name} must have 1 to 1024 heads, got {t.size(1)}")
    nodes, dim, dev = k.size(0), q.size(2), q.device
    _check(8 <= dim <= 256 and dim % 8 == 0, f"the head width must be a multiple of 8, 8 to 256, got {dim}")
    _check(q.size(0) <= nodes, f"q must have at most k's {nodes} rows, got {q.size(0)}")
    _check(isinstance(positions, torch.Tensor) and positions.device == dev, f"positions must be a tensor on {dev}")
    _check(positions.dim() in (1, 2) and positions.size(0) == nodes,
           f"positions must have shape [{nodes}] or [{nodes}, axes], got {_shape(positions)}")
    _check(positions.dtype in _POSITIONS, f"positions must be float32, float64 or int64, got {positions.dtype}")
    _check(positions.dim() == 1 or 1 <= positions.size(1) <= 8, f"positions must have 1 to 8 axes, got {_shape(positions)}")
    _check(isinstance(frequencies, torch.Tensor) and frequencies.device == dev, f"frequencies must be a tensor on {dev}")
    _check(frequencies.dim() == 1 and 1 <= frequencies.size(0) <= dim // 2,
           f"frequencies must hold 1 to {dim // 2} pairs, got {_shape(frequencies)}")
    _check(frequencies.dtype == torch.float32, f"frequencies must be float32, got {frequencies.dtype}")
    _check(not (frequencies.requires_grad and torch.is_grad_enabled()), "frequencies have no gradient here: detach them")
    types = set()
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            _check(bool(norm), f"{name} comes with norm")
            _check(isinstance(t, torch.Tensor) and t.device == dev and t.shape == (dim,)
                   and t.dtype in (torch.float32, q.dtype), f"{name} must be float32 or {q.dtype} [{dim}] on {dev}")
            types.add(t.dtype)
    _check(len(types) < 2, "q_weight and k_weight must have one dtype")


def _rotate_is_fine(q, k, positions, frequencies, q_weight, k_weight, norm):
    """Whether _check_rotate would pass, without its messages' host time."""
    if not (type(q) in _TENSORS and type(k) in _TENSORS and type(positions) in _TENSORS and type(frequencies) in _TENSORS
            and q.dim() == 3 and k.dim() == 3 and positions.dim() == 2 and frequencies.dim() == 1 and q.is_cuda):
        return False
    (targets, heads, dim), (nodes, kv, kdim) = q.shape, k.shape
    dtype, dev = q.dtype, q.device
    if q_weight is not None or k_weight is not None:
        if not (norm and type(q_weight) in _TENSORS and type(k_weight) in _TENSORS):
            return False
        wtype = q_weight.dtype
        if not (k_weight.dtype == wtype and (wtype == dtype or wtype == torch.float32) and q_weight.shape == (dim,)
                and k_weight.shape == (dim,) and q_weight.device == dev and k_weight.device == dev):
            return False
    at = positions.shape
    return (targets <= nodes and dim == kdim and 8 <= dim <= 256 and dim % 8 == 0 and 1 <= heads <= 1024 and 1 <= kv <= 1024
            and dtype in _DTYPES and k.dtype == dtype and k.device == dev and positions.device == dev
            and at[0] == nodes and 1 <= at[1] <= 8 and positions.dtype in _POSITIONS
            and frequencies.device == dev and 1 <= frequencies.size(0) <= dim // 2 and frequencies.dtype == torch.float32
            and not frequencies.requires_grad)


def rotate_heads(q, k, positions, frequencies, sections=None, q_weight=None, k_weight=None, eps=1e-6, norm=True,
                 interleaved=False):
    """Queries and keys, each head normalised and rotated by angles that go with its atom's position.

      n        = x / sqrt(mean(x ** 2) + eps) * weight         over a head's channels (norm=False: n = x)
      theta[j] = positions[i, axis(j)] * frequencies[j]
      y[a]     = n[a] cos(theta[j]) - n[b] sin(theta[j])
      y[b]     = n[a] sin(theta[j]) + n[b] cos(theta[j])       (a, b) = (j, j + P), interleaved: (2 j, 2 j + 1)

    q [targets, heads, dim] and k [nodes, kv_heads, dim], float32 or bfloat16, any strides (rows
    that are whole and start at 16 bytes are read in place), dim a multiple of 8 up to 256; row i of both
    belongs to atom i, and q may have fewer rows (a rank's own atoms come first, then its ghosts).
    positions [nodes, axes] (or [nodes]: one axis), float32, float64 or int64: coordinates, or places in
    a sequence or a grid.  frequencies [P] float32, radians for a unit of the position, P up to dim // 2:
    the first sections[0] of them go with axis 0, the next sections[1] with axis 1 and so on (default:
    the same number for each axis).  Channels from 2 P on are not rotated.  q_weight and k_weight [dim],
    of the heads' type or float32 (default: ones).  Angles are worked out in 64 bits and squares summed in 32;
    results are rounded once.  Returns (q, k) of the inputs' shapes and type, contiguous.

    Differentiable in q, k, the weights and positions (in 32 bits, whatever their type), once, in reverse:
    a tensor with a forward-mode tangent is refused, and so are frequencies that require a gradient.  Sums have
    a fixed order: results repeat bit for bit.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents("rotate_heads", q, k, positions, frequencies, q_weight, k_weight)
    if not _rotate_is_fine(q, k, positions, frequencies, q_weight, k_weight, norm):
        _check_rotate(q, k, positions, frequencies, q_weight, k_weight, norm)
        if positions.dim() == 1:
            positions = positions.unsqueeze(1)
    axes, pairs = positions.size(1), frequencies.size(0)
    if sections is None:
        if pairs % axes:
            raise RuntimeError(f"{pairs} frequencies do not go into {axes} equal sections")
        sections = (pairs // axes,) * axes
    else:
        sections = tuple(int(n) for n in sections)
        _check(len(sections) == axes and min(sections) >= 0 and sum(sections) == pairs,
               f"sections must be {axes} numbers, not negative, that add up to {pairs}, got {sections}")
    _check(not norm or 0.0 <= eps <= 3e38, f"eps must be finite and not negative, got {eps}")
    positions, frequencies = positions.contiguous(), frequencies.contiguous()
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    how = sections, float(eps), int(bool(norm)), int(bool(interleaved))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or positions.requires_grad
                                    or q_weight is not None and q_weight.requires_grad
                                    or k_weight is not None and k_weight.requires_grad):
        return _Rotate.apply(q, k, positions, frequencies, q_weight, k_weight, *how)
    return _rotate_forward(q, k, positions, frequencies, q_weight, k_weight, *how)[3:]
