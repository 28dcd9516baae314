"""The steps of a transformer layer around ``neighbor_attention`` and ``grouped_linear``: heads
normalised and rotated by the atoms' positions, rows routed to experts, taken into their order and
back.

    q, k = rotate_heads(q, k, positions, frequencies)     # before neighbor_attention (periodic cells: see there)
    routing = route_rows(grouped_linear(x, router, natoms), k=2)
    rows = dispatch_rows(x, routing)                      # in the experts' order
    rows = grouped_linear(rows, weight, routing.sizes)    # a weight for each expert
    x = combine_rows(rows, routing, residual=x)

No counterpart in the reference.  The kernels are those of libdynamis_graph.so (dg_rotate_*, dg_route_*,
dg_exchange_*), called through _torch_layer.so, which holds their autograd nodes; there is no CPU path.  Everything runs on the current stream without synchronising the host and can be
captured in a HIP graph; tensors follow torch's rules for streams.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .. import _lib as L
from .dynamis_state_impl import _check, _shape
from .neighbor_ops import _DTYPES, _TENSORS, _refuse_tangents

_POSITIONS = torch.float32, torch.float64, torch.int64


@functools.lru_cache(maxsize=64)
def _sections(sections, axes, pairs):
    """Pairs of each axis."""
    if sections is None:
        _check(pairs % axes == 0, f"{pairs} frequencies do not go into {axes} equal sections")
        sections = (pairs // axes,) * axes
    _check(len(sections) == axes and min(sections) >= 0 and sum(sections) == pairs,
           f"sections must be {axes} numbers, not negative, that add up to {pairs}, got {sections}")
    return sections


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
    results are rounded once.  A mean square plus eps has to lie between 1e-38 and 3e38, or the head's result is
    zeros or not finite.  Returns (q, k) of the inputs' shapes and type, contiguous.

    Positions count as they are: an edge across the boundary of a periodic cell has the angle between the atoms
    themselves, not that to the image, unless all images of an atom have the same angles: fractional
    coordinates, positions @ inv(cell), and frequencies of 2 pi times whole numbers.

    Differentiable in q, k, the weights and positions (in 32 bits, float64 positions in 64), once, in reverse:
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
    sections = _sections(sections if sections is None else tuple(map(int, sections)), axes, pairs)
    if norm and not 0.0 <= eps <= 3e38:
        raise RuntimeError(f"eps must be finite and not negative, got {eps}")
    return L.torch_layer().rotate(q, k, positions, frequencies, q_weight, k_weight, sections, eps if norm else 0.0, bool(norm),
                                  bool(interleaved))


class Routing:
    """Which experts a batch's rows go to (see ``route_rows``).

    rows, num_experts, k;  weights [rows, k] float32;  experts [rows, k] int32 (-1: none);
    sizes [num_experts] int64, the rows of each expert, as ``grouped_linear`` takes them;
    places [rows, k] int32, where a choice lies in the experts' order (of a choice of none, -1 minus
    its place behind the last): together a permutation of [0, rows * k).

    ``dispatch_rows`` and ``combine_rows`` go by places and weights alone, which a caller may change or make.  A
    place past the rows is left out and none is read or written out of bounds; but a row of the experts'
    order that no place points to is not written (``dispatch_rows``' result there, and y's gradient in
    ``combine_rows``, are what the memory held), and one that two point to holds either.  A choice is
    dropped by turning its place p into -1 - p, which keeps the permutation."""

    def __init__(self, num_experts, weights, experts, sizes, places):
        (self.rows, self.k), self.num_experts = experts.shape, num_experts
        self.weights, self.experts, self.sizes, self.places = weights, experts, sizes, places


def _check_route(logits, k, scoring, bias, groups, top_groups, group_best, scale):
    """The refusals of route_rows, with their messages."""
    _check(isinstance(logits, torch.Tensor) and logits.is_cuda, "logits must be a CUDA tensor")
    _check(logits.dim() == 2, f"logits must have shape [rows, experts], got {_shape(logits)}")
    _check(logits.dtype in _DTYPES, f"logits must be float32 or bfloat16, got {logits.dtype}")
    rows, experts = logits.shape
    _check(1 <= experts <= 1024, f"there must be 1 to 1024 experts, got {experts}")
    _check(1 <= k <= min(64, experts), f"k must be 1 to {min(64, experts)}, got {k}")
    _check(rows * k < 1 << 31, f"rows times k must be below 2^31, got {rows} times {k}")
    _check(scoring in ("softmax", "sigmoid"), f'scoring must be "softmax" or "sigmoid", got {scoring!r}')
    _check(1 <= groups <= 64 and experts % groups == 0, f"groups must be 1 to 64 and divide the {experts} experts, got {groups}")
    _check(1 <= top_groups <= groups, f"top_groups must be 1 to {groups}, got {top_groups}")
    _check(group_best in (1, 2), f"group_best must be 1 or 2, got {group_best}")
    _check(-3e38 <= scale <= 3e38, f"scale must be finite, got {scale}")
    if bias is not None:
        _check(isinstance(bias, torch.Tensor) and bias.device == logits.device and bias.is_floating_point()
               and tuple(bias.shape) == (experts,), f"bias must be floating [{experts}] on {logits.device}")


def _route_is_fine(logits, k, scoring, bias, groups, top_groups, group_best, scale):
    """Whether _check_route would pass, without its messages' host time."""
    if not (type(logits) in _TENSORS and logits.is_cuda and logits.dim() == 2 and (bias is None or type(bias) in _TENSORS)):
        return False
    rows, experts = logits.shape
    return (logits.dtype in _DTYPES and 1 <= k <= 64 and k <= experts <= 1024 and rows * k < 1 << 31
            and (scoring == "softmax" or scoring == "sigmoid") and 1 <= groups <= 64 and experts % groups == 0
            and 1 <= top_groups <= groups and 1 <= group_best <= 2 and -3e38 <= scale <= 3e38
            and (bias is None or bias.device == logits.device and bias.is_floating_point() and bias.shape == (experts,)))


def route_rows(logits, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """The k experts of each row by its logits, their weights, and the experts' order of the rows.

      s       = softmax(logits) or sigmoid(logits)
      v       = logits, or with a bias s + bias, in 64 bits
      experts = the k largest v, NaN above all and the first of equals
      weights = scale s[experts], with renormalize divided by their sum over the row

    logits [rows, experts], float32 or bfloat16, 1 to 1024 experts; k up to 64; scoring "softmax" or
    "sigmoid".  bias [experts], used in float32, moves the choice alone and never the weights (it
    keeps the experts balanced).  groups > 1 parts the experts into as many neighbouring groups, each
    worth its largest v, or with group_best=2 the sum of its two largest s (+ bias); experts are chosen from the
    top_groups worthiest groups.

    An expert whose logit or bias is -inf is never chosen.  Where fewer than k are left (a row of
    padding, all -inf), the rest of the row's choices is -1 with weight 0, and takes no place among
    the experts' rows.  rows * k has to be below 2^31.

    Returns a Routing.  Nothing synchronises the host.  Its weights are differentiable in the logits (once, in
    reverse; the choice has no gradient, nor has the bias).  Results repeat bit for bit.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents("route_rows", logits, bias)
    k, groups, top_groups, group_best = int(k), int(groups), int(top_groups), int(group_best)
    if not _route_is_fine(logits, k, scoring, bias, groups, top_groups, group_best, scale):
        _check_route(logits, k, scoring, bias, groups, top_groups, group_best, scale)
    return Routing(logits.size(1), *L.torch_layer().route(logits, bias, k, scoring == "sigmoid", groups, top_groups, group_best,
                                                          bool(renormalize), scale))


def _check_routing(routing):
    """Rows and choices of a routing, by the places that its users read: a Routing can be made or changed by anyone."""
    _check(isinstance(routing, Routing), "routing must be a Routing")
    places = routing.places
    if not (type(places) in _TENSORS and places.is_cuda and places.dtype == torch.int32 and places.dim() == 2
            and 1 <= places.size(1) <= 64):
        raise RuntimeError("routing.places must be a CUDA tensor, int32 [rows, k]")
    return places.shape


def _check_rows(name, t, routing, rows):
    """The refusals of rows that go with a routing; their messages cost host time where one is due alone."""
    if type(t) in _TENSORS and t.dim() == 2 and t.size(0) == rows and t.dtype in _DTYPES \
            and t.device == routing.places.device and 1 <= t.size(1) <= 1 << 20:
        return
    _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dim() == 2 and t.size(0) == rows, f"{name} must have shape [{rows}, width], got {_shape(t)}")
    _check(t.dtype in _DTYPES, f"{name} must be float32 or bfloat16, got {t.dtype}")
    _check(t.device == routing.places.device, f"{name} must be on {routing.places.device}, got {t.device}")
    _check(1 <= t.size(1) <= 1 << 20, f"the width must be 1 to 2^20, got {t.size(1)}")


def dispatch_rows(x, routing):
    """Rows in the order of the experts that they are routed to: x[i] at each of routing.places[i].

    x [rows, width], float32 or bfloat16.  Returns [rows * k, width]: the first routing.sizes[0] rows are
    expert 0's, in the order of x, and so on, as ``grouped_linear`` takes them with routing.sizes; rows
    behind the last expert's (choices of none) are zeros.  Differentiable in x (once, in reverse): the
    gradient is the sum over a row's choices, in 32 bits and in their order.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents("dispatch_rows", x)
    rows, _ = _check_routing(routing)
    _check_rows("x", x, routing, rows)
    return L.torch_layer().dispatch(x, routing.places)


def combine_rows(y, routing, residual=None):
    """The experts' results back: out[i] = residual[i] + sum_j routing.weights[i, j] y[routing.places[i, j]].

    y [rows * k, width], in the order of ``dispatch_rows``, and residual [rows, width] (or None) of its
    type, float32 or bfloat16.  Choices of none add nothing, whatever y holds behind the last
    expert's rows.  Sums are 32 bits, in the choices' order, and rounded once.  Differentiable in y, the
    routing's weights (and so in the router's logits) and the residual, once, in reverse.
    """
    rows, k = _check_routing(routing)
    if forward_ad._current_level >= 0:
        _refuse_tangents("combine_rows", y, routing.weights, residual)
    _check_rows("y", y, routing, rows * k)
    if residual is not None:
        _check_rows("residual", residual, routing, rows)
        if residual.dtype != y.dtype or residual.size(1) != y.size(1):
            raise RuntimeError(f"residual must be {y.dtype} [{rows}, {y.size(1)}], "
                               f"got {residual.dtype} {_shape(residual)}")
    weights = routing.weights
    if not (type(weights) in _TENSORS and weights.dtype == torch.float32 and weights.shape == routing.places.shape
            and weights.device == y.device):
        raise RuntimeError(f"routing.weights must be float32 {_shape(routing.places)} on {y.device}")
    return L.torch_layer().combine(y, weights, residual, routing.places)
