"""Type stubs of a layer's operators around attention and grouped products (``layer_ops``)."""
from __future__ import annotations

import typing

import torch

def rotate_heads(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
                 sections: typing.Sequence[int] | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, norm: bool = True,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]: ...

class Routing:
    rows: int
    num_experts: int
    k: int
    weights: torch.Tensor
    experts: torch.Tensor
    sizes: torch.Tensor
    places: torch.Tensor
    def __init__(self, num_experts: int, weights: torch.Tensor, experts: torch.Tensor, sizes: torch.Tensor,
                 places: torch.Tensor) -> None: ...

def route_rows(logits: torch.Tensor, k: int, scoring: typing.Literal["softmax", "sigmoid"] = "softmax",
               bias: torch.Tensor | None = None, groups: int = 1, top_groups: int = 1, group_best: int = 1,
               renormalize: bool = True, scale: float = 1.0) -> Routing: ...
def dispatch_rows(x: torch.Tensor, routing: Routing) -> torch.Tensor: ...
def combine_rows(y: torch.Tensor, routing: Routing, residual: torch.Tensor | None = None) -> torch.Tensor: ...
