"""Type stubs of the operators on a built graph (``neighbor_ops``)."""
from __future__ import annotations

import typing

import torch

class NeighborPlan:
    device: torch.device
    num_nodes: int
    num_targets: int
    num_edges: int
    num_buckets: int
    symmetric: bool
    def record_stream(self, stream: torch.cuda.Stream) -> None: ...

def neighbor_plan(edge_index: torch.Tensor, num_nodes: int, num_targets: int | None = None,
                  distances: torch.Tensor | None = None,
                  boundaries: torch.Tensor | typing.Sequence[float] | None = None,
                  edge_mask: torch.Tensor | None = None, backward: bool = True) -> NeighborPlan: ...
@typing.overload
def neighbor_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: NeighborPlan,
                       bias_table: torch.Tensor | None = None, scale: float | None = None,
                       return_lse: typing.Literal[False] = False) -> torch.Tensor: ...
@typing.overload
def neighbor_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: NeighborPlan,
                       bias_table: torch.Tensor | None = None, scale: float | None = None, *,
                       return_lse: typing.Literal[True]) -> tuple[torch.Tensor, torch.Tensor]: ...
def grouped_linear(x: torch.Tensor, weight: torch.Tensor, sizes: torch.Tensor | typing.Sequence[int],
                   bias: torch.Tensor | None = None, activation: typing.Literal["silu", "gelu"] | None = None,
                   residual: torch.Tensor | None = None) -> torch.Tensor: ...
