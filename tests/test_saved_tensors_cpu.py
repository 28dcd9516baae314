"""What a backward pass takes from a hook: its strides are free, its shape, type and device are not (no GPU)."""
import pytest
import torch

from dynamis_amd.dynamis_state import neighbor_ops


def test_saved_tensors_of_another_make_are_refused():
    t, cpu = torch.zeros(4, 6), torch.device("cpu")
    neighbor_ops._came_back("op", cpu, (t, (4, 6), torch.float32), (torch.zeros(6, 4).t(), t.shape, torch.float32))
    for bad in (t[:3], t.double(), t.flatten(), torch.empty(4, 6, device="meta")):
        with pytest.raises(RuntimeError, match="op: a saved tensor came back"):
            neighbor_ops._came_back("op", cpu, (t, (4, 6), torch.float32), (bad, (4, 6), torch.float32))
