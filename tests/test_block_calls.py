"""Calls of the block operators that have no right answer, on the CPU: each is refused, and says why, before anything
looks for a device."""
import pytest
import torch

from lingbot_world_v2_realtime_amd import kernels
from lingbot_world_v2_realtime_amd.layers.linear import W4Linear


@pytest.fixture
def w4_module(monkeypatch):
    """A W4Linear of 1536 -> 32 with empty tiles (the quantisation itself needs the GPU)."""
    def tiles(w, group, fmt, zeros):
        shapes = kernels._w4_shapes(*w.shape, group)
        return torch.zeros(shapes[0], dtype=torch.uint8), torch.zeros(shapes[1], dtype=torch.bfloat16), None
    monkeypatch.setattr(kernels, "quant_w4", tiles)
    return W4Linear(torch.nn.Linear(1536, 32))


@pytest.mark.parametrize("width", [1500, 1409, 1535, 1408, 1537, 1])
def test_w4_linear_refuses_another_width(w4_module, width):
    """1409 to 1535 columns end in the weights' last tile of 128: the tiles alone do not tell them from 1536."""
    with torch.no_grad(), pytest.raises(ValueError, match=f"1536 .*{width}"):
        w4_module(torch.zeros(2, width, dtype=torch.bfloat16))
