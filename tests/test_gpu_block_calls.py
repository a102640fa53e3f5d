"""Calls that the block operators' documentation allows at the edges of their sizes, layouts and types, on the GPU against
the definitions in 64 bits (oracle/block.py), with the bounds of test_gpu_block.py."""
import pytest
import torch

from oracle import block
from test_gpu_block import DEV, DT, _qk, _rand, _within

pytestmark = pytest.mark.gpu


def test_rotary_axis_that_the_positions_do_not_hold():
    """A plan built by hand, of axes -1, 0, 1 and 2, with positions of two columns: pairs of axes 0 and 1 turn as they should,
    the others are NaN and not turned by another axis's position."""
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    for pairs in ("interleaved", "half"):
        freq = Rotary.build(32, DEV).freq
        axis = torch.tensor([0] * 5 + [1] * 5 + [2] * 5 + [-1], dtype=torch.int32, device=DEV)
        q, k = _qk(70, 2, 9, 3, 2, 40, "fp32")
        pos = torch.randint(0, 500, (2, 9, 2), device=DEV, generator=_rand(71))
        first = torch.arange(16, device=DEV)
        first, second = (2 * first, 2 * first + 1) if pairs == "interleaved" else (first, first + 16)
        held = torch.cat((first[:10], second[:10], torch.arange(32, 40, device=DEV)))
        for x, o in zip((q, k), rotary_embed(q, k, pos, Rotary(freq, axis, pairs))):
            want, mag = block.rotary(x, pos, freq, axis.clamp(0, 1), pairs)
            # (positions up to 500 of a frequency of 1: the 64-bit angle adds nothing to the 12 roundings)
            _within(o[..., held], (want[..., held], mag[..., held]), pairs, 13)
            assert bool(o[..., first[10:]].isnan().all()) and bool(o[..., second[10:]].isnan().all())
