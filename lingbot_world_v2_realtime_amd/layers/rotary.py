"""Rotary positions of q and k by themselves: any head size up to 512, whole heads or their first part, neighbouring or
half layout, one axis or several, frequencies stretched for contexts longer than the trained one; forward and backward.

layers/prologue.py rotates inside the quantisation of a chunk's q and k, from a table of the model's three axes; this is for
attention that is not quantised (training, other head sizes, single tokens) and for positions that no table holds: the
angles are formed in the kernel from the positions themselves.
"""
import math
from dataclasses import dataclass
from typing import Optional

import torch

from .. import kernels

__all__ = ["Rotary", "rotary_embed", "grid_positions"]


@dataclass
class Rotary:
    """A rotation's plan, on the device: float64 frequencies [pairs] (radians a position), the axis of each pair (int32, None
    with one axis), which channels are partners, the factor that cos and sin are multiplied by, and how many axes there
    are, so that positions of fewer can be refused (None: not known; a pair whose axis the positions do not hold comes out
    as NaN)."""
    freq: torch.Tensor
    axis: Optional[torch.Tensor] = None
    pairs: str = "interleaved"
    factor: float = 1.0
    axes: Optional[int] = None

    @classmethod
    def build(cls, dim, device, base=10000.0, pairs="interleaved", sections=None, scaling=None, stretch=1.0,
              trained_len=None, fast_turns=32.0, slow_turns=1.0):
        """The plan of `dim` rotated channels (even). sections: pairs of each axis (their sum dim / 2), every axis with
        frequencies base^(-i / pairs) of its own, as the model's frame / height / width sections have
        (reference/wan/modules/model.py:29-36); None: one axis.

        scaling, for contexts `stretch` times the trained length:
        - None: the frequencies as they are;
        - 'linear': all divided by `stretch`;
        - 'base': the base multiplied by stretch^(d / (d - 2)), d the axis's channels: the slowest pair is stretched in
          full, the fastest not at all;
        - 'ramp': by the turns a pair makes over `trained_len` tokens: pairs of more than `fast_turns` stay, pairs of
          fewer than `slow_turns` are divided, with a linear ramp between, and cos and sin grow by 1 + 0.1 ln(stretch)
          (the published YaRN rule)."""
        if dim < 2 or dim % 2:
            raise ValueError(f"dim must be even, got {dim}")
        if scaling not in (None, "linear", "base", "ramp"):
            raise ValueError(f"scaling must be None, 'linear', 'base' or 'ramp', got {scaling!r}")
        if not stretch >= 1.0:
            raise ValueError(f"stretch must be 1 or more, got {stretch}")
        if scaling == "ramp" and not (trained_len and trained_len > 0 and fast_turns > slow_turns):
            raise ValueError("'ramp' needs trained_len and fast_turns > slow_turns")
        parts = (dim // 2,) if sections is None else tuple(int(p) for p in sections)
        if sum(parts) != dim // 2 or min(parts) < 1:
            raise ValueError(f"sections {parts} must be positive and add up to {dim // 2} pairs")
        freq, axis = [], []
        for i, n in enumerate(parts):
            b = base * stretch ** (n / (n - 1)) if scaling == "base" and n > 1 else base
            f = b ** (-torch.arange(n, dtype=torch.float64) / n)
            if scaling == "linear":
                f = f / stretch
            elif scaling == "ramp":
                turns = trained_len * f / (2 * math.pi)
                keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
                f = f * keep + f / stretch * (1 - keep)
            freq.append(f)
            axis += [i] * n
        return cls(torch.cat(freq).to(device),
                   torch.tensor(axis, dtype=torch.int32, device=device) if len(parts) > 1 else None, pairs,
                   1.0 + 0.1 * math.log(stretch) if scaling == "ramp" else 1.0, len(parts))


def grid_positions(grid_size, start_frame=0, device="cuda"):
    """int32 [frames * h * w, 3]: the (frame, row, column) of each token of a chunk's grid (frames, h, w)."""
    f, h, w = (int(n) for n in grid_size)
    t = torch.arange(f * h * w, dtype=torch.int32, device=device)
    return torch.stack((start_frame + t // (h * w), t // w % h, t % w), dim=1)


def rotary_embed(q, k, positions, rope, tensor_layout="NHD", inplace=False):
    """q [B, L, Hq, D] and k [B, L, Hk, D] (or None) rotated by the plan `rope` ("HND": [B, H, L, D]; bf16, fp16 or fp32
    on the GPU, any strides with contiguous channels, any head counts). positions: int32 or int64 tensor [L] or [B, L]
    (with several axes [L, axes] or [B, L, axes]), or an int: the first token's position, the others following.
    Channels past the plan's are copied. Angles are formed in 64 bits, the rotation in fp32, with one rounding.
    inplace: q and k are overwritten and returned (refused where a gradient is recorded, or where two elements of them
    share memory). Returns (q, k); differentiable in both."""
    return kernels.block_binding().rotary_embed(q, k, positions, rope.freq, rope.axis, rope.pairs, rope.factor,
                                                tensor_layout, rope.axes, inplace)
