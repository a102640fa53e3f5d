"""The gated norm between two sub-layers of a block, forward and backward.

The reference's block adds each sub-layer's output to the residual stream through a gate, then normalises the stream
and modulates it for the next one (lingbot/models/lingbot_world/transformer.py:281-360), with one modulation row for every
latent frame. Written with torch operations that is a dozen passes over [B, L, C]; here it is one pass, and one more for all
gradients.
"""
from .. import kernels

__all__ = ["gated_norm"]


def gated_norm(x, y=None, gate=None, shift=None, scale=None, weight=None, bias=None, post_weight=None, norm="layer",
               post_norm=None, eps=1e-6, residual_scale=1.0, branch_scale=1.0, group_len=None):
    """The stream and the next sub-layer's input, in one pass:

        s = residual_scale * x + branch_scale * gate * (post_norm(y) * post_weight)
        h = (norm(s) * weight + bias) * (1 + scale) + shift

    x, y: [B, L, C] bf16, fp16 or fp32 on the GPU, any strides of B and L. norm, post_norm: 'layer', 'rms' or None, with
    `eps`. gate, shift, scale: [C], or [B, rows, C] with `group_len` tokens a row (default: ceil(L / rows)),
    e.g. slices of one projection's output. weight, bias, post_weight: [C]. Vectors are of x's dtype or fp32;
    where they differ among themselves all are taken in fp32. Every step is fp32 and each output is rounded once: the norm reads
    s before its rounding. C is at most 12288; the rows may be none.

    Returns (s, h), s alone where norm is None, and h alone where there is no y (s would be x scaled).
    Differentiable in x, y and every vector (once: there is no second derivative). The backward reads x and y again and
    keeps nothing else; the sums over rows are in fp32 and in a fixed order.
    """
    s, h = kernels.block_binding().norm(x, y, gate, shift, scale, weight, bias, post_weight, norm, post_norm, eps,
                                        residual_scale, branch_scale, group_len)
    return h if s is None else s if h is None else (s, h)
