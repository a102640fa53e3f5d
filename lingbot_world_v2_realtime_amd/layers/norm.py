"""The gated norm between two sub-layers of a block, forward and backward.

The reference's block adds each sub-layer's output to the residual stream through a gate, then normalises the stream
and modulates it for the next one (lingbot/models/lingbot_world/transformer.py:281-360), with one modulation row for every
latent frame. Written with torch operations that is a dozen passes over [B, L, C]; here it is one pass, and one more for all
gradients.
"""
import torch
from torch.autograd.function import once_differentiable

from .. import kernels
from .linear import _plain

__all__ = ["gated_norm"]

_VECTORS = ("gate", "shift", "scale", "weight", "bias", "post_weight")


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, opts, x, y, *vectors):
        named = dict(zip(_VECTORS, vectors))
        ctx.opts = {key: v for key, v in opts.items() if key != "want_stream"}
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, *vectors)
        return kernels.gated_norm(x, y, **named, **opts)

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, dh):
        x, y, *vectors = ctx.saved_tensors
        names = ("x", "y") + _VECTORS
        wants = [name for name, needed in zip(names, ctx.needs_input_grad[1:]) if needed]
        ds, dh = (d if d is None else d.contiguous() for d in (ds, dh))
        grads = kernels.gated_norm_bwd(x, ds, dh, y, **dict(zip(_VECTORS, vectors)), **ctx.opts, wants=wants)
        return (None, *(grads.get(name) for name in names))


def gated_norm(x, y=None, gate=None, shift=None, scale=None, weight=None, bias=None, post_weight=None, norm="layer",
               post_norm=None, eps=1e-6, residual_scale=1.0, branch_scale=1.0, group_len=None):
    """The stream and the next sub-layer's input, in one pass:

        s = residual_scale * x + branch_scale * gate * (post_norm(y) * post_weight)
        h = (norm(s) * weight + bias) * (1 + scale) + shift

    x, y: [B, L, C] bf16, fp16 or fp32 on the GPU, any strides of B and L. norm, post_norm: 'layer', 'rms' or None, with
    `eps`. gate, shift, scale: [C], or [B, rows, C] with `group_len` tokens a row (default: the rows share the L tokens
    evenly), e.g. slices of one projection's output. weight, bias, post_weight: [C]. Vectors are of x's dtype or fp32;
    where they differ among themselves all are taken in fp32. Every step is fp32 and each output is rounded once: the norm reads
    s before its rounding. C is at most 12288; the rows may be none.

    Returns (s, h), s alone where norm is None, and h alone where there is no y (s would be x scaled).
    Differentiable in x, y and every vector (once: there is no second derivative). The backward reads x and y again and
    keeps nothing else; the sums over rows are in fp32 and in a fixed order.
    """
    vectors = (gate, shift, scale, weight, bias, post_weight)
    dtypes = {v.dtype for v in vectors if v is not None}
    if len(dtypes) > 1:
        vectors = tuple(v if v is None or v.dtype == torch.float32 else v.float() for v in vectors)
    opts = {"norm": norm, "post_norm": post_norm, "eps": eps, "residual_scale": residual_scale,
            "branch_scale": branch_scale, "group_len": group_len, "want_stream": y is not None}
    if _plain(x, y, *vectors):
        s, h = kernels.gated_norm(x, y, **dict(zip(_VECTORS, vectors)), **opts)
    else:
        s, h = _GatedNorm.apply(opts, x, y, *vectors)
    return h if s is None else s if h is None else (s, h)
