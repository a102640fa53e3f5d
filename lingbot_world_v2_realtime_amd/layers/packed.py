"""Attention over sequences of different lengths packed one behind the other, causal, with grouped heads: the prompts of a
batch, or a training step's documents, without padding. layers/attention.py attends a batch of one length, not causally;
layers/kv4.py continues from here with single tokens.
"""
from .. import kernels

__all__ = ["packed_attention"]


def packed_attention(q, k, v, starts, k_starts=None, sm_scale=None, causal=True):
    """q [T, Hq, D] and k, v [Tk, Hk, D] (bf16 or fp16 on the GPU, D 64 or 128, Hq a multiple of Hk: head h of q reads head
    h // (Hq / Hk)). Rows starts[s] .. starts[s + 1] of q are sequence s, rows k_starts[s] .. k_starts[s + 1] of k and v its
    keys (int32 on the GPU, [sequences + 1], not falling; k_starts None: the same). With `causal` the last query of a sequence
    sees all of its keys and each query before it one less, whatever the two lengths are (a prefix that is in k and v
    alone; queries that see nothing); without, every query sees every key of its sequence. Rows that see nothing, and rows
    of no sequence, give 0. sm_scale: D^-1/2 by default. Returns [T, Hq, D] of q's type; differentiable in q, k and v.

    Products are of the inputs' type with fp32 sums, the softmax is fp32, its weights are rounded to the type before they
    meet v (and, in the gradient, d_out), and every output once; the gradient's other weights meet k in two parts of the type, and q
    in one (two where a sequence has up to 128 queries or keys). An infinity or NaN reaches the rows that see it and no others.
    Rows that are not 16-byte aligned are copied."""
    return kernels.block_binding().packed_attention(q, k, v, starts, k_starts, sm_scale, causal)
