"""A cache of K and V in 4 bits, in pages, and the attention that reads it: 4.25 bits a value where layers/kv_quant.py's chunk
memory takes 8 for K and 14 for V, token by token instead of by chunks, for sequences that grow by single tokens.
"""
from dataclasses import dataclass

import torch

from .. import kernels

__all__ = ["KV4Cache"]

PAGE = 64


@dataclass
class KV4Cache:
    """Pages of 64 tokens for each of `layers` layers (include/lbw_causal.h has the layout): K and V as e2m1 codes with a
    power of two for each 32 channels of a token (OCP MXFP4). Which pages a sequence holds is the caller's to say: `table`
    int32 [S, pages of a sequence] and `lens` int32 [S] on the GPU, the tokens of each sequence with those of the call. A
    call's tokens are the newest of each sequence: rows starts[s] .. starts[s + 1] (int32 [S + 1], not falling) of k, v or q,
    the last row the sequence's last token; starts None: one row for each sequence. What lies past a row of the table, or in a page that
    the cache does not have, is not written, reads as 0 and is not attended. Nothing here waits for the GPU, so all of
    it can be captured in a HIP graph, and lengths and tables may change between replays; table's width bounds them."""
    k: torch.Tensor          # uint8 [layers, pages, heads, 64, D / 2]
    k_scale: torch.Tensor    # uint8 [layers, pages, heads, 64, D / 32]
    v: torch.Tensor          # uint8 [layers, pages, heads, 64 * D / 2]
    v_scale: torch.Tensor    # uint8 [layers, pages, heads, 64 * D / 32]

    @classmethod
    def empty(cls, layers, pages, heads, head_dim=128, device="cuda"):
        """A cache of `pages` pages for `heads` heads of K and V of 64 or 128 channels, all of them 0."""
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if min(layers, pages, heads) < 1:
            raise ValueError(f"layers ({layers}), pages ({pages}) and heads ({heads}) must be 1 or more")
        shape = (layers, pages, heads)
        return cls(*(torch.zeros(*shape, *tail, dtype=torch.uint8, device=device) for tail in
                     ((PAGE, head_dim // 2), (PAGE, head_dim // 32), (PAGE * head_dim // 2,), (PAGE * head_dim // 32,))))

    def write(self, layer, k, v, table, lens, starts=None):
        """k, v [T, heads, D] (bf16 or fp16) into the pages: a group's scale is the least power of two at which none of its
        magnitudes is over 6, codes are the nearest, ties to even; a group with a value that is not finite is held as NaN. A
        page may be in the table once only for the tokens that a call writes. No gradient."""
        kernels.block_binding().kv4_write(self.k, self.k_scale, self.v, self.v_scale, layer, table, lens, starts, k, v)

    def read(self, layer, table, lens, starts=None, tokens=None):
        """What the cache holds of the call's tokens: (k, v) bf16 [tokens, heads, D], exact. tokens: how many rows there are,
        with starts (rows of no sequence are 0)."""
        return kernels.block_binding().kv4_read(self.k, self.k_scale, self.v, self.v_scale, layer, table, lens, starts, tokens)

    def attend(self, layer, q, table, lens, starts=None, sm_scale=None):
        """Attention of q [T, Hq, D] (bf16 or fp16, Hq a multiple of the cache's heads) over the pages, each row over the
        tokens up to its own (of those that the table holds): a decoder's next token of every sequence, or a few drafted ones
        at once. Returns [T, Hq, D] of q's type; rows that see nothing, and rows of no sequence, are 0. The cache's values
        enter the products exactly; softmax and sums are fp32, the softmax's weights are rounded to bf16 before they meet V
        where q is bf16, and held in two bf16 values where it is fp16. Many tokens of a sequence at once are better served
        by packed_attention over read(). No gradient."""
        return kernels.block_binding().kv4_attend(self.k, self.k_scale, self.v, self.v_scale, layer, table, lens, starts, q,
                                                  sm_scale)
