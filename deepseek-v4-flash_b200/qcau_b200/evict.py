"""Bounding the paged latent cache by accumulated attention weight.

Every decode (or verification) step adds to each cached token the attention
weight it received; when a sequence is over its budget, its first tokens, its
most recent ones and those of the largest sums stay.  A step with draft trees
(without mask and commit: a decode step, s = 1) of a PagedKVCache pc, sums
[sequences, positions] starting at 0:

    base = pc.seqlens.clone()
    slots = pc.append(seqs, [s] * len(seqs))  # kv_build writes the drafted rows there
    mask = tree_mask(parents)
    o, lse = tree_attn(q, pc.cache, pc.block_table, pc.seqlens, mask, softmax_scale=scale,
                       return_lse=True)
    # the lengths, rows and nodes that lse belongs to: before the step's end
    attn_weight_sums(q, pc.cache, pc.block_table, pc.seqlens, lse, mask, softmax_scale=scale,
                     sums=sums)
    # a path of each tree is accepted; its rows and their sums move up
    commit(pc.cache, pc.block_table, base, path, accepted, seqlens=pc.seqlens, sums=sums)
    pc.truncate(seqs, lengths)
    # sequences over the budget come down to it
    keep, lens = evict(pc.cache, pc.block_table, pc.seqlens, sums, budget, n_first=first,
                       n_recent=recent)
    pc.truncate(range(len(lens)), lens.tolist())

The latent row of a token is shared by all heads, so one choice is made per
sequence.  Rows keep the rotation of the position they were written at: a
sequence's positions go on counting from its uncut length.  The reference has
no eviction (its cache is a window plus compressed rows).
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import bind


def attn_weight_sums(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                     seqlens: torch.Tensor, lse: torch.Tensor,
                     mask: Optional[torch.Tensor] = None, *, softmax_scale: float,
                     tree_lens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None,
                     sums: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight that each cached token received in one step, summed
    over the step's query tokens and heads.

    q, cache, block_table, seqlens, mask, tree_lens, max_seqlen as tree_attn
    took them, lse [b, s, h] fp32 as it returned them (q [b, 1, h, d] and no
    mask: a decode step): the call belongs between the attention and the step's
    end, whose commit moves the rows and changes the lengths.  Returns sums [b, max_seqlen] fp32, 0 where no query
    sees; with `sums` given ([b, at least max_seqlen], rows may be strided) the
    weights are added to it instead, at positions below seqlens, and it is
    returned.  The same inputs give the same bits.
    """
    return bind().attn_weight_sums(q, cache, block_table, seqlens, lse, mask, softmax_scale, tree_lens,
                                   max_seqlen, sums)


def select_rows(sums: torch.Tensor, seqlens: torch.Tensor, budget: int, *, n_first: int = 0,
                n_recent: int = 0, sums_out: Optional[torch.Tensor] = None):
    """The tokens to keep of each sequence: (keep [b, budget] int32, counts [b]
    int32).

    Of the first seqlens[i] positions of sums [b, positions] fp32, the first
    n_first, the last n_recent and those of the largest sums, min(seqlens[i],
    budget) in all, ascending, -1 past the count.  Among equal sums the lower
    position stays; NaN ranks above every number.  sums_out (sums
    itself, or other memory) gets the kept sums in the new order and 0 behind
    them.
    """
    return bind().select_rows(sums, seqlens, budget, n_first, n_recent, sums_out)


def evict(cache: torch.Tensor, block_table: torch.Tensor, seqlens: torch.Tensor,
          sums: torch.Tensor, budget: int, *, n_first: int = 0, n_recent: int = 0,
          dst_cache: Optional[torch.Tensor] = None, dst_table: Optional[torch.Tensor] = None,
          sums_out: Optional[torch.Tensor] = None):
    """Bring sequences over `budget` tokens down to it: select_rows, then the
    cache's rows and the sums move together.

    In place (cache, block_table and sums) unless dst_cache / dst_table /
    sums_out name where they go; a sequence within its budget stays as it is.
    Returns (keep [b, budget] int32, lens [b] int32: the new lengths); seqlens
    is left to the caller (seqlens.copy_(lens), PagedKVCache.truncate).
    """
    return bind().evict(cache, block_table, seqlens, sums, budget, n_first, n_recent, dst_cache,
                        dst_table, sums_out)
