"""Speculative decoding with draft trees on the paged latent cache.

A drafting step proposes a tree of tokens per sequence: their latent rows are
appended to the cache (PagedKVCache.append + kv_build, node t at token base +
t), one attention verifies all of them, and the accepted path's rows move up
behind the sequence:

    mask = tree_mask(parents)                       # ancestors of each node
    o, lse = tree_attn(q, cache, block_table, seqlens, mask, softmax_scale=scale,
                       return_lse=True)             # seqlens counts the drafted rows
    ...                                             # accept a path per sequence
    commit(cache, block_table, base_lens, path, accepted, seqlens=seqlens)

(On a cache that is bounded by its attention weights, qcau_b200.evict shows where
their sums come in between.)

The reference has no speculative decoding; the attention is its sparse_attn
(Deepseek_origin/inference/kernel.py:276-352) with every cached token in place
of the index list and the tree in place of causality.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import bind, check, lib, require_cuda, stream_ptr


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """mask [b, s, s] bool of draft trees: True at each node's ancestors and at
    itself.  parents [b, s] int32: the index of the node's parent, which comes
    before it, or -1 for a child of the sequence's last token.  A parent that
    is no earlier node raises the device error bit DEVERR_INDEX."""
    require_cuda(parents)
    if parents.dim() != 2 or parents.size(1) == 0:
        raise ValueError("tree_mask: parents must be [batch, nodes]")
    if parents.dtype != torch.int32 or not parents.is_contiguous():
        raise ValueError("tree_mask: parents must be contiguous int32")
    b, s = parents.shape
    mask = torch.empty(b, s, s, device=parents.device, dtype=torch.bool)
    with torch.cuda.device(parents.device):
        check(lib().qcau_tree_mask(parents.data_ptr(), mask.data_ptr(), b, s,
                                   stream_ptr(parents.device)), "tree_mask")
    return mask


def tree_attn(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
              seqlens: torch.Tensor, mask: Optional[torch.Tensor] = None, *,
              softmax_scale: float, tree_lens: Optional[torch.Tensor] = None,
              attn_sink: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None,
              return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of s drafted tokens per sequence over the paged cache that
    holds their rows (verification of a draft tree).

    q [b, s, h, d] bf16 (d = 576 or 512, the cache's width; any s and h), cache
    [pages, page, d] bf16 (page a multiple of 64), block_table [b, max_pages]
    int32, seqlens [b] int32: cached tokens, of which the last tree_lens[i]
    (None: s, or none where seqlens[i] is 0, an idle slot) are the tree's nodes
    in the cache.  Node t attends to all tokens
    before the tree and to node j when mask[i, t, j]; mask is bool [b, s, s],
    or [s, s] for all sequences, or None for a chain (j <= t).  attn_sink [h].

    Returns o [b, s, h, 512] bf16 (written to `out` when given, other
    memory than q and the cache), and with
    return_lse the log-sum-exps [b, s, h] fp32 that attn_weight_sums takes.
    Nodes past tree_lens[i] get zeros and -inf.  max_seqlen bounds seqlens
    (None: what the block table holds) and sizes the launch.
    """
    return bind().tree_attn(q, cache, block_table, seqlens, mask, softmax_scale, tree_lens, attn_sink,
                            max_seqlen, return_lse, out)


def commit(cache: torch.Tensor, block_table: torch.Tensor, base_lens: torch.Tensor,
           path: torch.Tensor, accepted: torch.Tensor, *,
           seqlens: Optional[torch.Tensor] = None, sums: Optional[torch.Tensor] = None) -> None:
    """End a drafting step: the rows of each sequence's accepted path move up
    behind its base_lens[i] tokens, in place.

    path [b, k] int32: the accepted nodes from the root down (ascending, as a
    node comes after its parent; values past accepted[i] are ignored), accepted
    [b] int32: how many (0: none).  seqlens [b], when given, becomes base_lens
    + accepted (it may be base_lens itself); PagedKVCache.truncate returns the pages of the rest.
    sums [b, positions] fp32: the running weight sums of a cache that is also
    bounded by eviction (evict.attn_weight_sums, which has the step's weights
    added before this call).  The accepted nodes' sums move with their rows, and
    0 follows to the row's end, so that the tokens that come next inherit
    nothing from rejected nodes.
    """
    if base_lens is None:
        raise ValueError("commit: base_lens is needed")
    bind().keep_rows(cache, block_table, path, accepted, base_lens, None, None, seqlens, sums)
