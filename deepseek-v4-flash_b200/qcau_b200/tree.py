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

The reference has no speculative decoding; the attention is its sparse_attn
(Deepseek_origin/inference/kernel.py:276-352) with every cached token in place
of the index list and the tree in place of causality.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import (call_on, check, data, lib, pack_tree_args, require_cuda, stream_ptr,
                   workspace_size)
from .cache import _check_ints, _check_paged, keep_rows


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """mask [b, s, s] bool of draft trees: True at each node's ancestors and at
    itself.  parents [b, s] int32: the index of the node's parent, which comes
    before it, or -1 for a child of the sequence's last token.  A parent that
    is no earlier node raises the device error bit DEVERR_INDEX."""
    require_cuda(parents)
    if parents.dim() != 2 or parents.size(1) == 0:
        raise ValueError("tree_mask: parents must be [batch, nodes]")
    _check_ints("tree_mask", "parents", parents, parents.shape, parents.get_device())
    b, s = parents.shape
    mask = torch.empty(b, s, s, device=parents.device, dtype=torch.bool)
    with torch.cuda.device(parents.device):
        check(lib().qcau_tree_mask(parents.data_ptr(), mask.data_ptr(), b, s,
                                   stream_ptr(parents.device)), "tree_mask")
    return mask


def _check_step(what: str, q, cache, block_table, seqlens, mask, tree_lens, max_seqlen):
    """The checks that the attention and the weight sums share.  Returns the device
    index, q contiguous, its shape, the mask's sequence stride, (page size, pages
    of a sequence, pages) and the bound of the lengths."""
    index = q.get_device()
    if index < 0:
        require_cuda(q)
    num_pages, page, width, rows, max_pages = _check_paged(what, index, cache, block_table)
    shape = q.shape
    if len(shape) != 4 or q.dtype != torch.bfloat16:
        raise ValueError(f"{what}: q must be bf16 [batch, nodes, heads, width]")
    b, s, h, d = shape
    if s == 0 or h == 0:
        raise ValueError(f"{what}: q has no rows")
    if width != d:
        raise ValueError(f"{what}: q and the cache must have one width")
    if rows != b:
        raise ValueError(f"{what}: one block-table row per sequence is needed")
    _check_ints(what, "seqlens", seqlens, (b,), index)
    if tree_lens is not None:
        _check_ints(what, "tree_lens", tree_lens, (b,), index)
    stride = 0
    if mask is not None:
        dims = mask.shape
        if dims == (b, s, s):
            stride = s * s
        if dims not in ((b, s, s), (s, s)) or not mask.is_contiguous() \
                or mask.dtype not in (torch.bool, torch.uint8) or mask.get_device() != index:
            raise ValueError(f"{what}: the mask must be a contiguous bool [batch, nodes, nodes] or "
                             "[nodes, nodes] tensor on q's device")
    if not q.is_contiguous():
        q = q.contiguous()
    most = max_pages * page if max_seqlen is None else max_seqlen
    return index, q, shape, stride, (page, max_pages, num_pages), most


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
    (None: s) are the tree's nodes in the cache.  Node t attends to all tokens
    before the tree and to node j when mask[i, t, j]; mask is bool [b, s, s],
    or [s, s] for all sequences, or None for a chain (j <= t).  attn_sink [h].

    Returns o [b, s, h, 512] bf16 (written to `out` when given), and with
    return_lse the log-sum-exps [b, s, h] fp32 that attn_weight_sums takes.
    Nodes past tree_lens[i] get zeros and -inf.  max_seqlen bounds seqlens
    (None: what the block table holds) and sizes the launch.
    """
    index, q, (b, s, h, d), stride, pages, most = _check_step(
        "tree_attn", q, cache, block_table, seqlens, mask, tree_lens, max_seqlen)
    dev = q.device
    sink = attn_sink
    if sink is not None:
        if sink.numel() != h or sink.get_device() != index:
            raise ValueError("tree_attn: attn_sink needs one value per head, on q's device")
        if sink.dtype != torch.float32 or not sink.is_contiguous():
            sink = sink.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty((b, s, h, 512), dtype=torch.bfloat16, device=dev)
    elif out.shape != (b, s, h, 512) or out.dtype != torch.bfloat16 \
            or not out.is_contiguous() or out.get_device() != index:
        raise ValueError("tree_attn: out must be a contiguous bf16 [batch, nodes, heads, 512] tensor")
    lse = torch.empty((b, s, h), dtype=torch.float32, device=dev) if return_lse else None
    need = workspace_size("qcau_tree_attn_workspace_size", b, s, h, most)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    args = pack_tree_args(
        q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), seqlens.data_ptr(),
        data(tree_lens), data(mask), data(sink), out.data_ptr(), data(lse), 0, ws.data_ptr(), stride,
        b, s, h, d, 512, *pages, most, 0, need, softmax_scale, 0)
    call_on(index, "tree_attn", lib().qcau_tree_attn, args)
    return (out, lse) if return_lse else out


def commit(cache: torch.Tensor, block_table: torch.Tensor, base_lens: torch.Tensor,
           path: torch.Tensor, accepted: torch.Tensor, *,
           seqlens: Optional[torch.Tensor] = None) -> None:
    """End a drafting step: the rows of each sequence's accepted path move up
    behind its base_lens[i] tokens, in place.

    path [b, k] int32: the accepted nodes from the root down (ascending, as a
    node comes after its parent; values past accepted[i] are ignored), accepted
    [b] int32: how many (0: none).  seqlens [b], when given, becomes base_lens
    + accepted; PagedKVCache.truncate returns the pages of the rest.
    """
    if base_lens is None:
        raise ValueError("commit: base_lens is needed")
    keep_rows(cache, block_table, path, accepted, start=base_lens, seqlens=seqlens)
