"""Bounding the paged latent cache by accumulated attention weight.

Every decode (or verification) step adds to each cached token the attention
weight it received; when a sequence is over its budget, its first tokens, its
most recent ones and those of the largest sums stay:

    o, lse = tree_attn(q, cache, block_table, seqlens, softmax_scale=scale, return_lse=True)
    attn_weight_sums(q, cache, block_table, seqlens, lse, softmax_scale=scale, sums=sums)
    ...
    keep, lens = evict(cache, block_table, seqlens, sums, budget, n_first=4, n_recent=256)

The latent row of a token is shared by all heads, so one choice is made per
sequence.  Rows keep the rotation of the position they were written at: a
sequence's positions go on counting from its uncut length.  The reference has
no eviction (its cache is a window plus compressed rows).
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, lib, ptr, require_cuda, stream_ptr
from .cache import _check_ints, _check_move, keep_rows
from .tree import _check_step


def _check_sums(sums: torch.Tensor, b: int, device, what: str) -> None:
    if sums.dim() != 2 or sums.dtype != torch.float32 or sums.size(0) != b or sums.device != device \
            or sums.stride(1) != 1 or (b > 1 and sums.stride(0) < sums.size(1)):
        raise ValueError(f"{what}: sums must be fp32 [batch, positions] with contiguous rows, on "
                         f"{device}")


def attn_weight_sums(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                     seqlens: torch.Tensor, lse: torch.Tensor,
                     mask: Optional[torch.Tensor] = None, *, softmax_scale: float,
                     tree_lens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None,
                     sums: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight that each cached token received in one step, summed
    over the step's query tokens and heads.

    q, cache, block_table, seqlens, mask, tree_lens, max_seqlen as tree_attn
    takes them, lse [b, s, h] fp32 as it returned them (q [b, 1, h, d] and no
    mask: a decode step).  Returns sums [b, max_seqlen] fp32, 0 where no query
    sees; with `sums` given ([b, at least max_seqlen], rows may be strided) the
    weights are added to it instead, at positions below seqlens, and it is
    returned.  The same inputs give the same bits.
    """
    q, stride, most = _check_step("attn_weight_sums", q, cache, block_table, seqlens, mask,
                                  tree_lens, max_seqlen)
    require_cuda(lse, sums)
    b, s, h, d = q.shape
    dev = q.device
    if lse.dtype != torch.float32 or tuple(lse.shape) != (b, s, h) or not lse.is_contiguous() \
            or lse.device != dev:
        raise ValueError("attn_weight_sums: lse must be a contiguous fp32 [batch, nodes, heads] tensor")
    add = sums is not None
    if add:
        _check_sums(sums, b, dev, "attn_weight_sums")
    else:
        sums = torch.empty(b, most, device=dev, dtype=torch.float32)
    if sums.size(1) < most:
        raise ValueError("attn_weight_sums: a row of sums must hold max_seqlen values")
    L = lib()
    need = L.qcau_attn_weight_sums_workspace_size(b, s, h, most)
    with torch.cuda.device(dev):
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        check(L.qcau_attn_weight_sums(
            q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), seqlens.data_ptr(),
            lse.data_ptr(), ptr(tree_lens), ptr(mask), stride, sums.data_ptr(),
            max(sums.stride(0), sums.size(1)), int(add), b, s, h, d, cache.size(1),
            block_table.size(1), cache.size(0), most, softmax_scale, ptr(ws), need,
            stream_ptr(dev)), "attn_weight_sums")
    return sums


def select_rows(sums: torch.Tensor, seqlens: torch.Tensor, budget: int, *, n_first: int = 0,
                n_recent: int = 0, sums_out: Optional[torch.Tensor] = None):
    """The tokens to keep of each sequence: (keep [b, budget] int32, counts [b]
    int32).

    Of the first seqlens[i] positions of sums [b, positions] fp32, the first
    n_first, the last n_recent and those of the largest sums, min(seqlens[i],
    budget) in all, ascending, -1 past the count.  Among equal sums the lower
    position stays; NaN ranks above every number.  sums_out (may be sums itself)
    gets the kept sums in the new order and 0 behind them.
    """
    require_cuda(sums, seqlens, sums_out)
    b = seqlens.numel()
    dev = sums.device
    _check_ints(seqlens, (b,), dev, "select_rows: seqlens")
    _check_sums(sums, b, dev, "select_rows")
    n = sums.size(1)
    if sums_out is not None:
        _check_sums(sums_out, b, dev, "select_rows")
        if sums_out.size(1) != n:
            raise ValueError("select_rows: sums_out must have the shape of sums")
        if sums_out.data_ptr() == sums.data_ptr() and sums_out.stride(0) != sums.stride(0):
            raise ValueError("select_rows: in place, sums_out must be sums")
    keep = torch.empty(b, max(budget, 0), device=dev, dtype=torch.int32)
    counts = torch.empty(b, device=dev, dtype=torch.int32)
    with torch.cuda.device(dev):
        check(lib().qcau_evict_select(
            sums.data_ptr(), max(sums.stride(0), n), seqlens.data_ptr(), keep.data_ptr(),
            counts.data_ptr(), ptr(sums_out),
            0 if sums_out is None else max(sums_out.stride(0), n), b, n, budget, n_first, n_recent,
            stream_ptr(dev)), "evict_select")
    return keep, counts


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
    # every refusal comes before the sums are touched
    dc, dt = _check_move("evict", cache, block_table, dst_cache, dst_table)
    if seqlens.numel() != dt.size(0) or sums.device != cache.device:
        raise ValueError("evict: one length per block-table row, and all tensors on one device")
    n = sums.size(-1)
    if n > block_table.size(1) * cache.size(1) or min(budget, n) > dt.size(1) * dc.size(1):
        raise ValueError("evict: a block table does not hold the positions of sums, or the budget")
    keep, counts = select_rows(sums, seqlens, budget, n_first=n_first, n_recent=n_recent,
                               sums_out=sums if sums_out is None else sums_out)
    keep_rows(cache, block_table, keep, counts, dst_cache=dst_cache, dst_table=dst_table)
    return keep, counts
