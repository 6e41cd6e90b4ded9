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

from ._lib import (call_on, data, lib, pack_select_args, pack_tree_args, require_cuda,
                   workspace_size)
from .cache import _check_ints, _check_move, _launch_keep
from .tree import _check_step


def _check_sums(what: str, sums: torch.Tensor, b: int, index: int) -> int:
    """The row stride of sums [b, positions]."""
    if sums.dim() != 2 or sums.dtype != torch.float32 or sums.get_device() != index:
        raise ValueError(f"{what}: sums must be fp32 [batch, positions] on the device of the lengths")
    (rows, n), (step, one) = sums.shape, sums.stride()
    if rows != b or (n > 1 and one != 1) or (b > 1 and step < n):
        raise ValueError(f"{what}: sums needs one contiguous row per sequence")
    return max(step, n)


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
    q, stride, pages, most = _check_step("attn_weight_sums", q, cache, block_table, seqlens, mask,
                                         tree_lens, max_seqlen)
    b, s, h, d = q.shape
    index = q.get_device()
    if lse.dtype != torch.float32 or lse.shape != (b, s, h) or not lse.is_contiguous() \
            or lse.get_device() != index:
        raise ValueError("attn_weight_sums: lse must be a contiguous fp32 [batch, nodes, heads] tensor")
    add = sums is not None
    if add:
        sums_stride = _check_sums("attn_weight_sums", sums, b, index)
        if sums.size(1) < most:
            raise ValueError("attn_weight_sums: a row of sums must hold max_seqlen values")
    else:
        sums = torch.empty((b, most), dtype=torch.float32, device=q.device)
        sums_stride = most
    need = workspace_size("qcau_attn_weight_sums_workspace_size", b, s, h, most)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    args = pack_tree_args(
        q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), seqlens.data_ptr(),
        data(tree_lens), data(mask), 0, 0, lse.data_ptr(), sums.data_ptr(), data(ws), stride, b, s, h,
        d, 512, *pages, most, sums_stride, need, softmax_scale, add)
    call_on(index, "attn_weight_sums", lib().qcau_attn_weight_sums, args)
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
    b, index = seqlens.numel(), seqlens.get_device()
    if index < 0:
        require_cuda(seqlens)
    _check_ints("select_rows", "seqlens", seqlens, (b,), index)
    stride = _check_sums("select_rows", sums, b, index)
    n, out_stride = sums.size(1), 0
    if sums_out is sums:
        out_stride = stride
    elif sums_out is not None:
        out_stride = _check_sums("select_rows", sums_out, b, index)
        if sums_out.size(1) != n:
            raise ValueError("select_rows: sums_out must have the shape of sums")
        if sums_out.data_ptr() == sums.data_ptr() and out_stride != stride:
            raise ValueError("select_rows: in place, sums_out must be sums")
    keep = torch.empty((b, max(budget, 0)), dtype=torch.int32, device=seqlens.device)
    counts = torch.empty_like(seqlens)
    args = pack_select_args(sums.data_ptr(), seqlens.data_ptr(), keep.data_ptr(), counts.data_ptr(),
                            data(sums_out), stride, out_stride, b, n, budget, n_first, n_recent)
    call_on(index, "evict_select", lib().qcau_evict_select, args)
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
    if seqlens.numel() != dt.size(0) or sums.get_device() != cache.get_device():
        raise ValueError("evict: one length per block-table row, and all tensors on one device")
    n = sums.size(-1)
    if n > block_table.size(1) * cache.size(1) or min(budget, n) > dt.size(1) * dc.size(1):
        raise ValueError("evict: a block table does not hold the positions of sums, or the budget")
    keep, counts = select_rows(sums, seqlens, budget, n_first=n_first, n_recent=n_recent,
                               sums_out=sums if sums_out is None else sums_out)
    _launch_keep(cache, block_table, dc, dt, keep, counts, None, None)
    return keep, counts
