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


def _check_sums(what: str, sums: torch.Tensor, b: int, index: int):
    """(positions, row stride) of sums [b, positions]."""
    shape = sums.shape
    if len(shape) != 2 or sums.dtype != torch.float32 or sums.get_device() != index:
        raise ValueError(f"{what}: sums must be fp32 [batch, positions] on the device of the others")
    (rows, n), (step, one) = shape, sums.stride()
    if rows != b or (n > 1 and one != 1) or (b > 1 and step < n):
        raise ValueError(f"{what}: sums needs one contiguous row per sequence")
    return n, max(step, n)


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
    index, q, (b, s, h, d), stride, pages, most = _check_step(
        "attn_weight_sums", q, cache, block_table, seqlens, mask, tree_lens, max_seqlen)
    if lse.dtype != torch.float32 or lse.shape != (b, s, h) or not lse.is_contiguous() \
            or lse.get_device() != index:
        raise ValueError("attn_weight_sums: lse must be a contiguous fp32 [batch, nodes, heads] tensor")
    add = sums is not None
    if add:
        n, sums_stride = _check_sums("attn_weight_sums", sums, b, index)
        if n < most:
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
    index = seqlens.get_device()
    if index < 0:
        require_cuda(seqlens)
    out = _check_select("select_rows", index, sums, seqlens, seqlens.numel(), sums_out)
    return _launch_select(index, sums, seqlens, budget, n_first, n_recent, sums_out, out)


def _check_select(what: str, index: int, sums, seqlens, b: int, sums_out):
    """(sequences, positions, row strides of sums and sums_out)."""
    _check_ints(what, "seqlens", seqlens, (b,), index)
    n, stride = _check_sums(what, sums, b, index)
    if sums_out is None:
        return b, n, stride, 0
    if sums_out is sums:
        return b, n, stride, stride
    out_n, out_stride = _check_sums(what, sums_out, b, index)
    if out_n != n or (sums_out.data_ptr() == sums.data_ptr() and out_stride != stride):
        raise ValueError(f"{what}: sums_out must have the shape of sums, and be sums or other memory")
    return b, n, stride, out_stride


def _launch_select(index, sums, seqlens, budget, n_first, n_recent, sums_out, sizes):
    b, n, stride, out_stride = sizes
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
    if sums_out is None:
        sums_out = sums
    index = cache.get_device()
    move = _check_move("evict", cache, block_table, dst_cache, dst_table)
    _, _, (_, page, _, b, max_pages), _, dst_max = move
    sizes = _check_select("evict", index, sums, seqlens, b, sums_out)
    n = sizes[1]
    if n > max_pages * page or min(budget, n) > dst_max * page:
        raise ValueError("evict: a block table does not hold the positions of sums, or the budget")
    keep, counts = _launch_select(index, sums, seqlens, budget, n_first, n_recent, sums_out, sizes)
    _launch_keep(index, cache, block_table, move, keep, budget, counts, 0, 0)
    return keep, counts
