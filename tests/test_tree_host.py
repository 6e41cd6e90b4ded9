"""Draft-tree and eviction entry points without a GPU: workspace sizes, the C
ABI's refusals before any device work, and the page bookkeeping."""
import numpy as np
import pytest
import torch

from qcau_b200 import _lib
from qcau_b200.cache import PagedKVCache

_HOST = [np.zeros(1 << 16, dtype=np.uint8) for _ in range(8)]
P = [int((a.ctypes.data + 15) // 16 * 16) for a in _HOST]

no_device = pytest.mark.skipif(torch.cuda.is_available(),
                               reason="argument checks with host buffers run without a device")


def _expect(rc, exc, text):
    with pytest.raises(exc) as e:
        _lib.check(rc, "call")
    assert text in str(e.value), str(e.value)


def test_workspaces_do_not_grow_with_the_batch():
    """Two slots of 128 rows per CTA pair whatever the batch; none of the partial
    sums while a sequence's rows are one group."""
    L = _lib.lib()
    pair = 2 * 128 * (512 + 2) * 4 + 16
    assert L.qcau_tree_attn_workspace_size(1, 1, 16, 1) == pair
    assert L.qcau_tree_attn_workspace_size(64, 64, 128, 32768) == 74 * pair
    assert L.qcau_attn_weight_sums_workspace_size(32, 1, 128, 16384) == 0
    assert L.qcau_attn_weight_sums_workspace_size(7, 24, 32, 6001) == 3 * 7 * 6004 * 4


@no_device
def test_tree_attn_refusals():
    L = _lib.lib()
    good = dict(q=P[0], cache=P[1], table=P[2], seqlens=P[3], nodes=0, mask=0, sink=0, o=P[4], lse=0, sums=0, ws=P[5],
                stride=0, b=1, s=4, h=16, d=576, dv=512, page=64, max_pages=4, num_pages=8, most=200, sums_stride=0,
                ws_bytes=1 << 30, scale=0.07, accumulate=0)

    def call(**change):
        return L.qcau_tree_attn(_lib.TreeArgs(*{**good, **change}.values()), None)

    _expect(L.qcau_tree_attn(None, None), ValueError, "NULL")

    for change, exc, text in (
            (dict(q=0), ValueError, "NULL"), (dict(o=0), ValueError, "NULL"), (dict(s=0), ValueError, "bad shape"),
            (dict(h=0), ValueError, "bad shape"), (dict(b=-1), ValueError, "bad shape"), (dict(most=0), ValueError, "max_seqlen"),
            (dict(most=257), ValueError, "max_seqlen"), (dict(d=128), NotImplementedError, "d_qk"),
            (dict(page=16), ValueError, "max_seqlen"), (dict(page=96), NotImplementedError, "page_size"),
            (dict(mask=P[6], stride=15), ValueError, "stride"), (dict(scale=0.0), ValueError, "softmax_scale"),
            (dict(scale=float("nan")), ValueError, "softmax_scale"), (dict(q=P[0] + 2), ValueError, "aligned"),
            (dict(cache=P[1] + 8), ValueError, "aligned"), (dict(o=P[4] + 4), ValueError, "aligned"),
            (dict(ws_bytes=100), ValueError, "workspace"), (dict(ws=0), ValueError, "workspace"),
            (dict(b=1 << 17), NotImplementedError, "too large"), (dict(s=1 << 22), NotImplementedError, "too large"),
            (dict(num_pages=1 << 31), NotImplementedError, "too large")):
        _expect(call(**change), exc, text)
    assert call(b=0) == 0


@no_device
def test_weight_sums_refusals():
    L = _lib.lib()
    good = dict(q=P[0], cache=P[1], table=P[2], seqlens=P[3], nodes=0, mask=0, sink=0, o=0, lse=P[4], sums=P[5], ws=0,
                stride=0, b=1, s=4, h=16, d=576, dv=512, page=64, max_pages=4, num_pages=8, most=200, sums_stride=200,
                ws_bytes=0, scale=0.07, accumulate=0)

    def call(**change):
        return L.qcau_attn_weight_sums(_lib.TreeArgs(*{**good, **change}.values()), None)

    _expect(L.qcau_attn_weight_sums(None, None), ValueError, "NULL")

    for change, exc, text in (
            (dict(lse=0), ValueError, "NULL"), (dict(sums=0), ValueError, "NULL"), (dict(sums_stride=199), ValueError, "row of sums"),
            (dict(page=32), ValueError, "max_seqlen"), (dict(page=100), NotImplementedError, "page_size"),
            (dict(d=64), NotImplementedError, "d_qk"), (dict(scale=-1.0), ValueError, "softmax_scale"),
            (dict(s=40), ValueError, "workspace")):
        _expect(call(**change), exc, text)
    assert call(b=0) == 0


@no_device
def test_select_and_keep_refusals():
    L = _lib.lib()
    good = dict(sums=P[0], seqlens=P[1], keep=P[2], counts=P[3], out=0, stride=100, out_stride=0, b=1, n=100, budget=10,
                first=2, recent=3)

    def select(**change):
        return L.qcau_evict_select(_lib.SelectArgs(*{**good, **change}.values()), None)

    _expect(L.qcau_evict_select(None, None), ValueError, "NULL")

    for change, text in ((dict(keep=0), "NULL"), (dict(budget=0), "bad shape"), (dict(n=0), "bad shape"),
                         (dict(first=8), "budget"), (dict(first=-1), "budget"), (dict(recent=-1), "budget"),
                         (dict(stride=99), "row of sums"), (dict(out=P[4], out_stride=99), "row of sums")):
        _expect(select(**change), ValueError, text)
    assert select(b=0) == 0
    good_rows = dict(cache=P[0], table=P[1], dst=P[0], dst_table=P[1], keep=P[2], counts=P[3], start=0, lens=0, max_pages=4,
                     num_pages=8, dst_max_pages=4, dst_num_pages=8, keep_stride=5, b=1, k=5, d=576, page=64)

    def rows(**change):
        return L.qcau_keep_rows(_lib.KeepArgs(*{**good_rows, **change}.values()), None)

    _expect(L.qcau_keep_rows(None, None), ValueError, "NULL")

    for change, exc, text in ((dict(dst=0), ValueError, "NULL"), (dict(k=0), ValueError, "bad shape"),
                              (dict(keep_stride=4), ValueError, "bad shape"), (dict(page=0), ValueError, "bad shape"),
                              (dict(d=24), ValueError, "multiple of 16"), (dict(cache=P[0] + 2), ValueError, "aligned"),
                              (dict(b=70000), NotImplementedError, "too large"),
                              (dict(max_pages=1 << 26), NotImplementedError, "too large")):
        _expect(rows(**change), exc, text)
    assert rows(b=0) == 0
    _expect(L.qcau_tree_mask(None, P[0], 1, 4, None), ValueError, "NULL")
    _expect(L.qcau_tree_mask(P[0], P[1], 1, 0, None), ValueError, "bad shape")


def test_truncate_returns_pages():
    pc = PagedKVCache(num_pages=12, max_seqs=2, max_pages=8, width=16, device="cpu")
    pc.append([0, 1], [300, 100])
    assert pc.free_pages == 12 - 5 - 2
    table = pc.block_table.clone()
    pc.truncate([0, 1], [129, 100])
    assert pc.free_pages == 12 - 3 - 2 and pc.length(0) == 129 and pc.seqlens.tolist() == [129, 100]
    assert torch.equal(pc.block_table[0, :3], table[0, :3]) and pc.block_table[0, 3:].eq(0).all()
    rows = pc.append([0], [63])  # fills the last page
    assert rows[0] == int(table[0, 2]) * 64 + 1 and pc.free_pages == 7
    pc.truncate([0], [0])
    assert pc.free_pages == 10 and pc.length(0) == 0
    for bad in (-1, 101):
        with pytest.raises(ValueError):
            pc.truncate([0, 1], [0, bad])
    assert pc.length(1) == 100


def test_truncate_takes_each_sequence_once():
    """A second, longer length of a sequence would name pages already returned."""
    pc = PagedKVCache(num_pages=12, max_seqs=2, max_pages=8, width=16, device="cpu")
    pc.append([0, 1], [300, 100])
    for seqs, lengths in (([0, 0], [10, 200]), ([0, 1], [10]), ([0], [10, 20])):
        with pytest.raises(ValueError):
            pc.truncate(seqs, lengths)
        assert pc.length(0) == 300 and pc.free_pages == 5


@no_device
def test_overlapping_results_are_refused():
    L = _lib.lib()
    step = dict(q=P[0], cache=P[1], table=P[2], seqlens=P[3], nodes=0, mask=0, sink=0, o=P[0] + 512, lse=0, sums=0, ws=P[5],
                stride=0, b=1, s=1, h=2, d=512, dv=512, page=64, max_pages=4, num_pages=8, most=200, sums_stride=0,
                ws_bytes=1 << 30, scale=0.07, accumulate=0)
    for o in (P[0], P[0] + 2032, P[0] - 2032):
        _expect(L.qcau_tree_attn(_lib.TreeArgs(*{**step, "o": o}.values()), None), ValueError, "overlap")
    rows = dict(cache=P[0], table=P[1], dst=P[0], dst_table=P[1], keep=P[2], counts=P[3], start=P[4], lens=0, max_pages=4,
                num_pages=8, dst_max_pages=4, dst_num_pages=8, keep_stride=5, b=3, k=5, d=576, page=64)
    for lens in (P[3] + 4, P[3] - 8, P[4] + 8, P[4] - 4):
        _expect(L.qcau_keep_rows(_lib.KeepArgs(*{**rows, "lens": lens}.values()), None), ValueError, "overlap")


@no_device
def test_sizes_past_64_bits_are_refused():
    L = _lib.lib()
    step = dict(q=P[0], cache=P[1], table=P[2], seqlens=P[3], nodes=0, mask=0, sink=0, o=P[4], lse=0, sums=0, ws=P[5],
                stride=0, b=1, s=1, h=2, d=576, dv=512, page=64, max_pages=4, num_pages=8, most=200, sums_stride=0,
                ws_bytes=1 << 30, scale=0.07, accumulate=0)
    for change in (dict(max_pages=(1 << 58) + 4), dict(page=(1 << 62) + 64, max_pages=8)):
        _expect(L.qcau_tree_attn(_lib.TreeArgs(*{**step, **change}.values()), None), ValueError, "bad shape")


def test_the_binding_refuses_host_tensors_and_other_types():
    """The compiled binding loads without a device, and refuses before any device work."""
    from qcau_b200 import evict as E
    from qcau_b200 import tree as T

    q = torch.zeros(1, 2, 4, 576, dtype=torch.bfloat16)
    cache, table = torch.zeros(2, 64, 576, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32)
    lens, sums = torch.ones(1, dtype=torch.int32), torch.zeros(1, 128)
    with pytest.raises(ValueError, match="CUDA"):
        T.tree_attn(q, cache, table, lens, softmax_scale=0.07)
    with pytest.raises(ValueError, match="CUDA"):
        E.attn_weight_sums(q, cache, table, lens, torch.zeros(1, 2, 4), softmax_scale=0.07)
    with pytest.raises(ValueError, match="CUDA"):
        E.select_rows(sums, lens, 10)
    with pytest.raises(ValueError, match="CUDA"):
        E.evict(cache, table, lens, sums, 10)
    with pytest.raises(ValueError, match="CUDA"):
        T.commit(cache, table, lens, table, lens)
    with pytest.raises(TypeError, match="q must be a tensor"):
        T.tree_attn(None, cache, table, lens, softmax_scale=0.07)
    with pytest.raises(TypeError, match="mask must be a tensor or None"):
        T.tree_attn(q, cache, table, lens, 3, softmax_scale=0.07)
    with pytest.raises(TypeError, match="softmax_scale"):
        T.tree_attn(q, cache, table, lens, softmax_scale="x")
    with pytest.raises(ValueError, match="base_lens"):
        T.commit(cache, table, None, table, lens)


@no_device
def test_keep_rows_sums_refusals():
    L = _lib.lib()
    good = dict(cache=P[0], table=P[1], dst=P[0], dst_table=P[1], keep=P[2], counts=P[3], start=0, lens=0, max_pages=4,
                num_pages=8, dst_max_pages=4, dst_num_pages=8, keep_stride=5, b=1, k=5, d=576, page=64)

    def call(sums=P[4], stride=100, n=100, **change):
        return L.qcau_keep_rows_sums(_lib.KeepArgs(*{**good, **change}.values()), sums, stride, n, None)

    _expect(L.qcau_keep_rows_sums(None, P[4], 100, 100, None), ValueError, "NULL")
    for change, exc, text in ((dict(sums=0), ValueError, "NULL"), (dict(stride=99), ValueError, "row of sums"),
                              (dict(n=0), ValueError, "row of sums"), (dict(n=1 << 31, stride=1 << 31), NotImplementedError, "too large"),
                              (dict(keep=0), ValueError, "NULL"), (dict(k=6), ValueError, "bad shape"),
                              (dict(d=24), ValueError, "multiple of 16"), (dict(cache=P[0] + 2), ValueError, "aligned"),
                              (dict(b=70000), NotImplementedError, "too large")):
        _expect(call(**change), exc, text)
    assert call(b=0) == 0


@no_device
def test_evict_refuses_before_anything_is_launched():
    """What the move of the rows refuses is refused before the selection runs: it
    changes the sums.  (A launch without a device would be another error.)"""
    L = _lib.lib()
    select = dict(sums=P[0], seqlens=P[1], keep=P[2], counts=P[3], out=P[0], stride=100, out_stride=100, b=1, n=100, budget=10,
                  first=2, recent=3)
    rows = dict(cache=P[4], table=P[5], dst=P[4], dst_table=P[5], keep=0, counts=0, start=0, lens=0, max_pages=4,
                num_pages=8, dst_max_pages=4, dst_num_pages=8, keep_stride=0, b=0, k=0, d=576, page=64)

    def call(s={}, r={}):
        return L.qcau_evict(_lib.SelectArgs(*{**select, **s}.values()), _lib.KeepArgs(*{**rows, **r}.values()), None)

    _expect(L.qcau_evict(None, None, None), ValueError, "NULL")
    for s, r, exc, text in ((dict(budget=0), {}, ValueError, "bad shape"), (dict(first=9), {}, ValueError, "budget"),
                            ({}, dict(cache=P[4] + 2), ValueError, "aligned"), ({}, dict(dst=P[4] + 8), ValueError, "aligned"),
                            ({}, dict(d=24), ValueError, "multiple of 16"), ({}, dict(table=0), ValueError, "NULL"),
                            (dict(b=70000), {}, NotImplementedError, "too large"),
                            ({}, dict(num_pages=1 << 26), NotImplementedError, "too large"),
                            (dict(n=257, stride=257, out_stride=257), {}, ValueError, "does not hold"),
                            (dict(budget=80), dict(dst_max_pages=1), ValueError, "does not hold")):
        _expect(call(s, r), exc, text)
    assert call(dict(b=0)) == 0


def _rows(start, stride, b, n):
    return {start + i * stride + j for i in range(b) for j in range(n)}


@no_device
def test_sums_out_that_overlaps_sums_is_refused():
    """A block of one sequence would write what another's has not read.  Rows between the
    other's rows share nothing; every offset of both is tried against the set of places."""
    L = _lib.lib()

    def refused(off, stride, out_stride, b, n):
        at = P[0] + (1 << 14)
        # (a misaligned cache: what passes the overlap check must not launch)
        args = dict(sums=at, seqlens=P[1], keep=P[2], counts=P[3], out=at + 4 * off, stride=stride, out_stride=out_stride, b=b,
                    n=n, budget=1, first=0, recent=0)
        cache = dict(cache=P[4] + 2, table=P[5], dst=P[4], dst_table=P[5], keep=0, counts=0, start=0, lens=0, max_pages=4,
                     num_pages=8, dst_max_pages=4, dst_num_pages=8, keep_stride=0, b=0, k=0, d=576, page=64)
        rc = L.qcau_evict(_lib.SelectArgs(*args.values()), _lib.KeepArgs(*cache.values()), None)
        with pytest.raises(ValueError) as e:
            _lib.check(rc, "call")
        assert "overlap" in str(e.value) or "aligned" in str(e.value)
        return "overlap" in str(e.value)

    for stride, b, n in ((10, 1, 10), (10, 3, 10), (20, 3, 10), (21, 3, 10), (17, 4, 10), (40, 2, 7)):
        for off in range(-4 * stride - 3, 4 * stride + 4):
            want = off != 0 and bool(_rows(0, stride, b, n) & _rows(off, stride, b, n))
            assert refused(off, stride, stride, b, n) == want, (off, stride, b, n)
    # other strides: by the extents, and the same pointer too
    for off, want in ((0, True), (5, True), (29, True), (30, False), (-34, False), (-33, True)):
        assert refused(off, 10, 12, 3, 10) is want, off


@no_device
def test_output_over_the_cache_is_refused():
    L = _lib.lib()
    step = dict(q=P[0], cache=P[1], table=P[2], seqlens=P[3], nodes=0, mask=0, sink=0, o=P[1], lse=0, sums=0, ws=P[5],
                stride=0, b=1, s=1, h=2, d=512, dv=512, page=64, max_pages=1, num_pages=1, most=64, sums_stride=0,
                ws_bytes=1 << 30, scale=0.07, accumulate=0)
    for o in (P[1], P[1] + 65536 - 16, P[1] - 2032):
        _expect(L.qcau_tree_attn(_lib.TreeArgs(*{**step, "o": o}.values()), None), ValueError, "overlap the cache")
