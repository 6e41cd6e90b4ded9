"""Attention weight sums and eviction on the paged cache (qcau_b200.evict)
against their 64-bit forms: decode steps and trees, groups of rows that are
full, partial and several, the selection's ties, specials and protected tokens
at every size class, moves in place and into other pages, refusals."""
import math

import pytest
import torch

import tree_reference as R
from test_gpu_tree import SCALE, build, masks_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from qcau_b200 import _lib
    from qcau_b200.cache import PagedKVCache, keep_rows
    from qcau_b200.evict import attn_weight_sums, evict, select_rows
    from qcau_b200.tree import tree_attn, tree_mask


def lse_of(x):
    """The log-sum-exps in 64 bits, rounded to the operator's fp32 input."""
    out = []
    masks = masks_of(x)
    for i, r in enumerate(x["rows"]):
        out.append(R.attention(x["q"][i].cpu(), r, x["nodes"][i], None if masks is None else masks[i].cpu(),
                               None if x["sink"] is None else x["sink"].cpu(), SCALE)[1])
    return torch.stack(out).float().cuda()


def check_sums(x, lse, got, before=None, most=None):
    """A weight's exponent may be off by the scores' tolerance; the fp32 sum over
    n rows loses n * 2^-24 of it at most (they are added 256 at a time: fewer)."""
    masks = masks_of(x)
    for i, r in enumerate(x["rows"]):
        n, q = r.size(0), x["q"][i].cpu()
        s, h = q.shape[:2]
        m = None if masks is None else masks[i].cpu()
        _, _, _, _, g = R.attention(q, r, x["nodes"][i], m, None, SCALE)
        xs = torch.einsum("thd,nd->thn", q.double(), r.double()) * SCALE
        vis = R.seen(n, x["nodes"][i], s, m)[:, None, :].expand(s, h, n)
        w = torch.where(vis, torch.exp(xs - lse[i].double().cpu()[:, :, None]), torch.zeros_like(xs))
        want = w.sum((0, 1))
        tol = (w * 2 * R.score_tolerance(g, lse[i].double().cpu())[:, :, None]).sum((0, 1)) + s * h * 2.0 ** -24 * want
        if before is not None:
            want = want + before[i, :n].double().cpu()
            tol = tol + 2.0 ** -24 * want.abs()
        diff = (got[i, :n].double().cpu() - want).abs()
        assert bool((diff <= tol + 1e-30).all()), (i, float((diff / (tol + 1e-30)).max()))
        rest = got[i, n:most]
        assert bool((rest == (0 if before is None else before[i, n:most])).all())


CASES = [
    dict(lens=[1], nodes=[1], s=1, h=1),
    dict(lens=[63, 64, 65, 200], nodes=[1, 1, 1, 1], s=1, h=16),
    dict(lens=[130, 300], nodes=[1, 1], s=1, h=128, sink=True),
    dict(lens=[130, 77], nodes=[1, 1], s=1, h=100),
    dict(lens=[300, 150], nodes=[5, 3], s=5, h=7, mask="tree"),
    dict(lens=[200, 9, 400, 13], nodes=[13, 9, 4, 13], s=13, h=16, mask="tree"),
    dict(lens=[190, 191], nodes=[70, 69], s=70, h=1, mask="tree"),
    dict(lens=[300, 280], nodes=[6, 0], s=6, h=16, mask="any"),
    dict(lens=[200, 150, 140], nodes=[9, 4, 9], s=9, h=64, mask="tree"),
    dict(lens=[700], nodes=[5], s=5, h=128, mask=None),
    dict(lens=[500, 400], nodes=[17, 17], s=17, h=16, mask="one", d=512, page=128),
    dict(lens=[9000], nodes=[1], s=1, h=16),
    dict(lens=[5100, 5000], nodes=[6, 6], s=6, h=64, mask="tree"),
    dict(lens=[129 + 7 * i for i in range(300)], nodes=[1 + i % 3 for i in range(300)], s=3, h=8, mask="tree"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"b{len(c['lens'])}-s{c['s']}-h{c['h']}-{c.get('mask')}-{max(c['lens'])}")
def test_weight_sums_vs_64_bits(case):
    x = build(case)
    lse = lse_of(x)
    args = (x["q"], x["cache"], x["table"], x["seqlens"], lse, x["mask"])
    got = attn_weight_sums(*args, softmax_scale=SCALE, tree_lens=x["tree_lens"])
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert got.shape == (len(x["rows"]), x["table"].size(1) * x["cache"].size(1))
    check_sums(x, lse, got)
    # added to sums of a wider buffer, whose other positions stay
    wide = torch.rand(got.size(0), got.size(1) + 13, device="cuda")
    before = wide.clone()
    most = max(case["lens"])
    back = attn_weight_sums(*args, softmax_scale=SCALE, tree_lens=x["tree_lens"], max_seqlen=most, sums=wide)
    assert back is wide
    check_sums(x, lse, wide, before, most)
    assert torch.equal(wide[:, most:], before[:, most:])
    # no atomics: the same bits again
    assert torch.equal(attn_weight_sums(*args, softmax_scale=SCALE, tree_lens=x["tree_lens"]), got)
    assert _lib.device_error() == 0


def test_queries_of_missing_nodes_and_unseen_rows_may_hold_anything():
    x = build(dict(lens=[200, 150], nodes=[4, 2], s=4, h=16, mask="tree"))
    lse = lse_of(x)
    args = (x["cache"], x["table"], x["seqlens"], lse, x["mask"])
    want = attn_weight_sums(x["q"], *args, softmax_scale=SCALE, tree_lens=x["tree_lens"])
    x["q"][1, 2:] = float("nan")
    lse[1, 2:] = float("nan")
    got = attn_weight_sums(x["q"], *args, softmax_scale=SCALE, tree_lens=x["tree_lens"])
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())


def test_weights_of_one_step_sum_to_its_rows():
    """With the attention's own log-sum-exps every row's weights sum to 1, so all
    of a step's to rows (each off by its exponent's error: under 1e-4 here)."""
    x = build(dict(lens=[777, 2000], nodes=[1, 1], s=1, h=128))
    _, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], softmax_scale=SCALE, return_lse=True)
    w = attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], lse, softmax_scale=SCALE)
    assert torch.allclose(w.double().sum(1), torch.full((2,), 128.0, dtype=torch.float64, device="cuda"), rtol=1e-4)


# ---------------------------------------------------------------- selection


def plain_select(sums, lens, budget, n_first, n_recent):
    """Stable sort of one row at a time, from the definition."""
    keep = torch.full((len(lens), budget), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        key = sums[i, :n].cpu().clone()
        key = torch.where(torch.isnan(key), torch.full_like(key, math.inf), key).double()
        key[torch.isnan(sums[i, :n].cpu())] = 2.0 ** 200  # above infinity's place below
        key = torch.where(torch.isinf(key) & (key > 0), torch.full_like(key, 2.0 ** 199), key)
        key[:n_first] = 2.0 ** 300
        if n_recent:
            key[max(0, n - n_recent):] = 2.0 ** 300
        order = torch.sort(key, descending=True, stable=True).indices[:budget]
        at = torch.sort(order).values
        keep[i, :len(at)] = at.to(torch.int32)
    return keep


@pytest.mark.parametrize("width", [1, 65, 1024, 4096, 4097, 8193, 16384, 16385, 32768, 32769, 70001, 270001])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "specials"])
def test_selection_equals_the_stable_sort(width, kind):
    g = torch.Generator().manual_seed(width)
    lens = [width, max(1, width // 3), max(1, width - 1), 1, 0]
    sums = torch.rand(len(lens), width, generator=g).pow(6)
    if kind == "ties":
        sums = torch.randint(0, 4, sums.shape, generator=g).float() / 4
    elif kind == "equal":
        sums = torch.full_like(sums, 0.25)
    elif kind == "specials":
        sums = sums - 0.1
        sums[:, ::5], sums[:, 1::7], sums[:, 2::11] = float("nan"), math.inf, -math.inf
        sums[:, 3::9], sums[:, 4::13] = 0.0, -0.0
    for budget, first, recent in ((1, 0, 0), (max(1, width // 4), min(4, width // 8), min(16, width // 9)),
                                  (max(1, width - 2), 0, 1), (width, 0, 0), (width + 3, 1, 1)):
        if first + recent > budget:
            continue
        dev = sums.cuda()
        out = torch.full_like(dev, 5.0)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        keep, counts = select_rows(dev, n, budget, n_first=first, n_recent=recent, sums_out=out)
        want = plain_select(sums, lens, budget, first, recent)
        assert torch.equal(keep.cpu(), want), (budget, first, recent)
        assert counts.tolist() == [min(v, budget) for v in lens]
        moved = torch.zeros_like(sums)
        for i, c in enumerate(counts.tolist()):
            moved[i, :c] = sums[i, want[i, :c].long()]
        assert torch.equal(torch.nan_to_num(out.cpu(), nan=7.0), torch.nan_to_num(moved, nan=7.0))
        # the sums' own buffer
        again, _ = select_rows(dev, n, budget, n_first=first, n_recent=recent, sums_out=dev)
        assert torch.equal(again, keep) and torch.equal(torch.nan_to_num(dev, nan=7.0), torch.nan_to_num(out, nan=7.0))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("b,width", [(160, 5000), (80, 9000), (40, 20000), (160, 40000)])
def test_selection_of_many_sequences(b, width):
    """More sequences than SMs: one block each, or clusters of two and four."""
    g = torch.Generator().manual_seed(b)
    lens = torch.randint(1, width + 1, (b,), generator=g).tolist()
    lens[0] = width
    sums = torch.randint(0, 3000, (b, width), generator=g).float()
    budget = width // 3
    keep, counts = select_rows(sums.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), budget, n_first=2,
                               n_recent=7)
    assert torch.equal(keep.cpu(), plain_select(sums, lens, budget, 2, 7))
    assert counts.tolist() == [min(n, budget) for n in lens]


def test_lengths_out_of_range_are_flagged():
    sums = torch.rand(2, 100, device="cuda")
    for lens in ([100, 101], [-1, 100]):
        keep, counts = select_rows(sums, torch.tensor(lens, dtype=torch.int32, device="cuda"), 10)
        assert counts.tolist() == [min(max(v, 0), 10) for v in lens]
        assert _lib.device_error() == _lib.DEVERR_INDEX


# ---------------------------------------------------------------- the cache


@pytest.mark.parametrize("lens,budget,d,page", [([700, 64, 1500, 1], 300, 576, 64), ([5000], 2000, 576, 64),
                                                ([900, 3000], 2999, 512, 128), ([300] * 40, 100, 64, 16),
                                                ([12000], 9001, 576, 64), ([9000, 9500, 20], 8000, 512, 128)])
@pytest.mark.parametrize("inplace", [True, False])
def test_evict_moves_rows_and_sums(lens, budget, d, page, inplace):
    cache, table, rows = R.paged(lens, d, page, seed=2, stale=3.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    sums = torch.rand(len(lens), max(lens), device="cuda", generator=g)
    for i, n in enumerate(lens):
        sums[i, n:] = 0
    first_sums, first_cache = sums.clone(), cache.clone()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = plain_select(sums, lens, budget, 2, 5 if budget > 7 else 0)
    kw = {}
    if not inplace:
        dst, dtab, _ = R.paged([min(budget, max(lens))] * len(lens), d, page, seed=5, stale=-4.0)
        dst.fill_(-4.0)
        kw = dict(dst_cache=dst, dst_table=dtab, sums_out=torch.full_like(sums, 5.0))
    keep, counts = evict(cache, table, n, sums, budget, n_first=2, n_recent=5, **kw)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert torch.equal(keep.cpu(), want)
    to, to_table = (cache, table) if inplace else (kw["dst_cache"], kw["dst_table"])
    expect = first_cache.clone() if inplace else torch.full_like(to, -4.0)
    moved = torch.zeros_like(sums)
    for i, c in enumerate(counts.tolist()):
        at = want[i, :c].long()
        moved[i, :c] = first_sums[i, at.cuda()]
        for p in range(0, c, page):
            expect[to_table[i, p // page], :min(page, c - p)] = rows[i][at[p:p + page]].cuda()
    assert torch.equal(to, expect)
    assert torch.equal(sums if inplace else kw["sums_out"], moved)
    if not inplace:
        assert torch.equal(cache, first_cache) and torch.equal(sums, first_sums)


def test_decode_with_a_bounded_cache():
    """Steps of decode over a growing cache: attention, its weights into the running
    sums, an eviction when the budget is passed, and attention again.  The
    kept rows and sums are those a plain loop keeps."""
    dev, d, h, budget = "cuda", 576, 16, 96
    pc = PagedKVCache(num_pages=12, max_seqs=2, max_pages=4, device=dev)
    g = torch.Generator(device=dev).manual_seed(9)
    flat = pc.cache.view(-1, d)
    most = pc.max_pages * pc.page_size
    sums = torch.zeros(2, most, device=dev)
    kept = [torch.empty(0, d, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    held = [torch.zeros(0, dtype=torch.float64, device=dev) for _ in range(2)]
    evictions = 0
    for step, new in enumerate(([90, 60], [1, 1], [5, 1], [1, 40], [1, 1], [1, 1])):
        slots = pc.append([0, 1], new)
        fresh = torch.randn(sum(new), d, device=dev, generator=g).to(torch.bfloat16)
        flat[slots.long()] = fresh
        for i in range(2):
            kept[i] = torch.cat([kept[i], fresh[:new[0]] if i == 0 else fresh[new[0]:]])
            held[i] = torch.cat([held[i], torch.zeros(new[i], dtype=torch.float64, device=dev)])
        q = torch.randn(2, 1, h, d, device=dev, generator=g).to(torch.bfloat16)
        o, lse = tree_attn(q, pc.cache, pc.block_table, pc.seqlens, softmax_scale=SCALE, return_lse=True)
        attn_weight_sums(q, pc.cache, pc.block_table, pc.seqlens, lse, softmax_scale=SCALE, sums=sums)
        for i in range(2):
            want, wl, p, mag, gg = R.attention(q[i].cpu(), kept[i].cpu(), 1, None, None, SCALE)
            assert bool(((o[i].double().cpu() - want).abs() <= (2.0 ** -7 + 2.0 ** -10) * mag).all())
            held[i] = held[i] + p.sum((0, 1)).cuda()
            assert torch.allclose(sums[i, :len(held[i])].double(), held[i], rtol=1e-4, atol=1e-9)
        if max(pc.length(0), pc.length(1)) > budget:
            evictions += 1
            before = sums.clone()
            keep, lens = evict(pc.cache, pc.block_table, pc.seqlens, sums, budget, n_first=2, n_recent=8)
            pc.truncate([0, 1], lens.tolist())
            for i in range(2):
                at = plain_select(before, [len(kept[0]), len(kept[1])], budget, 2, 8)[i]
                at = at[at >= 0].long().cuda()
                kept[i], held[i] = kept[i][at], held[i][at]
                assert torch.equal(R.gather(pc.cache, pc.block_table, i, len(at)), kept[i])
    assert evictions >= 2 and pc.seqlens.tolist() == [len(kept[0]), len(kept[1])]
    assert _lib.device_error() == 0


def test_captured_step_replays():
    """Attention, weights and eviction captured in one graph and replayed on new
    contents give the eager calls' bits."""
    x = build(dict(lens=[700, 650], nodes=[4, 4], s=4, h=16, mask="tree"), stale=0.0)
    sums = torch.rand(2, 704, device="cuda")
    dst, dtab, _ = R.paged([300, 300], 576, 64, seed=4, stale=0.0)
    out = torch.zeros_like(sums)

    def step():
        _, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE, return_lse=True)
        w = attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], lse, x["mask"], softmax_scale=SCALE)
        keep, lens = evict(x["cache"], x["table"], x["seqlens"], w, 300, n_first=1, n_recent=9, dst_cache=dst,
                           dst_table=dtab, sums_out=out)
        return keep, lens

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError):  # the sums' rows must have the positions of the weights
        step_bad = torch.zeros(2, 703, device="cuda")
        attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], torch.zeros(2, 4, 16, device="cuda"),
                         softmax_scale=SCALE, sums=step_bad)
    with torch.cuda.graph(graph):
        keep, lens = step()
    x["q"].copy_(torch.randn(x["q"].shape, device="cuda").to(torch.bfloat16))
    x["seqlens"].sub_(100)
    graph.replay()
    torch.cuda.synchronize()
    got = [keep.clone(), lens.clone(), dst.clone(), out.clone()]
    dst.zero_()
    k2, l2 = step()
    torch.cuda.synchronize()
    assert torch.equal(got[0], k2) and torch.equal(got[1], l2) and torch.equal(got[3], out)
    for i, n in enumerate(l2.tolist()):
        for p in range(0, n, 64):
            m = min(64, n - p)
            assert torch.equal(got[2][dtab[i, p // 64], :m], dst[dtab[i, p // 64], :m])
    assert _lib.device_error() == 0


# ---------------------------------------------------------------- refusals


def test_refusals():
    x = build(dict(lens=[100, 90], nodes=[4, 4], s=4, h=16), stale=0.0)
    lse = torch.zeros(2, 4, 16, device="cuda")

    def no(fn, *a, exc=ValueError, **k):
        with pytest.raises(exc):
            fn(*a, **k)

    base = (x["q"], x["cache"], x["table"], x["seqlens"])
    no(attn_weight_sums, *base, lse.double(), softmax_scale=SCALE)
    no(attn_weight_sums, *base, lse[:, :3], softmax_scale=SCALE)
    no(attn_weight_sums, *base, lse.cpu(), softmax_scale=SCALE)
    no(attn_weight_sums, *base, lse, softmax_scale=-SCALE)
    no(attn_weight_sums, *base, lse, softmax_scale=SCALE, sums=torch.zeros(2, 100, device="cuda"))
    no(attn_weight_sums, *base, lse, softmax_scale=SCALE, sums=torch.zeros(2, 128, device="cuda", dtype=torch.float64))
    no(attn_weight_sums, *base, lse, softmax_scale=SCALE, sums=torch.zeros(128, 2, device="cuda").t())
    no(attn_weight_sums, *base, lse, softmax_scale=SCALE, sums=torch.zeros(1, 128, device="cuda").expand(2, 128))
    sums, n = torch.rand(2, 128, device="cuda"), x["seqlens"]
    kept = sums.clone()
    no(select_rows, sums, n, 0)
    no(select_rows, sums, n, -1)
    no(select_rows, sums, n, 10, n_first=6, n_recent=5)
    no(select_rows, sums, n, 10, n_first=-1)
    no(select_rows, sums.half(), n, 10)
    no(select_rows, sums, n.long(), 10)
    no(select_rows, sums[:1], n, 10)
    no(select_rows, sums, n, 10, sums_out=sums[:, :64])
    no(evict, x["cache"], x["table"][:1], n, sums, 10)
    no(evict, x["cache"], x["table"], n[:1], sums, 10)
    no(evict, x["cache"], x["table"], n, torch.rand(2, 129, device="cuda"), 10)
    no(evict, x["cache"].half(), x["table"], n, sums, 10)
    no(evict, x["cache"], x["table"], n, sums, 100, dst_table=x["table"][:, :1].contiguous())
    no(evict, x["cache"], x["table"], n, sums, 10, dst_cache=torch.zeros(4, 32, 576, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(sums, kept)  # nothing was touched
    assert _lib.device_error() == 0


def test_empty_batch():
    cache = torch.zeros(2, 64, 576, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    n = torch.zeros(0, dtype=torch.int32, device="cuda")
    w = attn_weight_sums(torch.zeros(0, 3, 16, 576, device="cuda", dtype=torch.bfloat16), cache, table, n,
                         torch.zeros(0, 3, 16, device="cuda"), softmax_scale=SCALE)
    assert w.shape == (0, 128)
    keep, lens = evict(cache, table, n, w, 5)
    assert keep.shape == (0, 5) and lens.shape == (0,)
    keep_rows(cache, table, keep, lens)
    assert tree_mask(torch.zeros(0, 4, dtype=torch.int32, device="cuda")).shape == (0, 4, 4)


def test_a_step_with_idle_slots():
    """A decode step of a cache whose other slots are empty: no error, sums of 0
    there, nothing kept."""
    pc = PagedKVCache(num_pages=16, max_seqs=4, max_pages=6)
    g = torch.Generator().manual_seed(8)
    slots = pc.append([1, 3], [300, 130])
    pc.cache.view(-1, 576)[slots.long()] = torch.randn(430, 576, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(4, 1, 16, 576, generator=g).to(torch.bfloat16).cuda()
    o, lse = tree_attn(q, pc.cache, pc.block_table, pc.seqlens, softmax_scale=SCALE, return_lse=True)
    sums = attn_weight_sums(q, pc.cache, pc.block_table, pc.seqlens, lse, softmax_scale=SCALE)
    total = sums.sum(1)
    assert total[[0, 2]].eq(0).all() and o[[0, 2]].eq(0).all()
    # 16 rows' weights, 1 in all each: an exponent is off by 2^-19 of sum |q k| * scale
    # (576 * 0.64 * 0.073 = 27) plus 2^-20 * (1 + lse), under 2^-13; sums lose less
    assert (total[[1, 3]] - 16).abs().max() < 16 * 2.0 ** -12
    before = pc.cache.clone()
    keep, lens = evict(pc.cache, pc.block_table, pc.seqlens, sums, 128, n_first=4, n_recent=16)
    torch.cuda.synchronize()
    assert lens.tolist() == [0, 128, 0, 128] and keep[[0, 2]].eq(-1).all()
    for i in (1, 3):
        rows = R.gather(before, pc.block_table, i, 300)
        assert torch.equal(R.gather(pc.cache, pc.block_table, i, 128), rows[keep[i].long()])
    assert _lib.device_error() == 0


def test_sums_of_pages_far_into_a_cache():
    """Rows whose offsets pass 32 bits: a cache of 5 GB."""
    pages, d = 68000, 576
    cache = torch.empty(pages, 64, d, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 31 and cache.numel() * 2 > 2 ** 32
    at = [pages - 1, 5, pages - 2, 60000, 0, pages - 4]
    small = torch.randn(6, 64, d, device="cuda").to(torch.bfloat16)
    cache[at] = small
    table = torch.tensor([at], dtype=torch.int32, device="cuda")
    near = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    lens = torch.tensor([350], dtype=torch.int32, device="cuda")
    for h in (16, 128, 400):
        q = torch.randn(1, 1, h, d, device="cuda").to(torch.bfloat16)
        lse = tree_attn(q, small, near, lens, softmax_scale=SCALE, return_lse=True)[1]
        w = attn_weight_sums(q, cache, table, lens, lse, softmax_scale=SCALE)
        assert torch.equal(w, attn_weight_sums(q, small, near, lens, lse, softmax_scale=SCALE))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("b,s,h", [(32, 1, 16), (33, 1, 16), (100, 2, 64), (40, 5, 64), (257, 1, 8)])
def test_sums_of_many_sequences(b, s, h):
    g = torch.Generator().manual_seed(b)
    lens = [0 if i % 5 == 3 else int(torch.randint(1, 900, (1,), generator=g)) for i in range(b)]
    x = build(dict(lens=lens, nodes=[min(n, 1 + i % s) for i, n in enumerate(lens)], s=s, h=h, mask="tree"))
    lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE,
                    tree_lens=x["tree_lens"], return_lse=True)[1]
    got = attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], lse, x["mask"], softmax_scale=SCALE,
                           tree_lens=x["tree_lens"])
    torch.cuda.synchronize()
    live = [i for i, n in enumerate(lens) if n]
    some = dict(rows=[x["rows"][i] for i in live], nodes=[x["nodes"][i] for i in live], q=x["q"][live], mask=x["mask"][live])
    check_sums(some, lse[live], got[live])
    assert got[[i for i, n in enumerate(lens) if not n]].eq(0).all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("s,h,n", [(60, 1, 500), (64, 4, 200), (37, 1, 40), (90, 2, 300), (70, 3, 129)])
def test_sums_of_trees_of_few_heads(s, h, n):
    """Many nodes in a group of rows, their masks read several at a time."""
    x = build(dict(lens=[n, max(s, n // 2)], nodes=[min(s, n), min(s, max(s, n // 2)) - 3], s=s, h=h, mask="any"))
    lse = lse_of(x)
    got = attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], lse, x["mask"], softmax_scale=SCALE,
                           tree_lens=x["tree_lens"])
    torch.cuda.synchronize()
    check_sums(x, lse, got)
    assert _lib.device_error() == 0


def test_calls_in_a_row_see_what_ran_before_them():
    """Launches overlap the kernels before them; inputs that change between calls, by
    kernels of torch and of this package, are read as they then are."""
    g = torch.Generator().manual_seed(12)
    b, s, h, most = 3, 4, 16, 2000
    x = build(dict(lens=[most] * b, nodes=[s] * b, s=s, h=h, mask="tree"), stale=0.0)
    q, lens, nodes = x["q"].clone(), x["seqlens"].clone(), x["tree_lens"].clone()
    steps = [(torch.randint(s, most + 1, (b,), generator=g).to(torch.int32).cuda(),
              torch.randn(q.shape, generator=g).to(torch.bfloat16).cuda()) for _ in range(12)]

    def step(n, qs, cache):
        lens.copy_(n)
        q.copy_(qs)
        o, lse = tree_attn(q, cache, x["table"], lens, x["mask"], softmax_scale=SCALE, tree_lens=nodes, return_lse=True)
        w = attn_weight_sums(q, cache, x["table"], lens, lse, x["mask"], softmax_scale=SCALE, tree_lens=nodes)
        keep, counts = evict(cache, x["table"], lens, w, 500, n_first=2, n_recent=8)
        o2 = tree_attn(q, cache, x["table"], counts, x["mask"], softmax_scale=SCALE, tree_lens=nodes)
        return o, lse, w, keep, counts, o2

    caches = [x["cache"].clone(), x["cache"].clone()]
    slow = []
    for n, qs in steps:
        caches[0].copy_(x["cache"])
        out = step(n, qs, caches[0])
        torch.cuda.synchronize()
        slow.append([t.clone() for t in out] + [caches[0].clone()])
    fast = []
    for _ in range(3):
        for k, (n, qs) in enumerate(steps):
            caches[1].copy_(x["cache"])
            fast.append((k, [*step(n, qs, caches[1]), caches[1].clone()]))
    torch.cuda.synchronize()
    for k, got in fast:
        for a, c in zip(got, slow[k]):
            assert torch.equal(a, c), k
    assert _lib.device_error() == 0


def test_a_refused_eviction_changes_nothing():
    """A cache view that is not 16-byte aligned, or whose pages are too many, is refused
    before the sums are compacted in place."""
    n = torch.full((1,), 128, dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    flat = torch.randn(2 * 64 * 64 + 8, device="cuda").to(torch.bfloat16)
    odd, even = flat[1:1 + 2 * 64 * 64].view(2, 64, 64), flat[:2 * 64 * 64].view(2, 64, 64)
    sums = torch.rand(1, 128, device="cuda")
    rows_before, sums_before = flat.clone(), sums.clone()
    for cache, dst in ((odd, None), (even, odd)):
        with pytest.raises(ValueError, match="aligned"):
            evict(cache, table, n, sums, 20, dst_cache=dst)
    many = 65536
    with pytest.raises(NotImplementedError, match="too large"):
        all_sums = sums.expand(many, 128).contiguous()
        evict(even, table.expand(many, 2).contiguous(), n.expand(many).contiguous(), all_sums, 20)
    torch.cuda.synchronize()
    assert torch.equal(all_sums, sums_before.expand(many, 128))
    assert torch.equal(sums, sums_before) and torch.equal(flat, rows_before)
    evict(even, table, n, sums, 20)
    assert not torch.equal(sums, sums_before)
    assert _lib.device_error() == 0


def test_sums_out_over_part_of_the_sums():
    """Views shifted against one another are refused and nothing is touched; the two
    halves of one buffer's rows are other memory."""
    buf = torch.rand(5, 200, device="cuda")
    before = buf.clone()
    n = torch.tensor([100, 90, 100], dtype=torch.int32, device="cuda")
    flat = buf.view(-1)
    for out in (buf[1:4, :100], buf[:3, 50:150], flat[1:601].view(3, 200)[:, :100], flat[:300].view(3, 100)):
        with pytest.raises(ValueError, match="overlap"):
            select_rows(buf[:3, :100], n, 20, sums_out=out)
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    keep, _ = select_rows(buf[:3, :100], n, 20, sums_out=buf[:3, 100:])
    assert torch.equal(keep.cpu(), plain_select(before, [100, 90, 100], 20, 0, 0))
    assert torch.equal(buf[:3, 100:120], before[:3].gather(1, keep.long()))
    assert torch.equal(buf[:3, :100], before[:3, :100]) and buf[:3, 120:].eq(0).all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("s,h,mask", [(1, 16, None), (5, 12, "tree"), (60, 1, "any"), (1, 128, None), (8, 16, "tree"), (25, 4, "any")])
@pytest.mark.parametrize("d,page", [(512, 64), (512, 128), (576, 128), (512, 192)])
def test_sums_of_both_widths_and_larger_pages(s, h, mask, d, page):
    """Groups of 64 and 128 rows, whose tiles are two blocks a CTA: blocks of one page, of
    two, and past the sequence's end; the last chain of a 512-wide row is shorter."""
    x = build(dict(lens=[700, 257, 128, max(s, 65)], nodes=[s, s, s, s - s // 3], s=s, h=h, mask=mask, d=d, page=page))
    lse = lse_of(x)
    got = attn_weight_sums(x["q"], x["cache"], x["table"], x["seqlens"], lse, x["mask"], softmax_scale=SCALE,
                           tree_lens=x["tree_lens"])
    torch.cuda.synchronize()
    check_sums(x, lse, got)
    assert _lib.device_error() == 0


def test_one_sequence_s_sums_in_place_whatever_the_stride():
    """A view of one row has no stride to speak of: the same memory is the same sums."""
    buf = torch.rand(1, 300, device="cuda")
    one = buf[:, :100]                       # stride 300
    same = torch.as_strided(buf, (1, 100), (100, 1))
    before, n = one.clone(), torch.tensor([100], dtype=torch.int32, device="cuda")
    keep, _ = select_rows(one, n, 20, sums_out=same)
    assert torch.equal(keep.cpu(), plain_select(before, [100], 20, 0, 0))
    assert torch.equal(buf[:, :20], before.gather(1, keep.long())) and buf[:, 20:100].eq(0).all()
    assert _lib.device_error() == 0
