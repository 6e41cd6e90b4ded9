"""Draft-tree attention on the paged cache (qcau_b200.tree) against its 64-bit
form: head counts that fill and do not fill a group of rows, one node to many,
one token to long caches, pages that end inside a tile, masks that leave a row
nothing, NaN behind the sequences and among unseen nodes, split and unsplit
schedules; its refusals; the commit of an accepted path."""
import math

import pytest
import torch

import tree_reference as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from qcau_b200 import _lib
    from qcau_b200.cache import PagedKVCache, keep_rows
    from qcau_b200.tree import commit, tree_attn, tree_mask

SCALE = 192 ** -0.5


def check_attention(o, lse, q, rows, nodes, masks, sink, scale):
    """o and lse of every sequence within the tolerances their roundings give.

    o: P is rounded to bf16 (half a step is 2^-8 of it), which moves the sum by
    2^-8 sum(p |v|) at most; the result is rounded to bf16 (2^-8 of it); the
    exponents' error acts on every p alike."""
    for i, r in enumerate(rows):
        want_o, want_lse, _, mag, g = R.attention(q[i].cpu(), r, nodes[i],
                                                  None if masks is None else masks[i].cpu(),
                                                  None if sink is None else sink.cpu(), scale)
        tol = R.score_tolerance(g, want_lse)
        got = lse[i].double().cpu()
        live = torch.isfinite(want_lse)
        assert torch.equal(torch.isfinite(got), live), i
        assert torch.equal(got[~live], want_lse[~live]), i
        off = (got - want_lse).abs()[live]
        assert bool((off <= tol[live]).all()), (i, float((off / tol[live]).max()))
        e = 2 * tol[:, :, None]
        bound = (2.0 ** -8 + e) * mag * (1 + 2.0 ** -8) + 2.0 ** -8 * want_o.abs() + 1e-30
        diff = (o[i].double().cpu() - want_o).abs()
        assert bool((diff <= bound).all()), (i, float((diff / bound).max()))


CASES = [
    # b lens, nodes, s, h, d, page, mask, sink
    dict(lens=[1], nodes=[1], s=1, h=1),
    dict(lens=[2, 1, 65], nodes=[2, 1, 2], s=2, h=3),
    dict(lens=[64, 63, 128, 129], nodes=[1, 1, 1, 1], s=1, h=16),
    dict(lens=[300], nodes=[7], s=7, h=5, sink=True),
    dict(lens=[130, 200], nodes=[8, 8], s=8, h=16, mask="tree"),
    dict(lens=[200, 9, 1000, 13], nodes=[13, 9, 4, 13], s=13, h=16, mask="tree", sink=True),
    dict(lens=[513, 700], nodes=[4, 3], s=4, h=128, mask="tree"),
    dict(lens=[190, 191, 192, 193], nodes=[70, 70, 70, 70], s=70, h=2, mask="tree"),
    dict(lens=[1500], nodes=[33], s=33, h=4, mask="tree", d=512, page=128, sink=True),
    dict(lens=[400, 90], nodes=[5, 5], s=5, h=64, mask="tree", d=512, page=192),
    dict(lens=[40, 50], nodes=[40, 50], s=50, h=8, mask="tree"),
    dict(lens=[300, 280], nodes=[6, 0], s=6, h=16, mask="tree"),
    dict(lens=[500, 300], nodes=[9, 7], s=9, h=16, mask="any"),
    dict(lens=[9, 5], nodes=[9, 5], s=9, h=16, mask="any", sink=True),
    dict(lens=[150, 150], nodes=[6, 6], s=6, h=20, mask="one"),
    # one row over many ranges; teams of two, three and five pairs; many sequences
    dict(lens=[9000], nodes=[8], s=8, h=16, mask="tree"),
    dict(lens=[5200], nodes=[2], s=2, h=128, mask="tree"),
    dict(lens=[5000, 4900], nodes=[3, 3], s=3, h=128, mask="tree", sink=True),
    dict(lens=[2300, 2200, 2100], nodes=[40, 40, 40], s=40, h=16, mask="tree"),
    dict(lens=[129 + 7 * i for i in range(300)], nodes=[1 + i % 3 for i in range(300)], s=3, h=8, mask="tree"),
]


def build(case, seed=1, stale=float("nan")):
    lens, nodes, s, h = case["lens"], case["nodes"], case["s"], case["h"]
    d, page = case.get("d", 576), case.get("page", 64)
    b = len(lens)
    cache, table, rows = R.paged(lens, d, page, seed=seed, stale=stale)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(b, s, h, d, generator=g) * (0.5 + 2 * torch.rand(1, 1, h, 1, generator=g))).to(torch.bfloat16)
    kind = case.get("mask")
    if kind == "tree":
        mask = R.random_tree(b, s, seed)[1]
    elif kind == "any":  # no tree at all: rows that see none of the nodes among them
        mask = torch.rand(b, s, s, generator=g) < 0.3
        mask[:, s // 2] = False
    elif kind == "one":
        mask = R.random_tree(1, s, seed)[1][0]
    else:
        mask = None
    sink = torch.randn(h, generator=g) * 2 if case.get("sink") else None
    return dict(cache=cache, table=table, rows=rows, q=q.cuda(), mask=None if mask is None else mask.cuda(),
                sink=None if sink is None else sink.cuda(),
                seqlens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                tree_lens=torch.tensor(nodes, dtype=torch.int32, device="cuda"), nodes=nodes)


def masks_of(x):
    m = x["mask"]
    return None if m is None else m if m.dim() == 3 else m.expand(len(x["rows"]), -1, -1)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"b{len(c['lens'])}-s{c['s']}-h{c['h']}-{c.get('mask')}-{max(c['lens'])}")
def test_tree_attention_vs_64_bits(case):
    x = build(case)
    o, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE,
                       tree_lens=x["tree_lens"], attn_sink=x["sink"], return_lse=True)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    check_attention(o, lse, x["q"], x["rows"], x["nodes"], masks_of(x), x["sink"], SCALE)
    for i, n in enumerate(x["nodes"]):
        assert bool((o[i, n:] == 0).all()) and bool((lse[i, n:] == -math.inf).all())


def test_rows_that_see_nothing():
    """A new sequence whose mask leaves node 1 nothing: zeros, and the sink's
    value or -inf as its log-sum-exp."""
    x = build(dict(lens=[4], nodes=[4], s=4, h=16))
    mask = torch.eye(4, dtype=torch.bool, device="cuda").unsqueeze(0).contiguous()
    mask[0, 1] = False
    for sink in (None, torch.linspace(-60, 60, 16, device="cuda")):
        o, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], mask, softmax_scale=SCALE,
                           attn_sink=sink, return_lse=True)
        assert bool((o[0, 1] == 0).all())
        if sink is None:
            assert bool((lse[0, 1] == -math.inf).all())
        else:
            assert torch.allclose(lse[0, 1], sink, rtol=2.0 ** -21, atol=0)
        check_attention(o, lse, x["q"], x["rows"], [4], mask, sink, SCALE)
    assert _lib.device_error() == 0


def test_sinks_far_above_and_below_the_scores():
    """A sink of 200 leaves outputs near zero and lse = 200; one of -200 changes nothing."""
    x = build(dict(lens=[300], nodes=[5], s=5, h=16, mask="tree"))
    args = (x["q"], x["cache"], x["table"], x["seqlens"], x["mask"])
    o0, l0 = tree_attn(*args, softmax_scale=SCALE, return_lse=True)
    o1, l1 = tree_attn(*args, softmax_scale=SCALE, attn_sink=torch.full((16,), -200.0, device="cuda"), return_lse=True)
    assert torch.equal(o0, o1) and torch.equal(l0, l1)
    o2, l2 = tree_attn(*args, softmax_scale=SCALE, attn_sink=torch.full((16,), 200.0, device="cuda"), return_lse=True)
    assert torch.allclose(l2, torch.full_like(l2, 200.0), rtol=2.0 ** -21, atol=0)
    assert bool(torch.isfinite(o2.float()).all()) and float(o2.float().abs().max()) < 1e-30


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_unseen_nodes_may_hold_anything(value):
    """Node 2's row is not finite: only the nodes that see it are touched."""
    x = build(dict(lens=[150], nodes=[6], s=6, h=16))
    parents = torch.tensor([[-1, 0, 0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    mask = tree_mask(parents)
    clean = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], mask, softmax_scale=SCALE)
    p = 150 - 6 + 2
    x["cache"][x["table"][0, p // 64], p % 64] = value
    o, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], mask, softmax_scale=SCALE, return_lse=True)
    apart = [0, 1, 3, 5]
    assert torch.equal(o[0, apart], clean[0, apart])
    assert bool(torch.isfinite(lse[0, apart]).all())
    if value != -float("inf"):
        assert bool(torch.isnan(o[0, [2, 4]].float()).all())
    assert _lib.device_error() == 0


def test_tree_mask_marks_ancestors():
    for b, s in ((1, 1), (3, 7), (2, 65), (5, 200)):
        parents, want = R.random_tree(b, s, seed=s)
        assert torch.equal(tree_mask(parents.cuda()).cpu(), want)
    assert _lib.device_error() == 0
    tree_mask(torch.tensor([[-1, 1]], dtype=torch.int32, device="cuda"))
    assert _lib.device_error() == _lib.DEVERR_INDEX


def test_chain_equals_causal_prefill():
    """Without a mask the tree is a chain: the causal attention that the prefill
    entry computes (same roundings, other groupings of rows)."""
    x = build(dict(lens=[333, 90], nodes=[9, 9], s=9, h=128), stale=0.0)
    o = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], softmax_scale=SCALE)
    L = _lib.lib()
    b, s, h, d = x["q"].shape
    most = x["table"].size(1) * 64
    want = torch.empty_like(o)
    need = L.qcau_prefill_attn_workspace_size(b, s, h, 512, most)
    ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
    _lib.check(L.qcau_prefill_attn_paged(
        x["q"].data_ptr(), x["cache"].data_ptr(), x["table"].data_ptr(), x["seqlens"].data_ptr(), None,
        want.data_ptr(), b, s, h, d, 512, d, 64, x["table"].size(1), x["cache"].size(0), most, SCALE,
        ws.data_ptr(), need, _lib.stream_ptr()), "prefill")
    # two roundings of P and two of the result, each half a bf16 step
    for i, r in enumerate(x["rows"]):
        _, _, _, mag, _ = R.attention(x["q"][i].cpu(), r, 9, None, None, SCALE)
        diff = (o[i].double() - want[i].double()).abs().cpu()
        assert bool((diff <= 2.0 ** -6 * mag).all())


def test_same_bits_again_on_another_stream_and_in_a_graph():
    x = build(dict(lens=[4000, 3000], nodes=[12, 10], s=12, h=16, mask="tree", sink=True))

    def call(out=None):
        return tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE,
                         tree_lens=x["tree_lens"], attn_sink=x["sink"], return_lse=True, out=out)

    o, lse = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o1, lse1 = call()
    side.synchronize()
    assert torch.equal(o, o1) and torch.equal(lse, lse1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, lse2 = call()
    for _ in range(2):
        o2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    # the replay reads the lengths live
    x["seqlens"].sub_(1000)
    graph.replay()
    o3, lse3 = call()
    torch.cuda.synchronize()
    assert torch.equal(o3, o2) and torch.equal(lse3, lse2)
    assert _lib.device_error() == 0


def test_strided_queries_and_given_output():
    x = build(dict(lens=[200, 300], nodes=[4, 4], s=4, h=16, mask="tree"))
    args = (x["cache"], x["table"], x["seqlens"], x["mask"])
    want = tree_attn(x["q"], *args, softmax_scale=SCALE)
    wide = torch.zeros(2, 4, 16, 640, device="cuda", dtype=torch.bfloat16)
    wide[..., :576] = x["q"]
    out = torch.full((2, 4, 16, 512), 7.0, device="cuda", dtype=torch.bfloat16)
    got = tree_attn(wide[..., :576], *args, softmax_scale=SCALE, out=out)
    assert got is out and torch.equal(out, want)


def test_lengths_and_pages_out_of_range_are_flagged():
    x = build(dict(lens=[100, 100], nodes=[3, 3], s=3, h=16), stale=0.0)

    def call(seqlens, tree_lens, table, most):
        o = tree_attn(x["q"], x["cache"], table, torch.tensor(seqlens, dtype=torch.int32, device="cuda"),
                      softmax_scale=SCALE, max_seqlen=most,
                      tree_lens=torch.tensor(tree_lens, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        return o

    call([100, 100], [3, 3], x["table"], 128)
    assert _lib.device_error() == 0
    for seqlens, nodes, most in (([100, 100], [3, 3], 90), ([100, -5], [3, 3], 128), ([100, 2], [3, 3], 128),
                                 ([100, 100], [3, 4], 128), ([100, 100], [-1, 3], 128)):
        call(seqlens, nodes, x["table"], most)
        assert _lib.device_error() == _lib.DEVERR_INDEX, (seqlens, nodes, most)
    bad = x["table"].clone()
    bad[1, 0] = x["cache"].size(0)
    good = call([100, 100], [3, 3], x["table"], 128)
    o = call([100, 100], [3, 3], bad, 128)
    assert _lib.device_error() == _lib.DEVERR_INDEX
    assert torch.equal(o[0], good[0])


# ---------------------------------------------------------------- commit


@pytest.mark.parametrize("d,page,k", [(576, 64, 8), (512, 128, 70), (64, 16, 5), (576, 48, 300)])
def test_commit_moves_the_path_in_place(d, page, k):
    b = 5
    base = [0, 1, page - 1, 3 * page, 2 * page + 5]
    cache, table, rows = R.paged([n + k for n in base], d, page, max_pages=(3 * page + k) // page + 1, seed=k, stale=9.0)
    g = torch.Generator().manual_seed(k)
    taken = [0, k, 1, min(k, 3), k // 2]
    path = torch.full((b, k), -7, dtype=torch.int32)
    want = cache.clone()
    for i in range(b):
        nodes = torch.sort(torch.randperm(k, generator=g)[:taken[i]]).values
        path[i, :taken[i]] = nodes.to(torch.int32)
        for j, node in enumerate(nodes.tolist()):
            p = base[i] + j
            want[table[i, p // page], p % page] = rows[i][base[i] + node].cuda()
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    commit(cache, table, torch.tensor(base, dtype=torch.int32, device="cuda"), path.cuda(),
           torch.tensor(taken, dtype=torch.int32, device="cuda"), seqlens=lens)
    torch.cuda.synchronize()
    assert torch.equal(cache, want)
    assert lens.tolist() == [x + y for x, y in zip(base, taken)]
    assert _lib.device_error() == 0


def test_a_path_out_of_order_or_range_is_flagged():
    cache, table, _ = R.paged([200], 64, 64, seed=1, stale=0.0)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for path, count, start in (([3, 2], 2, 10), ([1, 1], 2, 10), ([-1, 2], 2, 10), ([0, 400], 2, 10),
                               ([0, 1], 3, 10), ([0, 1], -1, 10), ([0, 1], 2, 255), ([0, 1], 2, -1)):
        keep_rows(cache, table, torch.tensor([path], dtype=torch.int32, device="cuda"), one * count, start=one * start)
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_INDEX, (path, count, start)
    keep_rows(cache, table, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), one * 2, start=one * 254)
    assert _lib.device_error() == 0


def test_a_drafting_step_end_to_end():
    """Two sequences: a tree is appended, verified and its accepted path
    committed; the next step's attention equals that of a cache that only ever
    held the accepted tokens."""
    dev, d, h = "cuda", 576, 16
    pc = PagedKVCache(num_pages=40, max_seqs=2, max_pages=16, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    lens = [100, 190]
    flat = pc.cache.view(-1, d)
    flat[pc.append([0, 1], lens).long()] = torch.randn(sum(lens), d, device=dev, generator=g).to(torch.bfloat16)
    base = pc.seqlens.clone()
    s = 7
    parents = torch.tensor([[-1, -1, 0, 1, 1, 4, 4], [-1, 0, 0, 2, 3, 3, 5]], dtype=torch.int32, device=dev)
    drafted = torch.randn(2 * s, d, device=dev, generator=g).to(torch.bfloat16)
    flat[pc.append([0, 1], [s, s]).long()] = drafted
    q = torch.randn(2, s, h, d, device=dev, generator=g).to(torch.bfloat16)
    o = tree_attn(q, pc.cache, pc.block_table, pc.seqlens, tree_mask(parents), softmax_scale=SCALE)
    path = torch.tensor([[1, 4, 6], [0, 2, 0]], dtype=torch.int32, device=dev)
    accepted = torch.tensor([3, 2], dtype=torch.int32, device=dev)
    # the accepted path's outputs are those of a chain of just these tokens
    want_rows = []
    for i, n in enumerate(lens):
        take = path[i, :int(accepted[i])].long()
        rows = torch.cat([R.gather(pc.cache, pc.block_table, i, n), drafted[i * s + take]])
        want_rows.append(rows)
        want, _, _, mag, gg = R.attention(q[i, take].cpu(), rows.cpu(), len(take), None, None, SCALE)
        diff = (o[i, take].double().cpu() - want).abs()
        assert bool((diff <= (2.0 ** -7 + 2.0 ** -10) * mag).all())
    commit(pc.cache, pc.block_table, base, path, accepted, seqlens=pc.seqlens)
    pc.truncate([0, 1], [lens[i] + int(accepted[i]) for i in range(2)])
    assert pc.seqlens.tolist() == [103, 192] and pc.length(1) == 192
    for i, rows in enumerate(want_rows):
        assert torch.equal(R.gather(pc.cache, pc.block_table, i, rows.size(0)), rows)
    assert _lib.device_error() == 0


# ---------------------------------------------------------------- refusals


def test_refusals():
    x = build(dict(lens=[100, 90], nodes=[4, 4], s=4, h=16), stale=0.0)
    good = dict(q=x["q"], cache=x["cache"], block_table=x["table"], seqlens=x["seqlens"], softmax_scale=SCALE)

    def refused(exc=ValueError, **change):
        with pytest.raises(exc):
            tree_attn(**{**good, **change})

    refused(q=x["q"].float())
    refused(q=x["q"].cpu())
    refused(q=x["q"][0])
    refused(q=x["q"][..., :512].contiguous())
    refused(q=x["q"][:, :0])
    refused(cache=x["cache"].half())
    refused(cache=x["cache"].transpose(0, 1))
    refused(block_table=x["table"].long())
    refused(block_table=x["table"][:1])
    refused(seqlens=x["seqlens"].long())
    refused(seqlens=x["seqlens"][:1])
    refused(tree_lens=x["tree_lens"].float())
    refused(mask=torch.ones(2, 4, 5, dtype=torch.bool, device="cuda"))
    refused(mask=torch.ones(2, 4, 4, device="cuda"))
    refused(mask=torch.ones(4, 4, 2, dtype=torch.bool, device="cuda").permute(2, 0, 1))
    refused(attn_sink=torch.zeros(15, device="cuda"))
    refused(out=torch.empty(2, 4, 16, 576, device="cuda", dtype=torch.bfloat16))
    refused(max_seqlen=0)
    refused(max_seqlen=x["table"].size(1) * 64 + 1)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(softmax_scale=scale)
    narrow = torch.zeros(4, 64, 128, device="cuda", dtype=torch.bfloat16)
    refused(NotImplementedError, q=x["q"][..., :128].contiguous(), cache=narrow)
    small = torch.zeros(16, 16, 576, device="cuda", dtype=torch.bfloat16)
    refused(NotImplementedError, cache=small, max_seqlen=16)
    with pytest.raises(ValueError):
        tree_mask(torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        tree_mask(torch.zeros(3, 4, device="cuda"))
    k = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    for args in ((k.long(), n), (k, n.long()), (k[0], n), (k, n[:1]), (k[:, :0].contiguous(), n)):
        with pytest.raises(ValueError):
            keep_rows(x["cache"], x["table"], *args)
    with pytest.raises(ValueError):
        keep_rows(x["cache"], x["table"], k, n, dst_cache=narrow)
    with pytest.raises(ValueError):
        commit(x["cache"], x["table"], None, k, n)
    assert _lib.device_error() == 0


def test_empty_batch():
    cache = torch.zeros(2, 64, 576, device="cuda", dtype=torch.bfloat16)
    o, lse = tree_attn(torch.zeros(0, 3, 16, 576, device="cuda", dtype=torch.bfloat16), cache,
                       torch.zeros(0, 2, dtype=torch.int32, device="cuda"),
                       torch.zeros(0, dtype=torch.int32, device="cuda"), softmax_scale=SCALE, return_lse=True)
    assert o.shape == (0, 3, 16, 512) and lse.shape == (0, 3, 16)


def test_idle_slots_have_no_nodes():
    """Without tree_lens a sequence of no tokens, an idle slot of a cache, has no
    nodes: zeros, -inf, and no error; the others as if it were not there."""
    x = build(dict(lens=[200, 300], nodes=[4, 4], s=4, h=16, mask="tree"))
    want, want_lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE, return_lse=True)
    q = torch.cat([x["q"][:1], torch.full_like(x["q"][:1], float("nan")), x["q"][1:]])
    table = torch.stack([x["table"][0], torch.full_like(x["table"][0], -1), x["table"][1]])
    mask = torch.stack([x["mask"][0], x["mask"][0], x["mask"][1]])
    lens = torch.tensor([200, 0, 300], dtype=torch.int32, device="cuda")
    o, lse = tree_attn(q, x["cache"], table, lens, mask, softmax_scale=SCALE, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert torch.equal(o[[0, 2]], want) and torch.equal(lse[[0, 2]], want_lse)
    assert o[1].eq(0).all() and lse[1].eq(-math.inf).all()


def test_two_calls_at_once():
    """Calls on two streams share nothing."""
    xs = [build(dict(lens=[4000, 3000], nodes=[12, 10], s=12, h=16, mask="tree"), seed=3),
          build(dict(lens=[6000], nodes=[3], s=3, h=64), seed=4)]

    def call(x):
        return tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE, tree_lens=x["tree_lens"])

    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(call(xs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])
    assert _lib.device_error() == 0


@pytest.mark.parametrize("k", [5, 300])
@pytest.mark.parametrize("into", ["start", "counts"])
def test_lengths_may_be_updated_in_place(k, into):
    b, page, d = 6, 64, 576
    base, taken = [0, 1, 63, 192, 133, 70], [0, k, 1, 3, k // 2, k]
    cache, table, rows = R.paged([n + k for n in base], d, page, max_pages=(192 + k) // page + 1, seed=k, stale=9.0)
    g = torch.Generator().manual_seed(k)
    path = torch.full((b, k), -7, dtype=torch.int32)
    want = cache.clone()
    for i in range(b):
        nodes = torch.sort(torch.randperm(k, generator=g)[:taken[i]]).values
        path[i, :taken[i]] = nodes.to(torch.int32)
        for j, node in enumerate(nodes.tolist()):
            p = base[i] + j
            want[table[i, p // page], p % page] = rows[i][base[i] + node].cuda()
    start = torch.tensor(base, dtype=torch.int32, device="cuda")
    counts = torch.tensor(taken, dtype=torch.int32, device="cuda")
    lens = start if into == "start" else counts
    commit(cache, table, start, path.cuda(), counts, seqlens=lens)
    torch.cuda.synchronize()
    assert torch.equal(cache, want)
    assert lens.tolist() == [x + y for x, y in zip(base, taken)]
    assert _lib.device_error() == 0


def test_pages_far_into_a_cache():
    """Rows whose offsets pass 32 bits: a cache of 5 GB, the sequence in its last
    pages and its first."""
    pages, d, s, h = 68000, 576, 4, 16
    cache = torch.empty(pages, 64, d, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 31 and cache.numel() * 2 > 2 ** 32
    at = [pages - 1, 5, pages - 2, 60000, 0, pages - 4]
    small, _, _ = R.paged([6 * 64], d, 64, seed=2, stale=0.0)
    small = small[:6].contiguous()
    small.nan_to_num_(0.0)
    cache[at] = small
    table = torch.tensor([at], dtype=torch.int32, device="cuda")
    near = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    lens = torch.tensor([350], dtype=torch.int32, device="cuda")
    q = torch.randn(1, s, h, d, device="cuda").to(torch.bfloat16)
    o = tree_attn(q, cache, table, lens, softmax_scale=SCALE)
    assert torch.equal(o, tree_attn(q, small, near, lens, softmax_scale=SCALE))
    for k in (40, 200):
        keep = torch.sort(torch.randperm(340)[:k]).values.to(torch.int32).view(1, k).cuda()
        n = torch.tensor([k], dtype=torch.int32, device="cuda")
        keep_rows(cache, table, keep, n)
        keep_rows(small, near, keep, n)
        torch.cuda.synchronize()
        assert torch.equal(cache[at], small)
    assert _lib.device_error() == 0


def test_output_over_the_queries_is_refused():
    x = build(dict(lens=[200], nodes=[4], s=4, h=16, d=512))
    with pytest.raises(ValueError, match="overlap"):
        tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], softmax_scale=SCALE, out=x["q"])


@pytest.mark.parametrize("b", [31, 32, 33, 100, 257])
def test_batches_around_the_plan_s_sizes(b):
    """Up to 32 sequences each warp plans for itself, above them the block does, above
    256 in several runs; idle slots among them."""
    g = torch.Generator().manual_seed(b)
    lens = [0 if i % 5 == 3 else int(torch.randint(1, 700, (1,), generator=g)) for i in range(b)]
    x = build(dict(lens=lens, nodes=[min(n, 1 + i % 3) for i, n in enumerate(lens)], s=3, h=8, mask="tree"))
    o, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE,
                       tree_lens=x["tree_lens"], return_lse=True)
    torch.cuda.synchronize()
    live = [i for i, n in enumerate(lens) if n]
    check_attention(o[live], lse[live], x["q"][live], [x["rows"][i] for i in live], [x["nodes"][i] for i in live],
                    x["mask"][live], None, SCALE)
    idle = [i for i, n in enumerate(lens) if not n]
    assert o[idle].eq(0).all() and lse[idle].eq(-math.inf).all()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("b,s,h,most", [(1, 3, 5, 5000), (1, 8, 16, 12000), (3, 8, 16, 6000), (5, 8, 16, 3000), (9, 4, 32, 2500),
                                        (18, 8, 16, 1500), (19, 8, 16, 1500), (2, 33, 8, 4000)])
def test_rows_cut_into_many_pieces(b, s, h, most):
    """Few groups of rows over all ranges: their merge gives a row eight warps, four,
    two or one."""
    g = torch.Generator().manual_seed(most)
    lens = [most] + [int(torch.randint(s, most, (1,), generator=g)) for _ in range(b - 1)]
    x = build(dict(lens=lens, nodes=[s - i % 2 for i in range(b)], s=s, h=h, mask="tree", sink=b % 2 == 1), seed=b)
    o, lse = tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], x["mask"], softmax_scale=SCALE,
                       tree_lens=x["tree_lens"], attn_sink=x["sink"], return_lse=True)
    torch.cuda.synchronize()
    check_attention(o, lse, x["q"], x["rows"], x["nodes"], x["mask"], x["sink"], SCALE)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("k,width,into", [(5, 300, None), (70, 271, None), (300, 600, "start"), (2500, 3000, None)])
def test_commit_moves_the_sums_with_the_rows(k, width, into):
    """The accepted nodes' sums follow their rows and nothing stays of the others,
    in rows of a wider buffer; the cache is moved as without sums."""
    b, page, d = 5, 64, 64
    base = [0, 1, 63, 192, 133]
    taken = [0, k, 1, min(k, 3), k // 2]
    cache, table, _ = R.paged([n + k for n in base], d, page, max_pages=(192 + k) // page + 1, seed=k, stale=9.0)
    g = torch.Generator().manual_seed(k)
    path = torch.full((b, k), -7, dtype=torch.int32)
    wide = torch.rand(b, width + 9, generator=g)
    want = wide.clone()
    want[:, :width] = 0
    for i in range(b):
        nodes = torch.sort(torch.randperm(min(k, width - base[i]), generator=g)[:taken[i]]).values
        taken[i] = len(nodes)
        path[i, :taken[i]] = nodes.to(torch.int32)
        want[i, :base[i]] = wide[i, :base[i]]
        want[i, base[i]:base[i] + taken[i]] = wide[i, base[i] + nodes]
    other, sums = cache.clone(), wide.cuda()
    start = torch.tensor(base, dtype=torch.int32, device="cuda")
    counts = torch.tensor(taken, dtype=torch.int32, device="cuda")
    commit(other, table, start, path.cuda(), counts)
    lens = start if into else torch.zeros_like(start)
    commit(cache, table, start, path.cuda(), counts, seqlens=lens, sums=sums[:, :width])
    torch.cuda.synchronize()
    assert torch.equal(sums.cpu(), want) and torch.equal(cache, other)
    assert lens.tolist() == [x + y for x, y in zip(base, taken)]
    assert _lib.device_error() == 0


def test_sums_of_a_path_out_of_order_or_range_are_flagged():
    """What is not moved raises the error bit; a refused sequence's sums stay, and the
    next one's move."""
    cache, table, _ = R.paged([200, 200], 64, 64, seed=1, stale=0.0)
    for path, count, start in (([3, 2], 2, 10), ([-1, 2], 2, 10), ([0, 90], 2, 10), ([0, 1], 3, 10), ([0, 1], -1, 10),
                               ([0, 1], 2, 255), ([0, 1], 2, 120)):
        sums = torch.rand(2, 100, device="cuda")
        before = sums.clone()
        keep = torch.tensor([path, [0, 4]], dtype=torch.int32, device="cuda")
        keep_rows(cache, table, keep, torch.tensor([count, 2], dtype=torch.int32, device="cuda"),
                  start=torch.tensor([start, 7], dtype=torch.int32, device="cuda"), sums=sums)
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_INDEX, (path, count, start)
        if not 0 <= count <= 2 or start > 100:
            assert torch.equal(sums[0], before[0])
        assert torch.equal(sums[1, :8], before[1, :8]) and sums[1, 8] == before[1, 11] and sums[1, 9:].eq(0).all()


def test_commit_refuses_other_sums():
    cache, table, _ = R.paged([200], 64, 64, seed=1, stale=0.0)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    path = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for sums in (torch.zeros(1, 100), torch.zeros(2, 100, device="cuda"), torch.zeros(100, device="cuda"),
                 torch.zeros(1, 100, device="cuda", dtype=torch.float64), torch.zeros(1, 0, device="cuda")):
        with pytest.raises(ValueError):
            commit(cache, table, one, path, one, sums=sums)
    with pytest.raises(TypeError):
        commit(cache, table, one, path, one, sums=3)


def test_output_over_the_cache_is_refused():
    x = build(dict(lens=[200], nodes=[4], s=4, h=16, d=512))
    before = x["cache"].clone()
    with pytest.raises(ValueError, match="overlap the cache"):
        tree_attn(x["q"], x["cache"], x["table"], x["seqlens"], softmax_scale=SCALE, out=x["cache"].view(-1)[:4 * 16 * 512].view(1, 4, 16, 512))
    torch.cuda.synchronize()
    assert torch.equal(x["cache"].view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("lens", [[60], [2500], [300] * 40])
def test_infinite_sinks_take_all_the_weight(lens):
    """A sink of +inf leaves its head zeros and lse = inf, one of -inf is none; the other
    heads as they are (rows written whole, and merged from pieces)."""
    x = build(dict(lens=lens, nodes=[5] * len(lens), s=5, h=16, mask="tree"))
    args = (x["q"], x["cache"], x["table"], x["seqlens"], x["mask"])
    sink = torch.linspace(-3, 3, 16, device="cuda")
    o, lse = tree_attn(*args, softmax_scale=SCALE, attn_sink=sink, return_lse=True)
    high, none, rest = [2, 9], [0, 15], [i for i in range(16) if i not in (0, 2, 9, 15)]
    bare, bare_lse = tree_attn(*args, softmax_scale=SCALE, return_lse=True)
    sink[high], sink[none] = math.inf, -math.inf
    o2, lse2 = tree_attn(*args, softmax_scale=SCALE, attn_sink=sink, return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(o2[:, :, rest], o[:, :, rest]) and torch.equal(lse2[:, :, rest], lse[:, :, rest])
    assert torch.equal(o2[:, :, none], bare[:, :, none]) and torch.equal(lse2[:, :, none], bare_lse[:, :, none])
    assert o2[:, :, high].eq(0).all() and lse2[:, :, high].eq(math.inf).all()
    assert _lib.device_error() == 0


def test_captured_behind_work_of_another_stream():
    """A capture whose call depends on kernels of two streams, and is waited for by a third."""
    x = build(dict(lens=[900, 700], nodes=[4, 4], s=4, h=16, mask="tree"), stale=0.0)
    base, other = torch.cuda.Stream(), torch.cuda.Stream()
    q, lens = x["q"].clone(), x["seqlens"].clone()
    want = tree_attn(x["q"] * 2, x["cache"], x["table"], x["seqlens"] - 40, x["mask"], softmax_scale=SCALE)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=base):
        other.wait_stream(base)
        q.copy_(x["q"] * 2)
        with torch.cuda.stream(other):
            lens.copy_(x["seqlens"] - 40)
        base.wait_stream(other)
        o = tree_attn(q, x["cache"], x["table"], lens, x["mask"], softmax_scale=SCALE)
        other.wait_stream(base)
        with torch.cuda.stream(other):
            twice = o.float() * 2
        base.wait_stream(other)
    for _ in range(3):
        q.zero_()
        lens.fill_(4)
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(twice, want.float() * 2)
    assert _lib.device_error() == 0
