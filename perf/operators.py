"""Speculative decoding and cache eviction on the paged latent cache: the calls that are measured.

Four operators over a paged cache of bf16 rows [pages, page, width] (576 = 512 latent + 64 rope values, V the first 512;
or 512-wide rows that are K and V), one latent row per token shared by all heads:

  tree      attention of a tree of drafted tokens over the cache (which holds their rows), with its log-sum-exp
  weights   the attention weight that every cached token received, summed over the query tokens and heads
  evict     the tokens to keep by those sums (the first and the most recent ones always), and the cache brought down to them
  commit    a drafting step's end: the rows of the accepted path move up behind the sequence, in place

Where `own` is false, run() computes them with elementary torch operations in 32 bits.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

VALUE = 512  # values of a row that are V


@functools.cache
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from qcau_b200 import evict, tree
    return tree, evict


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one user's request at low latency: a small draft tree, the heads of one of eight shards, a short cache
        dict(name="tree, one sequence", op="tree", b=1, s=8, h=16, d=576, len=1003, page=64, ragged=False, sink=False),
        # a serving batch with all heads on the GPU, trees and sequences of different sizes
        dict(name="tree, batch of 32", op="tree", b=32, s=8, h=128, d=576, len=4096, page=64, ragged=True, sink=False),
        # long contexts with the heads of one shard and a wide tree
        dict(name="tree, long contexts", op="tree", b=16, s=64, h=16, d=576, len=32768, page=64, ragged=False, sink=False),
        # 512-wide rows with an attention sink, odd sizes, larger pages, new sequences without a prefix among them
        dict(name="tree, 512 wide, sink", op="tree", b=23, s=13, h=64, d=512, len=2501, page=128, ragged=True, sink=True),
        # a decode step of a short sequence: one query token, 16 heads
        dict(name="weights, one sequence", op="weights", b=1, s=1, h=16, d=576, len=777, page=64, ragged=False, sink=False),
        # a decode step of a batch at long contexts, all heads
        dict(name="weights, decode batch", op="weights", b=32, s=1, h=128, d=576, len=16384, page=64, ragged=False, sink=False),
        # a verification step's weights: the rows of a tree, odd sizes
        dict(name="weights, tree", op="weights", b=7, s=24, h=32, d=576, len=6001, page=64, ragged=True, sink=False),
        # one sequence over its budget
        dict(name="evict, one sequence", op="evict", b=1, d=576, len=5003, budget=1024, first=4, recent=64, page=64, ragged=False),
        # a batch brought from 16384 tokens to a quarter
        dict(name="evict, batch of 32", op="evict", b=32, d=576, len=16384, budget=4096, first=16, recent=512, page=64, ragged=False),
        # ragged sequences, some below the budget, odd sizes
        dict(name="evict, ragged", op="evict", b=9, d=512, len=9001, budget=999, first=1, recent=33, page=128, ragged=True),
        # the end of a drafting step for one sequence
        dict(name="commit, one sequence", op="commit", b=1, s=8, d=576, len=1003, page=64, ragged=False),
        # the same for a batch
        dict(name="commit, batch of 128", op="commit", b=128, s=32, d=576, len=641, page=64, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "evict", "commit"])
    case = dict(op=op, d=rng.choice([576, 576, 512]), page=rng.choice([64, 64, 128]), ragged=rng.random() < 0.7)
    most = 524288  # cached tokens of all sequences
    if op in ("tree", "weights"):
        s = _log(rng, 1, 64)
        h = rng.choice([1, 5, 8, 16, 16, 32, 64, 128, 128])
        n = _log(rng, max(64, s), 32768)
        room = min(most, (16 if op == "tree" else 4) * 32768 * 1024 // (s * h)) // n
        case.update(b=_log(rng, 1, max(1, min(64, room))), s=s, h=h, len=n, sink=rng.random() < 0.3)
    elif op == "evict":
        n = _log(rng, 65, 32768)
        budget = _log(rng, max(1, n // 16), n)
        first = rng.randint(0, min(16, budget))
        recent = rng.randint(0, min(512, budget - first))
        case.update(b=_log(rng, 1, max(1, min(64, most // n))), len=n, budget=budget, first=first, recent=recent)
    else:
        s = _log(rng, 1, 64)
        n = _log(rng, max(64, s), 2048)
        case.update(b=_log(rng, 1, 128), s=s, len=n)
    return case


def _mean_len(case):
    return case["len"] * (0.625 if case["ragged"] else 1.0)


def work(case):
    b, d, n = case["b"], case["d"], _mean_len(case)
    if case["op"] in ("tree", "weights"):
        rows = b * case["s"] * case["h"]
        k, q = 2 * d * b * n, 2 * d * rows
        if case["op"] == "tree":  # the cache once, queries, outputs, their log-sum-exps
            return {"bytes": k + q + rows * (2 * VALUE + 4), "flops": 2.0 * rows * n * (d + VALUE)}
        return {"bytes": k + q + 4 * rows + 4 * b * case["len"], "flops": 2.0 * rows * n * d}
    if case["op"] == "evict":  # the sums read once and written once; each kept row read and written
        kept = b * min(case["budget"], n)
        return {"bytes": 4 * b * n + 4 * b * case["len"] + kept * (4 * d + 4), "flops": 0.0}
    moved = b * (1 + case["s"]) / 2  # written as drafted, the accepted ones read and written
    return {"bytes": moved * 8 * d, "flops": 0.0}


# ---------------------------------------------------------------- inputs


def _lengths(case, seed, least):
    r = np.random.RandomState(seed % (1 << 31))
    b, n = case["b"], case["len"]
    if not case["ragged"]:
        return np.full(b, n)
    got = r.randint(min(n, max(n // 4, least)), n + 1, b)
    got[r.randint(b)] = n
    return got


def _pages(case, g, dev, extra=0):
    """A cache with its pages in a random order, as a pool that has been in use hands them out."""
    per = -(-(case["len"] + extra) // case["page"])
    pages = case["b"] * per
    cache = torch.randn(pages, case["page"], case["d"], generator=g, device=dev)
    cache *= torch.rsqrt(cache.square().mean(-1, keepdim=True) + 1e-6)
    table = torch.randperm(pages, generator=g, device=dev).to(torch.int32).view(case["b"], per).contiguous()
    return cache.to(torch.bfloat16), table


def _tree(case, seed, dev):
    """Random draft trees: for each node the index of its parent (-1: the last token of the sequence)."""
    b, s = case["b"], case["s"]
    r = np.random.RandomState((seed + 77) % (1 << 31))
    parents = np.maximum(np.arange(s)[None, :] - 1 - r.randint(0, 4, (b, s)), -1)
    counts = np.full(b, s) if not case["ragged"] else r.randint(1, s + 1, b)
    a = torch.zeros(b, s, s + 1, device=dev)
    a.scatter_(2, torch.from_numpy(parents + 1).to(dev).unsqueeze(-1), 1.0)
    seen = a[:, :, 1:] + torch.eye(s, device=dev)
    for _ in range(max(1, s.bit_length())):
        seen = (seen @ seen > 0).float()
    return parents, counts, seen > 0


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    state = dict(case=case)
    if op in ("tree", "weights"):
        b, s, h, d = case["b"], case["s"], case["h"], case["d"]
        cache, table = _pages(case, g, dev)
        _, counts, mask = _tree(case, seed, dev)
        lens = np.maximum(_lengths(case, seed, s), counts)
        if case["ragged"] and b > 3:
            lens[b // 2] = counts[b // 2]  # a new sequence: nothing before its tree
        # heads differ in how sharply they attend
        sharp = 0.5 + 2.0 * torch.rand(1, 1, h, 1, generator=g, device=dev)
        state.update(
            q=(torch.randn(b, s, h, d, generator=g, device=dev) * sharp).to(torch.bfloat16),
            cache=cache, table=table, mask=mask, scale=192 ** -0.5,
            lens=torch.from_numpy(lens).to(dev, torch.int32), nodes=torch.from_numpy(counts).to(dev, torch.int32),
            sink=torch.randn(h, generator=g, device=dev) if case["sink"] else None)
        if op == "weights":  # what the attention that ran before left
            state["lse"] = _attention(state)[1]
    elif op == "evict":
        cache, table = _pages(case, g, dev)
        lens = _lengths(case, seed, 1)
        sums = torch.rand(case["b"], case["len"], generator=g, device=dev).pow(8) * 10 + 1e-4  # few tokens take most
        fresh = dict(case, len=case["budget"])
        kept, kept_table = _pages(fresh, g, dev)
        state.update(cache=cache, table=table, lens=torch.from_numpy(lens).to(dev, torch.int32), sums=sums,
                     kept=kept, kept_table=kept_table, kept_sums=torch.zeros_like(sums))
    else:
        b, s, d = case["b"], case["s"], case["d"]
        cache, table = _pages(case, g, dev, extra=s)
        base = _lengths(case, seed, 0)
        parents, counts, _ = _tree(case, seed, dev)
        r = np.random.RandomState((seed + 5) % (1 << 31))
        path, taken = np.full((b, s), -1), np.zeros(b, np.int64)
        for i in range(b):  # the accepted path ends at a random node
            at, back = r.randint(-1, counts[i]), []
            while at >= 0:
                back.append(at)
                at = parents[i, at]
            taken[i] = len(back)
            path[i, :len(back)] = back[::-1]
        pos = base[:, None] + np.arange(s)[None, :]
        slots = np.take_along_axis(table.cpu().numpy().astype(np.int64), pos // case["page"], 1) * case["page"] + pos % case["page"]
        state.update(cache=cache, table=table, base=torch.from_numpy(base).to(dev, torch.int32),
                     slots=torch.from_numpy(slots.reshape(-1)).to(dev),
                     drafted=torch.randn(b * s, d, generator=g, device=dev).to(torch.bfloat16),
                     path=torch.from_numpy(path).to(dev, torch.int32), taken=torch.from_numpy(taken).to(dev, torch.int32),
                     lens=torch.zeros(b, dtype=torch.int32, device=dev))
    return state


# ---------------------------------------------------------------- the plain form


def _seen(st, n):
    """Which cached positions [n] each query token sees [b, s, n]."""
    dev, s = st["q"].device, st["q"].size(1)
    pos = torch.arange(n, device=dev)
    base = (st["lens"] - st["nodes"]).long()
    at = pos[None, :] - base[:, None]                                     # node of each position
    inside = (at >= 0) & (at < st["nodes"][:, None])
    tree = st["mask"].gather(2, at.clamp(0, s - 1)[:, None, :].expand(-1, s, -1))
    seen = (at < 0)[:, None, :] | (tree & inside[:, None, :])
    return seen & (torch.arange(s, device=dev)[None, :, None] < st["nodes"][:, None, None])


def _scores(st):
    """The cached rows in token order [b, n, d], the scaled scores [b, s * h, n] and who sees what [b, s * h, n], all in 32 bits."""
    b, s, h, d = st["q"].shape
    n = st["case"]["len"]
    live = torch.arange(n, device=st["q"].device)[None, :] < st["lens"][:, None]
    rows = st["cache"][st["table"].long()].view(b, -1, d)[:, :n].float()
    rows = rows.masked_fill(~live[:, :, None], 0.0)
    scores = torch.bmm(st["q"].float().view(b, s * h, d), rows.transpose(1, 2)) * st["scale"]
    seen = _seen(st, n)[:, :, None, :].expand(b, s, h, n).reshape(b, s * h, n)
    return rows, scores, seen


def _attention(st):
    b, s, h, d = st["q"].shape
    rows, scores, seen = _scores(st)
    scores = scores.masked_fill(~seen, -math.inf)
    real = (torch.arange(s, device=scores.device)[None, :] < st["nodes"][:, None])[:, :, None].expand(b, s, h).reshape(b, s * h)
    sink = st["sink"].float().view(1, 1, h).expand(b, s, h).reshape(b, s * h) if st["sink"] is not None else torch.full_like(real, -math.inf, dtype=torch.float32)
    top = torch.maximum(scores.amax(-1), sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top[:, :, None])
    total = e.sum(-1) + torch.exp(sink - top)
    o = torch.bmm(e, rows[:, :, :VALUE]) / total.clamp_min(1e-38)[:, :, None]
    lse = torch.where(real, top + torch.log(total), torch.full_like(top, -math.inf))
    return o.to(torch.bfloat16).view(b, s, h, VALUE), lse.view(b, s, h)


def _weights(st):
    b, s, h, _ = st["q"].shape
    _, scores, seen = _scores(st)
    w = torch.exp(scores - st["lse"].view(b, s * h, 1))
    return torch.where(seen, w, torch.zeros_like(w)).sum(1)


def _rows_of(table, pos, page):
    return table.long().gather(1, pos // page) * page + pos % page


def _evict(st):
    case = st["case"]
    n, budget, page = case["len"], case["budget"], case["page"]
    pos = torch.arange(n, device=st["sums"].device)[None, :]
    lens = st["lens"][:, None]
    sure = (pos < case["first"]) | (pos >= lens - case["recent"])
    rank = torch.where(sure, math.inf, st["sums"])
    rank = torch.where(pos < lens, rank, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    counts = torch.minimum(st["lens"], torch.full_like(st["lens"], budget))
    i = torch.arange(budget, device=order.device)[None, :]
    live = i < counts[:, None]
    keep = torch.sort(torch.where(live, order, n), dim=1).values
    src = _rows_of(st["table"], keep.clamp(max=n - 1), page)
    dst = _rows_of(st["kept_table"], i.expand_as(keep), page)
    flat, kept = st["cache"].view(-1, case["d"]), st["kept"].view(-1, case["d"])
    kept[dst] = torch.where(live[:, :, None], flat[src], kept[dst])
    st["kept_sums"].zero_()
    st["kept_sums"][:, :budget] = torch.where(live, st["sums"].gather(1, keep.clamp(max=n - 1)), 0.0)
    return torch.where(live, keep, -1).to(torch.int32), counts, st["kept"], st["kept_sums"]


def _commit(st):
    case = st["case"]
    flat = st["cache"].view(-1, case["d"])
    flat.index_copy_(0, st["slots"], st["drafted"])
    i = torch.arange(case["s"], device=flat.device)[None, :]
    live = i < st["taken"][:, None]
    base = st["base"].long()[:, None]
    src = _rows_of(st["table"], base + torch.where(live, st["path"].long(), i), case["page"])
    dst = _rows_of(st["table"], base + i, case["page"])
    flat[dst] = flat[src]
    return st["cache"], st["base"] + st["taken"]


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        return {"tree": _attention, "weights": _weights, "evict": _evict, "commit": _commit}[op](st)
    tree, evict = _package()
    if op == "tree":
        return tree.tree_attn(st["q"], st["cache"], st["table"], st["lens"], st["mask"], softmax_scale=st["scale"],
                              tree_lens=st["nodes"], attn_sink=st["sink"], max_seqlen=st["case"]["len"], return_lse=True)
    if op == "weights":
        return evict.attn_weight_sums(st["q"], st["cache"], st["table"], st["lens"], st["lse"], st["mask"], softmax_scale=st["scale"],
                                      tree_lens=st["nodes"], max_seqlen=st["case"]["len"])
    if op == "evict":
        c = st["case"]
        keep, counts = evict.evict(st["cache"], st["table"], st["lens"], st["sums"], c["budget"], n_first=c["first"], n_recent=c["recent"],
                                   dst_cache=st["kept"], dst_table=st["kept_table"], sums_out=st["kept_sums"])
        return keep, counts, st["kept"], st["kept_sums"]
    st["cache"].view(-1, st["case"]["d"]).index_copy_(0, st["slots"], st["drafted"])
    tree.commit(st["cache"], st["table"], st["base"], st["path"], st["taken"], seqlens=st["lens"])
    return st["cache"], st["lens"]


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "commit":
        before = st["cache"].cpu().view(torch.int16).numpy().copy()
        new, page = st["drafted"].cpu().view(torch.int16).numpy().reshape(case["b"], case["s"], -1), case["page"]
        table, base = st["table"].cpu().numpy(), st["base"].cpu().numpy()
        path, taken = st["path"].cpu().numpy(), st["taken"].cpu().numpy()
        for i in range(case["b"]):
            for t in range(case["s"]):
                p = base[i] + t
                before[table[i, p // page], p % page] = new[i, path[i, t] if t < taken[i] else t]
        return torch.from_numpy(before).view(torch.bfloat16).double(), base + taken
    if case["op"] == "evict":
        sums, lens = st["sums"].double().cpu().numpy(), st["lens"].cpu().numpy()
        kept, page = st["kept"].cpu().view(torch.int16).numpy().copy(), case["page"]
        flat = st["cache"].cpu().view(torch.int16).numpy()
        table, to = st["table"].cpu().numpy(), st["kept_table"].cpu().numpy()
        keep, counts, out = np.full((case["b"], case["budget"]), -1, np.int32), np.minimum(lens, case["budget"]), np.zeros_like(sums)
        for i, n in enumerate(lens):
            key = sums[i, :n].copy()
            key[:case["first"]] = np.inf
            key[max(0, n - case["recent"]):] = np.inf
            at = np.sort(np.lexsort((np.arange(n), -key))[:counts[i]])
            keep[i, :counts[i]], out[i, :counts[i]] = at, sums[i, at]
            j = np.arange(counts[i])
            kept[to[i, j // page], j % page] = flat[table[i, at // page], at % page]
        return keep, counts, torch.from_numpy(kept).view(torch.bfloat16).double(), out
    b, s, h, d = st["q"].shape
    q, lens, nodes = st["q"].double(), st["lens"].tolist(), st["nodes"].tolist()
    o = torch.zeros(b, s, h, VALUE, dtype=torch.float64, device=q.device)
    lse = torch.full((b, s, h), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.zeros(b, case["len"], dtype=torch.float64, device=q.device)
    for i in range(b):
        n, c = lens[i], nodes[i]
        k = st["cache"][st["table"][i].long()].reshape(-1, d)[:n].double()
        hide = torch.zeros(c, n, dtype=torch.bool, device=q.device)
        hide[:, n - c:] = ~st["mask"][i, :c, :c]
        for t0 in range(0, c, 8):  # a few tokens at a time: the scores of all heads are large in 64 bits
            t1 = min(c, t0 + 8)
            x = torch.einsum("thd,nd->thn", q[i, t0:t1], k) * st["scale"]
            x.masked_fill_(hide[t0:t1, None, :], -math.inf)
            if case["op"] == "weights":
                w[i, :n] += torch.exp(x - st["lse"][i, t0:t1, :, None].double()).sum((0, 1))
                continue
            y = x if st["sink"] is None else torch.cat([x, st["sink"].double().view(1, h, 1).expand(t1 - t0, h, 1)], 2)
            lse[i, t0:t1] = torch.logsumexp(y, 2)
            p = torch.exp(x - lse[i, t0:t1, :, None])
            o[i, t0:t1] = torch.einsum("thn,nv->thv", torch.nan_to_num(p), k[:, :VALUE])
    return w if case["op"] == "weights" else (o, lse)
