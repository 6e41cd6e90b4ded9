"""Plain 64-bit forms of the draft-tree and eviction operators, and the inputs
their tests share (sequences in a paged cache whose pages are shuffled and whose
unused rows hold NaN)."""
from __future__ import annotations

import math

import torch


def paged(lens, d, page, max_pages=None, seed=0, device="cuda", stale=float("nan")):
    """(cache, table, rows): sequences of lens[i] random rows [lens[i], d] in a
    paged cache with shuffled pages; everything behind a sequence's end, and
    every page of none, holds `stale`."""
    g = torch.Generator().manual_seed(seed)
    per = max_pages or max(1, max((n + page - 1) // page for n in lens))
    num = len(lens) * per + 2
    cache = torch.full((num, page, d), stale, dtype=torch.bfloat16)
    table = torch.randperm(num, generator=g)[:len(lens) * per].view(len(lens), per).to(torch.int32)
    rows = []
    for i, n in enumerate(lens):
        x = torch.randn(n, d, generator=g).to(torch.bfloat16)
        rows.append(x)
        for p in range(0, n, page):
            cache[table[i, p // page], :min(page, n - p)] = x[p:p + page]
    return cache.to(device), table.to(device), rows


def gather(cache, table, i, n):
    """The first n rows of sequence i, in order."""
    return cache[table[i].long()].reshape(-1, cache.size(2))[:n]


def random_tree(b, s, seed=0, reach=4):
    """parents [b, s] int32 of random trees, and the mask their definition gives."""
    g = torch.Generator().manual_seed(seed)
    parents = torch.full((b, s), -1, dtype=torch.int32)
    mask = torch.zeros(b, s, s, dtype=torch.bool)
    for i in range(b):
        for t in range(s):
            up = max(-1, t - 1 - int(torch.randint(reach, (1,), generator=g)))
            parents[i, t] = up
            if up >= 0:
                mask[i, t] = mask[i, up]
            mask[i, t, t] = True
    return parents, mask


def seen(n, nodes, s, mask):
    """[s, n]: the tokens that each node of one sequence sees."""
    base = n - nodes
    vis = torch.zeros(s, n, dtype=torch.bool)
    for t in range(min(s, nodes)):
        vis[t, :base] = True
        vis[t, base:] = torch.arange(nodes) <= t if mask is None else mask[t, :nodes]
    return vis


def attention(q, rows, nodes, mask, sink, scale):
    """One sequence in 64 bits: o, lse, and what their tolerances need: the sum of
    p |v| per output, and the largest scale * sum |q k| over what a row sees."""
    s, h, d = q.shape
    q, k = q.double(), rows.double()
    n = k.size(0)
    vis = seen(n, nodes, s, mask)[:, None, :].expand(s, h, n)
    x = torch.einsum("thd,nd->thn", q, k) * scale
    x = torch.where(vis, x, torch.full_like(x, -math.inf))
    full = x if sink is None else torch.cat([x, sink.double().view(1, h, 1).expand(s, h, 1)], 2)
    lse = torch.logsumexp(full, 2) if full.size(2) else torch.full((s, h), -math.inf, dtype=torch.float64)
    lse[nodes:] = -math.inf
    p = torch.where(vis, torch.exp(x - lse[:, :, None]), torch.zeros_like(x))
    v = k[:, :512]
    # what a row does not see stays out of its sums whatever it holds
    v_all = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    o = torch.einsum("thn,nv->thv", p, v_all)
    mag = torch.einsum("thn,nv->thv", p, v_all.abs())
    reach = torch.einsum("thd,nd->thn", q.abs(), torch.nan_to_num(k, nan=0.0, posinf=0.0, neginf=0.0).abs()) * scale
    reach = torch.where(vis, reach, torch.zeros_like(reach))
    g = reach.amax(2) if n else torch.zeros(s, h, dtype=torch.float64)
    return o, lse, p, mag, g


def score_tolerance(g, lse):
    """How far an exponent x - lse may be off: the scores are fp32 sums of exact
    bf16 products on the tensor cores (2^-19 of the sum of their magnitudes; fp32
    additions of 36 partial sums lose 36 * 2^-24 at most, and twice that where the
    adder truncates), the exponent and the log-sum-exp are rounded to fp32 in base
    2 (2^-20 with their products), and 2^x has 2^-22."""
    return 2.0 ** -19 * g + 2.0 ** -20 * (1 + torch.nan_to_num(lse, neginf=0.0).abs())
