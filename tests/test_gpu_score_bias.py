"""The mean error of the scores behind the tree attention and the weight sums.  Tensor
cores truncate, which leaves scores short by a share per accumulation step; the kernels
take a mean of 1.35e-8 a step back in the softmax scale.  Sequences of one token show the
scores themselves: the log-sum-exp, or the logarithm of the weight with lse = 0."""
import functools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from qcau_b200 import _lib
    from qcau_b200.evict import attn_weight_sums
    from qcau_b200.tree import tree_attn

SHARE = 1.35e-8  # per step, as the kernels take it back
B = 2000


@functools.cache
def scores(d, h, lean):
    """q, cache, table, lengths and the exact q . k [B, h].  lean: the queries lean towards
    their token, so that their products add up and do not cancel."""
    g = torch.Generator(device="cuda").manual_seed(d + h)
    q = torch.randn(B, 1, h, d, device="cuda", generator=g)
    k = torch.randn(B, d, device="cuda", generator=g)
    if lean:
        q += (0.3 + 0.7 * torch.rand(B, 1, h, 1, device="cuda", generator=g)) * k[:, None, None, :]
    q, k = q.to(torch.bfloat16), k.to(torch.bfloat16)
    cache = torch.zeros(B, 64, d, device="cuda", dtype=torch.bfloat16)
    cache[:, 0] = k
    table = torch.arange(B, device="cuda", dtype=torch.int32).view(B, 1)
    dot = torch.einsum("bhd,bd->bh", q[:, 0].double(), k.double())
    return q, cache, table, torch.ones(B, device="cuda", dtype=torch.int32), dot


def mean_steps(d, chain):
    """Of a score's chains, weighted by their share of it: d / 16 steps in chains of `chain`."""
    n = d // 16
    return (n // chain * chain ** 2 + (n % chain) ** 2) / n


def rounding(scale, log2e, d, chain):
    """How far the kernels' factor of a score, scale * log2(e) with the share back, is
    moved by its one rounding to fp32 (up to 2^-24, as much as the shares of four steps)."""
    exact = scale * log2e * (1 + SHARE * mean_steps(d, chain))
    return torch.tensor(exact, dtype=torch.float64).float().double().item() / exact


def slope(op, d, h, chain, lean):
    """Least-squares slope of the scores' error over the scores, for 64 softmax scales whose
    own rounding is taken out."""
    q, cache, table, lens, dot = scores(d, h, lean)
    num = den = 0.0
    for i in range(64):
        scale = (0.03 if lean else 0.05) * (1 + i / 97)
        scale = torch.tensor(scale, dtype=torch.float32).double().item()
        x = dot * scale
        if op == "attention":
            got = tree_attn(q, cache, table, lens, softmax_scale=scale, return_lse=True)[1][:, 0].double()
            got /= rounding(scale, math.log2(math.e), d, chain)
        else:  # a weight is a sum over heads: all but one give 0
            j = i % h
            lse = torch.full((B, 1, h), math.inf, device="cuda")
            lse[:, 0, j] = 0
            x = x[:, j]
            got = attn_weight_sums(q, cache, table, lens, lse, softmax_scale=scale)[:, 0].double().log()
            # log2(e) is an fp32 constant there, for scores and log-sum-exps alike
            log2e = torch.tensor(math.log2(math.e), dtype=torch.float32).double().item()
            got /= rounding(scale, log2e, d, chain) * log2e / math.log2(math.e)
        num, den = num + float(((got - x) * x).sum()), den + float((x * x).sum())
    assert _lib.device_error() == 0
    return num / den


@pytest.mark.parametrize("lean", [False, True])
@pytest.mark.parametrize("d", [576, 512])
@pytest.mark.parametrize("op,h,chain", [("attention", 128, 36), ("weights", 64, 9), ("weights", 128, 18), ("weights", 256, 18)])
def test_scores_are_off_by_a_third_of_the_truncation_at_most(op, h, chain, d, lean):
    """The share that is lost depends on the data; what is taken back lies between
    queries that lean to their token and queries that do not, so that a third of it, or
    less, is left.  Without it, or with its sign turned, a whole or two would be."""
    off = slope(op, d, h, chain, lean)
    assert abs(off) <= SHARE * mean_steps(d, chain) / 3, off


def test_both_widths_are_corrected_by_their_own_steps():
    """512-wide rows have 4 steps fewer: their scores are off as those of 576-wide ones
    are, within half of these steps' share."""
    off = slope("attention", 576, 128, 36, False) - slope("attention", 512, 128, 36, False)
    assert abs(off) <= 4 * SHARE / 2, off
