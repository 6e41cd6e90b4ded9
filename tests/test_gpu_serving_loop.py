"""The serving step that qcau_b200.evict documents, run as it stands there over many
steps: draft trees verified on a bounded cache, their weights summed, the accepted
path committed with its sums, the cache brought down to its budget.  Rows, lengths and
sums are those of a plain loop in 64 bits."""
import textwrap

import pytest
import torch

import tree_reference as R
from test_gpu_tree import SCALE

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from qcau_b200 import _lib, evict as E
    from qcau_b200.cache import PagedKVCache
    from qcau_b200.tree import commit, tree_attn, tree_mask


def documented_step():
    """The indented lines of the module's documentation."""
    lines = [ln for ln in E.__doc__.splitlines() if ln.startswith("    ")]
    return compile(textwrap.dedent("\n".join(lines)), "evict", "exec")


class Filled(PagedKVCache if torch.cuda.is_available() else object):
    """A cache whose appended rows are written at once (kv_build's part)."""

    def append(self, seqs, counts):
        slots = super().append(seqs, counts)
        self.fresh = torch.randn(len(slots), self.width, generator=self.rng).to(torch.bfloat16)
        self.cache.view(-1, self.width)[slots.long()] = self.fresh.cuda()
        return slots


@pytest.mark.parametrize("s,h,budget", [(1, 16, 70), (7, 16, 96), (20, 5, 150)])
def test_documented_step_over_many_steps(s, h, budget):
    d, slots, seqs = 576, 4, [0, 2, 3]  # slot 1 is idle
    pc = Filled(num_pages=40, max_seqs=slots, max_pages=5)
    pc.rng = torch.Generator().manual_seed(s)
    rng = torch.Generator().manual_seed(s + 1)
    first = [60, 1, 130]
    pc.append(seqs, first)
    rows = dict(zip(seqs, pc.fresh.split(first)))
    held = {i: torch.zeros(n, dtype=torch.float64) for i, n in zip(seqs, first)}
    sums = torch.zeros(slots, pc.max_pages * pc.page_size, device="cuda")
    calls = []

    def evict(*a, **k):
        calls.append(a[3].clone())
        return E.evict(*a, **k)

    step, evicted = documented_step(), 0
    for t in range(6):
        parents, masks = R.random_tree(slots, s, seed=10 * s + t)
        q = torch.randn(slots, s, h, d, generator=rng).to(torch.bfloat16)
        # the accepted path ends at a random node, or nothing is accepted
        path, accepted, taken = torch.full((slots, s), -1, dtype=torch.int32), torch.zeros(slots, dtype=torch.int32), {}
        for i in seqs:
            at, back = int(torch.randint(0 if s == 1 else -1, s, (1,), generator=rng)), []
            while at >= 0:
                back.append(at)
                at = int(parents[i, at])
            taken[i] = back[::-1]
            path[i, :len(back)] = torch.tensor(taken[i], dtype=torch.int32)
            accepted[i] = len(back)
        before = {i: pc.length(i) for i in seqs}
        names = dict(pc=pc, seqs=seqs, s=s, parents=parents.cuda(), q=q.cuda(), scale=SCALE, sums=sums, path=path.cuda(),
                     accepted=accepted.cuda(), lengths=[before[i] + len(taken[i]) for i in seqs], budget=budget, first=2,
                     recent=9, tree_mask=tree_mask, tree_attn=tree_attn, commit=commit, evict=evict,
                     attn_weight_sums=E.attn_weight_sums)
        exec(step, names)
        torch.cuda.synchronize()
        assert _lib.device_error() == 0
        at_evict = calls[-1].double().cpu()
        for i, new in zip(seqs, pc.fresh.split(s)):
            n = before[i]
            drafted = torch.cat([rows[i], new])
            _, _, p, _, _ = R.attention(q[i], drafted, s, masks[i], None, SCALE)
            got = torch.cat([held[i], torch.zeros(s, dtype=torch.float64)]) + p.sum((0, 1))
            live = list(range(n)) + [n + j for j in taken[i]]
            rows[i], held[i] = drafted[live], got[live]
            # an exponent is off by under 2^-13 (2^-19 of sum |q k| * scale, about 27, and
            # 2^-20 * (1 + lse)), the log-sum-exp by as much: 2^-12 of a weight, and the
            # fp32 sums of s * h terms and six steps lose less than another 2^-13
            assert bool(((at_evict[i, :len(live)] - held[i]).abs() <= 2.0 ** -11.4 * held[i] + 1e-30).all())
            assert at_evict[i, len(live):].eq(0).all()
            # the choice is made by the sums as they are on the device
            key = at_evict[i, :len(live)].clone()
            key[:2], key[max(0, len(live) - 9):] = 1e30, 1e30
            order = torch.sort(key, descending=True, stable=True).indices[:budget]
            keep = torch.sort(order).values
            evicted += len(keep) < len(live)
            rows[i], held[i] = rows[i][keep], held[i][keep]
            assert pc.length(i) == len(keep) and int(pc.seqlens[i]) == len(keep)
            assert torch.equal(R.gather(pc.cache, pc.block_table, i, len(keep)).cpu(), rows[i])
            assert torch.equal(sums[i, :len(keep)].double().cpu(), at_evict[i][keep]) and sums[i, len(keep):].eq(0).all()
        assert pc.length(1) == 0 and sums[1].eq(0).all()
    assert evicted  # each case comes over its budget


def test_sequences_that_do_not_draft_are_brought_down_too():
    """A sequence with tokens and no nodes in this step: its weights, rows and length are
    kept as they are until it is over the budget."""
    d, h, s, budget = 576, 16, 3, 100
    pc = Filled(num_pages=20, max_seqs=2, max_pages=5)
    pc.rng = torch.Generator().manual_seed(5)
    pc.append([0, 1], [80, 150])
    rows = pc.fresh[80:]
    sums = torch.rand(2, 320, device="cuda")
    sums[0, 80:], sums[1, 150:] = 0, 0
    before = sums[1].clone()
    nodes = torch.tensor([s, 0], dtype=torch.int32, device="cuda")
    lacking = dict(tree_lens=nodes)
    names = dict(pc=pc, seqs=[0], s=s, parents=torch.tensor([[-1, 0, 0]] * 2, dtype=torch.int32, device="cuda"),
                 q=torch.randn(2, s, h, d, generator=pc.rng).to(torch.bfloat16).cuda(), scale=SCALE, sums=sums,
                 path=torch.tensor([[0, 2, -1]] * 2, dtype=torch.int32, device="cuda"),
                 accepted=torch.tensor([2, 0], dtype=torch.int32, device="cuda"), lengths=[82], budget=budget, first=2, recent=9,
                 tree_mask=tree_mask, tree_attn=lambda *a, **k: tree_attn(*a, **k, **lacking), commit=commit, evict=E.evict,
                 attn_weight_sums=lambda *a, **k: E.attn_weight_sums(*a, **k, **lacking))
    exec(documented_step(), names)
    torch.cuda.synchronize()
    key = before[:150].double().cpu()
    key[:2], key[141:] = 1e30, 1e30
    keep = torch.sort(torch.sort(key, descending=True, stable=True).indices[:budget]).values
    assert pc.length(0) == 82 and pc.length(1) == budget and pc.seqlens.tolist() == [82, budget]
    assert torch.equal(R.gather(pc.cache, pc.block_table, 1, budget).cpu(), rows[keep])
    assert torch.equal(sums[1, :budget].cpu(), before.cpu()[keep]) and sums[1, budget:].eq(0).all()
    assert _lib.device_error() == 0
