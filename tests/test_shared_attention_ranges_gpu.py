"""Long contexts whose every range of pages shows in the result: a unit that is left out, or counted twice, is told from rounding."""
import math
import random

import pytest
import torch

import test_shared_attention_gpu as A

pytestmark = pytest.mark.gpu
DEV, PAGE = "cuda:0", 16


def ranges_of(plan, row, tokens):
    """The ranges of pages, 64 at most, in which the kernels walk a row's context: a unit takes the ids of 64 pages at a time."""
    size = plan.units.numel() // max(plan.n_units, 1)
    whole = []
    for u in plan.units.view(plan.n_units, size).tolist() if plan.n_units else []:
        if row in u[8:8 + u[0]]:
            whole.append((u[1], u[1] + u[2]))
    first, have = int(plan.row_pages[row]), -(-tokens // PAGE)
    per = -(-max(have - first, 0) // plan.own_splits)
    whole += [(p, min(p + per, have)) for p in range(first, have, per or 1)]
    whole.sort()
    assert whole[0][0] == 0 and whole[-1][1] == have and all(a[1] == b[0] for a, b in zip(whole, whole[1:]))
    return [(p, min(p + 64, hi)) for lo, hi in whole for p in range(lo, hi, 64)]


CASES = [(8, 2, 128, [([0, 1, 2], 8000)], [128000 + 5, 128000 + 700, 128000 + 64], None),        # block units of 125 pages
         (8, 8, 64, [([0, 1], 8000)], [128000 + 1, 128000 + 5000], None),                         # units of single waves
         (8, 2, 128, [], [50000, 3], None),                                                       # own pages in 64 shares
         (8, 2, 128, [([0, 1], 10)], [40000, 300], [170, 170]),                                   # and in one: a plan that was outgrown
         (8, 2, 128, [([0, 1, 2], 4000), ([3, 4], 70)], [64005, 64700, 64064, 1120, 2000], None),
         (16, 1, 128, [(list(range(40)), 700)], [11200 + 100 * i for i in range(40)], None)]


@pytest.mark.parametrize("Hq,Hkv,D,groups,lens,first", CASES)
def test_every_range_counts(ops, Hq, Hkv, D, groups, lens, first):
    """One token of every range has nearly all the weight that it holds, others none at all: the result is a mean of as many values as there are ranges.

    A query is 8 in one dimension, so a product is exact; a score, up to 233 in powers of two, is off by four roundings (the scale's three and the product's),
    a weight by that twice (its own and the maximum's), by 2^-22 of the exponential and by 2^-22 of its two halves; a part's factor in the join as much again.  Sums of
    at most 200 nonzero terms add 200 half steps, twice (values and weights)."""
    print("case ranges", Hq, Hkv, D, [p for _, p in groups], lens[:5], flush=True)
    c = A.build(ops, 1, groups, lens, Hq, Hkv, D, garbage=False)
    if first is not None:
        c["plan"] = ops.SharedPrefixPlan(groups, first, Hq, Hkv, D, DEV)
    plan, rng = c["plan"], random.Random(Hq + len(lens))
    g = torch.Generator(DEV)
    g.manual_seed(5)
    c["qkv"].zero_()
    for h in range(Hq):
        c["qkv"][:, h, h] = 8.0
    c["k"].zero_()
    c["v"].normal_(generator=g)
    table = c["table"].cpu()
    peaks = {}                                                  # (page, slot) of the cache -> key; a shared page's peak is all its rows'
    rows = []
    slot_of = {}                                                # of the pages that have a peak
    for b, n in enumerate(lens):
        mine, pages = [], table[int(c["rows"][b])].tolist()
        for lo, hi in ranges_of(plan, b, n):
            have = [(pages[p], slot_of[pages[p]]) for p in range(lo, hi) if pages[p] in slot_of]
            if not have:
                at = rng.randrange(lo * PAGE, min(hi * PAGE, n))
                have = [(pages[at // PAGE], at % PAGE)]
                slot_of.update(have)
                peaks[have[0]] = 160.0 + rng.randrange(11) / 8
            mine.append(have)
        rows.append(mine)
    page, slot = (torch.tensor([p[i] for p in peaks], device=DEV) for i in (0, 1))
    key = torch.tensor(list(peaks.values()), device=DEV)
    for d in range(Hq):
        c["k"][page, :, d // 32, d % 32 // 8, slot, d % 8] = key[:, None].half()
    got = A.call(ops, c).double().cpu()
    v = c["v"].cpu()
    for b, mine in enumerate(rows):
        spots = [p for r in mine for p in r]
        s = torch.tensor([8 * peaks[p] / math.sqrt(D) for p in spots], dtype=torch.float64)
        w = (s - s.max()).exp()
        values = torch.stack([v[p[0], :, :, p[1]] for p in spots]).double()          # [spot, Hkv, D]
        owner = torch.tensor([i for i, r in enumerate(mine) for _ in r])
        want = (w[:, None, None] * values).sum(0) / w.sum()
        assert len(spots) <= 200
        u = 2.0 ** -24
        e = 2 * (2 * 4 * 233 * u * math.log(2) + 2 * 2.0 ** -22) + 2 * 200 * u
        most = 2 * e * values.abs().amax() + want.abs() * 2.0 ** -11 + 2.0 ** -25
        off = (got[b].view(Hkv, Hq // Hkv, D) - want[:, None]).abs()
        assert bool((off <= most[:, None]).all()), (b, float((off / most[:, None]).max()))
        for times in (0.0, 2.0) if len(mine) > 1 else ():       # a range left out, or twice
            f = torch.where(owner == torch.arange(len(mine))[:, None], times, 1.0) * w
            wrong = (f @ values.flatten(1)).view(len(mine), Hkv, D) / f.sum(1)[:, None, None]
            assert bool(((wrong - want).abs() > 2 * most).flatten(1).any(1).all()), (b, times)
