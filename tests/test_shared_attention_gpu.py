"""Decode attention over shared prefixes against the definition in 64 bits, and against the operator without sharing."""
import math
import random

import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 16


def build(ops, seed, groups, lens, Hq, Hkv, D, extra_blocks=2, garbage=True):
    """groups: (rows, pages); a pool in which the groups' rows name the same pages.  Slots behind a row's context hold NaN and infinities."""
    rng = random.Random(seed)
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    B = len(lens)
    pre = {r: p for rows, p in groups for r in rows}
    need = sum(p for _, p in groups) + sum(-(-n // PAGE) - pre.get(r, 0) for r, n in enumerate(lens))
    n_pages = need + 3
    free = list(range(n_pages))
    rng.shuffle(free)
    blocks = max([-(-n // PAGE) for n in lens] + [1]) + extra_blocks
    n_seq = B + 2
    slots = list(range(n_seq))
    rng.shuffle(slots)
    table = torch.full((n_seq, blocks), -1, dtype=torch.int32)
    for rows, p in groups:
        pages = [free.pop() for _ in range(p)]
        for r in rows:
            table[slots[r], :p] = torch.tensor(pages, dtype=torch.int32)
    for r, n in enumerate(lens):
        for j in range(pre.get(r, 0), -(-n // PAGE)):
            table[slots[r], j] = free.pop()
    k = torch.randn((n_pages, Hkv, D // 32, 4, PAGE, 8), generator=g, device=DEV).to(torch.float16)
    v = torch.randn((n_pages, Hkv, D, PAGE), generator=g, device=DEV).to(torch.float16)
    if garbage:
        for r, n in enumerate(lens):
            if n % PAGE:
                page = int(table[slots[r], n // PAGE])
                k[page, :, :, :, n % PAGE:] = float("nan")
                v[page, :, :, n % PAGE:] = float("inf")
        for p in free:
            k[p], v[p] = float("nan"), float("nan")
    qkv = (torch.randn((B, Hq + 2 * Hkv, D), generator=g, device=DEV) * 2).to(torch.float16)
    return dict(qkv=qkv, k=k, v=v, table=table.to(DEV), rows=torch.tensor(slots[:B], dtype=torch.int32, device=DEV),
                ctx=torch.tensor(lens, dtype=torch.int32, device=DEV), plan=ops.SharedPrefixPlan(groups, lens, Hq, Hkv, D, DEV), heads=(Hq, Hkv, D), lens=lens)


def call(ops, c, **kw):
    return ops.paged_attn_decode_shared(c["qkv"], c["k"], c["v"], c["table"], c["rows"], c["ctx"], c["plan"], *c["heads"], **kw)


def exact(c, lens=None):
    """(out, bound): a product q . k is off by at most D steps of fp32 over the sum of its terms' magnitudes, a score further by its scaling, its
    difference to the maximum and the exponential (2 ulp each of the hardware's exp2 and its argument); a weight so by a factor 1 +- e, the sums of n
    weights by another n steps, and the weights enter as 22 bits.  The result is a mean of values: off by at most 2 e max |v| and its own rounding."""
    Hq, Hkv, D = c["heads"]
    out, bounds = [], []
    for b, n in enumerate(lens or c["lens"]):
        if n == 0:
            out.append(torch.zeros(Hq * D, dtype=torch.float64, device=DEV))
            bounds.append(torch.zeros(Hq * D, dtype=torch.float64, device=DEV))
            continue
        pages = c["table"][int(c["rows"][b]), : -(-n // PAGE)].long()
        d = torch.float64
        k = c["k"][pages].to(d).permute(1, 0, 4, 2, 3, 5).reshape(Hkv, -1, D)[:, :n]
        v = c["v"][pages].to(d).permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :n]
        q = c["qkv"][b, :Hq].to(d).view(Hkv, Hq // Hkv, D)
        s = q @ k.transpose(1, 2).contiguous() / math.sqrt(D)
        mag = (q.abs() @ k.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True) / math.sqrt(D)
        o = torch.softmax(s, -1) @ v
        u = 2.0 ** -24
        e = (D + 4) * u * mag + 2 * (s.amax(-1, keepdim=True) - s.amin(-1, keepdim=True)) * u + 8 * u + (n + 64) * u + 2.0 ** -21
        out.append(o.reshape(-1))
        bounds.append((2 * e * v.abs().amax() + o.abs() * 2.0 ** -11 + 2.0 ** -25).reshape(-1))
    return torch.stack(out), torch.stack(bounds)


def close(got, c, lens=None):
    want, most = exact(c, lens)
    off = (got.double() - want).abs()
    assert bool(got.isfinite().all()) and bool((off <= most).all()), float((off / most.clamp_min(1e-30)).max())


HEADS = [(16, 16, 64), (32, 32, 128), (32, 8, 128), (12, 4, 64), (16, 1, 128), (10, 2, 64)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("groups,lens", [
    ([([0, 1], 1)], [17, 16]),                                         # one page; a row that ends with its prefix
    ([([2, 0, 3], 3), ([5, 4], 7)], [60, 0, 49, 48 + 33, 112, 300]),   # two groups, mixed order, an empty row between
    ([], [1, 15, 16, 200, 0]),                                         # nothing shared
    ([(list(range(1, 40)), 20)], [5] + [320 + 3 * i for i in range(39)]),
])
def test_against_64_bits(ops, Hq, Hkv, D, groups, lens):
    print("case shared", Hq, Hkv, D, groups, lens, flush=True)
    c = build(ops, Hq + len(lens), groups, lens, Hq, Hkv, D)
    got = call(ops, c)
    close(got, c)
    frag = call(ops, c, frag=True)
    assert torch.equal(frag.unpack(), got)
    out = torch.full_like(got, 9.0)
    assert call(ops, c, out=out) is out and torch.equal(out, got)


@pytest.mark.parametrize("members", [1, 8, 9, 16, 17, 31, 33, 64, 100, 129, 140, 260])
def test_group_sizes(ops, members):
    """Every number of row tiles that a unit's waves share, and groups of several units."""
    print("case members", members, flush=True)
    Hq, Hkv, D = (8, 8, 64)
    lens = [33 * PAGE + 1 + i % 50 for i in range(members)]
    c = build(ops, members, [(list(range(members)), 33)], lens, Hq, Hkv, D)
    close(call(ops, c), c)
    Hq, Hkv, D = (14, 2, 128)
    c = build(ops, members, [(list(range(members)), 33)], lens, Hq, Hkv, D)
    close(call(ops, c), c)


def test_long_contexts(ops):
    print("case long", flush=True)
    Hq, Hkv, D = (8, 2, 128)
    for groups, lens in (([([0, 1, 2], 4000)], [64000 + 5, 64000 + 700, 64000 + 64]), ([], [50000, 3]), ([([1, 2], 9)], [40000, 144, 20000])):
        c = build(ops, 3, groups, lens, Hq, Hkv, D)
        close(call(ops, c), c)


def test_peaked_scores_and_lowest_values(ops):
    """One token takes all the weight, in the prefix or behind it; scores far below."""
    print("case peaks", flush=True)
    Hq, Hkv, D = (8, 4, 64)
    c = build(ops, 8, [([0, 1, 2, 3], 6)], [96 + 10, 96, 97, 130], Hq, Hkv, D)
    c["qkv"] *= 30
    c["k"][:, :, 0, 0, 0, 0] = torch.where(c["k"][:, :, 0, 0, 0, 0].isnan(), c["k"][:, :, 0, 0, 0, 0], 300.0)
    close(call(ops, c), c)
    c["qkv"] = c["qkv"].abs() * 0 - 60000.0
    close(call(ops, c), c)


def test_same_as_without_sharing_and_growing_contexts(ops):
    """A plan stays good while its rows' contexts grow; against the operator that reads every row's pages for itself."""
    print("case growth", flush=True)
    Hq, Hkv, D = (16, 4, 128)
    lens = [160 + 7 * i for i in range(12)] + [40]
    full = [n + 150 for n in lens]
    c = build(ops, 5, [(list(range(12)), 10)], full, Hq, Hkv, D, garbage=False)
    c["plan"] = ops.SharedPrefixPlan([(list(range(12)), 10)], lens, Hq, Hkv, D, DEV)
    for grow in (0, 1, 6, 150):
        now = [n + grow for n in lens]
        c["ctx"].copy_(torch.tensor(now, dtype=torch.int32))
        got = call(ops, c)
        close(got, c, now)
        alone = ops.paged_attn_decode(c["qkv"], c["k"], c["v"], c["table"], c["rows"], c["ctx"], Hq, Hkv, D)
        want, most = exact(c, now)
        assert bool(((got.double() - alone.double()).abs() <= 2 * most).all())


def test_invalid_rows_and_pages(ops):
    """Rows with a sequence outside the table answer zero, pages outside the pool count for nothing."""
    print("case invalid", flush=True)
    Hq, Hkv, D = (8, 8, 64)
    c = build(ops, 6, [([0, 1, 2], 4)], [70, 80, 90, 50, 20], Hq, Hkv, D)
    want = call(ops, c)
    keep = c["rows"].clone()
    c["rows"][3], c["rows"][4] = -1, 7
    c["rows"][1] = 99
    got = call(ops, c)
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and bool((got[[1, 3, 4]] == 0).all())
    c["rows"].copy_(keep)
    c["rows"][0] = -1                                                  # the first of its group
    got = call(ops, c)
    assert torch.equal(got[1:], want[1:]) and bool((got[0] == 0).all())
    c["rows"].copy_(keep)
    c["ctx"].copy_(torch.tensor([70, 80, -5, 2 ** 30, 20], dtype=torch.int32))
    c["table"][int(keep[3]), 1:] = 2 ** 30
    got = call(ops, c)
    assert torch.equal(got[[0, 1, 4]], want[[0, 1, 4]]) and bool((got[2] == 0).all())
    close(got[3:4], {**c, "qkv": c["qkv"][3:4], "rows": keep[3:4], "lens": [16]})


def test_graph_replays_and_streams(ops):
    print("case graphs", flush=True)
    Hq, Hkv, D = (16, 8, 128)
    c = build(ops, 4, [([0, 2, 4], 5)], [100, 90, 120, 33, 81], Hq, Hkv, D)
    want = call(ops, c)
    outs = [torch.zeros_like(want) for _ in range(2)]
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(ops, c, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in outs]
    for _ in range(4):
        for o in outs:
            o.zero_()
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        assert torch.equal(call(ops, c), want)


def test_refusals(ops):
    print("case refusals", flush=True)
    for groups, lens in (([([0, 0], 1)], [40, 40]), ([([0], 1), ([0], 2)], [40, 40]), ([([2], 1)], [40, 40]), ([([0], 3)], [40, 40]), ([([], 1)], [40]),
                         ([([0], 0)], [40]), ([([-1], 1)], [40])):
        with pytest.raises(ValueError):
            ops.SharedPrefixPlan(groups, lens, 8, 8, 64, DEV)
    with pytest.raises(ValueError):
        ops.SharedPrefixPlan([], [4], 34, 2, 64, DEV)
    c = build(ops, 4, [([0, 1], 2)], [40, 50], 8, 8, 64)
    for change in ({"heads": (8, 4, 64)}, {"qkv": c["qkv"][:1]}, {"rows": c["rows"][:1]}, {"ctx": c["ctx"][:1]}, {"k": c["k"][:, :4]}, {"v": c["v"].transpose(2, 3)},
                   {"plan": ops.SharedPrefixPlan([], [4, 4, 4], 8, 8, 64, DEV)}):
        with pytest.raises(ValueError):
            call(ops, {**c, **change})
    with pytest.raises((ValueError, TypeError)):
        call(ops, {**c, "qkv": c["qkv"].float()})
    with pytest.raises(ValueError):
        call(ops, c, out=torch.zeros((2, 100), dtype=torch.float16, device=DEV))
    empty = ops.SharedPrefixPlan([], [], 8, 8, 64, DEV)
    assert ops.paged_attn_decode_shared(c["qkv"][:0], c["k"], c["v"], c["table"], c["rows"][:0], c["ctx"][:0], empty, 8, 8, 64).shape == (0, 512)


@pytest.mark.parametrize("Hq,Hkv,groups,lens", [(32, 8, [(list(range(8)), 40)], [640 + 30 * i for i in range(8)]), (8, 8, [([0, 1], 9), ([2, 3, 4], 5)], [150, 160, 80, 99, 200])])
def test_pages_far_into_a_cache(ops, Hq, Hkv, groups, lens):
    """Page ids whose elements lie beyond 32 bits give the bits of near ones."""
    print("case far", Hq, Hkv, flush=True)
    D = 128
    c = build(ops, 9, groups, lens, Hq, Hkv, D)
    want = call(ops, c)
    n = c["k"].shape[0]
    base = 2 ** 31 // (Hkv * D * PAGE) + 1000                  # (an element of page `base` has a number of 32 bits)
    far = {}
    for name in ("k", "v"):
        far[name] = torch.empty((base + n, *c[name].shape[1:]), dtype=torch.float16, device=DEV)
        far[name][0], far[name][base:] = float("nan"), c[name]
    table = torch.where(c["table"] >= 0, c["table"] + base, -1).to(torch.int32)
    assert torch.equal(call(ops, {**c, **far, "table": table}), want)


def test_plans_out_of_bounds_stay_within_the_call(ops):
    """A plan's arrays are bounded by the kernels: what they name outside the batch, the pages or the workspace counts for nothing, and other rows keep
    their results."""
    print("case damaged plan", flush=True)
    Hq, Hkv, D = (8, 2, 64)
    groups, lens = [(list(range(10)), 6), ([11, 12], 3)], [100 + i for i in range(10)] + [30, 60, 70]
    c = build(ops, 2, groups, lens, Hq, Hkv, D)
    want = call(ops, c)
    plan, n = c["plan"], c["plan"].units.numel() // 72
    keep = plan.data.clone()
    units = plan.units.view(n, 72)
    small = [u for u in range(plan.n_block, n)]                # the units of rows 11 and 12
    for at, value in ((1, 2 ** 20), (1, -5), (2, 2 ** 30), (3, 1000), (3, -1), (8, 10 ** 6), (8, -7), (0, -1)):
        units[small, at] = value
        got = call(ops, c)
        torch.cuda.synchronize()
        assert torch.equal(got[:11], want[:11])
        plan.data.copy_(keep)
    for at, value in ((1, 2 ** 20), (1, -5), (2, 2 ** 30), (3, 1000), (3, -1), (8, 10 ** 6), (8, -7), (0, -1), (0, 1000)):       # and of the others
        units[:plan.n_block, at] = value
        got = call(ops, c)
        torch.cuda.synchronize()
        assert torch.equal(got[10:], want[10:])
        plan.data.copy_(keep)
    for name, value in (("row_slots", 10 ** 6), ("row_slots", -3), ("row_pages", 2 ** 30), ("row_pages", -1)):
        getattr(plan, name)[11:] = value
        got = call(ops, c)
        torch.cuda.synchronize()
        assert torch.equal(got[:11], want[:11])
        plan.data.copy_(keep)
    assert torch.equal(call(ops, c), want)
