"""The selection of a beam search, the places in which beams go on, and copies of pages, against plain evaluations."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def best_of(logits, scores, k, ended=None, eos=None):
    """By 64-bit values, all candidates sorted."""
    R, W = scores.shape
    V = logits.shape[1]
    out = np.full((R, k), -np.inf), np.full((R, k), -1), np.full((R, k), -1)
    with np.errstate(all="ignore"):
        for r in range(R):
            z = logits[r * W:(r + 1) * W].astype(np.float64)
            m = z.max(1, keepdims=True)
            x = z - (m + np.log(np.exp(z - m).sum(1, keepdims=True))) + scores[r].astype(np.float64)[:, None]
            for w in range(W):
                if ended is not None and ended[r, w]:
                    x[w] = -np.inf
                    x[w, eos] = scores[r, w]
                if not scores[r, w] > -np.inf:
                    x[w] = -np.inf
            x = x.reshape(-1)
            x[np.isnan(x)] = -np.inf
            order = np.lexsort((np.arange(x.size), -x))[:k]
            order = order[x[order] > -np.inf]
            for o, a in zip(out, (x[order], order % V, order // V)):
                o[r, :len(order)] = a
    return out


def check(ops, logits, scores, k=None, ended=None, eos=None):
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)                        # noqa: E731
    got = ops.beam_select(logits if isinstance(logits, torch.Tensor) else up(logits), up(scores), ended=up(ended), eos=eos, k=k)
    host = logits.cpu().numpy() if isinstance(logits, torch.Tensor) else logits
    value, token, parent = best_of(host, scores, k or scores.shape[1], ended, eos)
    assert np.array_equal(got[1].cpu().numpy(), token) and np.array_equal(got[2].cpu().numpy(), parent), (logits.shape, scores.shape)
    g = got[0].cpu().numpy()
    fine = np.isfinite(value)
    assert np.array_equal(fine, np.isfinite(g)) and np.array_equal(g[~fine], value[~fine])
    # a logarithm of a sum of V exponentials (hardware's, 2^-22; sums of at most V / 64 and 64 terms in fp32, half a step each) and one rounding
    V = host.shape[1]
    assert (np.abs(g[fine] - value[fine]) <= 2.0 ** -24 * np.abs(value[fine]) + 2.0 ** -22 + (V / 64 + 64 + 2) * 2.0 ** -24).all()


@pytest.mark.parametrize("W,k", [(1, 1), (2, 2), (4, 4), (4, 8), (5, 3), (16, 16), (16, 32), (3, 32)])
@pytest.mark.parametrize("V", [1, 2, 5, 63, 1000, 1023, 1025, 4099, 32003])
def test_random_beams(ops, W, k, V):
    rng = np.random.default_rng(V * 100 + W)
    for R in (1, 3):
        logits = (rng.standard_normal((R * W, V)) * 2.5).astype(np.float32)
        scores = (-rng.random((R, W)) * 6).astype(np.float32)
        check(ops, logits, scores, k)
        ended = (rng.random((R, W)) < 0.4).astype(np.int32)
        check(ops, logits, scores, k, ended, int(rng.integers(V)))
        scores[:, 1:] = -np.inf                            # the first step: one beam
        check(ops, logits, scores, k)


def test_many_rows_of_many_tiles(ops):
    rng = np.random.default_rng(1)
    logits = (rng.standard_normal((520 * 8, 5000)) * 2).astype(np.float32)
    check(ops, logits, (-rng.random((520, 8)) * 3).astype(np.float32))
    logits = (rng.standard_normal((24, 128256)) * 2).astype(np.float32)
    check(ops, logits, (-rng.random((3, 8)) * 3).astype(np.float32), 16)
    # ascending columns: every one beats those before
    logits = np.tile(np.linspace(-8, 8, 40000, dtype=np.float32), (6, 1))
    check(ops, logits, (-rng.random((2, 3)) * 3).astype(np.float32), 32)
    check(ops, logits[:, ::-1].copy(), (-rng.random((2, 3)) * 3).astype(np.float32), 32)


def test_equal_values_and_values_that_are_none(ops):
    V = 3000
    z = np.zeros((6, V), np.float32)
    check(ops, z, np.zeros((2, 3), np.float32), 7)          # all alike: the first columns of the first beam
    z[:, 100::7] = 1
    check(ops, z, np.zeros((2, 3), np.float32), 32)
    check(ops, z, np.array([[0, 0, -1], [-1, 0, 0]], np.float32), 32)
    z = np.full((6, V), -np.inf, np.float32)
    check(ops, z, np.zeros((2, 3), np.float32), 4)          # nothing left
    z[0, 2999], z[3, 0], z[4, 5] = 1, -3, 2
    check(ops, z, np.zeros((2, 3), np.float32), 4)          # fewer than asked for
    z = np.random.default_rng(3).standard_normal((6, V)).astype(np.float32)
    z[1, 77], z[4, 2000] = np.nan, np.inf                   # such a beam has no candidate
    check(ops, z, np.zeros((2, 3), np.float32), 5)
    check(ops, z, np.full((2, 3), np.nan, np.float32), 5)
    check(ops, z * 40 + 3e3, np.zeros((2, 3), np.float32), 5)
    z = np.full((4, V), -1e30, np.float32)
    z[:, 1234] = 0
    check(ops, z, np.zeros((1, 4), np.float32), 4)


def test_strided_rows_and_all_alignments(ops):
    rng = np.random.default_rng(5)
    for V, ld, off in ((1000, 1003, 0), (1001, 1024, 1), (2047, 2051, 2), (777, 779, 3)):
        buf = torch.from_numpy((rng.standard_normal(off + 6 * ld + V) * 2).astype(np.float32)).to(DEV)
        view = torch.as_strided(buf, (6, V), (ld, 1), off)
        check(ops, view, (-rng.random((2, 3))).astype(np.float32))


def test_refusals(ops):
    z, s = torch.zeros((6, 50), device=DEV), torch.zeros((2, 3), device=DEV)
    e = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    for kw in (dict(logits=z[:5]), dict(logits=z.half()), dict(logits=z.t()), dict(scores=s.cpu()), dict(ended=e), dict(ended=e, eos=50), dict(ended=e, eos=-1),
               dict(ended=e[:1], eos=1)):
        with pytest.raises(ValueError):
            ops.beam_select(**{"logits": z, "scores": s, **kw})
    for kw in (dict(k=33), dict(k=0), dict(logits=torch.zeros((34, 9), device=DEV), scores=torch.zeros((2, 17), device=DEV))):
        with pytest.raises(RuntimeError):
            ops.beam_select(**{"logits": z, "scores": s, **kw})
    with pytest.raises(TypeError):
        ops.beam_select(z, s.double())
    with pytest.raises(TypeError):
        ops.beam_select(z, s, ended=e.long(), eos=1)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)                                           # noqa: E731
    for bad in ((i(2, 3), i(5), i(6, 4), i(6)), (i(2, 3), i(6), i(24), i(6)), (i(2, 3), i(6), i(6, 4), i(5)), (i(6), i(6), i(6, 4), i(6)), (i(2, 3), i(6).cpu(), i(6, 4), i(6))):
        with pytest.raises(ValueError):
            ops.beam_reorder(*bad)
    with pytest.raises(RuntimeError):
        ops.beam_reorder(i(1, 17), i(17), i(17, 4), i(17))
    p = torch.zeros((2, 9, 5), device=DEV)
    for bad in (([], i(2), i(2)), ([p] * 9, i(2), i(2)), ([p[0, 0]], i(2), i(2)), ([p], i(2), i(3)), ([p], i(2).cpu(), i(2)), ([p.transpose(0, 1)], i(2), i(2)), ([p[:0]], i(2), i(2)),
                ([p, p.cpu()], i(2), i(2))):
        with pytest.raises(ValueError):
            ops.copy_pages(*bad)
    with pytest.raises(TypeError):
        ops.copy_pages([p], i(2).long(), i(2))


def reordered(parents, slots, table, pos):
    """One beam after the other, on the host."""
    R, W = parents.shape
    table, new = table.copy(), np.empty_like(slots)
    moves = np.full((4, R * W), -1)
    for r in range(R):
        p, s = parents[r], slots[r * W:(r + 1) * W]
        dead = [w for w in range(W) if w not in p]
        seen = set()
        for c in range(W):
            at = r * W + c
            if 0 <= p[c] < W and p[c] not in seen:
                seen.add(p[c])
                new[at] = s[p[c]]
                continue
            new[at] = s[dead.pop(0)]
            if 0 <= p[c] < W:
                src, dst, j = s[p[c]], new[at], pos[r * W + p[c]] // 16
                moves[:2, at] = src, dst
                if 0 <= j < table.shape[1] and table[src, j] >= 0 and table[dst, j] >= 0:
                    moves[2:, at] = table[src, j], table[dst, j]
                table[dst, :max(min(j, table.shape[1]), 0)] = table[src, :max(min(j, table.shape[1]), 0)]
    return new, moves, table


def test_reordering(ops):
    rng = np.random.default_rng(7)
    for trial in range(60):
        R, W, blocks = int(rng.integers(1, 9)), int(rng.integers(1, 17)), int(rng.integers(1, 200))
        n = R * W + 3
        table = rng.permutation(n * blocks).reshape(n, blocks).astype(np.int32)
        slots = rng.permutation(n)[:R * W].astype(np.int32)
        pos = rng.integers(-1, blocks * 16, R * W).astype(np.int32)
        parents = rng.integers(0, W, (R, W)).astype(np.int32)
        if trial % 3 == 1:
            parents[rng.random((R, W)) < 0.3] = -1
        if trial % 5 == 2:
            table[rng.random(table.shape) < 0.1] = -1
        up = lambda a: torch.from_numpy(a.copy()).to(DEV)                                                          # noqa: E731
        t = up(table)
        new, moves = ops.beam_reorder(up(parents), up(slots), t, up(pos))
        e_new, e_moves, e_table = reordered(parents, slots, table, pos)
        assert np.array_equal(new.cpu().numpy(), e_new), (trial, parents)
        assert np.array_equal(torch.stack(list(moves)).cpu().numpy(), e_moves) and np.array_equal(t.cpu().numpy(), e_table), trial
        assert sorted(new.tolist()) == sorted(slots.tolist())
    e = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    assert ops.beam_reorder(e, e.view(-1), torch.zeros((2, 2), dtype=torch.int32, device=DEV), e.view(-1))[0].shape == (0,)


def test_copies_of_rows(ops):
    g = torch.Generator().manual_seed(1)
    rows = 400
    pools = [torch.randint(-128, 128, (3, rows, 2048), generator=g, dtype=torch.int8), torch.randn((3, rows, 8, 2), generator=g), torch.randn((1, rows, 8192 + 24), generator=g).half(),
             torch.randint(0, 9, (2, rows, 7), generator=g, dtype=torch.uint8), torch.randn((2, rows, 5, 3), generator=g).bfloat16(), torch.randn((2, rows, 1), generator=g).double(),
             torch.randint(0, 9, (1, rows), generator=g), torch.randn((1, rows, 20000), generator=g)]
    order = torch.randperm(rows, generator=g).to(torch.int32)
    src, dst = order[:150].clone(), order[150:300].clone()
    src[3], dst[5], src[7], dst[9] = -1, -1, rows, rows                 # rows that are none
    dst[11] = src[11]
    fine = (src >= 0) & (src < rows) & (dst >= 0) & (dst < rows)
    exp = [p.clone() for p in pools]
    for p in exp:
        p[:, dst[fine].long()] = p[:, src[fine].long()]
    dev = [p.to(DEV) for p in pools]
    ops.copy_pages(dev, src.to(DEV), dst.to(DEV))
    for p, e in zip(dev, exp):
        assert torch.equal(p.cpu(), e), p.shape
    ops.copy_pages(dev, src[:0].to(DEV), dst[:0].to(DEV))
    # one parent, many children; more pairs than a launch has rows of workgroups
    p = torch.arange(70001, dtype=torch.int32, device=DEV).view(1, -1, 1).repeat(1, 1, 3)
    ops.copy_pages([p], torch.zeros(70000, dtype=torch.int32, device=DEV), torch.arange(1, 70001, dtype=torch.int32, device=DEV))
    assert not p.any()


def test_copies_beyond_32_bits(ops):
    p = torch.empty((2, 3000, 1 << 20), dtype=torch.uint8, device=DEV)
    p[:, 2999], p[:, 5] = 7, 9
    p[1, 2999] = 8
    ops.copy_pages([p], torch.tensor([2999, 5], dtype=torch.int32, device=DEV), torch.tensor([0, 2998], dtype=torch.int32, device=DEV))
    assert bool((p[0, 0] == 7).all()) and bool((p[1, 0] == 8).all()) and bool((p[:, 2998] == 9).all())


def test_recorded_together(ops):
    """Selection, reordering and copies in one graph, replayed on changing inputs with other work between."""
    g = torch.Generator().manual_seed(3)
    R, W, V, blocks = 3, 4, 5000, 6
    table0 = torch.randperm(R * W * blocks, generator=g).view(R * W, blocks).to(torch.int32)
    pool0 = torch.randn((2, R * W * blocks, 96), generator=g)
    logits, scores = torch.empty((R * W, V), device=DEV), torch.empty((R, W), device=DEV)
    table, pool, slots = table0.to(DEV), pool0.to(DEV), torch.arange(R * W, dtype=torch.int32, device=DEV)
    pos = torch.full((R * W,), 37, dtype=torch.int32, device=DEV)

    def work():
        best, tokens, parents = ops.beam_select(logits, scores)
        new, moves = ops.beam_reorder(parents, slots, table, pos)
        ops.copy_pages([pool], moves.src_page, moves.dst_page)
        return best, tokens, parents, new

    logits.normal_(), scores.zero_()
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(6):
        z = torch.randn((R * W, V), generator=g) * 2
        s = -torch.rand((R, W), generator=g) * 4
        logits.copy_(z), scores.copy_(s), table.copy_(table0), pool.copy_(pool0)
        if i % 2:
            torch.cuda.synchronize()
            torch.randn((500, 500), device=DEV).sum()
        graph.replay()
        value, token, parent = best_of(z.numpy(), s.numpy(), W)
        assert np.array_equal(out[1].cpu().numpy(), token) and np.array_equal(out[2].cpu().numpy(), parent)
        e_new, e_moves, e_table = reordered(parent.astype(np.int32), np.arange(R * W, dtype=np.int32), table0.numpy(), pos.cpu().numpy())
        exp = pool0.clone()
        for a, b in zip(e_moves[2], e_moves[3]):
            if a >= 0:
                exp[:, b] = pool0[:, a]
        assert np.array_equal(out[3].cpu().numpy(), e_new) and np.array_equal(table.cpu().numpy(), e_table) and torch.equal(pool.cpu(), exp)
