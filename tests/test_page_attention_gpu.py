"""Attention over pages of 8 bits and under sliding windows, against 64 bits."""
import numpy as np
import pytest
import torch

from conftest import load_pkg
from page_cases import PAGE, Book, close, codes_of

pytestmark = pytest.mark.gpu

HEADS = [(16, 16, 64), (32, 8, 128), (16, 1, 128), (6, 2, 64), (4, 4, 128)]
SEEN = [(None, 0), (1, 0), (20, 0), (16, 3), (40, 17), (5, 1000), (100000, 4)]
LENS = [1, 2, 15, 16, 17, 31, 32, 33, 100, 250]


def step(ops, book, x, seqs, poss, window=None, sinks=0, **kw):
    args = (book.table, seqs, poss, book.cos, book.sin, book.Hq, book.Hkv, book.D)
    if book.quant:
        return ops.rope_attn_decode_q8(x, book.pages, *args, window=window, sinks=sinks, **kw)
    return ops.rope_attn_decode_window(x, book.kc, book.vc, *args, window=window, sinks=sinks, **kw)


def prompt(ops, book, x, seqs, poss, window=None, sinks=0, **kw):
    if book.quant:
        return ops.rope_attn_prefill_q8(x, book.pages, book.table, seqs, poss, book.cos, book.sin, book.Hq, book.Hkv, book.D, window=window, sinks=sinks, **kw)
    x = x.clone()
    if x.shape[0]:
        ops.rope_kv_append(x, book.kc, book.vc, book.table, seqs, poss, book.cos, book.sin, book.Hq, book.Hkv, book.D)
    return ops.paged_attn_prefill_window(x, book.kc, book.vc, book.table, seqs, poss, book.Hq, book.Hkv, book.D, window=window, sinks=sinks, **kw)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("heads", HEADS)
def test_steps_of_every_length(ops, heads, quant):
    for i, (window, sinks) in enumerate(SEEN):
        book = Book([n - 1 for n in LENS], *heads, quant, seed=i, room=1)
        x, seqs, poss, q = book.append(range(len(LENS)), [1] * len(LENS))
        keep = x.clone()
        for longest in (None, 250):
            out = step(ops, book, x, seqs, poss, window, sinks, longest=longest)
            close(out, book.expect(q, seqs, poss, window, sinks))
        assert torch.equal(x, keep)
        for b in range(len(LENS)):
            book.same_pages(b)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("heads", HEADS)
def test_prompts_of_every_length(ops, heads, quant):
    for i, (window, sinks) in enumerate(SEEN):
        book = Book([0] * len(LENS), *heads, quant, seed=i, room=250)
        x, seqs, poss, q = book.append(range(len(LENS)), LENS)
        out = prompt(ops, book, x, seqs, poss, window, sinks)
        close(out, book.expect(q, seqs, poss, window, sinks))
        for b in range(len(LENS)):
            book.same_pages(b)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("seen", [(None, 0), (37, 5)])
@pytest.mark.parametrize("cuts", [[200], [1, 199], [7, 9, 16, 1, 40, 127], [16] * 12 + [8], [130, 70], [33] + [1] * 30 + [137]])
def test_results_do_not_depend_on_how_a_prompt_is_cut(ops, quant, seen, cuts):
    book = Book([0, 21], 8, 2, 128, quant, seed=3, room=200)
    for n in cuts:
        x, seqs, poss, q = book.append([0, 1], [n, n])
        out = step(ops, book, x, seqs, poss, *seen) if n == 1 else prompt(ops, book, x, seqs, poss, *seen)
        close(out, book.expect(q, seqs, poss, *seen))
    book.same_pages(0), book.same_pages(1)


@pytest.mark.parametrize("quant", [True, False])
def test_shares_of_long_contexts(ops, quant):
    for lens, heads, seen in (([5000, 1, 2777], (8, 2, 64), (None, 0)), ([9001], (16, 1, 128), (None, 0)), ([6000, 6100], (4, 4, 64), (3000, 100)), ([3000], (32, 32, 64), (17, 2))):
        book = Book([n - 1 for n in lens], *heads, quant, seed=len(lens), room=1)
        x, seqs, poss, q = book.append(range(len(lens)), [1] * len(lens))
        exp = book.expect(q, seqs, poss, *seen)
        for longest in (None, max(lens), 16):
            close(step(ops, book, x, seqs, poss, *seen, longest=longest), exp)


@pytest.mark.parametrize("quant", [True, False])
def test_long_prompts(ops, quant):
    book = Book([0, 1000], 4, 2, 128, quant, seed=9, room=1300)
    x, seqs, poss, q = book.append([0, 1], [1300, 300])
    some = torch.randperm(1600, generator=torch.Generator().manual_seed(1))[:100].to(book.dev)
    for seen in ((None, 0), (400, 4), (64, 0)):
        ref = Book([0, 1000], 4, 2, 128, quant, seed=9, room=1300)
        x, seqs, poss, q = ref.append([0, 1], [1300, 300])
        out = prompt(ops, ref, x, seqs, poss, *seen)
        close(out[some], ref.expect(q[some], seqs[some], poss[some], *seen))


@pytest.mark.parametrize("quant", [True, False])
def test_fragment_order_and_given_results(ops, quant):
    for n in (1, 17, 40, 70):
        book = Book([30] * n, 4, 2, 64, quant, seed=n, room=70)
        x, seqs, poss, q = book.append(range(n), [1] * n)
        rows = step(ops, book, x, seqs, poss)
        frag = step(ops, book, x, seqs, poss, frag=True)
        assert torch.equal(frag.unpack(), rows)
        given = torch.empty_like(rows)
        assert step(ops, book, x, seqs, poss, out=given) is given and torch.equal(given, rows)
        book = Book([3], 4, 2, 64, quant, seed=n, room=n)
        x, seqs, poss, q = book.append([0], [n])
        rows = prompt(ops, book, x, seqs, poss)
        book = Book([3], 4, 2, 64, quant, seed=n, room=n)
        x, seqs, poss, q = book.append([0], [n])
        assert torch.equal(prompt(ops, book, x, seqs, poss, frag=True).unpack(), rows)


@pytest.mark.parametrize("quant", [True, False])
def test_rows_that_are_none(ops, quant):
    book = Book([40, 40, 40], 4, 2, 64, quant, seed=1, room=8, garbage=0.0)
    x, seqs, poss, q = book.append([0, 1, 2], [1, 1, 1])
    before = [t.clone() for t in ((book.pages.k, book.pages.v, book.pages.step, book.pages.tail_k, book.pages.tail_v) if quant else (book.kc, book.vc))]
    for s, p in ((-1, 40), (99, 40), (1, -1), (1, 48), (1, 1 << 20)):
        seqs[1], poss[1] = s, p
        for out in (step(ops, book, x, seqs, poss), prompt(ops, book, x, seqs, poss)):
            assert not out[1].any()
            e, tol = book.expect(q[[0, 2]], seqs[[0, 2]], poss[[0, 2]])
            close(out[[0, 2]], (e, tol))
    ids = book.table[1][book.table[1] >= 0].long()
    now = (book.pages.k, book.pages.v, book.pages.step, book.pages.tail_k, book.pages.tail_v) if quant else (book.kc, book.vc)
    for t, was in zip(now, before):
        at = torch.ones(1, dtype=torch.long, device=t.device) if quant and t.shape[0] == 4 else ids
        assert torch.equal(t[at], was[at])
    none = torch.empty((0, 8, 64), dtype=torch.float16, device=book.dev)
    e = torch.empty(0, dtype=torch.int32, device=book.dev)
    assert step(ops, book, none, e, e).shape == (0, 256) and prompt(ops, book, none, e, e).shape == (0, 256)


@pytest.mark.parametrize("quant", [True, False])
def test_pages_out_of_the_window_need_not_be_there(ops, quant):
    book = Book([299, 180], 4, 2, 128, quant, seed=1, room=40)
    x, seqs, poss, q = book.append([0, 1], [1, 1])
    window, sinks = 50, 20
    exp = book.expect(q, seqs, poss, window, sinks)
    book.table[0, 2:15] = -1                          # the window begins at token 250
    book.table[1, 2:7] = 1 << 28
    close(step(ops, book, x, seqs, poss, window, sinks), exp)
    x, seqs, poss, q = book.append([0, 1], [30, 30])
    exp = book.expect(q, seqs, poss, window, sinks)
    close(prompt(ops, book, x, seqs, poss, window, sinks), exp)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_infinities_that_nobody_sees(ops, quant, bad):
    """Tokens that are not finite, out of the window and behind the queries, touch nobody who does not see them; who sees them gets NaN.  A page of 8 bits that holds one
    is NaN throughout: there, who sees any of its tokens."""
    book = Book([100], 4, 2, 64, quant, seed=2, room=100)
    book.k[0][40], book.v[0][45] = bad, bad
    book.store()
    x, seqs, poss, q = book.append([0], [1])
    sinks = 32 if quant else 33                        # (token 32 lies in the page of the bad ones)
    close(step(ops, book, x, seqs, poss, 50, sinks), book.expect(q, seqs, poss, 50, sinks))       # sees 0 .. sinks - 1 and 51 .. 100
    if quant:
        assert torch.isnan(step(ops, book, x, seqs, poss, 50, 33)).all()
    assert not torch.isfinite(step(ops, book, x, seqs, poss, 60, sinks).float()).any()
    # in the middle of a pass: the tokens ahead of it do not see it
    y = book.draw(40, 8, 64)
    y[13, 4 + 2:] = bad                                # a value row of token 114
    x, seqs, poss, q = book.take(y, [0], [40], [0] * 40, list(range(101, 141)))
    out = prompt(ops, book, x, seqs, poss, 50, sinks)
    e, tol = book.expect(q[:13], seqs[:13], poss[:13], 50, sinks)
    close(out[:13], (e, tol))
    assert torch.isnan(out[13:].float()).any(1).all() if quant else not torch.isfinite(out[13:].float()).all(1).any()


def test_steps_of_very_different_sizes(ops):
    """Values of pages whose steps lie 2^20 apart, with all weight on the small ones; pages of zeros."""
    for sizes in ((1.0, 2.0 ** -10, 3e4), (2.0 ** -14, 1.0, 0.0), (0.0, 0.0, 0.0), (6e4, 2.0 ** -13, 6e4)):
        book = Book([0], 4, 2, 128, True, seed=4, room=96)
        y = book.draw(48, 8, 128)
        for j, s in enumerate(sizes):
            y[j * 16:(j + 1) * 16, 6:] = (torch.rand((16, 2, 128), generator=book.g).to(book.dev) * s).half()
        x, seqs, poss, q = book.take(y, [0], [48], [0] * 48, list(range(48)))
        close(prompt(ops, book, x, seqs, poss), book.expect(q, seqs, poss))
        # all weight on the second page: its keys are along the query
        y = book.draw(20, 8, 128)
        x, seqs, poss, q = book.append([0], [20])
        d = q.view(20, 2, 2, 128)[:, :, 0].float().mean(0)
        for t in range(16, 32):
            book.k[0][t] = (40 * d / d.norm(dim=-1, keepdim=True)).half()
        book.store()
        exp = book.expect(q, seqs, poss)
        close(prompt(ops, book, x, seqs, poss), exp)
        close(step(ops, book, x[19:], seqs[19:], poss[19:]), tuple(t[19:] for t in exp))


def test_values_of_pages(ops):
    book = Book([100, 33], 4, 2, 128, True, seed=5)
    ids = torch.tensor([int(book.table[0, 3]), int(book.table[1, 1]), int(book.table[0, 0])], dtype=torch.int32, device=book.dev)
    keys, values = book.pages.values(ids)
    for i, (b, j) in enumerate(((0, 3), (1, 1), (0, 0))):
        for got, src in ((keys, book.k), (values, book.v)):
            c, s = codes_of(src[b][j * PAGE:(j + 1) * PAGE])
            assert torch.equal(got[i].transpose(0, 1), (c.float() * s[None, :, None]).half())
    assert book.pages.values(ids[:0])[0].shape == (0, 2, 16, 128)
    keys, _ = book.pages.values(ids[:1].expand(70000).contiguous())
    assert torch.equal(keys[69999], keys[0])


def test_pages_beyond_32_bits(ops):
    """A pool of which the offsets of pages pass 2^32 bytes."""
    n, H, D = 280000, 8, 128
    pages = ops.QuantPages.empty(n, 2, H, D, "cuda:0")
    book = Book([199], 8, H, D, True, seed=6, room=9)
    far = torch.arange(n - 40, n - 40 + book.table.shape[1], dtype=torch.int32, device=book.dev)
    for name in ("k", "v", "step"):
        getattr(pages, name)[far.long()] = getattr(book.pages, name)[book.table[0].long().clamp_min(0)]
    pages.tail_k.copy_(book.pages.tail_k), pages.tail_v.copy_(book.pages.tail_v)
    x, seqs, poss, q = book.append([0], [1])
    book.table = torch.stack([far, far])
    exp = book.expect(q, seqs, poss)
    book.pages = pages
    close(step(ops, book, x, seqs, poss), exp)
    x, seqs, poss, q = book.append([0], [8])
    close(prompt(ops, book, x, seqs, poss), book.expect(q, seqs, poss))
    book.same_pages(0)


@pytest.mark.parametrize("quant", [True, False])
def test_recorded_steps_and_other_streams(ops, quant):
    """A step recorded once, replayed for the tokens of two pages, with other work and waits between; on a stream of its own."""
    book = Book([25, 3], 4, 2, 64, quant, seed=7, room=60)
    x = torch.empty((2, 8, 64), dtype=torch.float16, device=book.dev)
    seqs, poss = torch.tensor([0, 1], dtype=torch.int32, device=book.dev), torch.tensor([25, 3], dtype=torch.int32, device=book.dev)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    y, _, _, q = book.append([0, 1], [1, 1])
    x.copy_(y)
    step(ops, book, x, seqs, poss, 30, 2)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(ops, book, x, seqs, poss, 30, 2, longest=90)
    for i in range(36):
        if i:
            y, _, _, q = book.append([0, 1], [1, 1])
            x.copy_(y)
            poss.add_(1)
        if i % 5 == 4:
            torch.cuda.synchronize()
            torch.randn((1000, 1000), device=book.dev).sum()
        if i % 7 == 6:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        close(out, book.expect(q, seqs, poss, 30, 2))
    book.same_pages(0), book.same_pages(1)


def test_refusals(ops):
    book = Book([20, 20], 4, 2, 64, True, seed=8, room=4)
    x, seqs, poss, q = book.append([0, 1], [1, 1])
    for kw in (dict(window=0), dict(window=-1), dict(window=4, sinks=-1), dict(sinks=3), dict(window=1 << 31), dict(out=torch.empty((2, 128), dtype=torch.float16, device=book.dev))):
        with pytest.raises(ValueError):
            step(ops, book, x, seqs, poss, **kw)
    with pytest.raises(ValueError):
        step(ops, book, x[:, :7], seqs, poss)
    with pytest.raises(ValueError):
        step(ops, book, x, seqs[:1], poss)
    with pytest.raises(TypeError):
        step(ops, book, x, seqs.long(), poss)
    with pytest.raises(TypeError):
        step(ops, book, x.float(), seqs, poss)
    with pytest.raises(ValueError):
        step(ops, book, x, seqs.cpu(), poss)
    with pytest.raises(ValueError):
        ops.rope_attn_decode_q8(x, book.pages, book.table.t(), seqs, poss, book.cos, book.sin, 4, 2, 64)
    with pytest.raises(ValueError):
        ops.rope_attn_decode_q8(x, book.pages, book.table, seqs, poss, book.cos[:, :16], book.sin, 4, 2, 64)
    with pytest.raises(ValueError):
        ops.rope_attn_decode_q8(x, book.pages, torch.cat([book.table] * 2), seqs, poss, book.cos, book.sin, 4, 2, 64)      # more rows than tails
    p = book.pages
    for bad in ((p.k.float(), p.v, p.step, p.tail_k, p.tail_v), (p.k, p.v, p.step.double(), p.tail_k, p.tail_v)):
        with pytest.raises(TypeError):
            ops.QuantPages(*bad)
    for bad in ((p.k[:1], p.v, p.step, p.tail_k, p.tail_v), (p.k, p.v, p.step, p.tail_k[:1], p.tail_v), (p.k, p.v, p.step.cpu(), p.tail_k, p.tail_v),
                (p.k, p.v, p.step.transpose(0, 1).contiguous().transpose(0, 1), p.tail_k, p.tail_v)):
        with pytest.raises(ValueError):
            ops.QuantPages(*bad)
    with pytest.raises(ValueError):
        ops.QuantPages.empty(4, 2, 2, 96, book.dev)


def test_quotients_half_way_between_two_codes(ops):
    """Pages of small whole numbers, whose 127 x / a are often exactly half-way: ties go to the even code, also beside a page of zeros and one with an infinity."""
    g = torch.Generator().manual_seed(11)
    for most in (254, 2, 127, 508, 1016, 6, 40, 2032):
        book = Book([0], 4, 2, 64, True, seed=most, room=70)
        y = torch.randint(-most, most + 1, (64, 8, 64), generator=g).to(book.dev).half()
        y[:, 6:, 0] = most
        y[5, 7, 3], y[20, 7, 9] = 0, most / 2
        y[32:48, 6] = 0
        x, seqs, poss, q = book.take(y, [0], [64], [0] * 64, list(range(64)))
        book.cos.fill_(1), book.sin.fill_(0)               # keys as they come
        book.k[0] = x[:, 4:6].clone()
        prompt(ops, book, x, seqs, poss)
        book.same_pages(0)
        one = Book([0], 4, 2, 64, True, seed=most, room=70)
        one.cos.fill_(1), one.sin.fill_(0)
        for t in range(64):
            step(ops, one, x[t:t + 1], seqs[t:t + 1], poss[t:t + 1])
        one.k, one.v, one.lens = book.k, book.v, book.lens
        one.same_pages(0)


@pytest.mark.parametrize("step", [0.4, 1.0, 1.7, 2.5, 40.0, -0.7])
@pytest.mark.parametrize("quant", [False, True])
def test_scores_that_climb(ops, quant, step):
    """The greatest score grows (or falls) from tile to tile by amounts around those for which sums are rescaled, in a prompt and in single tokens behind it."""
    print("case climb", quant, step, flush=True)
    Hq, Hkv, D, n = 4, 2, 64, 400
    b = Book([0], Hq, Hkv, D, quant, seed=4, room=n + 20)
    t = torch.arange(n + 20, device=b.dev, dtype=torch.float32) / 64
    if step < 0:
        t = t.flip(0)
    u = torch.randn(D, generator=b.g).to(b.dev)
    u /= u.norm()
    # a rotation-free direction would need no tables: the tables here are made of ones and zeros, so that scores are what is drawn
    b.cos.fill_(1)
    b.sin.fill_(0)
    size = (t * abs(step) * 0.6931 * D ** 0.5).sqrt()[:, None, None]
    x = b.draw(n + 20, Hq + 2 * Hkv, D)
    top = float(size.max())
    x[:, :Hq] = (x[:, :Hq] * 0.05 + u * top).half()                          # q . k / sqrt(D) / ln 2 = step * token / 64, a little apart
    x[:, Hq:Hq + Hkv] = (x[:, Hq:Hq + Hkv] * 0.01 + u * size * size / max(top, 1e-3)).half()
    for new in [n] + [1] * 20:
        at = b.lens[0]
        x1, seqs, poss, q = b.take(x[at:at + new].contiguous(), [0], [new], [0] * new, list(range(at, at + new)))
        if quant:
            fn = ops.rope_attn_prefill_q8 if new > 1 else ops.rope_attn_decode_q8
            out = fn(x1, b.pages, b.table, seqs, poss, b.cos, b.sin, Hq, Hkv, D)
        elif new > 1:
            ops.rope_kv_append(x1, b.kc, b.vc, b.table, seqs, poss, b.cos, b.sin, Hq, Hkv, D)
            out = ops.paged_attn_prefill_window(x1, b.kc, b.vc, b.table, seqs, poss, Hq, Hkv, D, window=300)
        else:
            out = ops.rope_attn_decode_window(x1, b.kc, b.vc, b.table, seqs, poss, b.cos, b.sin, Hq, Hkv, D, window=300)
        close(out, b.expect(q, seqs, poss, None if quant else 300))


@pytest.mark.parametrize("shift", [-24, -20, -14, -7, 0, 6])
def test_codes_of_every_magnitude(ops, shift):
    """Pages of fp16 numbers of any bits, down to the smallest there is: every code is the nearest whole number to 127 x / a."""
    print("case magnitudes", shift, flush=True)
    T = 2048
    b = Book([0], 8, 8, 128, True, seed=100 + shift, room=T)
    b.cos.fill_(1), b.sin.fill_(0)
    g = torch.Generator().manual_seed(shift + 50)
    low = max(0, (shift + 24 - 12) << 10) if shift > -14 else 0                # of bits: up to 2^13 below the largest
    high = (1 << (shift + 24)) + 3 if shift < -14 else (shift + 15) << 10
    bits = torch.randint(low, high, (T, 24, 128), generator=g, dtype=torch.int32)
    y = (bits | torch.randint(0, 2, bits.shape, generator=g, dtype=torch.int32) << 15).to(torch.int16).view(torch.float16).to(b.dev)
    y[:, :8] = 0                                                               # (scores are zero)
    x, seqs, poss, q = b.take(y, [0], [T], [0] * T, list(range(T)))
    b.k[0] = x[:, 8:16].clone()
    out = prompt(ops, b, x, seqs, poss)
    b.same_pages(0)
    keys, values = b.pages.values(b.table[0, :T // 16].contiguous())
    for got, want in ((keys, b.k[0]), (values, b.v[0])):
        step = want.view(-1, 16, 8, 128).abs().amax((1, 3)).double() / 127
        d = (got.transpose(1, 2).double() - want.view(-1, 16, 8, 128).double()).abs()
        # half a step, the step's rounding (up to 127 of them), fp16's rounding of what is given back
        assert bool((d <= step[:, None, :, None] * (0.5 + 127 * 2.0 ** -24) + want.view(-1, 16, 8, 128).double().abs() * 2.0 ** -10 + 2.0 ** -24).all())
