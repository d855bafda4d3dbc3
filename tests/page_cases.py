"""Sequences on paged caches with every key and value at hand, and their attention in 64 bits."""
import math

import numpy as np
import torch

from conftest import load_pkg

PAGE = 16


def rope(D, n, device):
    return [torch.from_numpy(t).to(device) for t in load_pkg("kv_cache").rope_tables(D, 1e4, n)]


def rotated(x, cos, sin):
    """fp16 rows [.., heads, D] rotated by tables [.., D / 2]: separately rounded fp32 products, then fp16."""
    a, b = x.float().chunk(2, -1)
    c, s = cos[..., None, :], sin[..., None, :]
    return torch.cat([a * c - b * s, b * c + a * s], -1).half()


def codes_of(x):
    """A page [16, Hkv, D] fp16 -> (codes [16, Hkv, D] int64, step [Hkv] fp32), by whole numbers: the nearest to 127 x / a, the even one of two."""
    bad = ~torch.isfinite(x).all(2).all(0)
    x = torch.where(bad[None, :, None], torch.zeros((), dtype=x.dtype, device=x.device), x)
    a = x.abs().amax((0, 2))
    f = (127 * x.double() / a.double().clamp_min(2.0 ** -24)[None, :, None])     # (fp64: 53 bits hold the quotient of 18 and 11 far apart from the halves)
    codes = f.round()                                                        # ties to even
    step = (a.double() / 127).float()
    return codes.long(), torch.where(bad, torch.nan, step)


class Book:
    """B sequences: their rotated keys and values [n, Hkv, D] fp16, and a cache that holds them in shuffled pages - of 8 bits or fp16 -, whatever else is in it."""

    def __init__(self, lens, Hq, Hkv, D, quant, seed=0, room=0, garbage=float("nan"), device="cuda:0", scale=1.0):
        self.g = torch.Generator().manual_seed(seed)
        self.dev, self.Hq, self.Hkv, self.D, self.quant = device, Hq, Hkv, D, quant
        self.lens = list(lens)
        B, blocks = len(lens), max(1, max(-(-(n + room) // PAGE) for n in lens))
        self.table = torch.full((B + 1, blocks), -1, dtype=torch.int32)
        need = [-(-(n + room) // PAGE) for n in lens]
        order = (torch.randperm(sum(need) + 2, generator=self.g) + 0).tolist()
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.table = self.table.to(device)
        self.n_pages = sum(need) + 2
        self.cos, self.sin = rope(D, blocks * PAGE, device)
        self.k = [self.draw(n, Hkv, D) * scale for n in lens]
        self.v = [self.draw(n, Hkv, D) * scale for n in lens]
        ops, H = load_pkg("ops"), Hkv
        if quant:
            self.pages = ops.QuantPages.empty(self.n_pages, B + 1, H, D, device)
            self.pages.k.fill_(77)
            self.pages.v.fill_(-77)
            for t in (self.pages.step, self.pages.tail_k, self.pages.tail_v):
                t.fill_(garbage)
        else:
            self.kc = torch.full((self.n_pages, H, D // 32, 4, PAGE, 8), garbage, dtype=torch.float16, device=device)
            self.vc = torch.full((self.n_pages, H, D, PAGE), garbage, dtype=torch.float16, device=device)
        self.store()

    def draw(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dev).half()

    def store(self):
        """The cache is made to hold the sequences as they are."""
        for b, n in enumerate(self.lens):
            for j in range(-(-n // PAGE)):
                k, v = (t[b][j * PAGE:(j + 1) * PAGE] for t in (self.k, self.v))
                m, id = k.shape[0], int(self.table[b, j])
                if not self.quant:
                    self.kc[id, ..., :m, :] = self.frag(k)
                    self.vc[id, ..., :m] = v.permute(1, 2, 0)
                    continue
                if m == PAGE:
                    (ck, sk), (cv, sv) = codes_of(k), codes_of(v)
                    D = self.D
                    self.pages.k[id] = ck.view(PAGE, self.Hkv, D // 64, 2, 4, 8).permute(1, 2, 4, 0, 3, 5).to(torch.int8)
                    self.pages.v[id] = cv.view(4, 4, self.Hkv, D // 64, 4, 16).permute(2, 3, 0, 5, 4, 1).to(torch.int8)
                    self.pages.step[id, :, 0], self.pages.step[id, :, 1] = sk, sv
                if j == (n - 1) // PAGE:
                    self.pages.tail_k[b, ..., :m, :] = self.frag(k)
                    self.pages.tail_v[b, ..., :m] = v.permute(1, 2, 0)

    def frag(self, k):
        return k.view(-1, self.Hkv, self.D // 32, 4, 8).permute(1, 2, 3, 0, 4)

    def append(self, rows, new):
        """qkv [T, ..] of `new` more tokens of the sequences `rows` (behind each other), which the sequences hold from now on; (qkv, table rows, positions, queries)."""
        xs, seqs, poss = [], [], []
        for b, n in zip(rows, new):
            x = self.draw(n, self.Hq + 2 * self.Hkv, self.D)
            xs.append(x)
            seqs += [b] * n
            poss += list(range(self.lens[b], self.lens[b] + n))
        return self.take(torch.cat(xs), rows, new, seqs, poss)

    def take(self, x, rows, new, seqs, poss):
        t = lambda a: torch.tensor(a, dtype=torch.int32, device=self.dev)                                         # noqa: E731
        at = torch.tensor(poss, device=self.dev)
        q = rotated(x[:, :self.Hq], self.cos[at], self.sin[at])
        k = rotated(x[:, self.Hq:self.Hq + self.Hkv], self.cos[at], self.sin[at])
        first = 0
        for b, n in zip(rows, new):
            self.k[b] = torch.cat([self.k[b], k[first:first + n]])
            self.v[b] = torch.cat([self.v[b], x[first:first + n, self.Hq + self.Hkv:]])
            self.lens[b] += n
            first += n
        return x, t(seqs), t(poss), q

    def expect(self, q, seqs, poss, window=None, sinks=0):
        """(attention [T, Hq * D] in 64 bits, how far fp32 sums and one rounding may be from it)."""
        H, G, D, f64 = self.Hkv, self.Hq // self.Hkv, self.D, torch.float64
        out = torch.zeros((q.shape[0], H, G, D), dtype=f64, device=self.dev)
        tol = torch.zeros_like(out)
        for b in set(seqs.tolist()):
            rows = (seqs == b).nonzero()[:, 0]
            p = poss[rows].long()[:, None]
            n = int(p.max()) + 1
            own = [t[b][:n].double().transpose(0, 1) for t in (self.k, self.v)]                     # [H, n, D]
            cached = [t.clone() for t in own]
            for x, src in zip(cached, (self.k[b], self.v[b])):
                for j in range(n // PAGE if self.quant else 0):
                    c, step = codes_of(src[j * PAGE:(j + 1) * PAGE])
                    x[:, j * PAGE:(j + 1) * PAGE] = (c.double() * step.double()[None, :, None]).transpose(0, 1)
            i = torch.arange(n, device=self.dev)
            see = i <= p
            if window is not None:
                see &= (i > p - window) | (i < sinks)
            mine = (i // PAGE == p // PAGE)[None, :, None]                                          # [1, rows, 1, n]
            x = q[rows].double().view(-1, H, G, D).transpose(0, 1)                                  # [H, rows, G, D]
            s, size = (torch.where(mine, *(y(x) @ y(k).transpose(1, 2)[:, None] for k in (own[0], cached[0]))) / math.sqrt(D) for y in (lambda t: t, torch.abs))
            see = see[None, :, None]
            w = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            w_own, w_cached = torch.where(mine & see, w, 0.0), torch.where(~mine & see, w, 0.0)
            vs = [torch.where(see.any((0, 1, 2))[None, :, None], v, 0.0) for v in (own[1], cached[1])]    # (what nobody sees may be infinite)
            o = w_own @ vs[0][:, None] + w_cached @ vs[1][:, None]
            # a score is a sum of D products in fp32 (each at most half a step of the sum of magnitudes off) and its weight off by the same; weights as two
            # halves 2^-22, the hardware's exponential 2^-22, sums of n terms; numerator and denominator.  Besides, a weight of 2^-39 of the greatest is less than half of
            # fp16's last step, where 2^14 stands for the greatest: so much may be missing of every value
            rel = 2 * 2.0 ** -24 * (D * size.masked_fill(~see, 0).amax(-1, keepdim=True) + n + 16)
            out[rows] = o.transpose(0, 1)
            lost = 2.0 ** -39 * torch.maximum(*(v.abs() for v in vs)).sum(1)[:, None, None]
            tol[rows] = (2.0 ** -11 * o.abs() + rel * (w_own @ vs[0].abs()[:, None] + w_cached @ vs[1].abs()[:, None]) + lost + 2.0 ** -24).transpose(0, 1)
        return out.view(-1, self.Hq * D), tol.view(-1, self.Hq * D)

    def same_pages(self, b):
        """Whether the cache holds what `store` would have put there, of a sequence."""
        n = self.lens[b]
        for j in range(n // PAGE if self.quant else 0):
            id = int(self.table[b, j])
            (ck, sk), (cv, sv) = (codes_of(t[b][j * PAGE:(j + 1) * PAGE]) for t in (self.k, self.v))
            k = self.pages.k[id].permute(3, 0, 1, 4, 2, 5).reshape(PAGE, self.Hkv, self.D)
            v = self.pages.v[id].permute(2, 5, 0, 1, 4, 3).reshape(PAGE, self.Hkv, self.D)
            step = self.pages.step[id]
            assert torch.equal(k.long(), ck) and torch.equal(v.long(), cv), (b, j)
            assert torch.equal(step.nan_to_num(-1), torch.stack([sk, sv], 1).nan_to_num(-1)), (b, j)
        j = (n - 1) // PAGE
        k, v = (t[b][j * PAGE:] for t in (self.k, self.v))
        m = k.shape[0]
        if self.quant:
            assert torch.equal(self.pages.tail_k[b, ..., :m, :], self.frag(k)) and torch.equal(self.pages.tail_v[b, ..., :m], v.permute(1, 2, 0)), b
        else:
            id = int(self.table[b, j])
            assert torch.equal(self.kc[id, ..., :m, :], self.frag(k)) and torch.equal(self.vc[id, ..., :m], v.permute(1, 2, 0)), b


def close(out, exp):
    ref, tol = exp
    assert out.shape == ref.shape
    d = (out.double() - ref).abs()
    assert not torch.isnan(out).any(), f"{int(torch.isnan(out).any(1).sum())} rows hold NaN"
    worst = (d / tol).max()
    assert bool((d <= tol).all()), f"{float(worst):.2f} times the bound, rows {torch.unique((d > tol).nonzero()[:, 0])[:8].tolist()}"
