"""The greedy token under penalties, biases and grammar masks against a plain evaluation: bit for bit in fp32 where the steps are the
same, and against 64 bits within the steps' roundings."""
import numpy as np
import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, B, V, cap, n_bias=0, n_masks=0, pad=0, grid=64.0):
    """Host arrays of a case; logits on a grid, so that ties happen."""
    g = np.random.default_rng(seed)
    c = {"logits": (np.round(g.standard_normal((B, V + pad)) * 4 * grid) / grid).astype(np.float32)}
    c["history"] = np.minimum((g.random((B, cap)) ** 3 * V), V - 1).astype(np.int32)
    c["lengths"] = g.integers(0, cap + 1, B).astype(np.int32)
    c["lengths"][0] = cap
    c["gen_start"] = (c["lengths"] * g.random(B)).astype(np.int32)
    for n, lo, hi in (("repetition", 0.8, 1.6), ("presence", -0.5, 1.0), ("frequency", -0.2, 0.6)):
        c[n] = g.uniform(lo, hi, B).astype(np.float32)
    if n_bias:
        c["bias_ids"] = g.integers(-1, V, (B, n_bias)).astype(np.int32)
        c["bias"] = (g.standard_normal((B, n_bias)) * 3).astype(np.float32)
    if n_masks:
        c["masks"] = g.integers(-2 ** 31, 2 ** 31, (n_masks, -(-V // 32)), dtype=np.int64).astype(np.int32)
        c["mask_row"] = g.integers(-1, n_masks, B).astype(np.int32)
    return c


def plain(c, V, dtype):
    """Ids and logits after the rules, step by step in `dtype`."""
    z = c["logits"][:, :V].astype(dtype)
    for b in range(z.shape[0]):
        if "history" in c:
            n = int(np.clip(c["lengths"][b], 0, c["history"].shape[1]))
            h = c["history"][b, :n]
            gen = c["gen_start"][b] if "gen_start" in c else 0
            ok = (h >= 0) & (h < V)
            p = {k: c[k][b].astype(dtype) if k in c else dtype(d) for k, d in (("repetition", 1), ("presence", 0), ("frequency", 0))}
            times = np.bincount(h[ok & (np.arange(n) >= gen)], minlength=V).astype(dtype)
            s = np.unique(h[ok])
            with np.errstate(over="ignore", invalid="ignore"):
                v = z[b, s]
                v = np.where(v > 0, v / p["repetition"], v * p["repetition"]).astype(dtype)
                z[b, s] = v - (p["frequency"] * times[s] + np.where(times[s] > 0, p["presence"], dtype(0)))
        if "bias" in c:
            sums = {}
            for v, x in zip(c["bias_ids"][b].tolist(), c["bias"][b]):
                if 0 <= v < V:
                    sums[v] = dtype(sums.get(v, dtype(0)) + dtype(x))
            for v, x in sums.items():
                z[b, v] = z[b, v] + x
        if "masks" in c and 0 <= c["mask_row"][b] < len(c["masks"]):
            words = c["masks"][c["mask_row"][b]].view(np.uint32)
            v = np.arange(V)
            z[b, ((words[v // 32] >> (v % 32).astype(np.uint32)) & 1) == 0] = -np.inf
    w = np.where(np.isnan(z), -np.inf, z)
    ids = np.where(w.max(1) > -np.inf, w.argmax(1), -1).astype(np.int32)
    return ids, z


def on_gpu(ops, c, **more):
    t = {k: torch.from_numpy(v).to(DEV) for k, v in c.items()}
    return t, ops.LogitRules(**{k: v for k, v in t.items() if k != "logits"}, **more)


def show(*what):
    print("case", *what, flush=True)


@pytest.mark.parametrize("B,V,cap,n_bias,n_masks,pad", [
    (1, 1, 1, 1, 1, 0), (3, 5, 7, 2, 2, 0), (2, 33, 64, 3, 1, 1), (1, 32000, 64, 4, 1, 0), (5, 32003, 900, 16, 3, 0), (4, 32765, 100, 0, 0, 3),
    (3, 32766, 300, 5, 2, 0), (2, 40961, 2000, 40, 2, 2), (7, 128256, 3001, 300, 4, 0), (3, 50257, 1, 1024, 2, 1), (70, 1023, 5000, 7, 5, 0),
    (2, 2045, 500, 5, 1, 0), (2, 2046, 500, 5, 1, 0), (9, 8189, 700, 9, 2, 1), (3, 8190, 700, 9, 2, 2), (4, 16381, 1200, 0, 3, 3), (4, 16382, 1200, 30, 0, 0), (192, 32765, 40, 3, 2, 1), (192, 32766, 40, 0, 1, 0),
])
def test_rules_bit_for_bit_and_against_64_bits(ops, B, V, cap, n_bias, n_masks, pad):
    show("rules", B, V, cap, n_bias, n_masks, pad)
    c = make(B * 1000 + V, B, V, cap, n_bias, n_masks, pad)
    t, rules = on_gpu(ops, c)
    logits = t["logits"][:, :V]
    out = torch.full((B, V), 7.0, device=DEV)
    ids = ops.constrained_argmax(logits, rules, out=out)
    alone = ops.constrained_argmax(logits, rules)
    torch.cuda.synchronize()
    want, z = plain(c, V, np.float32)
    assert np.array_equal(out.cpu().numpy(), z)
    assert np.array_equal(ids.cpu().numpy(), want) and torch.equal(ids, alone)
    # 64 bits: four roundings behind the logit (penalty, product and sum of the counted terms, difference) and one per bias, each half a step of
    # a term that is at most the sum of the magnitudes
    z64 = plain(c, V, np.float64)[1]
    fine = np.isfinite(z64)
    assert np.array_equal(fine, np.isfinite(z))
    most = np.abs(c["logits"][:, :V]) * 1.6 + 1.0 + 0.6 * cap + (np.abs(c["bias"]).sum(1, keepdims=True) if n_bias else 0)
    assert (np.abs(z - z64)[fine] <= ((4 + n_bias + 1) * 2.0 ** -24 * most)[fine]).all()
    # in place
    ops.constrained_argmax(logits, rules, out=logits)
    assert torch.equal(logits, out)
    if pad:
        assert np.array_equal(t["logits"][:, V:].cpu().numpy(), c["logits"][:, V:])


@pytest.mark.parametrize("V", [300, 32000, 33000])
def test_empty_rows_ties_infinities(ops, V):
    show("edges", V)
    W = -(-V // 32)
    B = 9
    z = np.zeros((B, V), np.float32)
    z[1] = -np.inf                                                     # nothing to choose from
    z[2] = np.nan
    z[3, 40:] = np.nan
    z[3, 41] = -5.0
    z[3, :40] = -np.inf
    z[4, 17] = np.inf
    z[5] = np.finfo(np.float32).min
    z[6] = np.finfo(np.float32).min
    z[6, 7] = -np.inf
    z[7, 3], z[7, 200] = np.nan, 1.0                                   # NaN in a masked place, and in one that is not
    z[8, [5, 250]] = 4.0
    masks = np.zeros((3, W), np.int32)
    masks[1, (V - 1) // 32] = np.uint32(1 << ((V - 1) % 32)).astype(np.int32)      # the last token alone
    masks[2] = -1
    masks[2, 0] = ~(1 << 3)
    c = {"logits": z, "masks": masks, "mask_row": np.array([0, -1, -1, 5, -1, 1, -1, 2, -2], np.int32)}
    t, rules = on_gpu(ops, c)
    out = torch.empty_like(t["logits"])
    ids = ops.constrained_argmax(t["logits"], rules, out=out).cpu().tolist()
    want, zz = plain(c, V, np.float32)
    assert ids == want.tolist() == [-1, -1, -1, 41, 17, V - 1, 0, 200, 5]
    assert np.array_equal(out.cpu().numpy(), zz, equal_nan=True)
    # a penalty of an infinite logit, and one that pushes a finite one over the edge
    c = {"logits": np.array([[np.inf, -np.inf, 3e38, -3e38] + [0.0] * (V - 4)], np.float32), "history": np.array([[0, 1, 3, 2, 2, -1, V, 2 ** 31 - 1]], np.int32),
         "lengths": np.array([99], np.int32), "repetition": np.array([1.5], np.float32), "frequency": np.array([-1.0], np.float32)}
    t, rules = on_gpu(ops, c)
    out = torch.empty_like(t["logits"])
    assert ops.constrained_argmax(t["logits"], rules, out=out).item() == 0
    assert np.array_equal(out.cpu().numpy(), plain(c, V, np.float32)[1]) and out[0, 3].item() == -np.inf


def test_parameters_alone_and_none(ops):
    show("subsets")
    V, B = 1000, 4
    full = make(5, B, V, 50, 6, 2)
    hist = ("history", "lengths")
    for keys in ((), hist, hist + ("gen_start", "presence"), hist + ("repetition",), hist + ("frequency",), ("bias_ids", "bias"), ("masks", "mask_row")):
        c = {k: full[k] for k in ("logits",) + keys}
        t, rules = on_gpu(ops, c)
        out = torch.empty_like(t["logits"])
        ids = ops.constrained_argmax(t["logits"], rules, out=out)
        want, z = plain(c, V, np.float32)
        assert np.array_equal(out.cpu().numpy(), z) and np.array_equal(ids.cpu().numpy(), want)
        if not keys:
            assert torch.equal(ids, ops.argmax(t["logits"]))
    none = torch.empty((0, V), device=DEV)
    assert ops.constrained_argmax(none, ops.LogitRules()).shape == (0,)
    e = torch.empty((B, 0), device=DEV)
    assert ops.constrained_argmax(t["logits"], ops.LogitRules(bias_ids=e.int(), bias=e)).tolist() == full["logits"].argmax(1).tolist()


@pytest.mark.parametrize("V", [700, 40000])
def test_append_and_replays(ops, V):
    """Tokens go behind their row's history, eagerly and from a graph; a full history and a row without a token stay as they are."""
    show("append", V)
    B, cap, steps = 5, 12, 6
    c = make(11, B, V, cap, 4, 2)
    c["lengths"] = np.array([0, 3, 11, 12, 6], np.int32)
    c["gen_start"] = np.minimum(c["gen_start"], c["lengths"])
    c["masks"][0] = 0
    c["mask_row"] = np.array([-1, 1, -1, 1, 0], np.int32)
    want, host = [], {k: v.copy() for k, v in c.items()}
    for _ in range(steps):
        ids, _ = plain(host, V, np.float32)
        want.append(ids)
        for b in range(B):
            if ids[b] >= 0 and host["lengths"][b] < cap:
                host["history"][b, host["lengths"][b]] = ids[b]
                host["lengths"][b] += 1
    def check(run):
        t, rules = on_gpu(ops, c, append=True)
        ids = torch.empty(B, dtype=torch.int32, device=DEV)
        start = {k: t[k].clone() for k in ("history", "lengths")}
        step = run(t, rules, ids)
        for k, v in start.items():
            t[k].copy_(v)
        for w in want:
            step()
            torch.cuda.synchronize()
            assert np.array_equal(ids.cpu().numpy(), w)
        assert np.array_equal(t["history"].cpu().numpy(), host["history"]) and np.array_equal(t["lengths"].cpu().numpy(), host["lengths"])
    check(lambda t, rules, ids: lambda: ops.constrained_argmax(t["logits"], rules, ids=ids))
    def captured(t, rules, ids):
        ops.constrained_argmax(t["logits"], rules, ids=ids)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.constrained_argmax(t["logits"], rules, ids=ids)
        return g.replay
    check(captured)


def test_two_streams_and_two_graphs(ops):
    """Rules that are only read serve two calls at once."""
    show("streams")
    V = 40000
    cases = [make(s, 6, V, 200, 8, 2) for s in (1, 2)]
    shared = {k: v for k, v in cases[0].items() if k != "logits"}
    want = [plain({**shared, "logits": c["logits"]}, V, np.float32)[0] for c in cases]
    t, rules = on_gpu(ops, cases[0])
    z = [t["logits"], torch.from_numpy(cases[1]["logits"]).to(DEV)]
    ids = [torch.empty(6, dtype=torch.int32, device=DEV) for _ in z]
    graphs = []
    for x, i in zip(z, ids):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.constrained_argmax(x, rules, ids=i)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in z]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i, w in zip(ids, want):
            assert np.array_equal(i.cpu().numpy(), w)
            i.fill_(-7)


def test_refusals(ops):
    show("refusals")
    lm = load_pkg("_lib")
    z = torch.zeros((2, 100), device=DEV)
    i, f = torch.zeros((2, 4), dtype=torch.int32, device=DEV), torch.zeros((2, 4), device=DEV)
    one = torch.zeros(2, dtype=torch.int32, device=DEV)
    bad = [dict(history=i), dict(lengths=one), dict(repetition=f[:, 0].contiguous()), dict(append=True), dict(history=i, lengths=one[:1]), dict(bias_ids=i),
           dict(bias_ids=i, bias=f[:, :3].contiguous()), dict(history=i.long(), lengths=one), dict(history=i[:, ::2], lengths=one), dict(masks=i),
           dict(history=i[:, :0].contiguous(), lengths=one), dict(bias_ids=i.cpu(), bias=f.cpu())]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.LogitRules(**kw)
    rules = ops.LogitRules(history=i, lengths=one)
    for logits, out in ((z[:1], None), (z.half(), None), (z, torch.zeros((2, 99), device=DEV)), (z.t().contiguous().t(), None), (z[:, :50], z[:, 10:60]),
                        (z.cpu(), None)):
        with pytest.raises(ValueError):
            ops.constrained_argmax(logits, rules, out=out)
    with pytest.raises(ValueError):
        ops.constrained_argmax(z, ops.LogitRules(masks=torch.zeros((1, 5), dtype=torch.int32, device=DEV), mask_row=one))
    many = torch.zeros((2, 1025), dtype=torch.int32, device=DEV)
    with pytest.raises(lm.MloraError) as e:
        ops.constrained_argmax(z, ops.LogitRules(bias_ids=many, bias=many.float()))
    assert e.value.code == -2 and "1025" in str(e.value)
