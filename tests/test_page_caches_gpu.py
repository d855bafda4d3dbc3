"""Caches in 8 bits, under windows and of beams as a serving program meets them: in the cache, the model, the sessions and the front end, together."""
import copy

import numpy as np
import pytest
import torch

from conftest import load_pkg
from page_cases import PAGE, Book, close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMS = [{"bits": 8}, {"window": 37, "sinks": 3}, {"bits": 8, "window": 50, "sinks": 20}, {"bits": 8, "window": 1}]


@pytest.fixture(scope="module")
def fp16():
    synth = load_pkg("synth")
    wl = synth.config1()
    return wl, load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV)


class Mirror:
    """A cache of one layer beside a book of what its sequences hold, by name."""

    def __init__(self, form, Hq, Hkv, D, seqs, pages, blocks=20, seed=0):
        self.form, self.Hq, self.Hkv, self.D = form, Hq, Hkv, D
        self.kv = load_pkg("kv_cache").PagedKVCache(1, pages, Hkv, D, seqs, blocks, 1e4, blocks * PAGE, DEV, n_q_heads=Hq, **form)
        self.book = Book([0] * seqs, Hq, Hkv, D, form.get("bits") == 8, seed, room=blocks * PAGE)
        self.at = {}

    def add(self, sid):
        self.kv.add_sequence(sid)
        self.at[sid] = len(self.at)

    def like(self, sid, of, n=None):
        """`sid` holds the first n tokens of `of`."""
        b, o = self.at.setdefault(sid, len(self.at)), self.at[of]
        n = self.book.lens[o] if n is None else n
        self.book.k[b], self.book.v[b], self.book.lens[b] = self.book.k[o][:n], self.book.v[o][:n], n

    def draw(self, sids, new):
        x, seqs, poss, q = self.book.append([self.at[s] for s in sids], new)
        return x, self.book.expect(q, seqs, poss, self.form.get("window"), self.form.get("sinks", 0))

    def go(self, sids, new, frag=False):
        x, exp = self.draw(sids, new)
        self.kv.begin_forward(sids, new)
        out = self.kv.attention_with_fused_qkv(0, x.clone(), self.Hq, frag=frag)
        self.kv.end_forward()
        close(out.unpack() if frag else out, exp)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 2, 128)])
def test_passes_forks_and_prefixes(form, Hq, Hkv, D):
    """Prompts in portions, steps, sequences that begin with another's pages or go on from another in the middle of a page, and pages handed on."""
    print("case passes", form, Hq, Hkv, D, flush=True)
    m = Mirror(form, Hq, Hkv, D, 6, 70)
    for s in "ab":
        m.add(s)
    m.go(["a"], [75])
    m.go(["b", "a"], [1, 30])
    m.go(["a", "b"], [1, 1])
    m.go(["b"], [40])
    m.kv.fork(["c", "d"], "a")
    m.like("c", "a"), m.like("d", "a")
    m.go(["d", "a", "c"], [1, 1, 1], frag=D == 128)
    m.kv.fork(["e"], "b")                                # (42 tokens)
    m.like("e", "b")
    m.go(["e"], [9])
    m.go(["c", "e", "b"], [20, 3, 1])
    m.kv.free_sequence("a")
    m.kv.add_sequence("f")
    n = m.kv.share_prefix("f", "d")
    assert n in (0, 96)
    m.like("f", "d", n)
    m.go(["f", "d"], [5, 5])
    for _ in range(20):
        m.go(["b", "c", "d", "e", "f"], [1] * 5)
    for s in "bcdef":
        m.kv.free_sequence(s)
    assert sorted(m.kv.free) == list(range(70)) and not m.kv._owners


@pytest.mark.parametrize("form", [{}] + FORMS)
@pytest.mark.parametrize("record", [False, True])
def test_beams_hold_what_their_parents_held(ops, form, record):
    """Steps of beams whose parents are drawn: every beam attends to its own path, whichever row it has by then, and the host's pages are those of the rows."""
    print("case beams", form, record, flush=True)
    R, W, Hq, Hkv, D = 3, 4, 4, 2, 64
    m = Mirror(form, Hq, Hkv, D, R * W + 1, 130, seed=3)
    rng = np.random.default_rng(5)
    sids = []
    for r, n in enumerate((30, 16, 1)):
        m.add(r)
        m.go([r], [n])
        forks = [(r, w) for w in range(1, W)]
        m.kv.fork(forks, r)
        sids += [r, *forks]
        for f in forks:
            m.like(f, r)
    m.add("x")
    kv, i32 = m.kv, dict(dtype=torch.int32, device=DEV)
    slots, pos = torch.tensor([kv.slot[s] for s in sids], **i32), torch.tensor([kv.lens[s] for s in sids], **i32)
    ctx, parents, x = pos + 1, torch.zeros(R, W, **i32), torch.zeros(R * W, Hq + 2 * Hkv, D, dtype=torch.float16, device=DEV)
    out = torch.zeros(R * W, Hq * D, dtype=torch.float16, device=DEV)

    def enqueue():
        kv.attention_with_fused_qkv(0, x.clone(), Hq, out=out)
        kv.reorder(sids, parents, slots, ctx)
        pos.add_(1)
        ctx.add_(1)

    graph = None
    for i in range(40):
        if any(kv.lacks_page(s) for s in sids):
            kv.reserve(sids, PAGE)
        new, exp = m.draw(sids, [1] * len(sids))
        x.copy_(new)
        chosen = rng.integers(0, W, (R, W)).astype(np.int32)
        if i == 7:
            chosen[1, 2] = -1                            # a beam that there is not
        parents.copy_(torch.from_numpy(chosen))
        kv.begin_forward(sids, [1] * len(sids), device_meta=(slots, pos, ctx))
        if record and i > 0:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    enqueue()
            graph.replay()
        else:
            enqueue()
        kv.end_forward()
        kv.adrift(sids, slots)
        close(out, exp)
        held = [(m.book.k[m.at[s]], m.book.v[m.at[s]]) for s in sids]
        for j, s in enumerate(sids):
            p = int(chosen.reshape(-1)[j])
            if p >= 0:
                m.book.k[m.at[s]], m.book.v[m.at[s]] = held[j // W * W + p]
        if i == 7:                                       # (any row that was left over: its own, with what its old beam had; give it a path again)
            kv.settle()
            lost = sids[1 * W + 2]
            assert sorted(kv.slot[s] for s in sids) == sorted(slots.tolist())
            src, dst = torch.tensor([kv.slot[sids[W]]], **i32), torch.tensor([kv.slot[lost]], **i32)
            full, part = kv.lens[lost] // PAGE, kv.lens[lost] % PAGE
            assert part
            for p, q in zip(kv.table_h[dst.item(), :full].tolist(), kv.table_h[src.item(), :full].tolist()):
                if p != q:
                    if p >= 0:
                        kv._own(p, -1)
                    if q >= 0:
                        kv._own(q, 1)
            kv.table_h[dst.item(), :full] = kv.table_h[src.item(), :full]
            kv._dirty = True
            if kv.bits == 8:
                ops.copy_pages([kv.tail_k, kv.tail_v], src, dst)
            else:
                at = kv.table_h[[src.item(), dst.item()], full]
                ops.copy_pages([kv.k, kv.v], *(torch.tensor([int(a)], **i32) for a in at))
            m.book.k[m.at[lost]], m.book.v[m.at[lost]] = held[W + int(chosen[1, 0])]
        if i % 13 == 12:
            m.go(["x"], [3])                             # another sequence, whose pass uploads the table
    for s in [*sids, "x"]:
        kv.free_sequence(s)
    assert sorted(kv.free) == list(range(130)) and not kv._owners


def begin(model, kv, sid, prompt):
    kv.add_sequence(sid)
    kv.begin_forward([sid], [len(prompt)])
    z, _ = model["prefill_no_adapter"](model.embed(torch.from_numpy(prompt)), kv)
    kv.end_forward()
    return z


def prompts_of(model, lens, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, model.shape.vocab_size, n).astype(np.int32) for n in lens]


@pytest.mark.parametrize("form", FORMS[:3])
def test_recorded_sessions_choose_what_eager_ones_choose(fp16, form):
    print("case sessions", form, flush=True)
    _, model = fp16
    ds = load_pkg("decode_session")
    prompts, out = prompts_of(model, (200, 17, 240)), {}
    for graph in (False, True):
        kv = model.create_paged_kv_cache(3, 3 * 400, 256, 16, max_seq_len=400, **form)
        first = [int(begin(model, kv, i, p).argmax()) for i, p in enumerate(prompts)]
        s = ds.DecodeSession(model, kv, [0, 1, 2], {}, first, use_graph=graph)
        for _ in range(40):                              # across the length for which the work is cut anew
            s.step(keep_history=True)
        out[graph] = torch.stack(s.history).cpu().numpy()
        assert kv.cut == 400 and (not graph or s._cut == 400)
        again = copy.deepcopy(kv)                        # and a copy decodes as the original
        z = []
        for c in (kv, again):
            c.begin_forward([2, 0], [1, 1])
            z.append(model["decode_no_adapter"](model.embed(torch.tensor([3, 4])), c)[0])
            c.end_forward()
        assert torch.equal(*z)
        with pytest.raises(ValueError):
            ds.NativeDecodeSession(model, kv, [0], None, [1])
    assert np.array_equal(out[True], out[False])


@pytest.mark.parametrize("form", [{}] + FORMS[:3])
def test_the_model_on_these_caches(fp16, form):
    """Prompt passes and steps of the whole model take the cache's attention: equal to a model whose attention is computed from all tokens in 64 bits, up to fp16 roundings of
    activations (every one half a step; they add up to a few 1e-3 of the logits' scale over the layers, as against the oracle)."""
    print("case model", form, flush=True)
    _, model = fp16
    s = model.shape
    prompts = prompts_of(model, (70, 5), 2)

    class Plain:
        """A cache that keeps every token apart."""

        def __init__(self):
            self.books = [Book([0, 0], s.num_attention_heads, s.num_key_value_heads, s.head_dim, form.get("bits") == 8, room=128) for _ in range(s.num_hidden_layers)]
            self.plan, self.n_layers = None, s.num_hidden_layers
            self.plain = False

        def begin(self, sids, new):
            self._cur = (sids, new, all(n == 1 for n in new), None, None, None)

        def attention_with_fused_qkv(self, layer, qkv, n_q_heads, out=None, frag=False, o_shrink=None):
            b, (sids, new) = self.books[layer], self._cur[:2]
            x = qkv.view(-1, s.num_attention_heads + 2 * s.num_key_value_heads, s.head_dim)
            seqs = [i for i, n in zip(sids, new) for _ in range(n)]
            poss = [b.lens[i] + j for i, n in zip(sids, new) for j in range(n)]
            x, seqs, poss, q = b.take(x, sids, new, seqs, poss)
            o = b.expect(q, seqs, poss, form.get("window"), form.get("sinks", 0))[0].half()
            return load_pkg("ops").FragActivation.pack(o) if frag else o

    plain, kv = Plain(), model.create_paged_kv_cache(2, 200, 128, 16, max_seq_len=128, **form)
    worst = 0.0
    for b in plain.books:
        b.cos, b.sin = kv.rope_cos, kv.rope_sin
    for i in (0, 1):
        kv.add_sequence(i)
    for sids, tokens in (([0], prompts[0][:33]), ([0], prompts[0][33:]), ([1], prompts[1]), ([1, 0], [7, 9]), ([0, 1], [1, 2])):
        new = [len(tokens)] if len(sids) == 1 else [1, 1]
        t = torch.as_tensor(np.asarray(tokens, dtype=np.int32))
        rows = None if len(sids) == 2 else torch.tensor([len(tokens) - 1], device=DEV)
        plain.begin(sids, new)
        want = model.forward(model.embed(t), plain, None, rows)
        kv.begin_forward(sids, new)
        got = model["decode_no_adapter"](model.embed(t), kv)[0] if rows is None else model["prefill_no_adapter"](model.embed(t), kv)[0]
        kv.end_forward()
        worst = max(worst, float((got - want).abs().max() / want.std()))
    print(f"logits {worst:.2e}")
    assert worst <= 1e-2


def naive_search(model, kv, prompts, wids, W, steps, eos):
    """The same search over sequences that the host forks and frees, chosen in 64 bits."""
    V = model.shape.vocab_size
    R, live, fresh = len(prompts), [], 0
    scores, ended, paths = np.zeros((R, W)), np.zeros((R, W), bool), [[[] for _ in range(W)] for _ in range(R)]
    z = []
    for r, p in enumerate(prompts):
        kv.add_sequence(("n", r))
        kv.begin_forward([("n", r)], [len(p)])
        h = model.embed(torch.from_numpy(p))
        z.append(model["prefill_no_adapter"](h, kv)[0] if wids is None else model["prefill_a0"](h, kv, [wids[r]])[0])
        kv.end_forward()
        live.append([("n", r)])
    z = torch.cat(z)[:, None]
    for i in range(steps + 1):
        lp = torch.log_softmax(z.double(), -1).cpu().numpy()
        nxt = []
        for r in range(R):
            value = (scores[r][:, None] if i else np.zeros((1, 1))) + lp[r]
            if i and eos is not None:
                for w in np.flatnonzero(ended[r]):
                    value[w] = -np.inf
                    value[w, eos] = scores[r][w]
            best = np.argsort(-value.reshape(-1), kind="stable")[:W]
            parent, token = best // V, best % V
            scores[r] = value.reshape(-1)[best].astype(np.float32)
            ended[r] = token == eos if eos is not None else False
            paths[r] = [paths[r][p] + [int(t)] for p, t in zip(parent, token)] if i else [[int(t)] for t in token]
            new = []
            for p in parent:
                new.append(("n", r, fresh := fresh + 1))
                kv.fork(new[-1:], live[r][p])
            for sid in live[r]:
                kv.free_sequence(sid)
            live[r] = new
            nxt += token.tolist()
        if i < steps:
            sids = [s for beams in live for s in beams]
            kv.begin_forward(sids, [1] * len(sids))
            h = model.embed(torch.tensor(nxt, dtype=torch.int32))
            z = model["decode_no_adapter"](h, kv)[0] if wids is None else model["decode_a0"](h, kv, np.repeat(wids, W).astype(np.int32))[0]
            kv.end_forward()
            z = z.view(R, W, V)
    return scores, paths


@pytest.mark.parametrize("form,eos,adapters", [({}, None, True), ({"bits": 8}, None, False), ({"bits": 8}, 11, True), ({"window": 37, "sinks": 3}, None, False)])
@pytest.mark.parametrize("graph", [False, True])
def test_search_finds_what_the_host_finds(fp16, form, eos, adapters, graph):
    print("case search", form, eos, adapters, graph, flush=True)
    wl, model = fp16
    ds = load_pkg("decode_session")
    W, steps, V = 4, 37, model.shape.vocab_size
    prompts = prompts_of(model, (40, 16, 3), 4)
    R, wids = len(prompts), [0, 1, 0] if adapters else None
    make = lambda: model.create_paged_kv_cache(2 * R * W, 2 * R * W * 112, 64, 16, max_seq_len=112, **form)                # noqa: E731
    want_scores, want = naive_search(model, make(), prompts, wids, W, steps, eos)
    kv = make()
    z = []
    for r, p in enumerate(prompts):
        kv.add_sequence(r)
        kv.begin_forward([r], [len(p)])
        h = model.embed(torch.from_numpy(p))
        z.append(model["prefill_no_adapter"](h, kv)[0] if wids is None else model["prefill_a0"](h, kv, [wids[r]])[0])
        kv.end_forward()
    ids = {} if wids is None else model._ids(R, {0: (None, wids)})
    s = ds.BeamSession(model, kv, list(range(R)), ids, torch.cat(z), W, eos=eos, steps=steps, use_graph=graph)
    for _ in range(steps):
        scores, tokens, parents = s.step()
    got = s.answers()
    # every step's log-sum is a sum of V positive terms in fp32 (V 2^-24 of itself, in the worst order) and its value is rounded once
    tol = (steps + 1) * (V * 2.0 ** -24 + 2.0 ** -24 * np.abs(want_scores).max())
    for r in range(R):
        assert [t for _, t in got[r]] == [p[:p.index(eos) + 1] if eos in p else p for p in want[r]], r
        assert np.abs(np.array([v for v, _ in got[r]]) - want_scores[r]).max() <= tol
    s.close()
    assert sorted(kv.slot) == list(range(R))
    for r in range(R):
        kv.free_sequence(r)
    assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners


def test_one_beam_is_greedy(fp16):
    print("case one beam", flush=True)
    _, model = fp16
    ds = load_pkg("decode_session")
    prompts = prompts_of(model, (20, 33), 6)
    out = []
    for beams in (False, True):
        kv = model.create_paged_kv_cache(2, 200, 64, 16, bits=8)
        z = torch.cat([begin(model, kv, i, p) for i, p in enumerate(prompts)])
        if beams:
            s = ds.BeamSession(model, kv, [0, 1], {}, z, 1)
        else:
            s = ds.DecodeSession(model, kv, [0, 1], {}, z.argmax(-1).int())
            first = z.argmax(-1).cpu()
        for _ in range(20):
            s.step() if beams else s.step(keep_history=True)
        out.append([b[0][1] for b in s.answers()] if beams else torch.stack([first, *(h.cpu() for h in s.history)], 1).tolist())
    assert out[0] == out[1]


def front_end(model, prompts, wids, limits, eos=None, **config):
    ab, xg, lora = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), load_pkg("lora")
    b = ab.LlamaAutoBatcherClass()
    b.set_model(model)
    b.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=24, page_size=16, dense_lora=False, **config))
    b.set_eos_token_id(eos)
    lt, out = model.lora_types[0], []
    for p, w, n in zip(prompts, wids, limits):
        var = b.create_var(p)
        if w is not None:
            b.set_adapter(lora.LoraConfig(r=lt.r, alpha=lt.scaling * lt.r), wid=w)
        out.append(b.generate(var, max_gen_len=n))
    b.compile()
    b.execute()
    return [list(map(int, o.var)) for o in out], b


@pytest.mark.parametrize("config", [{"cache_bits": 8}, {"window": 30, "sinks": 4}, {"cache_bits": 8, "window": 30, "sinks": 4, "share_prefix": True}])
def test_front_end_on_these_caches(fp16, config):
    """Requests with and without adapters: the recorded steps of the front end choose what one call per step chooses."""
    print("case front end", config, flush=True)
    _, model = fp16
    prompts, wids, limits = prompts_of(model, (60, 20, 40, 33), 8), [0, None, 1, 0], [24, 24, 10, 24]
    prompts[3] = np.concatenate([prompts[0][:32], prompts[3]])[:64]
    got, b = front_end(model, prompts, wids, limits, **config)
    want, _ = front_end(model, prompts, wids, limits, native_decode=False, **config)
    assert got == want and [len(g) for g in got] == limits
    assert not b.graph.kv_cache.plain


def test_front_end_searches(fp16):
    """Answers of the front end are the best beams of searches over the same requests, up to the end token."""
    print("case front end beams", flush=True)
    _, model = fp16
    prompts, limits = prompts_of(model, (60, 20, 40), 9), [20, 20, 6]
    got, b = front_end(model, prompts, [None] * 3, limits, beams=3, cache_bits=8)
    kv = model.create_paged_kv_cache(20, 20 * 112, 64, 16, bits=8, max_seq_len=88)
    for group, n in (([0, 1], 20), ([2], 6)):
        order = b.seq_info.order_seqs(group)[0]
        _, want = naive_search(model, kv, [prompts[i] for i in order], None, 3, n - 1, None)
        assert [got[i] for i in order] == [w[0] for w in want]
    assert sorted(b.graph.kv_cache.slot) == [0, 1, 2]
    eos = got[0][9]
    ended, _ = front_end(model, prompts, [0, None, 1], limits, eos=eos, beams=3, window=50)
    assert all(g.index(eos) == len(g) - 1 if eos in g else len(g) == n for g, n in zip(ended, limits))


def test_searches_refuse(fp16):
    _, model = fp16
    ds, tr = load_pkg("decode_session"), load_pkg("token_rules")
    kv = model.create_paged_kv_cache(2, 100, 64, 16)
    z = begin(model, kv, 0, prompts_of(model, (5,))[0])
    for beams in (0, 17):
        with pytest.raises(ValueError):
            ds.BeamSession(model, kv, [0], {}, z, beams)
    with pytest.raises(ValueError):
        ds.BeamSession(model, kv, [0], {}, z.repeat(2, 1), 2)
    with pytest.raises(RuntimeError):
        ds.BeamSession(model, kv, [0], {}, z, 3)                      # (the cache has two rows)
    assert list(kv.slot) == [0]
    ab, xg = load_pkg("auto_batcher"), load_pkg("llama_exec_graph")
    b = ab.LlamaAutoBatcherClass()
    b.set_model(model)
    b.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=4, page_size=16, beams=2))
    b.set_rules(tr.TokenRules(repetition=1.5))
    b.generate(b.create_var(prompts_of(model, (5,))[0]))
    b.compile()
    with pytest.raises(ValueError):
        b.execute()


def test_two_streams_fork_and_decode(fp16):
    """A fork made while a step runs on another stream, and steps on either."""
    print("case streams", flush=True)
    _, model = fp16
    prompts = prompts_of(model, (50, 21), 12)

    def run(streams):
        kv = model.create_paged_kv_cache(4, 400, 64, 16, bits=8)
        z = []
        with torch.cuda.stream(streams[0]):
            for i, p in enumerate(prompts):
                begin(model, kv, i, p)
        for j in range(6):
            with torch.cuda.stream(streams[j % 2]):
                sids = [0, 1] if j < 2 else [0, 2, 1]
                if j == 2:
                    kv.fork([2], 0)
                kv.begin_forward(sids, [1] * len(sids))
                z.append(model["decode_no_adapter"](model.embed(torch.arange(len(sids)) + j), kv)[0])
                kv.end_forward()
        torch.cuda.synchronize()
        return torch.cat(z)

    one = torch.cuda.Stream()
    assert torch.equal(run([one, one]), run([torch.cuda.Stream(), torch.cuda.Stream()]))


@pytest.mark.parametrize("record", [False, True])
def test_beams_behind_a_long_prompt_read_it_once(record):
    """The plan over the prompt's pages serves every step, however the beams' rows change behind them."""
    print("case long prompt", record, flush=True)
    W, Hq, Hkv, D, i32 = 5, 4, 2, 64, dict(dtype=torch.int32, device=DEV)
    m = Mirror({}, Hq, Hkv, D, W, 170, blocks=140, seed=8)
    m.add(0)
    m.go([0], [2070])
    sids = [0, *(("f", w) for w in range(1, W))]
    m.kv.fork(sids[1:], 0)
    for s in sids[1:]:
        m.like(s, 0)
    kv, rng = m.kv, np.random.default_rng(2)
    slots, pos = torch.tensor([kv.slot[s] for s in sids], **i32), torch.full((W,), 2070, **i32)
    ctx, parents, x = pos + 1, torch.zeros(1, W, **i32), torch.zeros(W, Hq + 2 * Hkv, D, dtype=torch.float16, device=DEV)
    out, graph, plans = torch.zeros(W, Hq * D, dtype=torch.float16, device=DEV), None, set()
    for i in range(36):
        if kv.lacks_page(0):
            kv.reserve(sids, PAGE)
        new, exp = m.draw(sids, [1] * W)
        x.copy_(new)
        chosen = rng.integers(0, W, W).astype(np.int32)
        parents.copy_(torch.from_numpy(chosen)[None])
        kv.begin_forward(sids, [1] * W, device_meta=(slots, pos, ctx))
        plans.add(id(kv.plan))
        assert kv.plan is not None

        def enqueue():
            kv.attention_with_fused_qkv(0, x.clone(), Hq, out=out)
            kv.reorder(sids, parents, slots, ctx)
            pos.add_(1)
            ctx.add_(1)

        if record and i > 0:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    enqueue()
            graph.replay()
        else:
            enqueue()
        kv.end_forward()
        kv.adrift(sids, slots)
        close(out, exp)
        held = [(m.book.k[m.at[s]], m.book.v[m.at[s]]) for s in sids]
        for j, s in enumerate(sids):
            m.book.k[m.at[s]], m.book.v[m.at[s]] = held[chosen[j]]
    assert len(plans) == 1
    for s in sids:
        kv.free_sequence(s)
    assert sorted(kv.free) == list(range(170)) and not kv._owners


@pytest.mark.parametrize("form", FORMS[:3])
def test_a_wide_batch_in_fragment_order(form):
    print("case wide", form, flush=True)
    m = Mirror(form, 4, 2, 64, 75, 400, blocks=6, seed=9)
    for s in range(75):
        m.add(s)
    m.go(list(range(75)), [1 + s for s in range(75)], frag=True)
    for _ in range(2):
        m.go(list(range(74, -1, -1)), [1] * 75, frag=True)


@pytest.mark.parametrize("sinks", [1, 17, 40, 64, 70, 130])
@pytest.mark.parametrize("quant", [False, True])
def test_sinks_and_window_in_one_block(sinks, quant):
    """Sinks of one to nine pages, with pages in between that nobody sees, or that only some tokens of a portion see."""
    print("case sinks", sinks, quant, flush=True)
    form = {"window": 45, "sinks": sinks, **({"bits": 8} if quant else {})}
    m = Mirror(form, 8, 2, 128, 2, 60, blocks=26, seed=sinks)
    m.add("a")
    m.add("b")
    m.go(["a"], [130])
    m.go(["a", "b"], [77, 200])
    m.go(["b"], [1])
    m.go(["b", "a"], [33, 140])
    m.go(["a"], [1])


@pytest.mark.parametrize("form", [{}, {"bits": 8}, {"bits": 8, "window": 40, "sinks": 2}])
@pytest.mark.parametrize("graph", [False, True])
def test_searches_beside_each_other(fp16, form, graph):
    """Two searches and a greedy batch take turns on one cache, from which sequences come and go meanwhile: each gives what it gives alone."""
    print("case beside", form, graph, flush=True)
    _, model = fp16
    ds = load_pkg("decode_session")
    prompts, steps = prompts_of(model, (45, 14, 30, 20), 15), 40

    def made(kv, which):
        out = {}
        for i in which:
            z = begin(model, kv, i, prompts[i])
            if i < 2:
                out[i] = ds.BeamSession(model, kv, [i], {}, z, 3 + i, use_graph=graph)
            elif i == 2:
                out[i] = ds.DecodeSession(model, kv, [i], {}, z.argmax(-1).int(), use_graph=graph)
        return out

    def result(s):
        return s.answers() if isinstance(s, ds.BeamSession) else torch.stack(s.history).tolist()

    make = lambda: model.create_paged_kv_cache(10, 10 * 128, 64, 16, max_seq_len=128, **form)                              # noqa: E731
    alone = {}
    for i in range(3):
        s = made(make(), [i])[i]
        for _ in range(steps):
            s.step(**({"keep_history": True} if i == 2 else {}))
        alone[i] = result(s)
    kv = make()
    sessions = made(kv, range(3))
    for j in range(steps):
        for i, s in sessions.items():
            s.step(**({"keep_history": True} if i == 2 else {}))
        if j % 7 == 3:
            begin(model, kv, "x", prompts[3])
        if j % 7 == 5:
            kv.free_sequence("x")
    for i, s in sessions.items():
        got = result(s)
        if i < 2:
            assert [[t for _, t in r] for r in got] == [[t for _, t in r] for r in alone[i]] and [[v for v, _ in r] for r in got] == [[v for v, _ in r] for r in alone[i]]
            s.close()
        else:
            assert got == alone[i]
    for i in list(kv.slot):
        kv.free_sequence(i)
    assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners


def test_all_together_on_a_4_bit_model():
    """A search by the front end over a model with 4-bit linears and adapters, on a cache in 8 bits under a window, whose prompts begin alike."""
    print("case together", flush=True)
    synth = load_pkg("synth")
    wl = synth.config1()
    model = load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV, quant_group=64)
    prompts = prompts_of(model, (50, 50, 21), 20)
    prompts[1] = np.concatenate([prompts[0][:40], prompts[1][:10]])
    form = {"bits": 8, "window": 36, "sinks": 2}
    got, b = front_end(model, prompts, [1, 1, 1], [24, 24, 24], beams=3, cache_bits=8, window=36, sinks=2, share_prefix=True)
    order = b.seq_info.order_seqs([0, 1, 2])[0]
    kv = model.create_paged_kv_cache(20, 20 * 112, 64, 16, max_seq_len=88, **form)
    # prompts that are prefilled whole: the last ten tokens of the second take other kernels in the front end, so that its logits differ by roundings
    scores, want = naive_search(model, kv, [prompts[i] for i in order], [1, 1, 1], 3, 23, None)
    for i, w, s in zip(order, want, scores):
        assert got[i] == w[0] or i == 1 and len(got[i]) == 24, i
    assert len(b.graph.kv_cache.slot) == 3 and all(len(b.graph.kv_cache.pages_of(i)) <= 1 + 36 // 16 + 3 for i in range(3))
