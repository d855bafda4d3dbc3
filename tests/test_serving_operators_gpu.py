"""4-bit linears, shared prefixes and rules as a serving program meets them: in the model, the cache, the decode sessions and the front
end, alone and together."""
import numpy as np
import pytest
import torch

import oracle
from conftest import load_pkg
from helpers import n_pages_for

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def fp16():
    synth = load_pkg("synth")
    wl = synth.config1()
    return wl, load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV), synth.prompts(wl)


@pytest.fixture(scope="module")
def four_bit(fp16):
    wl, _, prompts = fp16
    return wl, load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV, quant_group=64), prompts


def oracle_of(wl, model, mode):
    """The oracle on the weights that the 4-bit model stands for."""
    synth = load_pkg("synth")
    s = wl.shape
    w = {k: v.float().numpy() for k, v in synth.base_weights(wl.seed, s, torch.float16, "cpu").items()}
    for l, L in enumerate(model.layers):
        q, k, v = L["qkv"].dequantize().cpu().split([s.q_size, s.kv_size, s.kv_size])
        gate, up = L["gate_up"].dequantize().cpu().chunk(2)
        for name, t in zip(("q", "k", "v", "o", "gate", "up", "down"), (q, k, v, L["o"].dequantize().cpu(), gate, up, L["down"].dequantize().cpu())):
            w[f"layers.{l}.{name}_proj"] = t.numpy()
    lw = synth.lora_weights(wl.seed, s, wl.lora, torch.float16, "cpu", tag="a0")
    return oracle.LlamaRef(s, w, {k: v.float().numpy() for k, v in lw.items()}, {"a0": wl.lora.scaling}, mode=mode)


def prefill(model, kv, sid, prompt, wid=None, skip=0):
    kv.begin_forward([sid], [len(prompt) - skip])
    h = model.embed(torch.from_numpy(np.ascontiguousarray(prompt[skip:])))
    logits, _ = model["prefill_no_adapter"](h, kv) if wid is None else model["prefill_a0"](h, kv, [int(wid)])
    kv.end_forward()
    return logits


def decode(model, kv, sids, tokens, wids=None):
    kv.begin_forward(sids, [1] * len(sids))
    h = model.embed(torch.as_tensor(np.asarray(tokens, dtype=np.int32)))
    logits, _ = model["decode_no_adapter"](h, kv) if wids is None else model["decode_a0"](h, kv, np.asarray(wids, dtype=np.int32))
    kv.end_forward()
    return logits


def err(got, want):
    return float(np.abs(got - want).max() / want.std())


def test_four_bit_model_against_oracle(four_bit):
    """Prompts and a decode step with adapters on a 4-bit base: the whole-model bound of the fp16 model (operators agree to an fp16 ulp; their rounding
    flips add up to a few 1e-3 of the logits' scale)."""
    print("case four-bit model", flush=True)
    wl, model, prompts = four_bit
    B, P = prompts.shape
    assert not model.native_step and model.weight_bytes_per_step() < 2 * 4096 * 11008 * 40
    for mode, most in (("mixed", 1e-2), ("fp32", 1.5e-2)):
        ref = oracle_of(wl, model, mode)
        n = n_pages_for(wl, 4)
        rk = ref.new_cache(n, 16, P + 8, np.arange(n))
        kv = model.create_paged_kv_cache(B, B * (P + 16), P, 16)
        for s in range(B):
            rk.add_sequence(s)
            kv.add_sequence(s)
        rk.begin_forward(list(range(B)), [P] * B)
        want = ref.forward(prompts.reshape(-1), rk, {"a0": np.repeat(wl.adapter_ids, P)}, logits_rows=np.arange(B) * P + P - 1)
        rk.end_forward()
        kv.begin_forward(list(range(B)), [P] * B)
        got, _ = model["prefill_a0"](model.embed(torch.from_numpy(prompts.reshape(-1))), kv, wl.adapter_ids)
        kv.end_forward()
        e0 = err(got.cpu().numpy(), want)
        nxt = want.argmax(-1)
        rk.begin_forward(list(range(B)), [1] * B)
        want = ref.forward(nxt, rk, {"a0": wl.adapter_ids})
        rk.end_forward()
        e1 = err(decode(model, kv, list(range(B)), nxt, wl.adapter_ids).cpu().numpy(), want)
        print(f"logits vs {mode} oracle: prefill {e0:.2e} decode {e1:.2e}")
        assert e0 <= most and e1 <= most


def test_four_bit_model_refuses_fp16_forms(four_bit):
    wl, model, _ = four_bit
    ds = load_pkg("decode_session")
    kv = model.create_paged_kv_cache(1, 64, 32, 16)
    kv.add_sequence(0)
    for call in (model.interleaved_gate_up, model.dense_lora_weights, lambda: ds.NativeDecodeSession(model, kv, [0], None, [1]),
                 lambda: type(model)(wl.shape, DEV, quant_group=48)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("rows,shared", [(3, 5), (20, 130), (40, 30)])
def test_shared_prefixes_in_the_cache(fp16, monkeypatch, rows, shared):
    """Sequences that took over another's pages decode as sequences with pages of their own that hold the same."""
    print("case shared cache", rows, shared, flush=True)
    wl, model, _ = fp16
    rng = np.random.default_rng(rows)
    head = rng.integers(0, wl.shape.vocab_size, shared * 16 + 3).astype(np.int32)
    tails = [rng.integers(0, wl.shape.vocab_size, 1 + int(rng.integers(0, 40))).astype(np.int32) for _ in range(rows)]
    prompts = [np.concatenate([head, t]) for t in tails]
    longest = max(map(len, prompts)) + 8
    kv = model.create_paged_kv_cache(rows, rows * longest, longest, 16, max_seq_len=longest)
    apart = model.create_paged_kv_cache(rows, rows * longest, longest, 16, max_seq_len=longest)
    for i, p in enumerate(prompts):
        kv.add_sequence(i)
        skip = kv.share_prefix(i, 0, len(head)) if i else 0
        assert skip == (shared * 16 if i else 0)
        prefill(model, kv, i, p, skip=skip)
    used = len(set(range(kv.n_pages)) - set(kv.free))
    assert used == sum(-(-len(p) // 16) for p in prompts) - (rows - 1) * shared
    # the same cache contents on pages of their own
    for i, p in enumerate(prompts):
        apart.add_sequence(i)
        apart.begin_forward([i], [len(p)])
        apart.end_forward()
        src, dst = (torch.tensor(c.pages_of(i), device=DEV) for c in (kv, apart))
        apart.k[:, dst], apart.v[:, dst] = kv.k[:, src], kv.v[:, src]
    kvm = load_pkg("kv_cache")
    made = []
    whole = kvm.ops.paged_attn_decode_shared
    monkeypatch.setattr(kvm.ops, "paged_attn_decode_shared", lambda *a, **k: made.append(1) or whole(*a, **k))
    sids = list(rng.permutation(rows))
    sids = [int(s) for s in sids]
    tokens = rng.integers(0, wl.shape.vocab_size, rows)
    got, want = decode(model, kv, sids, tokens), decode(model, apart, sids, tokens)
    assert len(made) == (wl.shape.num_hidden_layers if kv.shared_plan(sids) is not None else 0)
    assert (kv.shared_plan(sids) is not None) == (shared >= 128)
    assert err(got.cpu().numpy(), want.cpu().numpy()) <= 1e-2          # (whole-model bound, as against the oracle)
    # a sequence goes, the others' prefix stays
    kv.free_sequence(0)
    left = [s for s in sids if s]
    again = decode(model, kv, left, tokens[1:])
    apart.free_sequence(0)
    assert err(again.cpu().numpy(), decode(model, apart, left, tokens[1:]).cpu().numpy()) <= 1e-2


def test_shared_prefixes_of_wide_batches_with_adapters():
    """More than 64 rows, whose o deltas otherwise ride on the attention, in two groups and alone: as without a plan."""
    print("case wide shared", flush=True)
    synth = load_pkg("synth")
    wl = synth.config1()
    model = load_pkg("llama").LlamaForCausalLM.from_synthetic(6, wl.shape, [synth.LoraSpec(r=16, alpha=8.0, n_adapters=4)], DEV)
    rng = np.random.default_rng(4)
    rows, heads = 80, [rng.integers(0, wl.shape.vocab_size, n * 16).astype(np.int32) for n in (130, 20)]
    who = [(0, 1, None, 0)[i % 4] for i in range(rows)]
    wids = np.array([-1 if i % 7 == 3 else (2 if who[i] else 1) for i in range(rows)], dtype=np.int32)
    kv = model.create_paged_kv_cache(rows, 3000 + rows * 100, 2200, 16, max_seq_len=2200)
    first = {}
    for i in range(rows):
        g = who[i]
        prompt = np.concatenate([heads[g] if g is not None else heads[1][:9], rng.integers(0, wl.shape.vocab_size, 1 + i % 30).astype(np.int32)])
        kv.add_sequence(i)
        skip = 0 if g is None or g not in first else kv.share_prefix(i, first[g], len(heads[g]))
        first.setdefault(g, i)
        prefill(model, kv, i, prompt, 1, skip)
    sids, tokens = list(range(rows)), rng.integers(0, wl.shape.vocab_size, rows)
    def step():
        kv.begin_forward(sids, [1] * rows)
        z = model.forward(model.embed(torch.as_tensor(tokens.astype(np.int32))), kv, {0: torch.from_numpy(wids).to(DEV)})
        plan, kv._cur = kv.plan, None                        # the same step again: its keys and values are written anew
        return z.cpu().numpy(), plan
    got, plan = step()
    assert plan is not None and sorted(len(r) for r, _ in kv.prefix_groups(sids)) == [20, 40]
    kv._plans[tuple(sids)] = None
    want, plan = step()
    assert plan is None and err(got, want) <= 1e-2           # (whole-model bound, as against the oracle)


def plain_ids(logits, rules, prompts, answers):
    """The rules evaluated on the host, in the operator's order of roundings."""
    out = []
    for z, r, p, a in zip(logits.cpu().numpy().astype(np.float32), rules, prompts, answers):
        f = np.float32
        z = z.copy()
        if r is not None:
            seen = np.unique(np.concatenate([p, np.asarray(a, dtype=np.int64)]).astype(np.int64))
            times = np.bincount(np.asarray(a, dtype=np.int64), minlength=len(z)).astype(f)
            v = np.where(z[seen] > 0, z[seen] / f(r.repetition), z[seen] * f(r.repetition))
            z[seen] = v - (f(r.frequency) * times[seen] + np.where(times[seen] > 0, f(r.presence), f(0)))
            for t, x in (r.bias or {}).items():
                z[t] = z[t] + f(x)
            allowed = None if r.grammar is None else r.grammar(list(a))
            if allowed is not None:
                keep = np.zeros(len(z), bool)
                keep[list(allowed)] = True
                z[~keep] = -np.inf
        out.append(int(z.argmax()) if z.max() > -np.inf else -1)
    return out


def some_rules(vocab):
    tr = load_pkg("token_rules")
    word = [5, 9, 5, 700, vocab - 1]
    spell = lambda a: [word[len(a)]] if len(a) < len(word) else []                         # one word, then the end
    odd = lambda a: range(1, vocab, 2) if len(a) % 2 else None
    return [tr.TokenRules(repetition=1.3, presence=0.4, frequency=0.2), None, tr.TokenRules(grammar=spell), tr.TokenRules(bias={7: 100.0, 11: -3.0}, frequency=60.0),
            tr.TokenRules(grammar=odd, repetition=2.0)]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("adapters", [False, True])
def test_front_end_with_rules(fp16, native, adapters):
    """Every token is what the rules, evaluated on the host, make of the model's own logits along the same path."""
    print("case rules", native, adapters, flush=True)
    wl, model, _ = fp16
    ab, xg, lora, ops = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), load_pkg("lora"), load_pkg("ops")
    V, steps = wl.shape.vocab_size, 10
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, V, 20 + 7 * i).astype(np.int32) for i in range(5)]
    rules = some_rules(V)
    batcher = ab.LlamaAutoBatcherClass()
    batcher.set_model(model)
    batcher.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=steps, page_size=16, native_decode=native, dense_lora=False))
    lt = model.lora_types[0]
    out = []
    for i, (p, r) in enumerate(zip(prompts, rules)):
        var = batcher.create_var(p)
        if adapters:
            batcher.set_adapter(lora.LoraConfig(r=lt.r, alpha=lt.scaling * lt.r), wid=i % lt.n_adapters)
        if r is not None:
            batcher.set_rules(r)
        out.append(batcher.generate(var, max_gen_len=steps - i))
    batcher.compile()
    batcher.execute()
    got = [list(map(int, o.var)) for o in out]
    assert got[2] == [5, 9, 5, 700, V - 1]                                                  # the grammar's word, whatever the model says
    assert got[3][0] == 7 and len(set(got[3])) > 1 and all(t % 2 for t in got[4][1::2])
    assert [len(g) for g in got] == [10, 9, 5, 7, 6]
    # the same path, token by token; batches shrink as the front end's do
    kv = model.create_paged_kv_cache(5, 5 * 80, 64, 16)
    wids = [i % lt.n_adapters if adapters else None for i in range(5)]
    answers = [[] for _ in range(5)]
    for i, p in enumerate(prompts):
        kv.add_sequence(i)
        answers[i] += plain_ids(prefill(model, kv, i, p, wids[i]), [rules[i]], [p], [[]])
    order = batcher.seq_info.order_seqs(list(range(5)))[0]
    live = list(order)
    while live:
        z = decode(model, kv, live, [answers[i][-1] for i in live], [wids[i] for i in live] if adapters else None)
        nxt = plain_ids(z, [rules[i] for i in live], [prompts[i] for i in live], [answers[i] for i in live])
        for i, t in zip(live, nxt):
            if t >= 0:
                answers[i].append(t)
        live = [i for i, t in zip(live, nxt) if t >= 0 and len(answers[i]) < steps - i]
    if native and adapters:
        # once the ruled requests are done the native step may take over, whose bits are those of the operators
        assert [g[:5] for g in got] == [a[:5] for a in answers]
    else:
        assert got == answers


def test_answer_that_ends_before_its_first_token(fp16):
    print("case nothing allowed", flush=True)
    wl, model, prompts = fp16
    ab, xg, tr = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), load_pkg("token_rules")
    batcher = ab.LlamaAutoBatcherClass()
    batcher.set_model(model)
    batcher.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=4, page_size=16))
    out = []
    for i in range(2):
        if i == 0:
            batcher.set_rules(tr.TokenRules(grammar=lambda a: []))
        out.append(batcher.generate(batcher.create_var(prompts[i][:30])))
    batcher.compile()
    batcher.execute()
    assert len(out[0].var) == 0 and len(out[1].var) == 4
    with pytest.raises(ValueError):
        tr.BatchRules([tr.TokenRules(bias={wl.shape.vocab_size: 1.0})], [[1]], [[]], 1, wl.shape.vocab_size, DEV)
    with pytest.raises(ValueError):
        tr.BatchRules([tr.TokenRules(grammar=lambda a: [-1])], [[1]], [[]], 1, wl.shape.vocab_size, DEV)


@pytest.mark.parametrize("quantised", [False, True])
def test_front_end_with_shared_prefixes(fp16, four_bit, quantised):
    """Requests behind one instruction, of two adapters and none: pages are taken over from a request of the same adapter alone, and every token is the
    model's own choice along the path (up to near ties: the shorter prefill sums in another order)."""
    print("case front end shared", quantised, flush=True)
    wl, model, _ = four_bit if quantised else fp16
    ab, xg, lora = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), load_pkg("lora")
    V, steps = wl.shape.vocab_size, 9
    rng = np.random.default_rng(8)
    head = rng.integers(0, V, 16 * 130 + 5).astype(np.int32)
    prompts = [np.concatenate([head, rng.integers(0, V, 3 + 5 * i).astype(np.int32)]) for i in range(7)] + [head[:16 * 40].copy(), head.copy()]
    who = [None, 0, 1, 0, None, 1, 0, 0, None]
    lt = model.lora_types[0]
    results = {}
    for share in (False, True):
        batcher = ab.LlamaAutoBatcherClass()
        batcher.set_model(model)
        batcher.set_exec_config(xg.LlamaExecConfig(max_prompt_len=2200, max_gen_len=steps, page_size=16, share_prefix=share, dense_lora=False))
        out = []
        for p, w in zip(prompts, who):
            if w is not None:
                batcher.set_adapter(lora.LoraConfig(r=lt.r, alpha=lt.scaling * lt.r), wid=w)
            out.append(batcher.generate(batcher.create_var(p)))
        batcher.compile()
        batcher.execute()
        results[share] = [list(map(int, o.var)) for o in out]
        kv = batcher.graph.kv_cache
        if share:
            full = {s: len(p) // 16 for s, p in enumerate(prompts)}
            first = {w: who.index(w) for w in (None, 0, 1)}
            for s, w in enumerate(who):
                mine, src = kv.pages_of(s), kv.pages_of(first[w])
                n = 0 if s == first[w] else min(130, (len(prompts[s]) - 1) // 16, full[s])
                assert mine[:n] == src[:n] and (s == first[w] or mine[n] != src[n])
            assert len(kv._owners) == 3 * 130 and kv.shared_plan(list(range(9))) is not None
    # teacher-forced: each token of the sharing run is within a near tie of the best along its own path without sharing
    kv = model.create_paged_kv_cache(9, 9 * 2300, 2200, 16, max_seq_len=2300)
    for s, (p, w) in enumerate(zip(prompts, who)):
        kv.add_sequence(s)
        z = prefill(model, kv, s, p, w)[0]
        for t in results[True][s]:
            assert float(z.max() - z[t]) <= 2e-2 * float(z.std())
            z = decode(model, kv, [s], [t], None if w is None else [w])[0]


def test_all_together_in_a_recorded_session(four_bit):
    """A 4-bit base with adapters, requests behind shared pages, rules: steps replayed from a graph choose what eager steps choose, whose tokens are
    those that the host evaluates from the step's logits."""
    print("case together", flush=True)
    wl, model, _ = four_bit
    tr, ds = load_pkg("token_rules"), load_pkg("decode_session")
    V, rows, steps = wl.shape.vocab_size, 24, 7
    rng = np.random.default_rng(12)
    head = rng.integers(0, V, 16 * 130).astype(np.int32)
    prompts = [np.concatenate([head, rng.integers(0, V, 2 + 3 * i).astype(np.int32)]) for i in range(rows)]
    rules = [tr.TokenRules(repetition=1.2 + 0.01 * i, frequency=0.3) if i % 3 else None for i in range(rows)]
    rules[4] = tr.TokenRules(bias={i: -50.0 for i in range(100)}, presence=1.0)
    wids = np.zeros(rows, np.int32)
    def start():
        kv = model.create_paged_kv_cache(rows, 4096 + rows * 120, 2300, 16, max_seq_len=2300)
        firsts = []
        for i, p in enumerate(prompts):
            kv.add_sequence(i)
            skip = kv.share_prefix(i, 0, len(head)) if i else 0
            firsts.append(int(prefill(model, kv, i, p, 0, skip).argmax()))
        return kv, firsts
    def run(graph):
        kv, firsts = start()
        batch = tr.BatchRules(rules, prompts, [[f] for f in firsts], steps, V, DEV)
        s = ds.DecodeSession(model, kv, list(range(rows)), {0: wids}, firsts, use_graph=graph, rules=batch)
        for _ in range(steps):
            s.step(keep_history=True)
            assert kv.plan is not None
        torch.cuda.synchronize()
        return firsts, torch.stack(s.history).cpu().numpy(), batch
    firsts, eager, _ = run(False)
    again, replayed, batch = run(True)
    assert again == firsts and np.array_equal(eager, replayed)
    assert batch.args.lengths.tolist() == [len(p) + 1 + steps for p in prompts]
    with pytest.raises(RuntimeError):                        # the histories have no place for another token
        batch.take()
    kv, _ = start()
    answers = [[f] for f in firsts]
    for step in range(steps):
        z = decode(model, kv, list(range(rows)), [a[-1] for a in answers], wids)
        for a, t in zip(answers, plain_ids(z, rules, prompts, answers)):
            a.append(t)
    assert [a[1:] for a in answers] == eager.T.tolist()


def test_four_bit_decode_of_wide_mixed_batches():
    """More than 64 requests of two adapter types and none on a 4-bit base: rows as alone."""
    print("case wide mixed", flush=True)
    synth = load_pkg("synth")
    wl = synth.config1()
    specs = [synth.LoraSpec(r=16, alpha=8.0, n_adapters=4), synth.LoraSpec(r=8, alpha=16.0, n_adapters=3, targets=("q_proj", "o_proj", "gate_proj", "down_proj"))]
    model = load_pkg("llama").LlamaForCausalLM.from_synthetic(5, wl.shape, specs, DEV, quant_group=32)
    rng = np.random.default_rng(5)
    rows = 70
    prompts = [rng.integers(0, wl.shape.vocab_size, 3 + i % 9).astype(np.int32) for i in range(rows)]
    who = [(None, 0)[i % 2] if i % 3 else 1 for i in range(rows)]
    kv = model.create_paged_kv_cache(2 * rows, 2 * rows * 16, 16, 16)
    for copy in range(2):
        for i, p in enumerate(prompts):
            sid = copy * rows + i
            kv.add_sequence(sid)
            kv.begin_forward([sid], [len(p)])
            h = model.embed(torch.from_numpy(p))
            _ = model["prefill_no_adapter"](h, kv) if who[i] is None else model[f"prefill_a{who[i]}"](h, kv, [i % 3])
            kv.end_forward()
    tokens = rng.integers(0, wl.shape.vocab_size, rows)
    pairs = []
    for tid in (0, 1):
        at = [i for i in range(rows) if who[i] == tid]
        pairs += [at, [i % 3 for i in at]]
    kv.begin_forward(list(range(rows)), [1] * rows)
    wide, _ = model["mixed_decode_a0_a1"](model.embed(torch.from_numpy(tokens.astype(np.int32))), kv, *pairs)
    kv.end_forward()
    for i in range(rows):
        sid = rows + i
        kv.begin_forward([sid], [1])
        h = model.embed(torch.as_tensor(tokens[i:i + 1].astype(np.int32)))
        alone, _ = model["decode_no_adapter"](h, kv) if who[i] is None else model[f"decode_a{who[i]}"](h, kv, np.array([i % 3], dtype=np.int32))
        kv.end_forward()
        assert err(wide[i].cpu().numpy(), alone[0].cpu().numpy()) <= 1e-2          # (whole-model bound, as against the oracle)
    wide = decode(model, kv, list(range(rows)), tokens, np.arange(rows) % 4)       # all of one type
    for i in range(0, rows, 7):
        assert err(wide[i].cpu().numpy(), decode(model, kv, [rows + i], tokens[i:i + 1], np.array([i % 4]))[0].cpu().numpy()) <= 1e-2


def test_latent_pages_are_shared_too():
    """A cache of latents: a sequence on another's pages has the logits of the whole prompt."""
    print("case latent", flush=True)
    import safolorn_cases as C
    from oracle import safolorn_ref as R
    name, cfg = next(iter(C.CONFIGS.items()))
    weights = C.weights(cfg, 3, 1.0)
    model = load_pkg("safolorn").SafolornForCausalLM.from_weights(cfg, C.tensors(weights), torch.float32, DEV)
    rng = np.random.default_rng(9)
    head, tails = rng.integers(0, cfg["vocab"], 70), [rng.integers(0, cfg["vocab"], n) for n in (5, 20)]
    kv = model.create_paged_kv_cache(4, 1024, 1024, 16)
    def run(sid, t):
        kv.begin_forward([sid], [len(t)])
        out = model.forward(model.embed(torch.from_numpy(np.asarray(t).astype(np.int32))), kv, None)
        kv.end_forward()
        return out.double().cpu().numpy()
    kv.add_sequence(0)
    run(0, np.concatenate([head, tails[0]]))
    kv.add_sequence(1)
    skip = kv.share_prefix(1, 0, len(head))
    assert skip == 64
    prompt = np.concatenate([head, tails[1]])
    got = run(1, prompt[skip:])
    kv.free_sequence(0)
    got = np.concatenate([got, run(1, [int(tails[0][0])])])
    want = R.forward(np.concatenate([prompt, tails[0][:1]]), cfg, weights)[skip:]
    d = got - want
    assert np.abs(d).max() <= 2e-5 * 5 * want.std()          # rms 2e-5 of the logits' scale (the model's bound in fp32), five times that at most


def test_four_bit_linear_refuses_other_results():
    ops = load_pkg("ops")
    w = ops.quantize(torch.randn(32, 64, device=DEV), 32)
    x = torch.randn(3, 64, device=DEV).half()
    for kw in ({"out_dtype": torch.bfloat16}, {"out": torch.empty(3, 32, dtype=torch.bfloat16, device=DEV)}):
        with pytest.raises(TypeError):
            ops.linear(x, w, **kw)
    with pytest.raises(ValueError):
        ops.linear(x, w, kernel="gemm")
