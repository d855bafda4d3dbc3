"""Plans over shared prefixes as batches live: rows that outgrow them, copies of a cache, steps recorded with them."""
import copy

import numpy as np
import pytest
import torch

import test_shared_attention_gpu as A
from conftest import load_pkg

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def model():
    synth = load_pkg("synth")
    wl = synth.config1()
    return load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV)


def behind_one_prefix(model, rows, pages, room, seed=0):
    """A cache whose sequences share `pages` pages of keys and values, and have a few tokens of their own."""
    rng = np.random.default_rng(seed)
    V = model.shape.vocab_size
    head = rng.integers(0, V, 16 * pages).astype(np.int32)
    longest = 16 * pages + room
    kv = model.create_paged_kv_cache(rows, 16 * pages + rows * (room + 32), longest, 16, max_seq_len=longest)
    for i in range(rows):
        kv.add_sequence(i)
        skip = kv.share_prefix(i, 0, len(head)) if i else 0
        prompt = np.concatenate([head, rng.integers(0, V, 2 + 3 * i).astype(np.int32)])
        kv.begin_forward([i], [len(prompt) - skip])
        model["prefill_no_adapter"](model.embed(torch.from_numpy(np.ascontiguousarray(prompt[skip:]))), kv)
        kv.end_forward()
    return kv


@pytest.mark.parametrize("Hq,Hkv,D,own", [(32, 8, 128, (130, 700, 40, 1)), (8, 8, 64, (2000, 3, 500))])
def test_plans_of_either_length(ops, Hq, Hkv, D, own):
    """The plan of the first step and the one for the contexts as they have become give results within their bounds of the definition."""
    print("case either plan", Hq, Hkv, D, own, flush=True)
    rows = len(own)
    lens = [160 + n for n in own]
    c = A.build(ops, rows, [(list(range(rows)), 10)], lens, Hq, Hkv, D)
    early = ops.SharedPrefixPlan([(list(range(rows)), 10)], [161] * rows, Hq, Hkv, D, DEV)
    assert early.outgrown(lens) and early.own_splits == 1 and not c["plan"].outgrown(lens)
    A.close(A.call(ops, c), c)
    A.close(A.call(ops, {**c, "plan": early}), c)


def test_recorded_sessions_follow_their_plan(model):
    """A batch that outgrows its plan twice: replayed steps choose what eager ones choose, on the plan that the cache has by then."""
    print("case outgrown", flush=True)
    ds = load_pkg("decode_session")
    rows, steps = 4, 420
    out, plans = {}, {}
    for graph in (False, True):
        kv = behind_one_prefix(model, rows, 128, steps + 40)
        s = ds.DecodeSession(model, kv, list(range(rows)), {}, [5, 6, 7, 8], use_graph=graph)
        plans[graph] = []
        for _ in range(steps):
            s.step(keep_history=True)
            if not plans[graph] or kv.plan is not plans[graph][-1]:
                plans[graph].append(kv.plan)
            assert not graph or s._eager_steps == 1
        assert not graph or s._plan is kv.plan
        out[graph] = torch.stack(s.history).cpu().numpy()
    assert [p.own_splits for p in plans[True]] == [p.own_splits for p in plans[False]] == [1, 2, 4]
    assert np.array_equal(out[True], out[False])


def test_copy_of_a_cache_decodes_when_the_original_is_gone(model):
    print("case copied cache", flush=True)
    rows = 3
    kv = behind_one_prefix(model, rows, 130, 80)
    sids, tokens = list(range(rows)), torch.tensor([3, 4, 5], dtype=torch.int32)

    def step(cache):
        cache.begin_forward(sids, [1] * rows)
        logits, _ = model["decode_no_adapter"](model.embed(tokens), cache)
        cache.end_forward()
        assert cache.plan is not None
        return logits

    step(kv)
    other = copy.deepcopy(kv)
    want = step(kv)
    old = kv.plan.data
    kv.plan, kv._plans = None, {}
    old.fill_(-1)                                            # what the original's plan said
    del kv, old
    assert torch.equal(step(other), want)


@pytest.mark.parametrize("adapters,dense,pages,once", [(False, False, 300, True), (True, True, 300, True), (True, False, 300, True), (True, True, 140, False)])
def test_front_end_reads_shared_pages_once_where_that_pays(model, monkeypatch, adapters, dense, pages, once):
    """A batch that the native step could serve goes through the attention over shared prefixes where that pays, and there alone; every token is the model's own
    choice along its path (up to near ties: shorter prefills sum in another order)."""
    print("case front end once", adapters, dense, pages, flush=True)
    ab, xg, lora, kvm = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), load_pkg("lora"), load_pkg("kv_cache")
    made, shared = [], kvm.ops.paged_attn_decode_shared
    monkeypatch.setattr(kvm.ops, "paged_attn_decode_shared", lambda *a, **k: made.append(1) or shared(*a, **k))
    V, steps, rows = model.shape.vocab_size, 10, 4
    rng = np.random.default_rng(pages)
    head = rng.integers(0, V, 16 * pages).astype(np.int32)
    prompts = [np.concatenate([head, rng.integers(0, V, 2 + 7 * i).astype(np.int32)]) for i in range(rows)]
    longest = 16 * pages + 60
    lt = model.lora_types[0]
    batcher = ab.LlamaAutoBatcherClass()
    batcher.set_model(model)
    batcher.set_exec_config(xg.LlamaExecConfig(max_prompt_len=longest, max_gen_len=steps, page_size=16, share_prefix=True, dense_lora=dense))
    out = []
    for p in prompts:
        if adapters:
            batcher.set_adapter(lora.LoraConfig(r=lt.r, alpha=lt.scaling * lt.r), wid=1)
        out.append(batcher.generate(batcher.create_var(p)))
    batcher.compile()
    batcher.execute()
    assert (len(made) >= model.shape.num_hidden_layers) == once and bool(made) == once
    kv = model.create_paged_kv_cache(rows, rows * (longest + 32), longest, 16, max_seq_len=longest + 32)
    def tokens_of(sid, toks, kind):
        kv.begin_forward([sid], [len(toks)])
        h = model.embed(torch.from_numpy(np.ascontiguousarray(toks)))
        if adapters:
            z, _ = model[f"{kind}_a0"](h, kv, [1] if kind == "prefill" else np.array([1], dtype=np.int32))
        else:
            z, _ = model[f"{kind}_no_adapter"](h, kv)
        kv.end_forward()
        return z[0]
    for s, p in enumerate(prompts):
        kv.add_sequence(s)
        z = tokens_of(s, p, "prefill")
        answer = list(map(int, out[s].var))
        assert len(answer) == steps
        for t in answer:
            assert float(z.max() - z[t]) <= 2e-2 * float(z.std())
            z = tokens_of(s, np.array([t], dtype=np.int32), "decode")


@pytest.mark.parametrize("planned", [False, True])
def test_pass_begun_inside_a_capture(model, planned):
    """Recorded with the plan that is there or with none, a step's replays give what an eager step gives."""
    print("case pass in a capture", planned, flush=True)
    rows = 3
    kv = behind_one_prefix(model, rows, 130, 80)
    sids, tokens = list(range(rows)), torch.tensor([3, 4, 5], dtype=torch.int32, device=DEV)

    def step(meta):
        kv.begin_forward(sids, [1] * rows, device_meta=meta)
        logits = model.forward(model.embed(tokens), kv, {})
        kv._cur = None                                       # the same step again: its keys and values are written anew
        return logits

    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    at = [kv.lens[s] for s in sids]
    meta = i32([kv.slot[s] for s in sids]), i32(at), i32([n + 1 for n in at])
    want = step(meta)
    plan = kv.plan
    assert plan is not None
    if not planned:
        kv._plans.clear()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(meta)
    assert kv.plan is (plan if planned else None)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        if planned:
            assert torch.equal(got, want)
        else:
            assert float((got - want).abs().max() / want.std()) <= 1e-2          # (whole-model bound, as against the oracle)
        again = step(meta)
        assert kv.plan is not None and torch.equal(again, want)
        if not planned:
            kv._plans.clear()
