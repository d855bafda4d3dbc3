"""Searches by beams and what runs beside them, on the device: orders that values do not tell, the front end on every kind of cache, adapters of several types."""
import numpy as np
import pytest
import torch

from conftest import load_pkg
from test_page_caches_gpu import begin, front_end, prompts_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def selected(ops, z, scores, k):
    scores, tokens, parents = ops.beam_select(torch.from_numpy(z).to(DEV), torch.tensor(scores, dtype=torch.float32, device=DEV), k=k)
    return scores.cpu(), tokens.cpu().tolist(), parents.cpu().tolist()


def test_logits_closer_than_their_values(ops):
    """Logits so small that their values are one number in 64 bits: a beam's order is still that of its logits, whatever columns they are in."""
    V = 5000
    z = np.zeros((1, V), np.float32)
    z[0, [4000, 10, 20, 4999, 700]] = 2e-20, 1e-20, 3e-20, 2e-20, -1e-20
    _, tokens, parents = selected(ops, z, [[-1.0]], 6)
    assert tokens == [[20, 4000, 4999, 10, 0, 1]] and parents == [[0] * 6]
    # descending columns, more of them than are asked for: the greatest, not the first
    z = np.zeros((1, V), np.float32)
    z[0, 100:140] = np.arange(1, 41, dtype=np.float32) * np.float32(2.0 ** -70)
    assert selected(ops, z, [[0.0]], 32)[1] == [list(range(139, 107, -1))]
    # between beams such values are equal, and the lower beam goes first
    z = np.zeros((3, V), np.float32)
    z[0, 77], z[1, 5], z[2, 9] = 1e-20, 9e-20, 5e-20
    _, tokens, parents = selected(ops, z, [[0.0, 0.0, 0.0]], 4)
    assert tokens == [[77, 0, 1, 2]] and parents == [[0, 0, 0, 0]]
    _, tokens, parents = selected(ops, z, [[-1.0, 0.0, -2.0]], 3)
    assert tokens == [[5, 0, 1]] and parents == [[1, 1, 1]]


@pytest.fixture(scope="module")
def two_types():
    """A model with adapters of two types and ranks."""
    synth = load_pkg("synth")
    wl = synth.config1()
    specs = [wl.lora, synth.LoraSpec(r=16, alpha=8.0, n_adapters=3, targets=("q_proj", "k_proj", "o_proj"))]
    return load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, specs, DEV)


def host_search(model, kv, sids, z, adapters, W, steps):
    """The search of prefilled sequences with logits z [R, V], over forks that the host makes and frees, chosen in 64 bits; adapters: {type: ids [R]}.  Scores [R, W], tokens."""
    V, R = z.shape[1], len(sids)
    ids = model._merge_types({t: i.repeat_interleave(W) for t, i in adapters.items()}) if adapters else {}
    live, z, made = [[s] for s in sids], z[:, None], 0
    scores, paths = np.zeros((R, 1)), [[[]] for _ in range(R)]
    for i in range(steps + 1):
        lp, tokens, found = torch.log_softmax(z.double(), -1).cpu().numpy(), [], []
        for r in range(R):
            value = scores[r][:, None] + lp[r]
            best = np.argsort(-value.reshape(-1), kind="stable")[:W]
            found.append(value.reshape(-1)[best].astype(np.float32))
            paths[r] = [paths[r][b // V] + [int(b % V)] for b in best]
            new = []
            for b in best:
                made += 1
                new.append(("host", made))
                kv.fork(new[-1:], live[r][b // V])
            for s in live[r]:
                kv.free_sequence(s)
            live[r] = new
            tokens += (best % V).tolist()
        scores = np.stack(found).astype(np.float64)
        if i < steps:
            flat = [s for beams in live for s in beams]
            kv.begin_forward(flat, [1] * len(flat))
            z = model.forward(model.embed(torch.tensor(tokens, dtype=torch.int32)), kv, ids).view(R, W, V)
            kv.end_forward()
    return scores, paths


def alike(model, got, scores, paths, steps):
    """Answers (score, tokens) of a session are those of host_search: each step's sum of V exponentials in fp32 is off by V half steps at most, and its value is rounded once."""
    V = model.shape.vocab_size
    tol = (steps + 1) * (V * 2.0 ** -24 + 2.0 ** -24 * np.abs(scores).max())
    for answers, s, p in zip(got, scores, paths):
        assert [t for _, t in answers] == p
        assert np.abs(np.array([v for v, _ in answers]) - s).max() <= tol


@pytest.mark.parametrize("form", [{}, {"bits": 8}])
@pytest.mark.parametrize("graph", [False, True])
def test_search_over_adapters_of_several_types(two_types, form, graph):
    """Beside each other: a request of each type, one without, and one more of the first."""
    model, W, steps = two_types, 3, 20
    ds = load_pkg("decode_session")
    prompts, kinds = prompts_of(model, (40, 16, 3, 25), 31), [(0, 1), (1, 2), None, (0, 3)]

    def prefilled():
        kv = model.create_paged_kv_cache(2 * 4 * W, 2 * 4 * W * 112, 64, 16, max_seq_len=112, **form)
        z = []
        for i, (p, kind) in enumerate(zip(prompts, kinds)):
            kv.add_sequence(i)
            kv.begin_forward([i], [len(p)])
            h = model.embed(torch.from_numpy(p))
            z.append(model["prefill_no_adapter"](h, kv)[0] if kind is None else model[f"prefill_a{kind[0]}"](h, kv, [kind[1]])[0])
            kv.end_forward()
        return kv, torch.cat(z)

    pairs = {t: ([i for i, k in enumerate(kinds) if k and k[0] == t], [k[1] for k in kinds if k and k[0] == t]) for t in (0, 1)}
    adapters = model._ids(4, pairs)
    kv, z = prefilled()
    scores, paths = host_search(model, kv, range(4), z, adapters, W, steps)
    kv, z = prefilled()
    s = ds.BeamSession(model, kv, range(4), adapters, z, W, steps=steps, use_graph=graph)
    for _ in range(steps):
        s.step()
    alike(model, s.answers(), scores, paths, steps)
    s.close()
    # the types matter: a request answers otherwise without its adapter
    kv, z = prefilled()
    bare = ds.BeamSession(model, kv, range(4), {}, z, W, steps=steps)
    for _ in range(steps):
        bare.step()
    assert bare.answers()[2][0][1] == paths[2][0] and any(bare.answers()[i][0][1] != paths[i][0] for i in (0, 1, 3))


@pytest.mark.parametrize("config", [{}, {"share_prefix": True}, {"cache_bits": 8}, {"window": 30, "sinks": 4}])
def test_front_end_searches_on_every_cache(two_types, config):
    """From the prompts to the answers, with two adapters of one type and a request without: what the host's search finds on a cache that was filled by the same passes."""
    model, W, limit = two_types, 3, 20
    prompts, wids = prompts_of(model, (60, 20, 45), 33), [0, 2, 0]
    prompts[2] = np.concatenate([prompts[0][:32], prompts[2][:13]])
    got, b = front_end(model, prompts, wids, [limit] * 3, beams=W, **config)
    order = b.seq_info.order_seqs([0, 1, 2])[0]
    form = {k: v for k, v in (("bits", config.get("cache_bits", 16)), ("window", config.get("window")), ("sinks", config.get("sinks", 0)))}
    kv = model.create_paged_kv_cache(2 * 3 * W, 2 * 3 * W * 112, 64, 16, max_seq_len=88, **form)
    z = {}
    for i, (p, w) in enumerate(zip(prompts, wids)):
        kv.add_sequence(i)
        n = kv.share_prefix(i, 0, 32) if i == 2 and "share_prefix" in config else 0
        assert n == (32 if i == 2 and "share_prefix" in config else 0)
        kv.begin_forward([i], [len(p) - n])
        z[i] = model["prefill_a0"](model.embed(torch.from_numpy(p[n:])), kv, [w])[0]
        kv.end_forward()
    ids = model._ids(3, {0: (None, [wids[i] for i in order])})
    # (one type: rows of one bucket, as the front end's decode has them)
    _, paths = one_type_search(model, kv, order, torch.cat([z[i] for i in order]), ids[0], W, limit - 1)
    assert [got[i] for i in order] == [p[0] for p in paths]
    assert sorted(b.graph.kv_cache.slot) == [0, 1, 2]


def one_type_search(model, kv, sids, z, ids, W, steps):
    class One:
        shape, embed, _merge_types = model.shape, model.embed, staticmethod(lambda t: t)

        @staticmethod
        def forward(h, kv, adapters):
            return model.forward(h, kv, adapters)

    return host_search(One, kv, sids, z, {0: ids}, W, steps)


@pytest.mark.parametrize("form", [{"window": 40, "sinks": 2}, {"bits": 8, "window": 33}, {"window": 20}])
@pytest.mark.parametrize("graph", [False, True])
def test_searches_beside_sequences_that_give_pages_back(two_types, form, graph):
    """Greedy sequences of many lengths give pages back under a window while searches' rows are known on the device alone: each gives what it gives by itself."""
    model, steps = two_types, 45
    ds = load_pkg("decode_session")
    lens = {"p": 48, "q": 30, "a": 49, "b": 55, "c": 61, "d": 64}
    prompts = dict(zip(lens, prompts_of(model, lens.values(), 35)))

    def made(which):
        kv, out = model.create_paged_kv_cache(12, 12 * 128, 64, 16, max_seq_len=128, **form), {}
        for i in which:
            z = begin(model, kv, i, prompts[i])
            out[i] = ds.BeamSession(model, kv, [i], {}, z, 4, steps=steps, use_graph=graph) if i in "pq" else \
                ds.DecodeSession(model, kv, [i], {}, z.argmax(-1).int(), use_graph=graph)
        return kv, out

    def result(s):
        return s.answers() if isinstance(s, ds.BeamSession) else torch.stack(s.history).tolist()

    def run(sessions):
        for _ in range(steps):
            for i, s in sessions.items():
                s.step(**({} if i in "pq" else {"keep_history": True}))
        return {i: result(s) for i, s in sessions.items()}

    alone = {}
    for i in lens:
        alone.update(run(made([i])[1]))
    kv, sessions = made(lens)
    assert run(sessions) == alone
    for i in "pq":
        sessions[i].close()
    for i in lens:
        kv.free_sequence(i)
    assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners


def test_together_on_a_4_bit_model_that_shares_prefixes():
    """Every request's answer: the second's prompt is prefilled behind the pages that it takes over, here as in the front end."""
    synth = load_pkg("synth")
    wl = synth.config1()
    model = load_pkg("llama").LlamaForCausalLM.from_synthetic(wl.seed, wl.shape, [wl.lora], DEV, quant_group=64)
    prompts = prompts_of(model, (50, 50, 21), 37)
    prompts[1] = np.concatenate([prompts[0][:40], prompts[1][:10]])
    got, b = front_end(model, prompts, [1, 1, 1], [24] * 3, beams=3, cache_bits=8, window=36, sinks=2, share_prefix=True)
    order = b.seq_info.order_seqs([0, 1, 2])[0]
    kv = model.create_paged_kv_cache(20, 20 * 112, 64, 16, max_seq_len=88, bits=8, window=36, sinks=2)
    z = {}
    for i, p in enumerate(prompts):
        kv.add_sequence(i)
        n = kv.share_prefix(i, 0, 40) if i == 1 else 0
        kv.begin_forward([i], [len(p) - n])
        z[i] = model["prefill_a0"](model.embed(torch.from_numpy(p[n:])), kv, [1])[0]
        kv.end_forward()
    _, paths = one_type_search(model, kv, order, torch.cat([z[i] for i in order]), model._ids(3, {0: (None, [1, 1, 1])})[0], 3, 23)
    assert [got[i] for i in order] == [p[0] for p in paths]


def searched(ds, model, kv, prompts, W, steps, **kw):
    z = torch.cat([begin(model, kv, i, p) for i, p in enumerate(prompts)])
    return ds.BeamSession(model, kv, range(len(prompts)), {}, z, W, steps=steps, **kw)


@pytest.mark.parametrize("form", [{}, {"bits": 8, "window": 40, "sinks": 2}])
def test_searches_whose_prompts_ran_at_once(two_types, form):
    """The front end with batch_prefill, against a search behind the same pass over all prompts."""
    model, W, limit = two_types, 3, 20
    prompts, wids = prompts_of(model, (60, 20, 45), 41), [0, 2, 0]
    config = {"cache_bits": form.get("bits", 16), "window": form.get("window"), "sinks": form.get("sinks", 0)}
    got, b = front_end(model, prompts, wids, [limit] * 3, beams=W, batch_prefill=True, **config)
    order = b.seq_info.order_seqs([0, 1, 2])[0]
    kv = model.create_paged_kv_cache(2 * 3 * W, 2 * 3 * W * 112, 64, 16, max_seq_len=88, **form)
    lens = [len(p) for p in prompts]
    for i in range(3):
        kv.add_sequence(i)
    kv.begin_forward([0, 1, 2], lens)
    ids = model._ids(sum(lens), {0: (None, np.repeat(np.array(wids, np.int32), lens))})
    z = model.forward(model.embed(torch.from_numpy(np.concatenate(prompts))), kv, ids, model._last_rows(kv))
    kv.end_forward()
    _, paths = one_type_search(model, kv, order, z[torch.tensor(order, device=DEV)], model._ids(3, {0: (None, [wids[i] for i in order])})[0], W, limit - 1)
    assert [got[i] for i in order] == [p[0] for p in paths]


@pytest.mark.parametrize("form", [{}, {"bits": 8}, {"window": 40, "sinks": 2}])
@pytest.mark.parametrize("graph", [False, True])
def test_searches_on_another_stream_and_again(two_types, form, graph):
    """On a stream of their own, with the default stream's passes and closed searches in between: the same answers."""
    model, steps, W = two_types, 36, 4
    ds = load_pkg("decode_session")
    prompts = prompts_of(model, (47, 30), 43)
    make = lambda: model.create_paged_kv_cache(10, 10 * 112, 64, 16, max_seq_len=112, **form)                              # noqa: E731
    s = searched(ds, model, make(), prompts, W, steps)
    for _ in range(steps):
        s.step()
    want = s.answers()
    side, kv = torch.cuda.Stream(), make()
    for again in range(2):
        with torch.cuda.stream(side):
            s = searched(ds, model, kv, prompts, W, steps, use_graph=graph)
        for j in range(steps):
            with torch.cuda.stream(side):
                s.step()
            if j % 9 == 4:
                begin(model, kv, "x", prompts[1][:20 + j])
            if j % 9 == 7:
                kv.free_sequence("x")
        with torch.cuda.stream(side):
            got = s.answers()
        assert got == want, again
        s.close()
        for i in (0, 1):
            kv.free_sequence(i)
    assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners


def test_a_step_that_fails_on_the_device_s_side(two_types, monkeypatch):
    """Behind the reordering's launch: the rows are read back, the forks go, and the cache serves the next search as a new one does."""
    model, steps, W = two_types, 20, 4
    ds, ops = load_pkg("decode_session"), load_pkg("ops")
    prompts = prompts_of(model, (47, 30), 45)
    answers = []
    for broken in (True, False):
        kv = model.create_paged_kv_cache(10, 10 * 112, 64, 16, max_seq_len=112)
        if broken:
            s = searched(ds, model, kv, prompts, W, steps)
            for _ in range(5):
                s.step()

            def refuse(*a):
                raise RuntimeError("refused")

            with monkeypatch.context() as m:
                m.setattr(ops, "copy_pages", refuse)
                with pytest.raises(RuntimeError, match="refused"):
                    s.step()
            with pytest.raises(RuntimeError):
                s.step()
            s.close()
            table = kv.block_table[torch.tensor(kv.rows_of([0, 1]), device=DEV).long()].cpu().numpy()
            assert (table == kv.table_h[kv.rows_of([0, 1])]).all()
            for i in (0, 1):
                kv.free_sequence(i)
            assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners
        s = searched(ds, model, kv, prompts, W, steps)
        for _ in range(steps):
            s.step()
        answers.append(s.answers())
    assert answers[0] == answers[1]


def test_requests_whose_numbers_are_gone(two_types):
    """Logits that are NaN, or infinite in every row: no beams, no answer, and the other request's is its own."""
    model, steps = two_types, 12
    ds = load_pkg("decode_session")
    prompts = prompts_of(model, (47, 30, 12), 47)
    make = lambda: model.create_paged_kv_cache(12, 12 * 112, 64, 16, max_seq_len=112)                                      # noqa: E731
    s = searched(ds, model, make(), prompts[:1], 3, steps, eos=5)
    for _ in range(steps):
        s.step()
    want = s.answers()
    kv = make()
    z = torch.cat([begin(model, kv, i, p) for i, p in enumerate(prompts)])
    z[1], z[2, 77] = torch.nan, torch.inf
    for graph in (False, True):
        kv2 = make()
        for i, p in enumerate(prompts):
            begin(model, kv2, i, p)
        s = ds.BeamSession(model, kv2, range(3), {}, z, 3, eos=5, steps=steps, use_graph=graph)
        for _ in range(steps):
            s.step()
        assert not s.done()
        got = s.answers()
        assert [t for _, t in got[0]] == [t for _, t in want[0]] and got[1:] == [[], []]
        s.close()
        assert sorted(kv2.slot) == [0, 1, 2]
    s = ds.BeamSession(model, kv, [1, 2], {}, z[1:], 3)
    s.step()
    assert s.done()


@pytest.mark.parametrize("form", [{}, {"bits": 8}, {"window": 24, "sinks": 1}])
def test_wide_searches(two_types, form):
    """96 rows, for which a step takes its forms for wide batches: requests of 16 beams, with adapters."""
    model, W, steps = two_types, 16, 18
    ds = load_pkg("decode_session")
    prompts, wids = prompts_of(model, (40, 31, 3, 25, 16, 64), 51), [0, 1, 2, 3, 0, 1]

    def prefilled():
        kv = model.create_paged_kv_cache(2 * 6 * W, 2 * 6 * W * 112, 64, 16, max_seq_len=112, **form)
        z = []
        for i, (p, w) in enumerate(zip(prompts, wids)):
            kv.add_sequence(i)
            kv.begin_forward([i], [len(p)])
            z.append(model["prefill_a0"](model.embed(torch.from_numpy(p)), kv, [w])[0])
            kv.end_forward()
        return kv, torch.cat(z)

    ids = model._ids(6, {0: (None, wids)})
    kv, z = prefilled()
    scores, paths = one_type_search(model, kv, range(6), z, ids[0], W, steps)
    for graph in (False, True):
        kv, z = prefilled()
        s = ds.BeamSession(model, kv, range(6), ids, z, W, steps=steps, use_graph=graph)
        for _ in range(steps):
            s.step()
        alike(model, s.answers(), scores, paths, steps)
        s.close()
        for i in range(6):
            kv.free_sequence(i)
        assert sorted(kv.free) == list(range(kv.n_pages)) and not kv._owners
