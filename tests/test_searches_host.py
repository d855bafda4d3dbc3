"""Searches beside other work on one cache, and searches that fail: the host's side of them, on the CPU."""
import numpy as np
import pytest
import torch

from conftest import load_pkg
from test_page_caches_host import PAGE, Device, cache, grow, sound


def begun(kv, sid, n, W):
    """A sequence of n tokens and its W - 1 forks (whose last page's contents the CPU does not copy)."""
    kv.add_sequence(sid)
    grow(kv, sid, n - n % PAGE)
    kv.fork([(sid, w) for w in range(1, W)], sid)
    sids = [sid] + [(sid, w) for w in range(1, W)]
    for s in sids if n % PAGE else ():
        grow(kv, s, n % PAGE)
    return Device(kv, sids, W)


def visible(kv, beams):
    """Of the beams' rows on the device, the blocks that their next tokens see (others may have gone back)."""
    j = torch.arange(kv.max_blocks)
    seen = (j >= max(0, kv.lens[beams.sids[0]] - kv.window + 1) // PAGE) | (j < -(-kv.sinks // PAGE))
    return kv.block_table[beams.slots.long()][:, seen].clone()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window", range(33, 49))
def test_passes_of_others_leave_the_rows_of_beams(window, bits):
    """Sequences of every length modulo 16 give pages back, by passes whose arrays are on the device, while a search's rows are known there alone."""
    rng = np.random.default_rng(window)
    released = 0
    for first in range(48, 64):
        kv = cache(pages=90, seqs=9, blocks=10, bits=bits, window=window, sinks=window % 3)
        beams = begun(kv, "p", 30, 4)
        kv.add_sequence("x")
        grow(kv, "x", first)
        slot = torch.tensor([kv.slot["x"]], dtype=torch.int32)
        for i in range(40):
            if i % 16 == 0:
                kv.reserve(beams.sids, PAGE)
            beams.step(rng, i)
            before, gone = visible(kv, beams), kv._gone.get("x")
            kv.begin_forward(["x"], [1], device_meta=(slot, None, None))
            kv.end_forward()
            released += kv._gone.get("x") != gone
            assert torch.equal(visible(kv, beams), before), (first, i)
        kv.settle()
        sound(kv)
        assert [kv.slot[s] for s in beams.sids] == beams.slots.tolist()
    assert released > 16


@pytest.mark.parametrize("window,sinks,lens", [(40, 2, (48, 30)), (40, 2, (60, 21)), (20, 0, (60, 16)), (36, 5, (35, 60))])
def test_searches_under_a_window_beside_each_other(window, sinks, lens):
    rng = np.random.default_rng(window + lens[0])
    kv = cache(pages=120, seqs=9, blocks=12, window=window, sinks=sinks)
    both = [begun(kv, s, n, 4) for s, n in zip("pq", lens)]
    for i in range(80):
        for one, other in (both, both[::-1]):
            if kv.lacks_page(one.sids[0]):
                kv.reserve(one.sids, PAGE)
            before = visible(kv, other)
            one.step(rng, i)
            assert i == 0 or torch.equal(visible(kv, other), before), i        # (ahead of its first step a search's rows are on the host alone)
    kv.settle()
    sound(kv)


class Model:
    """Logits from a table, a row for every token; `fails` raises instead."""

    cache_forms, device = True, "cpu"

    def __init__(self, V=50, seed=0):
        self.table = torch.randn((V, V), generator=torch.Generator().manual_seed(seed))
        self.fails = False

    def embed(self, tokens):
        return self.table[tokens.long()]

    def forward(self, hidden, kv, tok_adapter):
        if self.fails:
            raise RuntimeError("a forward pass that fails")
        return hidden


def select(logits, scores, ended=None, eos=None, k=None):
    """ops.beam_select on the CPU."""
    (R, W), V = scores.shape, logits.shape[1]
    k = W if k is None else k
    value = scores.double()[..., None] + logits.double().log_softmax(-1).view(R, W, V)
    if ended is not None:
        only = torch.where(torch.arange(V) == eos, scores.double()[..., None], -torch.inf)
        value = torch.where(ended[..., None] != 0, only, value)
    value = torch.where(value > -torch.inf, value, -torch.inf).view(R, W * V)
    value = torch.nn.functional.pad(value, (0, max(0, k - W * V)), value=-torch.inf)
    best, at = value.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k].int()
    none = best == -torch.inf
    return best.float(), torch.where(none, -1, at % V), torch.where(none, -1, at // V)


def reorder(parents, slots, table, ctx):
    """ops.beam_reorder on the CPU, without the moves."""
    (R, W), new, old = parents.shape, slots.clone(), table.clone()
    for r in range(R):
        p, mine = parents[r].tolist(), slots.view(R, W)[r].tolist()
        dead, block = [w for w in range(W) if w not in p], int(ctx[r * W]) // PAGE
        for w in range(W):
            stays = p[w] >= 0 and p[w] not in p[:w]
            to = mine[p[w]] if stays else mine[dead.pop(0)]
            if p[w] >= 0 and not stays:
                table[to, :block] = old[mine[p[w]], :block]
            new[r * W + w] = to
    return new, load_pkg("ops").BeamMoves(new, new, new, new)


@pytest.fixture
def on_cpu(monkeypatch):
    ops = load_pkg("ops")
    monkeypatch.setattr(ops, "beam_select", select)
    monkeypatch.setattr(ops, "beam_reorder", reorder)
    monkeypatch.setattr(ops, "copy_pages", lambda *a: None)
    return load_pkg("decode_session")


def prompts(kv, lens):
    for sid, n in lens.items():
        kv.add_sequence(sid)
        grow(kv, sid, n)


def test_a_search_gives_back_its_own_forks_alone(on_cpu):
    """Whatever the caller's sequences are called, and however often a search is closed."""
    kv = cache(pages=60, seqs=12)
    prompts(kv, {0: 32, ("beam", "mine"): 48, ("beam", 7, 1): 16})
    model = Model()
    ids = [0, ("beam", "mine"), ("beam", 7, 1)]
    s = on_cpu.BeamSession(model, kv, ids, {}, model.table[:3], 3)
    for _ in range(20):
        s.step()
    s.close()
    assert list(kv.slot) == ids
    sound(kv)
    s.close()
    assert list(kv.slot) == ids and [len(kv.pages_of(i)) for i in ids] == [4, 5, 3]
    again = on_cpu.BeamSession(model, kv, ids, {}, model.table[:3], 4)
    again.step()
    again.close()
    assert list(kv.slot) == ids
    sound(kv)


def test_a_search_that_does_not_begin_leaves_nothing(on_cpu, monkeypatch):
    """Refused logits, adapters that cannot be merged, no memory for what a search holds: the forks go back, and the next search begins."""
    kv = cache(pages=60, seqs=12)
    prompts(kv, {0: 32, 1: 48})
    model, ops, rows = Model(), load_pkg("ops"), torch.zeros(2, dtype=torch.int32)

    def refuse(*a, **k):
        raise RuntimeError("refused")

    def attempt(adapters):
        with pytest.raises(RuntimeError):
            on_cpu.BeamSession(model, kv, [0, 1], adapters, model.table[:2], 4)
        assert list(kv.slot) == [0, 1]
        sound(kv)

    model._merge_types = refuse
    attempt({0: rows, 1: rows})
    for of, name in ((ops, "beam_select"), (torch, "zeros"), (torch, "empty")):
        with monkeypatch.context() as m:
            m.setattr(of, name, refuse)
            if name != "zeros":                       # (flags of beams that have ended are made where there is an end)
                attempt({0: rows})
            else:
                with pytest.raises(RuntimeError):
                    on_cpu.BeamSession(model, kv, [0, 1], {0: rows}, model.table[:2], 4, eos=3)
                assert list(kv.slot) == [0, 1]
    s = on_cpu.BeamSession(model, kv, [0, 1], {0: rows}, model.table[:2], 4)
    s.step()
    s.close()
    sound(kv)


@pytest.mark.parametrize("kw", [{}, {"bits": 8}, {"window": 20, "sinks": 2}])
def test_a_fork_whose_copy_fails_leaves_nothing(kw):
    """The copy of the last page's contents is refused where the cache is not on the current device (here on none)."""
    kv = cache(pages=60, seqs=12, **kw)
    prompts(kv, {"a": 53})
    table = kv.table_h.copy()
    with pytest.raises(ValueError):
        kv.fork(["b", "c"], "a")
    assert list(kv.slot) == ["a"] and kv.lens == {"a": 53} and (kv.table_h == table).all() and len(kv.free_slots) == 11
    assert set(kv._gone) <= {"a"}
    sound(kv)


@pytest.mark.parametrize("where", ["forward", "beam_select", "beam_reorder", "copy_pages"])
@pytest.mark.parametrize("kw", [{}, {"window": 20, "sinks": 2}])
def test_a_step_that_fails_ends_the_search(on_cpu, monkeypatch, where, kw):
    """Wherever it fails, the host knows the rows that the device has, and forks and pages go back."""
    kv = cache(pages=60, seqs=12, **kw)
    prompts(kv, {0: 32, 1: 48, "x": 5})
    model, ops = Model(), load_pkg("ops")
    s = on_cpu.BeamSession(model, kv, [0, 1], {}, model.table[:2], 4)
    for _ in range(5):
        s.step()

    def refuse(*a, **k):
        raise RuntimeError("refused")

    with monkeypatch.context() as m:
        if where == "forward":
            model.fails = True
        else:
            m.setattr(ops, where, refuse)
        with pytest.raises(RuntimeError):
            s.step()
    model.fails = False
    assert kv.lens[0] == 37 and kv.lens[1] == 53
    with pytest.raises(RuntimeError):                 # (its state may be of half a step)
        s.step()
    table = kv.block_table.clone()
    grow(kv, "x", 1)                                  # another's pass, which reads the rows back
    kv.settle()
    rows = [kv.slot[i] for i in s.seq_ids]
    assert torch.equal(torch.from_numpy(kv.table_h[rows]), table[rows])
    sound(kv)
    s.close()
    assert list(kv.slot) == [0, 1, "x"]
    sound(kv)


def test_a_step_without_room_can_be_taken_again(on_cpu):
    """No page for the next token: nothing has been queued, and the search goes on when there is one."""
    kv = cache(pages=10, seqs=6)
    prompts(kv, {0: 32, "x": 64})
    model = Model()
    want = cache(pages=30, seqs=6)
    prompts(want, {0: 32})
    both = [on_cpu.BeamSession(model, c, [0], {}, model.table[:1], 4) for c in (kv, want)]
    for _ in range(16):
        for s in both:
            s.step()
    with pytest.raises(RuntimeError):                 # (four pages are wanted; the four of the first 16 tokens are not all given up)
        both[0].step()
    kv.free_sequence("x")
    for _ in range(9):
        for s in both:
            s.step()
    assert both[0].answers() == both[1].answers()
    both[0].close()
    sound(kv)


class Served(dict):
    """The front end's model: entry points by name."""

    cache_forms, native_step, lora_types, device, vocab_size = True, False, (), "cpu", 50

    def __init__(self, kv, bad=()):
        super().__init__(create_paged_kv_cache=lambda *a, **k: kv, embed=lambda t: Model.embed(self, t.reshape(-1)), prefill_no_adapter=self.prefill)
        self.table, self.fails, self.bad, self.kv = Model().table, False, set(bad), kv

    def prefill(self, hidden, kv):
        logits = hidden[-1:].clone()
        if kv._cur[0][0] in self.bad:
            logits[:] = torch.nan
        return logits, None

    embed, forward = Model.embed, Model.forward

    def _ids(self, n, pairs):
        return {}


def front_end(kv, lens, bad=(), rules=None, **config):
    """(batcher, answers) of requests of these lengths, whose limits are 20 tokens."""
    ab, xg = load_pkg("auto_batcher"), load_pkg("llama_exec_graph")
    b = ab.LlamaAutoBatcherClass()
    b.set_model(Served(kv, bad))
    b.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=24, page_size=16, native_decode=False, **config))
    out = []
    for i, n in enumerate(lens):
        if rules is not None and rules[i] is not None:
            b.set_rules(rules[i])
        out.append(b.generate(b.create_var(np.arange(n, dtype=np.int32) % 50), max_gen_len=20))
    b.compile()
    return b, out


@pytest.fixture
def served(on_cpu, monkeypatch):
    class Eager(on_cpu.BeamSession):
        def __init__(self, *a, use_graph, **kw):
            super().__init__(*a, **kw)

    monkeypatch.setattr(on_cpu, "BeamSession", Eager)
    monkeypatch.setattr(load_pkg("ops"), "argmax", lambda z: z.argmax(-1).int())


def test_a_front_end_search_that_fails_leaves_its_requests_alone(served):
    """Out of pages in the middle: the searches' rows and pages go back."""
    kv = cache(pages=12, seqs=8)
    b, _ = front_end(kv, (32, 48), beams=3)
    with pytest.raises(RuntimeError, match="out of pages"):
        b.execute()
    assert sorted(kv.slot) == [0, 1]
    sound(kv)


@pytest.mark.parametrize("eos", [None, 7])
def test_a_request_without_beams_has_no_answer(served, eos):
    """Logits that are NaN leave a request no beam: its answer is empty, and the others' are what they are without it."""
    answers = []
    for lens, bad in (((32, 48, 16), (1,)), ((32, 16), ())):
        kv = cache(pages=90, seqs=12)
        b, out = front_end(kv, lens, bad, beams=3)
        b.graph.eos_token_id = eos
        b.execute()
        assert sorted(kv.slot) == list(range(len(lens)))
        sound(kv)
        answers.append([o.var.tolist() for o in out])
        assert all(o.var.dtype == np.int64 for o in out)
    assert answers[0] == [answers[1][0], [], answers[1][1]]
    assert all(len(a) == 20 or a[-1] == eos for a in answers[1])


def test_a_search_is_done_where_no_beam_is_left(on_cpu):
    """A request without beams has none that could go on, whether or not there is an end token."""
    model, eos = Model(), 5
    model.table[:, eos] = 30.0                        # every beam ends soon
    logits = model.table[:2].clone()
    logits[1] = torch.nan
    kv = cache(pages=60, seqs=12)
    prompts(kv, {0: 32, 1: 48})
    s = on_cpu.BeamSession(model, kv, [0, 1], {}, logits, 3, eos=eos)
    for _ in range(3):
        s.step()
    assert s.done() and [len(b) for b in s.answers()] == [3, 0]
    s.close()
    for z, want in ((logits, False), (logits[1:].repeat(2, 1), True)):
        s = on_cpu.BeamSession(model, kv, [0, 1], {}, z, 3)
        s.step()
        assert s.done() is want
        s.close()


class Ruled:
    """Rules of which the batch below leaves nothing."""


@pytest.mark.parametrize("batch_prefill", [False, True])
@pytest.mark.parametrize("ruled", [0, 1])
def test_a_search_under_rules_is_refused_ahead_of_its_prompts(served, monkeypatch, ruled, batch_prefill):
    """Also where the rules leave a request no token at all."""
    xg = load_pkg("llama_exec_graph")

    class Nothing:
        def __init__(self, rules, *a):
            self.n = len(rules)

        def choose(self, logits):
            return torch.full((self.n,), -1, dtype=torch.int32)

    monkeypatch.setattr(xg, "BatchRules", Nothing)
    kv = cache(pages=90, seqs=12)
    rules = [None, None]
    rules[ruled] = Ruled()
    b, _ = front_end(kv, (32, 48), rules=rules, beams=3, batch_prefill=batch_prefill)
    with pytest.raises(ValueError, match="rules"):
        b.execute()
    assert not kv.slot
    graph = b.graph
    graph.kv_cache.add_sequence(0), graph.kv_cache.add_sequence(1)
    decode = graph.op_nodes[[op.op_type for op in graph.op_nodes].index("decode")]
    for var, first in zip(decode.input_vars, (5, 5)):
        var.var = -1 if decode.seqids[decode.input_vars.index(var)] == ruled else first
    with pytest.raises(ValueError, match="rules"):                  # the decode alone
        graph.execute_decode(decode)


@pytest.mark.parametrize("bits", [16, 8])
def test_sinks_without_a_window_are_refused(bits):
    """As PagedKVCache refuses them, on caches of 16 bits too."""
    with pytest.raises(ValueError, match="sinks"):
        front_end_cache(cache_bits=bits, sinks=4)
    assert front_end_cache(cache_bits=bits).sinks == 0
    assert front_end_cache(cache_bits=bits, window=32, sinks=4).sinks == 4


def front_end_cache(**config):
    xg, si = load_pkg("llama_exec_graph"), load_pkg("seq_info")
    vm = Served(None)
    vm["create_paged_kv_cache"] = lambda n, total, chunk, page, free_pages, max_seq_len, **form: cache(**form)
    g = xg.LlamaExecGraph()
    g.set_exec_vars(vm, "cpu", None, None, si.LlamaSeqInfo(8), xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=24, page_size=16, **config))
    return g.kv_cache


def test_sessions_take_the_rows_that_beams_have_now(on_cpu):
    """A sequence of a search that is still open lies in whatever row its beam has come to."""
    model, moved = Model(seed=3), 0
    for seed in range(6):
        kv = cache(pages=60, seqs=12)
        prompts(kv, {0: 32, 1: 48})
        s = on_cpu.BeamSession(model, kv, [0, 1], {}, model.table[seed:seed + 2], 4)
        for _ in range(7):
            s.step()
        assert kv._adrift
        moved += s.slots.tolist() != [kv.slot[i] for i in s.seq_ids]
        rows = {i: n for i, n in zip(s.seq_ids, s.slots.tolist())}
        if seed % 2:
            assert on_cpu.DecodeSession(model, kv, [1, 0], {}, [3, 4]).rows.tolist() == [rows[1], rows[0]]
        else:
            assert on_cpu.BeamSession(model, kv, [1, 0], {}, model.table[:2], 1).slots.tolist() == [rows[1], rows[0]]
        assert kv.rows_of(s.seq_ids) == s.slots.tolist() and not kv._adrift
    assert moved > 2


def test_groups_of_shared_pages_are_of_the_rows_that_beams_have_now(on_cpu):
    model = Model(seed=3)
    kv = cache(pages=90, seqs=12)
    prompts(kv, {0: 32})
    s = on_cpu.BeamSession(model, kv, [0], {}, model.table[:1], 4, steps=60)
    for _ in range(14):
        s.step()
    kv.settle()
    kv.reserve(s.seq_ids, 48)                         # (so that no step reads the rows back)
    for _ in range(40):
        s.step()
    assert kv._adrift
    groups = kv.prefix_groups(s.seq_ids)
    table = kv.block_table[s.slots.long(), :kv.lens[0] // PAGE]
    for members, pages in groups:
        assert pages == 0 or (table[members, :pages] == table[members[0], :pages]).all()
    kv.settle()
    assert groups == kv.prefix_groups(s.seq_ids) and max(p for _, p in groups) > 2


@pytest.mark.parametrize("W", [1, 3])
def test_a_sequence_is_searched_once(on_cpu, W):
    """The same sequence twice would be two rows that store into one page."""
    model = Model()
    kv = cache(pages=60, seqs=12)
    prompts(kv, {0: 32, 1: 48})
    for ids in ([0, 0], [1, 0, 1]):
        with pytest.raises(ValueError, match="twice"):
            on_cpu.BeamSession(model, kv, ids, {}, model.table[:len(ids)], W)
        assert list(kv.slot) == [0, 1]
    sound(kv)


@pytest.mark.parametrize("sinks", [0, 1, 16, 33])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 30, 33, 48])
def test_the_front_end_s_cache_has_room_for_its_searches(served, window, sinks):
    """The pool is sized for what is seen, not for what is written: no search runs out of it, whatever its prompts' lengths."""
    for lens, limit, beams in (((64, 63, 1), 200, 4), ((33, 48), 90, 3), ((17,), 150, 16)):
        ab, xg, made = load_pkg("auto_batcher"), load_pkg("llama_exec_graph"), []
        b = ab.LlamaAutoBatcherClass()
        vm = Served(None)

        def create(n, total, chunk, page, free_pages, max_seq_len, **form):
            made.append(cache(-(-total // page) + n, n, -(-max_seq_len // page), **form))
            return made[-1]

        vm["create_paged_kv_cache"] = create
        b.set_model(vm)
        b.set_exec_config(xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=limit, page_size=16, native_decode=False, window=window, sinks=sinks, beams=beams))
        out = [b.generate(b.create_var(np.arange(n, dtype=np.int32) % 50)) for n in lens]
        b.compile()
        b.execute()
        assert [len(o.var) for o in out] == [limit] * len(lens)
        sound(made[-1])
