"""Caches in 8 bits, under windows and of beams: the host's side of them, on the CPU."""
import copy
import pickle

import numpy as np
import pytest
import torch

from conftest import load_pkg

PAGE = 16


def cache(pages=40, seqs=4, blocks=20, **kw):
    return load_pkg("kv_cache").PagedKVCache(1, pages, 2, 64, seqs, blocks, 1e4, blocks * PAGE, device="cpu", **kw)


def grow(kv, sid, n, at_once=None):
    while n:
        m = min(n, at_once or n)
        kv.begin_forward([sid], [m])
        kv.end_forward()
        n -= m


def sound(kv):
    """Every page is in the pool, or has as many owners as rows hold it."""
    held = {}
    for row in kv.slot.values():
        for p in kv.table_h[row][kv.table_h[row] >= 0].tolist():
            held[p] = held.get(p, 0) + 1
    assert sorted(kv.free + list(held)) == list(range(kv.n_pages))
    assert kv._owners == {p: n for p, n in held.items() if n > 1}


@pytest.mark.parametrize("kw", [{"bits": 4}, {"window": 0}, {"sinks": 3}, {"window": 5, "sinks": -1}, {"window": 1 << 31}])
def test_forms_that_are_none(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_heads_of_other_sizes():
    kc = load_pkg("kv_cache")
    for kw in ({"bits": 8}, {"window": 8}):
        with pytest.raises(ValueError):
            kc.PagedKVCache(1, 4, 2, 32, 1, 4, 1e4, 64, device="cpu", **kw)
    assert kc.PagedKVCache(1, 4, 2, 32, 1, 4, 1e4, 64, device="cpu").plain


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 1), (40, 16), (33, 17), (1000, 4)])
@pytest.mark.parametrize("at_once", [1, 7, 64])
def test_pages_behind_the_window_go_back(window, sinks, at_once):
    kv = cache(window=window, sinks=sinks)
    kv.add_sequence("a")
    for _ in range(300 // at_once):
        first = kv.lens["a"]                        # of the pass that comes
        grow(kv, "a", at_once)
        blocks = np.flatnonzero(kv.table_h[kv.slot["a"]] >= 0)
        seen = [j for j in range(-(-kv.lens["a"] // PAGE)) if j * PAGE < sinks or (j + 1) * PAGE > first - window + 1]
        assert blocks.tolist() == seen, (first, window, sinks)
        sound(kv)
        assert (kv.block_table.numpy() == kv.table_h).all()
    kv.free_sequence("a")
    sound(kv)


def test_prefix_of_a_row_that_has_gone_on():
    """What the next token of the new sequence sees has to be there still."""
    kv = cache(window=40, sinks=4)
    for s in "abcd":
        kv.add_sequence(s)
    grow(kv, "a", 100)
    assert kv.share_prefix("b", "a", 90) == 80
    sound(kv)
    grow(kv, "b", 1)
    assert np.flatnonzero(kv.table_h[kv.slot["b"]] >= 0).tolist() == [0, 2, 3, 4, 5]       # token 80 sees 41 .. and the first page
    sound(kv)
    grow(kv, "a", 100, 1)                                                                  # token 199 saw 160 .. and the first page
    assert kv.share_prefix("c", "a", 90) == 0 and kv.share_prefix("c", "a") == 0           # (token 192 would see 153 ..)
    grow(kv, "a", 8, 1)
    assert kv.share_prefix("c", "a") == 208                                                # (token 208 sees 169 .., as 207 saw 168 ..)
    sound(kv)
    grow(kv, "c", 3)
    for s in "abcd":
        kv.free_sequence(s)
    sound(kv)


def test_refusals():
    kv = cache(pages=6, seqs=3, bits=8)
    kv.add_sequence("a")
    grow(kv, "a", 32)
    with pytest.raises(ValueError):
        kv.fork(["b", "b"], "a")
    with pytest.raises(ValueError):
        kv.fork(["a"], "a")
    with pytest.raises(RuntimeError):
        kv.fork(["b", "c", "d"], "a")
    kv.begin_forward(["a"], [1])
    with pytest.raises(RuntimeError):
        kv.fork(["b"], "a")
    with pytest.raises(ValueError):
        kv.attention_with_fused_qkv(0, torch.zeros(1, 6, 64, dtype=torch.float16), 2, o_shrink=(None, None))
    kv.end_forward()
    grow(kv, "a", 30)
    assert len(kv.free) == 2 and list(kv.slot) == ["a"]
    with pytest.raises(RuntimeError):                # two slots, but the third page that would be needed is not there
        kv.free.pop() and kv.fork(["b", "c"], "a")
    assert list(kv.slot) == ["a"]


def test_forks_of_whole_pages_and_reserved_ones():
    kv = cache(pages=12, seqs=4)
    kv.add_sequence("a")
    grow(kv, "a", 48)
    kv.fork(["b", "c"], "a")
    sound(kv)
    assert kv.lens["c"] == 48 and kv.lacks_page("b") and len(kv.free) == 9
    kv.reserve(["a", "b", "c"], 40)
    assert len(kv.free) == 0 and not kv.lacks_page("b")
    sound(kv)
    kv.reserve(["a"], 49)                            # more than there is: nothing
    kv.reserve(["a"], 48)
    assert not kv.free and kv.pages_of("a")[:3] == kv.pages_of("b")[:3]
    grow(kv, "c", 5)
    kv.free_sequence("b")
    sound(kv)


class Device:
    """`reorder` on the CPU's block table: a parent's first child stays, others take rows of beams without any."""

    def __init__(self, kv, sids, W):
        self.kv, self.sids, self.W = kv, list(sids), W
        self.slots = torch.tensor([kv.slot[s] for s in sids], dtype=torch.int32)
        self.paths = [[] for _ in sids]

    def step(self, rng, token):
        kv, W = self.kv, self.W
        kv.begin_forward(self.sids, [1] * len(self.sids), device_meta=(self.slots, None, None))
        kv.end_forward()
        table, new, paths = kv.block_table, self.slots.clone(), list(self.paths)
        for r in range(0, len(self.sids), W):
            parents = rng.integers(0, W, W)
            dead = [w for w in range(W) if w not in parents]
            block = kv.lens[self.sids[r]] // PAGE
            old = table.clone()
            for w, p in enumerate(parents):
                first = p not in parents[:w]
                new[r + w] = self.slots[r + (p if first else dead.pop(0))]
                if not first:
                    table[new[r + w], :block] = old[self.slots[r + p], :block]
                paths[r + w] = self.paths[r + p] + [(token, int(p))]
        self.slots.copy_(new)
        self.paths = paths
        kv.adrift(self.sids, self.slots)


@pytest.mark.parametrize("kw", [{}, {"bits": 8}, {"window": 20, "sinks": 2}, {"bits": 8, "window": 3}])
def test_rows_of_beams_are_read_back(kw):
    """Whatever the host does meanwhile: pages have as many owners as rows, those that nobody holds are in the pool, and a row's pages stay its own."""
    rng = np.random.default_rng(len(kw))
    kv = cache(pages=90, seqs=9, blocks=10, **kw)
    kv.add_sequence("x")
    for sid, n in (("p", 21), ("q", 32)):
        kv.add_sequence(sid)
        grow(kv, sid, n - n % PAGE)
        kv.fork([(sid, w) for w in range(1, 4)], sid)
    sids = [s if w == 0 else (s, w) for s in "pq" for w in range(4)]
    grow_all = lambda: [grow(kv, s, 5) for s in sids[:4]]                                  # noqa: E731
    grow_all()
    beams = Device(kv, sids, 4)
    for i in range(70):
        if i % 16 == 3 and i < 60:
            kv.reserve(sids, PAGE)
        beams.step(rng, i)
        if i % 5 == 4:
            kv.settle()
            sound(kv)
            assert [kv.slot[s] for s in sids] == beams.slots.tolist()
            own = [kv.table_h[kv.slot[s], kv.lens[s] // PAGE] for s in sids]
            assert all(n == 1 for p, n in zip(*np.unique([p for p in own if p >= 0], return_counts=True)))
        if i % 11 == 7:                              # another sequence's pass uploads the table
            grow(kv, "x", 3)
            assert not kv._adrift
    assert kv.pages_of("q")
    copied = copy.deepcopy(kv)
    again = pickle.loads(pickle.dumps(kv))
    for s in sids:
        kv.free_sequence(s)
    sound(kv)
    sound(copied)
    sound(again)
    assert copied.slot != kv.slot and not copied._adrift


def test_beams_take_no_plan_from_rows_that_change():
    """Pages that beams have come to share are not theirs to share for long: no plan is made of them, whatever it would save."""
    rng = np.random.default_rng(1)
    kv = cache(pages=1200, seqs=4, blocks=300, n_q_heads=2)
    kv.add_sequence("p")
    grow(kv, "p", 3)                                 # (no whole page that the beams share)
    sids = ["p", "b", "c", "d"]
    for s in sids[1:]:                               # as forks, whose copies the CPU does not make
        kv.add_sequence(s)
        grow(kv, s, 3)
    beams = Device(kv, sids, 4)
    kv.reserve(sids, 2320)                           # (so that the host hears of the rows at the end alone)
    for i in range(2300):
        beams.step(rng, i)
    kv.settle()
    sound(kv)
    assert max(p for _, p in kv.prefix_groups(sids)) >= 128
    kv.begin_forward(sids, [1] * 4, device_meta=(beams.slots, None, None))
    assert kv.plan is None and kv.shared_plan(sids) is None


def test_a_search_that_finds_no_room_leaves_nothing():
    ds = load_pkg("decode_session")

    class Model:
        cache_forms, device = True, "cpu"

    kv = cache(pages=12, seqs=5)
    for s in "ab":
        kv.add_sequence(s)
        grow(kv, s, 32)
    with pytest.raises(RuntimeError):                # rows for one more beam of each, not for two
        ds.BeamSession(Model, kv, ["a", "b"], {}, torch.zeros(2, 50), 3)
    assert sorted(kv.slot) == ["a", "b"]
    sound(kv)


def test_pages_of_a_copied_cache_are_its_own():
    kv = cache(bits=8)
    kv.pages(0)
    for other in (copy.deepcopy(kv), pickle.loads(pickle.dumps(kv))):
        other.pages(0).k.fill_(5)
        other.pages(0).tail_v.fill_(2)
        assert (other.k == 5).all() and (other.tail_v == 2).all() and not kv.k.any() and not kv.tail_v.any()


def test_steps_are_cut_by_powers_of_two():
    kv = cache(pages=200, blocks=190, window=10)
    kv.add_sequence(0)
    cuts = []
    for n in (250, 1, 6, 1, 255, 1):
        grow(kv, 0, n)
        cuts.append(kv.cut)
    assert cuts == [250, 256, 257, 512, 513, 1024]                                         # (a pass of several tokens is cut for what it is)
    kv2 = cache(pages=200, blocks=190, bits=8)
    kv2.add_sequence(0)
    seen = set()
    for _ in range(600):
        grow(kv2, 0, 1)
        seen.add(kv2.cut)
        assert kv2.cut >= kv2.lens[0]
    assert seen == {256, 512, 1024}
    plain = cache()
    plain.add_sequence(0)
    grow(plain, 0, 20)
    assert plain.cut is None


def test_bytes_of_a_step():
    full = cache(pages=60, blocks=40)
    q8, win = cache(pages=60, blocks=40, bits=8), cache(pages=60, blocks=40, window=64, sinks=16)
    for kv in (full, q8, win):
        kv.add_sequence(0)
        grow(kv, 0, 320)
    per = 2 * 2 * 64 * 2
    assert full.kv_bytes_read_per_step([0]) == 321 * per
    assert q8.kv_bytes_read_per_step([0]) == per + 320 * (per // 2 + 1)
    assert win.kv_bytes_read_per_step([0]) == 80 * per


def test_front_end_refuses():
    xg, si = load_pkg("llama_exec_graph"), load_pkg("seq_info")

    class Model(dict):
        lora_types = ()

    def graph(forms, **kw):
        made = []
        vm = Model(create_paged_kv_cache=lambda *a, **k: made.append((a, k)) or "cache")
        vm.__dict__["cache_forms"] = forms
        info = si.LlamaSeqInfo(8)
        for s in range(3):
            info.add_sequence(s)
        g = xg.LlamaExecGraph()
        g.set_exec_vars(vm, "cpu", None, None, info, xg.LlamaExecConfig(max_prompt_len=64, max_gen_len=1000, page_size=16, **kw))
        return made[0]

    assert graph(False) == ((3, 3 * 1064, 64, 16), {"free_pages": None, "max_seq_len": 1064})
    assert graph(True, cache_bits=8)[1] == {"free_pages": None, "max_seq_len": 1064, "bits": 8, "window": None, "sinks": 0}
    a, k = graph(True, window=128, sinks=4, beams=2)
    assert a[:2] == (6, 6 * (128 + 4 + 48)) and k["max_seq_len"] == 1064 and k["bits"] == 16
    for bad in ({"cache_bits": 8}, {"window": 3}, {"beams": 2}):
        with pytest.raises(ValueError):
            graph(False, **bad)
    for bad in ({"beams": 0}, {"beams": 17}):
        with pytest.raises(ValueError):
            graph(True, **bad)
