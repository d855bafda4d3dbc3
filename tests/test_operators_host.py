"""Argument checks of the operators of a wide decode step that need no GPU: every call below is refused ahead of a launch."""
import ctypes as C

from conftest import load_pkg


def test_constrained_argmax_refusals():
    lm = load_pkg("_lib")
    lib = lm.lib()
    def call(B=2, V=50000, ld=50000, out=None, ld_out=0, ws=16, nb=1 << 20, **kw):
        r = lm.LogitRulesArgs(**kw)
        return lib.mlora_constrained_argmax(16, out, ld_out, 16, ld, C.byref(r), B, V, ws, nb, None)
    assert lib.mlora_constrained_argmax_workspace_bytes(2, 50000) == 2 * 25 * 8 and lib.mlora_constrained_argmax_workspace_bytes(2, 2000) == 0
    assert lib.mlora_constrained_argmax(16, None, 0, None, 10, C.byref(lm.LogitRulesArgs()), 1, 10, None, 0, None) == -1
    assert call(B=-1) == -1 and call(B=65536) == -1 and call(V=0) == -1 and call(ld=49999) == -1
    assert call(out=16, ld_out=100) == -1
    assert call(history=16) == -1 and call(history=16, lengths=16, cap=0) == -1
    assert call(repetition=16) == -1 and call(append=1) == -1
    assert call(n_bias=1025, bias_ids=16, bias=16) == -2 and call(n_bias=3, bias_ids=16) == -1
    assert call(masks=16, n_masks=1) == -1 and call(masks=16, mask_row=16) == -1
    assert call(ws=None) == -3 and call(nb=2 * 25 * 8 - 1) == -3 and call(ws=20) == -3
    assert call(B=0) == 0


def test_linear4_refusals():
    lib = load_pkg("_lib").lib()
    sizes = [C.c_size_t() for _ in range(2)]
    assert lib.mlora_linear4_sizes(40, 352, 32, *(C.byref(s) for s in sizes)) == 0
    assert [s.value for s in sizes] == [9 * 1024, 9 * 16 * 4 * 3]
    assert lib.mlora_linear4_sizes(40, 352, 32, None, None) == 0
    assert lib.mlora_linear4_sizes(40, 352, 64, None, None) == -2 and lib.mlora_linear4_sizes(40, 96, 96, None, None) == -2
    assert lib.mlora_linear4_sizes(0, 32, 32, None, None) == -2 and lib.mlora_linear4_sizes(1, 0, 32, None, None) == -2
    def call(y=16, dt=0, mode=0, x=16, lay=0, ldx=128, q=16, m=16, group=128, T=4, K=128, N=32, ws=None, nb=0):
        return lib.mlora_linear4(y, dt, mode, x, lay, ldx, q, m, group, T, K, N, ws, nb, None)
    assert call(y=None) == -1 and call(m=None) == -1 and call(group=16) == -2 and call(T=-1) == -1 and call(dt=3) == -1
    assert call(mode=1) == -2 and call(mode=2) == -2 and call(ldx=120) == -1 and call(ldx=132) == -1 and call(lay=2) == -1
    assert call(x=24) == -1 and call(y=17) == -1 and call(dt=1, y=18) == -1
    need = lib.mlora_linear4_workspace_bytes(64, 4096, 4096)
    assert need % (64 * 4096 * 4) == 0 and need > 0 and lib.mlora_linear4_workspace_bytes(1, 4096, 4096) == 0
    big = dict(T=64, K=4096, N=4096, ldx=4096)
    assert call(**big) == -3 and call(ws=16, nb=need - 1, **big) == -3 and call(ws=24, nb=need, **big) == -3
    assert call(T=0) == 0


def test_shared_attention_refusals():
    lib = load_pkg("_lib").lib()
    assert lib.mlora_shared_attn_unit_rows() == 64 and lib.mlora_shared_attn_record_ints() == 72
    need = lib.mlora_shared_attn_workspace_bytes(4, 8, 128, 3)
    assert need == 4 * 8 * 3 * 130 * 4 and lib.mlora_shared_attn_workspace_bytes(0, 8, 128, 3) == 0
    def call(out=16, lay=0, units=16, n_block=1, n_units=1, row_pages=16, own=2, slots=3, B=4, Hq=8, Hkv=8, D=128, ws=16, nb=need):
        return lib.mlora_paged_attn_decode_shared(out, lay, 16, 16, 16, 16, 4, 16, 16, units, n_block, n_units, row_pages, 16, own, slots, B, Hq, Hkv, D,
                                                  5, 4, ws, nb, None)
    assert call(out=None) == -1 and call(row_pages=None) == -1 and call(units=None) == -1 and call(n_units=-1) == -1 and call(n_block=2) == -1 and call(n_block=-1) == -1
    assert call(D=96) == -2 and call(Hkv=3) == -1 and call(Hq=34, Hkv=2) == -2 and call(lay=5) == -1
    assert call(own=0) == -1 and call(slots=1) == -1 and call(B=-1) == -1 and call(B=70000) == -1
    assert call(ws=None) == -3 and call(nb=need - 1) == -3 and call(ws=24) == -3
    assert call(B=0) == 0


def _cache(**kw):
    kvc = load_pkg("kv_cache")
    return kvc.PagedKVCache(1, 40, 2, 64, max_seqs=8, max_blocks=12, rope_theta=1e4, max_pos=192, device="cpu", **kw)


def _fill(kv, sid, n):
    kv.add_sequence(sid)
    kv.begin_forward([sid], [n])
    kv.end_forward()


def test_shared_pages_have_owners_and_go_back_with_the_last():
    kv = _cache()
    free = set(kv.free)
    _fill(kv, "a", 70)
    kv.add_sequence("b")
    assert kv.share_prefix("b", "a", 69) == 64 and kv.lens["b"] == 64 and kv.pages_of("b") == kv.pages_of("a")[:4]
    kv.add_sequence("c")
    assert kv.share_prefix("c", "b") == 64
    kv.add_sequence("d")
    assert kv.share_prefix("d", "a", 15) == 0 and kv.lens["d"] == 0 and kv.pages_of("d") == []
    kv.begin_forward(["b", "c", "a"], [3, 20, 1])
    kv.end_forward()
    shared, own_a = kv.pages_of("a")[:4], kv.pages_of("a")[4:]
    assert kv.pages_of("b")[:4] == shared and kv.pages_of("c")[:4] == shared and kv.lens["c"] == 84
    assert len({*kv.pages_of("a"), *kv.pages_of("b"), *kv.pages_of("c")}) == 4 + 1 + 1 + 2
    assert (kv.block_table[kv.slot["c"], :4] == kv.block_table[kv.slot["a"], :4]).all()
    kv.free_sequence("a")
    assert set(own_a) <= set(kv.free) and not set(shared) & set(kv.free)
    kv.free_sequence("c")
    assert not set(shared) & set(kv.free)
    kv.free_sequence("b")
    kv.free_sequence("d")
    assert set(kv.free) == free and len(kv.free) == len(free) and not kv._owners


def test_share_prefix_refusals():
    import pytest
    kv = _cache()
    _fill(kv, 0, 40)
    _fill(kv, 1, 5)
    kv.add_sequence(2)
    for sid, of in ((1, 0), (0, 0), (2, 2)):
        with pytest.raises(ValueError):
            kv.share_prefix(sid, of)
    with pytest.raises(KeyError):
        kv.share_prefix(2, 7)
    kv.begin_forward([1], [1])
    with pytest.raises(RuntimeError):
        kv.share_prefix(2, 0)
    kv.end_forward()
    assert kv.share_prefix(2, 0, -3) == 0 and kv.share_prefix(2, 0, 1000) == 32
    time_mix = load_pkg("time_mix")
    state = load_pkg("kv_cache").PagedStateCache([time_mix.TimeMixSpec(2, 8)], 64, 4, 2, 4, 64, dtype=__import__("torch").float32, device="cpu")
    state.add_sequence(0)
    state.add_sequence(1)
    with pytest.raises(ValueError):
        state.share_prefix(1, 0)


def test_prefix_groups_save_most():
    kv = _cache()
    _fill(kv, 0, 16 * 6)
    for sid, of, n in ((1, 0, 16 * 6), (2, 0, 16 * 2), (3, 0, 16 * 5)):
        kv.add_sequence(sid)
        kv.share_prefix(sid, of, n)
    _fill(kv, 4, 20)
    kv.begin_forward([0, 1, 2, 3], [1, 1, 40, 1])
    kv.end_forward()
    # all four share two pages (saves 6); 0, 1 and 3 share five (saves 10)
    assert kv.prefix_groups([0, 1, 2, 3, 4]) == [([0, 1, 3], 5)]
    assert kv.prefix_groups([4, 2, 0]) == [([1, 2], 2)]
    assert kv.prefix_groups([4]) == [] and kv.prefix_groups([0]) == [] and kv.prefix_groups([]) == []
    for sid in (5, 6):
        kv.add_sequence(sid)
        kv.share_prefix(sid, 4)
    assert sorted(kv.prefix_groups([5, 0, 6, 3, 1])) == [([0, 2], 1), ([1, 3, 4], 5)]


def test_plans_of_a_cache_live_with_their_sequences():
    kv = _cache(n_q_heads=2)
    _fill(kv, 0, 33)
    kv.add_sequence(1)
    kv.share_prefix(1, 0)
    assert kv.shared_plan([0, 1]) is None and (0, 1) in kv._plans          # two pages do not pay
    kv.free_sequence(1)
    assert not kv._plans and kv.shared_plan([0]) is None
    kv.add_sequence(2)
    kv._plans[(0, 2)] = None                                             # asked before there was anything to share
    kv.share_prefix(2, 0)
    assert not kv._plans


def test_grammar_masks_and_rules_on_the_host():
    import pytest
    tr = load_pkg("token_rules")
    with pytest.raises(ValueError):
        tr.TokenRules(repetition=0.0)
    si = load_pkg("seq_info").LlamaSeqInfo(4)
    si.add_sequence(0)
    assert si.get_rules(0) is None
    r = tr.TokenRules(bias={3: 1.0})
    si.set_rules(0, r)
    assert si.get_rules(0) is r


def _on_shared_pages(rows=3, pages=130, own=5):
    """A cache on the CPU whose sequences share enough pages for a plan, and its batch."""
    kvc = load_pkg("kv_cache")
    kv = kvc.PagedKVCache(1, pages + 2 * rows, 2, 64, max_seqs=rows, max_blocks=pages + 4, rope_theta=1e4, max_pos=16 * (pages + 4), device="cpu", n_q_heads=4)
    for sid in range(rows):
        kv.add_sequence(sid)
        skip = kv.share_prefix(sid, 0) if sid else 0
        kv.begin_forward([sid], [16 * pages + (own if sid else 0) - skip])
        kv.end_forward()
    return kv, tuple(range(rows))


def test_copies_of_a_cache_with_a_plan_have_its_arrays_for_themselves():
    """What a copied or unpickled cache hands to the kernels lies in its own arrays and holds the same plan."""
    import copy
    import pickle
    import torch
    kv, batch = _on_shared_pages()
    kv.begin_forward(batch, [1] * len(batch))
    kv.end_forward()
    plan = kv.shared_plan(batch)
    assert plan is not None and kv.plan is plan
    for make in (copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))):
        other = make(kv)
        mine = other.shared_plan(batch)
        assert mine is not plan and other.plan is mine and torch.equal(mine.data, plan.data) and mine.data.data_ptr() != plan.data.data_ptr()
        for name in ("units", "row_pages", "row_slots"):
            a, b = getattr(mine, name), getattr(plan, name)
            assert torch.equal(a, b) and a.untyped_storage().data_ptr() == mine.data.untyped_storage().data_ptr()
        assert mine._args == (mine.units.data_ptr(), plan.n_block, plan.n_units, mine.row_pages.data_ptr(), mine.row_slots.data_ptr(), plan.own_splits, plan.slots)
        assert not {mine._args[i] for i in (0, 3, 4)} & {plan._args[i] for i in (0, 3, 4)}


def _tree_of_prefixes(seqs):
    """A cache whose sequences begin like one another: seqs are (of, pages taken over, own pages) in order."""
    kvc = load_pkg("kv_cache")
    most = 1 + max(taken + own for _, taken, own in seqs)
    kv = kvc.PagedKVCache(1, 1 + sum(own + 1 for _, _, own in seqs), 1, 32, max_seqs=len(seqs), max_blocks=most, rope_theta=1e4, max_pos=16 * most, device="cpu")
    for sid, (of, taken, own) in enumerate(seqs):
        kv.add_sequence(sid)
        if of is not None and taken:
            kv.share_prefix(sid, of, 16 * taken)
        kv.begin_forward([sid], [16 * own])
        kv.end_forward()
    return kv


def _pages_saved(kv, seq_ids, groups):
    """Of groups that are sound: a sequence in one at most, each of several with the same pages."""
    rows = [r for members, _ in groups for r in members]
    assert len(rows) == len(set(rows))
    for members, pages in groups:
        heads = {tuple(kv.pages_of(seq_ids[r])[:pages]) for r in members}
        assert len(members) > 1 and pages > 0 and len(heads) == 1 and all(kv.lens[seq_ids[r]] >= 16 * pages for r in members)
    return sum((len(members) - 1) * pages for members, pages in groups)


def test_prefix_groups_keep_those_outside_a_deeper_group():
    """Eleven sequences share ten pages, two of them 160: the two are one group, the nine others another."""
    kv = _tree_of_prefixes([(None, 0, 10), (0, 10, 150), (1, 160, 1)] + [(0, 10, 1)] * 8)
    ids = [0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 1]
    assert sorted(kv.prefix_groups(ids)) == [([0, 2, 3, 4, 5, 6, 7, 8, 9], 10), ([1, 10], 160)]


def test_prefix_groups_against_every_choice():
    """Small trees of prefixes: the most that any choice of a depth for every sequence saves."""
    import itertools
    import random
    for seed in range(60):
        rng = random.Random(seed)
        seqs = [(None, 0, rng.randint(1, 4))]
        for sid in range(1, rng.randint(2, 6)):
            of = rng.randrange(sid)
            has = seqs[of][1] + seqs[of][2]
            seqs.append((of, rng.randint(0, has), rng.randint(0, max(0, 4 - has) + 1)))
        seqs = [(of, taken, own if taken + own else 1) for of, taken, own in seqs]
        kv = _tree_of_prefixes(seqs)
        ids = list(range(len(seqs)))
        rng.shuffle(ids)
        pages = [kv.pages_of(s) for s in ids]
        most = 0
        for depths in itertools.product(*(range(min(len(p), 5) + 1) for p in pages)):
            groups = {}
            for r, d in enumerate(depths):
                groups.setdefault(tuple(pages[r][:d]), []).append(r)
            most = max(most, sum((len(m) - 1) * len(head) for head, m in groups.items()))
        assert max(map(len, pages)) <= 9 and _pages_saved(kv, ids, kv.prefix_groups(ids)) == max(most, 0)


def test_prefix_groups_of_a_long_chain():
    """Every sequence begins with all of the one before."""
    kv = _tree_of_prefixes([(None, 0, 1)] + [(i, i + 1, 1) for i in range(1299)])
    ids = list(range(1300))
    saved = _pages_saved(kv, ids, kv.prefix_groups(ids))
    # groups at depths d1 < d2 < .. of a chain: sum over them of d (number of sequences up to the next - 1); one at half the chain saves 650 x 650
    assert saved >= 650 * 650
    assert saved == _chain_most(1300)


def _chain_most(n):
    """The most that a chain saves: by a recursion over the deepest group, of sequences d - 1 .. e - 1 at depth d."""
    import numpy as np
    most = np.zeros(n + 1, np.int64)                          # of the sequences 0 .. e - 1
    for e in range(1, n + 1):
        d = np.arange(1, e + 1)
        most[e] = max(most[e - 1], int((most[d - 1] + (e - d) * d).max()))
    return int(most[n])


def test_linear4_cuts_by_the_order_of_x():
    """17 to 32 tokens in rows: which kernel takes a product, told by its partial sums; either order finds room in the general size."""
    lib = load_pkg("_lib").lib()
    of, either = lib.mlora_linear4_workspace_bytes_of, lib.mlora_linear4_workspace_bytes
    for T, K, N, slices in ((32, 4096, 4096, True), (24, 4096, 1024, True), (20, 6144, 3000, True), (17, 6144, 1024, True),       # two groups of waves, in slices
                            (28, 4096, 4096, False), (17, 4096, 1024, False), (32, 4096, 8192, False), (32, 2048, 1024, False), (24, 6144, 8192, False)):
        rows, frag = of(T, K, N, 0), of(T, K, N, 1)
        assert (rows > 0) == slices and frag == 0 and either(T, K, N) == rows, (T, K, N)
    for T, K, N in ((64, 4096, 4096), (33, 11008, 4096), (16, 4096, 4096), (30, 11008, 4096)):
        assert of(T, K, N, 0) == of(T, K, N, 1) == either(T, K, N)
    need = of(32, 4096, 4096, 0)
    def call(lay, ws, nb, T=32, K=4096, N=4096):
        return lib.mlora_linear4(16, 0, 0, 16, lay, K, 16, 16, 128, T, K, N, ws, nb, None)
    assert call(0, None, 0) == -3 and call(0, 16, need - 1) == -3


def test_plans_are_cut_anew_when_their_rows_outgrow_them():
    """As the rows' own pages grow the cache's plan is that of a new batch of these lengths (up to a factor of two in its shares); those before it stay as
    they are for the steps that were recorded with them, and go with the batch."""
    kvc, ops = load_pkg("kv_cache"), load_pkg("ops")
    kv = kvc.PagedKVCache(1, 1000, 8, 64, max_seqs=8, max_blocks=300, rope_theta=1e4, max_pos=4800, device="cpu", n_q_heads=32)
    batch = tuple(range(8))
    for sid in batch:
        kv.add_sequence(sid)
        skip = kv.share_prefix(sid, 0, 2048) if sid else 0
        kv.begin_forward([sid], [2048 + 5 + sid - skip])
        kv.end_forward()
    seen, before = [], []
    for step in range(1400):
        kv.begin_forward(batch, [1] * 8)
        assert kv.plan is kv.shared_plan(batch)
        if not seen or kv.plan is not seen[-1]:
            seen.append(kv.plan)
            before.append((kv.plan._args, kv.plan.data.clone()))
        kv.end_forward()
        new = ops.SharedPrefixPlan([(list(batch), 128)], [kv.lens[s] for s in batch], 32, 8, 64, "cpu")
        assert kv.plan.own_splits <= new.own_splits and (kv.plan.own_splits * 2 > new.own_splits or (kv.lens[0] - 1) % 16)
        assert kv.plan.groups == [(list(batch), 128)] and kv.plan.saved_bytes == seen[0].saved_bytes
    assert [p.own_splits for p in seen] == [1, 2, 4, 8]
    assert all(b.earlier is a for a, b in zip(seen, seen[1:])) and seen[0].earlier is None
    for p, (args, data) in zip(seen, before):
        assert p._args == args and (p.data == data).all() and p.units.data_ptr() == args[0]
    kv.free_sequence(3)
    assert not kv._plans


def test_when_a_batch_gives_up_the_native_step_for_shared_pages():
    """The choice on measured batches of both sides: rows, longest shared prefix, saved MB a layer, heads, dense adapters."""
    import types
    xg = load_pkg("llama_exec_graph").LlamaExecGraph
    graph = xg.__new__(xg)
    for rows, pages, mb, heads, dense, pays in ((4, 512, 101, (16, 16), True, True), (2, 1024, 67, (16, 16), True, True), (32, 256, 520, (16, 16), True, False),
                                                (16, 256, 252, (16, 16), True, False), (64, 128, 528, (16, 16), True, True), (64, 128, 528, (16, 16), False, True),
                                                (32, 64, 520, (32, 32), True, False), (32, 64, 520, (32, 32), False, True), (16, 256, 1007, (32, 32), True, True),
                                                (32, 256, 520, (32, 8), True, False), (32, 256, 520, (32, 8), False, True), (8, 128, 59, (32, 8), True, False),
                                                (8, 512, 235, (32, 8), True, True), (128, 64, 533, (32, 8), False, True)):
        plan = types.SimpleNamespace(groups=[([0, 1], 3), (list(range(rows)), pages)], saved_bytes=mb * 1e6, Hq=heads[0], Hkv=heads[1])
        graph.kv_cache = types.SimpleNamespace(shared_plan=lambda seqs: plan)
        assert graph._shared_pays(list(range(rows)), dense) == pays, (rows, pages, mb, heads, dense)
    graph.kv_cache = types.SimpleNamespace(shared_plan=lambda seqs: None)
    assert not graph._shared_pays([0, 1], False)
    graph.kv_cache = types.SimpleNamespace()
    assert not graph._shared_pays([0, 1], False)


def test_finished_sequences_are_told_by_their_new_tokens():
    """-1 (no token left) ends an answer wherever it stands among the new tokens; the rest of an answer is not looked at again."""
    import types

    class Answer(list):
        def __contains__(self, x):
            raise AssertionError("an answer is searched")

        def index(self, *a):
            raise AssertionError("an answer is searched")

    xg = load_pkg("llama_exec_graph").LlamaExecGraph
    graph = xg.__new__(xg)
    graph.eos_token_id, graph._ended, graph.seq_info = 2, set(), types.SimpleNamespace(get_max_gen_len=lambda sid: 6)
    out = {0: Answer([5, 6, 7]), 1: Answer([5, 6, -1]), 2: Answer([5, 6, 2]), 3: Answer([-1])}
    assert graph.check_seqs_finished([0, 1, 2, 3], out) == [0] and out[1] == [5, 6] and out[3] == [] and graph._ended == {1, 3}
    out = {0: Answer([5, 6, 7, 8]), 4: Answer([5, -1, 9, -1]), 5: Answer([1, 2, 3, 4, 5, 6]), 6: Answer([5, 6, 7, -1])}
    assert graph.check_seqs_finished([0, 4, 5, 6], out, 3) == [0] and out[4] == [5] and out[6] == [5, 6, 7] and graph._ended == {1, 3, 4, 6}


def test_short_allocation_only_where_it_means_what_it_did():
    import torch
    ops = load_pkg("ops")
    right = lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype)
    cpu = torch.device("cpu")
    assert ops._short_or_plain(right, cpu) is right
    for wrong in (None, lambda size, stride: right(size, stride, torch.float16), lambda size, stride, dtype: right(size, stride, torch.float32),
                  lambda size, stride, dtype: right(size, (1, 2), dtype), lambda size, stride, dtype: right((3, 2), (2, 1), dtype),
                  lambda size, stride, dtype: right(size, stride, dtype).requires_grad_()):
        assert ops._short_or_plain(wrong, cpu) is ops._plain_empty
    assert ops._short_or_plain(right, torch.device("cuda", 0)) is ops._plain_empty


def test_a_recorded_pass_makes_no_plan(monkeypatch):
    """A pass begun inside a capture, with arrays on the device, reads shared pages for every row where no plan is there yet, and takes the one that is."""
    import torch
    kv, batch = _on_shared_pages()
    kv.begin_forward(batch, [1] * len(batch))
    kv.end_forward()
    plan, kv._plans = kv.shared_plan(batch), {}
    assert plan is not None
    kv.device = torch.device("cuda")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    kv.begin_forward(batch, [1] * len(batch), device_meta=(None, None, None))
    kv.end_forward()
    assert kv.plan is None and not kv._plans
    kv._plans[batch] = plan
    kv.begin_forward(batch, [1] * len(batch), device_meta=(None, None, None))
    kv.end_forward()
    assert kv.plan is plan
