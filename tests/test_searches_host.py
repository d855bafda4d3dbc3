"""Searches beside other work on one cache, and searches that fail: the host's side of them, on the CPU."""
import numpy as np
import pytest
import torch

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
