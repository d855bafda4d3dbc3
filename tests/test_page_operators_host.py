"""Argument checks of the operators on paged caches and beams that need no GPU: every call below is refused ahead of a launch."""
import ctypes as C
import struct

from conftest import load_pkg


def _attn(lib, fn, **kw):
    a = dict(out=16, qkv=16, k=16, v=16, step=16, tail_k=16, tail_v=16, table=16, seq=16, pos=16, cos=16, sin=16, ws=0, nb=0, lay=0, max_blocks=4, max_pos=64, T=2, Hq=8, Hkv=8,
             D=128, n_pages=4, n_seq=2, window=0, sinks=0, splits=1)
    assert not set(kw) - set(a)
    a.update(kw)
    return getattr(lib, fn)(struct.pack("@13PN12i", *a.values()), None)


def test_page_attention_refusals():
    lib = load_pkg("_lib").lib()
    for fn in ("mlora_page_attn_decode", "mlora_page_attn_prefill"):
        call = lambda **kw: _attn(lib, fn, **kw)                                                                   # noqa: E731
        assert getattr(lib, fn)(None, None) == -1
        for name in ("out", "qkv", "k", "v", "table", "seq", "pos", "cos", "sin", "tail_k", "tail_v"):
            assert call(**{name: 0}) == -1, name
        for name in ("out", "qkv", "k", "v", "tail_k", "tail_v", "cos", "sin"):
            assert call(**{name: 24}) == -1, name
        assert call(step=20) == -1 and call(T=-1) == -1 and call(max_pos=0) == -1 and call(n_pages=0) == -1 and call(n_seq=0) == -1 and call(max_blocks=0) == -1
        assert call(D=96) == -2 and call(Hq=9, Hkv=2) == -1 and call(window=-1) == -1 and call(sinks=-1) == -1 and call(lay=5) == -1
        assert call(T=0) == 0
    assert _attn(lib, "mlora_page_attn_decode", Hq=34, Hkv=2) == -2 and _attn(lib, "mlora_page_attn_decode", T=70000) == -1
    need = lib.mlora_page_attn_workspace_bytes(2, 8, 128, 3)
    assert need == 2 * 8 * 3 * 130 * 4 and lib.mlora_page_attn_workspace_bytes(2, 8, 128, 1) == 0 and lib.mlora_page_attn_workspace_bytes(0, 8, 128, 3) == 0
    for fn in ("mlora_page_attn_decode", "mlora_page_attn_prefill"):
        assert _attn(lib, fn, splits=0) == -1 and _attn(lib, fn, splits=65) == -1 and _attn(lib, fn, T=70000, splits=2, ws=16, nb=1 << 40) == -1
        for ws, nb in ((0, need), (16, need - 1), (24, need)):
            assert _attn(lib, fn, splits=3, ws=ws, nb=nb) == -3
    assert _attn(lib, "mlora_page_attn_prefill", step=0, cos=0, sin=0, T=0) == 0 and _attn(lib, "mlora_page_attn_prefill", T=1 << 24) == -2
    assert _attn(lib, "mlora_page_attn_prefill", Hq=130, Hkv=2) == -2
    for prompt in (0, 1):
        splits = lambda *a: lib.mlora_page_attn_splits(prompt, *a)                                                 # noqa: E731
        assert splits(0, 8, 8, 100) == 1 and splits(1, 8, 8, 1) == 1 and 1 < splits(1, 8, 8, 1 << 20) <= 64 and splits(70000, 8, 8, 1 << 20) == 1 and splits(4, 8, 0, 9) == 1
    assert lib.mlora_page_values(16, 16, 16, 16, 16, 16, 1, 8, 96, 4, None) == -2 and lib.mlora_page_values(16, 16, 16, 16, None, 16, 1, 8, 64, 4, None) == -1
    assert lib.mlora_page_values(16, 16, 16, 16, 16, None, 1, 8, 64, 4, None) == -1 and lib.mlora_page_values(16, 16, 16, 16, 16, 16, 65536, 8, 64, 4, None) == -1
    assert lib.mlora_page_values(16, 16, 16, 16, 16, None, 0, 8, 64, 4, None) == 0


def test_copy_refusals():
    lib = load_pkg("_lib").lib()
    pool = lambda *a: struct.pack("@Plii", *a)                                                                     # noqa: E731
    good = pool(16, 64, 2, 9)
    assert lib.mlora_copy_pages(None, 1, 16, 16, 1, None) == -1 and lib.mlora_copy_pages(good, 1, None, 16, 1, None) == -1 and lib.mlora_copy_pages(good, 0, 16, 16, 1, None) == -1
    assert lib.mlora_copy_pages(good * 9, 9, 16, 16, 1, None) == -1 and lib.mlora_copy_pages(good, 1, 16, 16, -1, None) == -1
    for bad in (pool(0, 64, 2, 9), pool(16, 0, 2, 9), pool(16, 64, 0, 9), pool(16, 64, 2, 0), pool(16, (1 << 30) + 1, 2, 9)):
        assert lib.mlora_copy_pages(bad, 1, 16, 16, 1, None) == -1
    assert lib.mlora_copy_pages(pool(16, 1 << 30, 1 << 14, 9), 1, 16, 16, 1, None) == -2
    assert lib.mlora_copy_pages(good, 1, None, None, 0, None) == 0


def test_beam_refusals():
    lib = load_pkg("_lib").lib()
    need = lib.mlora_beam_select_workspace_bytes(2, 3, 500, 4)
    assert need > 0 and need % 8 == 0 and lib.mlora_beam_select_workspace_bytes(0, 3, 500, 4) == 0

    def call(out=16, logits=16, ld=500, scores=16, ended=None, eos=0, R=2, W=3, V=500, k=4, ws=16, nb=1 << 20):
        return lib.mlora_beam_select(out, 16, 16, logits, ld, scores, ended, eos, R, W, V, k, ws, nb, None)
    assert call(out=None) == -1 and call(scores=None) == -1 and call(logits=18) == -1 and call(ld=499) == -1 and call(V=0) == -1 and call(R=-1) == -1
    assert call(W=17) == -2 and call(W=0) == -2 and call(k=33) == -2 and call(k=0) == -2 and call(R=30000) == -2
    assert call(ended=16, eos=500) == -1 and call(ended=16, eos=-1) == -1
    assert call(ws=None) == -3 and call(nb=need - 1) == -3 and call(ws=20) == -3 and call(R=0) == 0
    order = lambda p=16, R=2, W=3, n=6, mb=4: lib.mlora_beam_reorder(16, 16, 16, 16, 16, p, 16, 16, 16, R, W, n, mb, None)   # noqa: E731
    assert order(p=None) == -1 and order(R=-1) == -1 and order(W=17) == -2 and order(n=0) == -1 and order(mb=0) == -1 and order(R=0) == 0
