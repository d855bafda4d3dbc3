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
