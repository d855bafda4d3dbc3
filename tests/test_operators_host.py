"""Argument checks of the operators of a wide decode step that need no GPU: every call below is refused ahead of a launch."""
import ctypes as C

from conftest import load_pkg


def test_constrained_argmax_refusals():
    lm = load_pkg("_lib")
    lib = lm.lib()
    def call(B=2, V=50000, ld=50000, out=None, ld_out=0, ws=16, nb=1 << 20, **kw):
        r = lm.LogitRulesArgs(**kw)
        return lib.mlora_constrained_argmax(16, out, ld_out, 16, ld, C.byref(r), B, V, ws, nb, None)
    assert lib.mlora_constrained_argmax_workspace_bytes(2, 50000) == 2 * 13 * 8 and lib.mlora_constrained_argmax_workspace_bytes(2, 32000) == 0
    assert lib.mlora_constrained_argmax(16, None, 0, None, 10, C.byref(lm.LogitRulesArgs()), 1, 10, None, 0, None) == -1
    assert call(B=-1) == -1 and call(B=65536) == -1 and call(V=0) == -1 and call(ld=49999) == -1
    assert call(out=16, ld_out=100) == -1
    assert call(history=16) == -1 and call(history=16, lengths=16, cap=0) == -1
    assert call(repetition=16) == -1 and call(append=1) == -1
    assert call(n_bias=1025, bias_ids=16, bias=16) == -2 and call(n_bias=3, bias_ids=16) == -1
    assert call(masks=16, n_masks=1) == -1 and call(masks=16, mask_row=16) == -1
    assert call(ws=None) == -3 and call(nb=2 * 13 * 8 - 1) == -3 and call(ws=20) == -3
    assert call(B=0) == 0
