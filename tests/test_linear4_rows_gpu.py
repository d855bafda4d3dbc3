"""4-bit linears of 17 to 32 tokens, either side of the borders between the two kernels, in rows and in fragment order."""
import pytest
import torch

import test_linear4_gpu as L
from conftest import load_pkg

pytestmark = pytest.mark.gpu

# K and N beside the borders; groups of every size
SIZES = [(512, 70, 32), (544, 70, 32), (1024, 4096, 64), (1024, 4112, 64), (1056, 48, 32), (2048, 200, 128), (2080, 170, 32), (4096, 1024, 128), (4096, 4100, 64),
         (4096, 5400, 32), (4224, 4096, 128), (4224, 4080, 64), (6144, 6150, 64), (6208, 40, 64)]


@pytest.mark.parametrize("K,N,group", SIZES)
def test_either_order_of_x(ops, K, N, group):
    """Stored and added, against 64 bits."""
    lib = load_pkg("_lib").lib()
    x, q, scale, zero = L.make(K + N, 32, K, N, group)
    W = ops.QuantWeight(q, scale, zero)
    y, mag = L.exact(x, q, scale, zero, group)
    for T in (17, 20, 21, 24, 25, 28, 29, 32):
        print("case rows", T, K, N, group, lib.mlora_linear4_workspace_bytes_of(T, K, N, 0), flush=True)
        a = x[:T].contiguous()
        wide = torch.full((T, K + 24), float("nan"), dtype=torch.float16, device=L.DEV)
        wide[:, 8:8 + K] = a
        for xs in (a, wide[:, 8:8 + K], ops.FragActivation.pack(a)):
            for out in (torch.float16, torch.float32):
                got = ops.linear(xs, W, out_dtype=out)
                assert bool(((got.double() - y[:T]).abs() <= L.bound(y[:T], mag[:T], K, group, out)).all())
        acc = torch.randn((T, N), device=L.DEV)
        want = acc.double() + y[:T]
        most = L.bound(y[:T], mag[:T] + want.abs() + y[:T].abs(), K, group, torch.float32)
        assert bool(((ops.linear(a, W, out=acc, accumulate=True).double() - want).abs() <= most).all())


@pytest.mark.parametrize("N,K", [(256, 384), (250, 352)])
def test_weights_in_any_order(ops, N, K):
    """q, scale and zero, or the weight that is rounded, as transposed or cut views: the same packed weight."""
    print("case strided weights", N, K, flush=True)
    group = 32
    x, q, scale, zero = L.make(N, 4, K, N, group)
    want = ops.QuantWeight(q, scale, zero)
    turned = [t.t().contiguous().t() for t in (q, scale, zero)]
    cut = [torch.cat([t, t], 1)[:, :t.shape[1]] for t in (q, scale, zero)]
    for views in (turned, cut):
        assert not views[0].is_contiguous()
        W = ops.QuantWeight(*views)
        assert torch.equal(W.q, want.q) and torch.equal(W.meta, want.meta)
    w = torch.randn((N, K), device=L.DEV).half()
    want = ops.quantize(w, group)
    for view in (w.t().contiguous().t(), torch.cat([w, w], 1)[:, :K], w.float().t().contiguous().t()):
        W = ops.quantize(view, group)
        assert torch.equal(W.q, want.q) and torch.equal(W.meta, want.meta)
