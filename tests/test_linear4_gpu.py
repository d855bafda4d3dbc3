"""Linears with 4-bit weights against the definition in 64 bits."""
import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, T, K, N, group):
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    x = torch.randn((T, K), generator=g, device=DEV).to(torch.float16)
    q = torch.randint(0, 16, (N, K), generator=g, device=DEV, dtype=torch.uint8)
    scale = (0.01 * torch.randn((N, K // group), generator=g, device=DEV).exp()).to(torch.float16)
    zero = torch.randint(0, 16, (N, K // group), generator=g, device=DEV, dtype=torch.uint8)
    return x, q, scale, zero


def exact(x, q, scale, zero, group):
    """(y, sum of the terms' magnitudes) in 64 bits."""
    d = torch.float64
    w = scale.to(d).repeat_interleave(group, 1) * (q.to(d) - zero.to(d).repeat_interleave(group, 1))
    return x.to(d) @ w.t(), x.to(d).abs() @ w.abs().t()


def bound(y, mag, K, group, out):
    """Products are exact.  A term passes through at most `group` additions of its group's sum, the scaling, the sums over a wave's groups and over
    eight waves (and the one into y): each half a step of at most the sum of the magnitudes; then the result's own rounding."""
    depth = group + 2 + -(-K // 128) * (128 // group) + 9
    return depth * 2.0 ** -24 * mag + (y.abs() * 2.0 ** -11 + 2.0 ** -25 if out == torch.float16 else 0)


SIZES = [(1, 32, 1, 32), (1, 64, 16, 64), (2, 96, 5, 32), (3, 128, 40, 128), (16, 352, 33, 32), (17, 192, 64, 64), (33, 1024, 100, 128), (64, 4096, 48, 128),
         (65, 256, 17, 64), (130, 640, 1000, 128), (1, 11008, 4096, 128), (16, 4096, 9000, 64), (31, 4096, 256, 32), (200, 2080, 2050, 32), (257, 128, 18000, 128)]


@pytest.mark.parametrize("T,K,N,group", SIZES)
def test_linear4_against_64_bits(ops, T, K, N, group):
    print("case linear4", T, K, N, group, flush=True)
    x, q, scale, zero = make(T + K + N, T, K, N, group)
    W = ops.QuantWeight(q, scale, zero)
    y, mag = exact(x, q, scale, zero, group)
    assert torch.equal(W.dequantize().double(), scale.double().repeat_interleave(group, 1) * (q.double() - zero.double().repeat_interleave(group, 1)))
    wide = torch.zeros((T, K + 40), dtype=torch.float16, device=DEV)
    wide[:, 8:8 + K] = x
    frag = ops.FragActivation.pack(x)
    for name, a in (("rows", x), ("strided", wide[:, 8:8 + K]), ("off 16 bytes", _shifted(x)), ("fragments", frag)):
        for out in (torch.float16, torch.float32):
            got = ops.linear(a, W, out_dtype=out)
            assert got.dtype == out and got.shape == (T, N)
            off = (got.double() - y).abs()
            assert bool((off <= bound(y, mag, K, group, out)).all()), (name, out, float((off / bound(y, mag, K, group, out)).max()))
    acc = torch.randn((T, N), device=DEV)
    want = acc.double() + y
    got = ops.linear(x, W, out=acc, accumulate=True)
    assert got is acc
    assert bool(((acc.double() - want).abs() <= bound(y, mag + want.abs() + y.abs(), K, group, torch.float32)).all())
    # into rows of a larger buffer, whose neighbours stay
    buf = torch.full((T * N + 7,), 3.0, dtype=torch.float32, device=DEV)
    ops.linear(x, W, out=buf[3:3 + T * N].view(T, N))
    assert torch.equal(buf[3:3 + T * N].view(T, N), ops.linear(x, W, out_dtype=torch.float32)) and bool((buf[:3] == 3).all()) and bool((buf[3 + T * N:] == 3).all())


# every cut of the kernel for more than 16 tokens: one to three row tiles a wave, K in slices, whole and broken last blocks for either group of
# waves, token blocks of 32 and 64 that are not full; and of the other one tiles of every count, waves with and without the end of K
CUTS = [(200, 160, 12200, 32), (193, 192, 12250, 64), (250, 256, 12288, 128), (100, 160, 16300, 32), (20, 1056, 12300, 32), (64, 2080, 300, 32), (48, 4160, 70, 64),
        (25, 2048, 700, 128), (17, 128, 40000, 128), (16, 1056, 4100, 32), (9, 288, 8200, 32), (5, 320, 12290, 64), (16, 192, 16400, 64), (3, 96, 24600, 32), (2, 128, 33000, 128),
        (1, 2016, 50, 32), (8, 1152, 33000, 64), (30, 192, 8200, 64), (18, 288, 16400, 32), (32, 96, 22100, 32), (27, 128, 24576, 64), (19, 6144, 40, 128), (17, 6176, 33, 32)]


@pytest.mark.parametrize("T,K,N,group", CUTS)
def test_every_cut(ops, T, K, N, group):
    print("case cut", T, K, N, group, flush=True)
    x, q, scale, zero = make(T + K + N, T, K, N, group)
    W = ops.QuantWeight(q, scale, zero)
    y, mag = exact(x, q, scale, zero, group)
    for a in (x, ops.FragActivation.pack(x)):
        for out in (torch.float16, torch.float32):
            got = ops.linear(a, W, out_dtype=out)
            assert bool(((got.double() - y).abs() <= bound(y, mag, K, group, out)).all())
            assert torch.equal(got, ops.linear(a, W, out_dtype=out))


def _shifted(x):
    flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=x.device)
    flat[1:] = x.reshape(-1)
    return flat[1:].view(x.shape)


@pytest.mark.parametrize("T", [1, 20, 64, 70])
def test_rows_do_not_touch_each_other(ops, T):
    """An infinite or NaN row stays in its row, and a row's bits do not depend on the others."""
    print("case rows", T, flush=True)
    x, q, scale, zero = make(3, T, 512, 300, 64)
    W = ops.QuantWeight(q, scale, zero)
    clean = ops.linear(x, W)
    x[T // 2, 7] = float("nan")
    x[0, 511] = float("inf")
    for a in (x, ops.FragActivation.pack(x)):
        y = ops.linear(a, W)
        keep = [t for t in range(T) if t not in (0, T // 2)]
        assert torch.equal(y[keep], clean[keep]) and not bool(y[T // 2].isfinite().any())
    big = torch.full((2, 512), 65504.0, dtype=torch.float16, device=DEV)     # sums beyond fp16 come out as infinities, in fp32 whole
    z = ops.linear(big, W, out_dtype=torch.float32)
    assert bool(z.isfinite().all())


def test_extreme_weights(ops):
    print("case extremes", flush=True)
    K, N = 256, 32
    x = torch.ones((4, K), dtype=torch.float16, device=DEV)
    for q, z in ((0, 15), (15, 0), (7, 7)):
        W = ops.QuantWeight(torch.full((N, K), q, dtype=torch.uint8, device=DEV), torch.full((N, 2), 2.0 ** -24, dtype=torch.float16, device=DEV),
                            torch.full((N, 2), z, dtype=torch.uint8, device=DEV))
        assert bool((ops.linear(x, W, out_dtype=torch.float32) == (q - z) * K * 2.0 ** -24).all())


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(ops, group):
    """Rounded to steps of a sixteenth of a group's range (0 included): half a step, half a step of the moved zero and what the scale's fp16 rounding adds."""
    print("case quantize", group, flush=True)
    g = torch.Generator(DEV)
    g.manual_seed(group)
    w = torch.randn((70, 512), generator=g, device=DEV) * 0.02
    w[3, :group] = 0
    w[4, group:2 * group] = w[4, group:2 * group].abs() + 0.01
    W = ops.quantize(w.half(), group)
    w = w.half().float()
    v = w.view(70, -1, group)
    step = (v.amax(2).clamp_min(0) - v.amin(2).clamp_max(0)) / 15
    off = (W.dequantize() - w).view(70, -1, group).abs()
    assert bool((off <= step[..., None] * (1 + 16 * 2.0 ** -10) + 2.0 ** -24).all())
    assert bool((W.dequantize()[3, :group] == 0).all())


def test_graph_streams_and_empty(ops):
    print("case graphs", flush=True)
    x, q, scale, zero = make(9, 5, 512, 320, 128)
    W = ops.QuantWeight(q, scale, zero)
    want = ops.linear(x, W)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.linear(x, W, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.linear(x, W)
    s.synchronize()
    assert torch.equal(other, want)
    assert ops.linear(x[:0], W).shape == (0, 320)


def test_refusals(ops):
    print("case refusals", flush=True)
    x, q, scale, zero = make(1, 4, 256, 32, 128)
    W = ops.QuantWeight(q, scale, zero)
    for args in ((q, scale[:, :1], zero[:, :1]), (q, scale, zero[:, :1]), (q[:, :250], scale, zero), (q, scale[:31], zero[:31]), (q.cpu(), scale.cpu(), zero.cpu()),
                 (q + 16, scale, zero), (q, scale, zero + 9), (q.int(), scale, zero), (q, scale.float(), zero)):
        with pytest.raises((ValueError, TypeError)):
            ops.QuantWeight(*args)
    for a, kw in ((x[:, :128], {}), (x.float(), {}), (x.bfloat16(), {}), (x.cpu(), {}), (x, {"out": torch.zeros((3, 32), device=DEV)}), (x, {"accumulate": True}),
                  (x, {"out": torch.zeros((4, 64), device=DEV)[:, ::2]})):
        with pytest.raises(ValueError):
            ops.linear(a, W, **kw)
    lm = load_pkg("_lib")
    with pytest.raises(lm.MloraError):
        ops.linear(x, W, out=torch.zeros((4, 32), dtype=torch.float16, device=DEV), accumulate=True)
    with pytest.raises(ValueError):
        ops.quantize(torch.zeros((16, 100), device=DEV), 64)
