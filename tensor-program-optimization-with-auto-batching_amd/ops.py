"""Operator surface over the C ABI: torch tensors supply device memory and the stream, nothing else.

Each function validates dtypes/contiguity on the host, hands raw pointers to libmlora_hip.so and
enqueues on torch's current stream.  None of them has a CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import struct
import typing

import torch

from . import _lib
from ._lib import F16, F32, ROWMAJOR, FRAG, STORE, ACCUMULATE, GLU_SILU, GLU_CLIPPED, lib

_BUCKET = struct.Struct("@PPiif4x")          # mlora_lora_bucket
_PAGE_ATTN = struct.Struct("@13PN12i")       # mlora_page_attn
_PAGE_POOL = struct.Struct("@Plii")          # mlora_page_pool
_LIB_OF = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}


def lib_of(dtype: torch.dtype):
    """The kernel library whose element type is `dtype`."""
    return lib(_LIB_OF[dtype])


def check(code: int, dtype: torch.dtype = torch.float16) -> None:
    _lib.check(code, _LIB_OF[dtype])


def _stream() -> int:
    """The current stream of the current device, without the object around it (6 us less per call)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _bucket(A, B, r, n_ad, scaling) -> bytes:
    """A mlora_lora_bucket (a scaling beyond fp32 is infinite, which struct alone refuses)."""
    return _BUCKET.pack(A, B, r, n_ad, ctypes.c_float(float(scaling)).value)


def upload(t: torch.Tensor, device, dtype=None) -> torch.Tensor:
    """A host tensor's copy on `device`, queued on the current stream; the host does not wait.  The values go through pinned memory
    of torch's pool, which keeps it until the copy has run.  (A copy from pageable memory waits for all that the stream holds: four
    of them left the GPU idle for 100 to 400 us of an eager pass.)  Above 64 KiB the host waits as it did: the copy engine that
    takes those makes the next release of device memory, as a capture begins with, 3 ms longer.  A capture refuses the copy as it
    did: its replays would read memory given back."""
    dtype = dtype or t.dtype
    if (t.is_cuda or not 0 < t.numel() * dtype.itemsize <= 65536 or torch.device(device).type != "cuda"
            or torch.cuda.is_current_stream_capturing()):
        return t.to(device, dtype)
    return torch.empty(t.shape, dtype=dtype, pin_memory=True).copy_(t).to(device, non_blocking=True)


@functools.lru_cache(maxsize=4096)
def _size(dtype, fn, *args):
    """A sizing or shape-rule function of the library (they depend on their integer arguments alone)."""
    return getattr(lib_of(dtype), fn)(*args)


def _dev(t: torch.Tensor, dtype=None, name="tensor") -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _here(device, who):
    """`device`, where work queued on the current stream runs."""
    if device.type != "cuda":
        raise ValueError(f"{who}: tensors must live on the GPU (no CPU path)")
    if device.index != torch._C._cuda_getDevice():
        raise ValueError(f"{who}: tensors on {device} while cuda:{torch._C._cuda_getDevice()} is current")
    return device


# A contiguous uninitialised tensor on the current device: what torch.empty gives, by the entry that torch's own compiled code uses (0.8 us instead of 1.7 a
# tensor, of which an operator of a few microseconds makes two).  It is torch's own affair: where it is absent, or gives anything else than it
# is asked for, the public function takes its place.  It goes past dispatch modes and the filling of new memory, which the operators can do
# without: they take addresses, and write every element of what they return.
def _plain_empty(size, stride, dtype):
    return torch.empty_strided(size, stride, dtype=dtype, device=torch.device("cuda", torch._C._cuda_getDevice()))


def _short_or_plain(short, device):
    try:
        t = short((2, 3), (3, 1), torch.float16)
        good = (t.shape, t.stride(), t.dtype, t.device, t.requires_grad) == ((2, 3), (3, 1), torch.float16, device, False)
    except Exception:
        good = False
    return short if good else _plain_empty


def _empty_strided_cuda(size, stride, dtype):
    """(The first call: chooses what takes its place.)"""
    global _empty_strided_cuda
    try:
        from torch._C._dynamo.guards import _empty_strided_cuda as short
    except ImportError:
        short = None
    _empty_strided_cuda = _short_or_plain(short, torch.device("cuda", torch._C._cuda_getDevice()))
    return _empty_strided_cuda(size, stride, dtype)


def _dt(t: torch.Tensor) -> int:
    if t.dtype in (torch.float16, torch.bfloat16):
        return F16
    if t.dtype == torch.float32:
        return F32
    raise TypeError(f"expected a 16-bit float type or float32, got {t.dtype}")


class FragActivation:
    """A [T, K] 16-bit activation block stored in matrix-core fragment order (MLORA_FRAG)."""

    def __init__(self, T: int, K: int, device, data: torch.Tensor = None, dtype: torch.dtype = torch.float16):
        self.T, self.K = T, K
        n = _size(dtype if data is None else data.dtype, "mlora_frag_activation_elems", T, K)
        self.data = torch.empty(n, dtype=dtype, device=device) if data is None else data
        if self.data.numel() < n:
            raise ValueError("FragActivation: buffer too small")

    @property
    def shape(self):
        return (self.T, self.K)

    @property
    def device(self):
        return self.data.device

    @property
    def dtype(self):
        return self.data.dtype

    def _tiles(self) -> int:
        return 1 if self.T <= 16 else (2 if self.T <= 32 else (4 if self.T <= 64 else -(-self.T // 16)))

    def columns(self, k0: int, K: int) -> "FragActivation":
        """Columns k0 .. k0 + K - 1 as a block of their own (multiples of 32: whole k-blocks, contiguous in this order)."""
        if k0 % 32 or K % 32 or k0 + K > self.K:
            raise ValueError("FragActivation.columns: whole 32-column blocks")
        return FragActivation(self.T, K, self.device, self.data[k0 * 16 * self._tiles():])

    @classmethod
    def pack(cls, x: torch.Tensor, out: "FragActivation" = None):
        """Row-major [T, K] (unit inner stride) -> fragment order."""
        T, K = x.shape
        out = cls(T, K, x.device, dtype=x.dtype) if out is None else out
        ld = x.stride(0) if T > 1 else max(K, x.stride(0))
        check(lib_of(x.dtype).mlora_pack_activation(out.data.data_ptr(), x.data_ptr(), ld, T, K, _stream()), x.dtype)
        return out

    def unpack(self) -> torch.Tensor:
        """Back to row-major [T, K] (host-side index arithmetic on the device tensor; for tests)."""
        TT = self._tiles()
        v = self.data[: TT * 16 * self.K].view(self.K // 32, TT, 4, 16, 8)
        return v.permute(1, 3, 0, 2, 4).reshape(TT * 16, self.K)[: self.T].contiguous()


def _x_arg(x, name="x"):
    """(pointer, layout, T, K) of a row-major tensor or a FragActivation."""
    if isinstance(x, FragActivation):
        return x.data.data_ptr(), FRAG, x.T, x.K
    return _dev(x, torch.float16, name), ROWMAJOR, x.shape[0], x.shape[1]


def gather_mm_workspace(T: int, K: int, r: int, device) -> torch.Tensor:
    n = _size(torch.float16, "mlora_gather_mm_workspace_bytes", T, K, r)
    return torch.empty(max(n, 16) // 4, dtype=torch.float32, device=device)


def gather_mm(y, x, A, B, tok_adapter, scaling: float, workspace=None):
    """y[t] += scaling * B[id_t] @ (A[id_t] @ x[t]) in place.  y [T,N] f16|f32 (rows may be strided: a
    column slice of a wider buffer), x [T,K] f16, A [n_ad,r,K] f16, B [n_ad,N,r] f16,
    tok_adapter [T] int32 (-1 = no adapter)."""
    xptr, xlay, T, K = _x_arg(x)
    n_ad, r, K2 = A.shape
    N = B.shape[1]
    if K2 != K or B.shape != (n_ad, N, r) or y.shape != (T, N) or tok_adapter.shape != (T,):
        raise ValueError(f"gather_mm: inconsistent shapes y{tuple(y.shape)} x{tuple(x.shape)} A{tuple(A.shape)} "
                         f"B{tuple(B.shape)} ids{tuple(tok_adapter.shape)}")
    if T == 0:
        return y                                   # an empty batch: nothing to add (an empty tensor has no device pointer)
    if workspace is None:
        workspace = gather_mm_workspace(T, K, r, x.device)
    if not y.is_cuda or y.stride(1) != 1:
        raise ValueError("gather_mm: y must be a GPU tensor with unit inner stride")
    ldy = y.stride(0) if T > 1 else max(N, y.stride(0))
    check(lib().mlora_gather_mm(y.data_ptr(), _dt(y), ldy, xptr, xlay, _dev(A, torch.float16, "A"),
                                _dev(B, torch.float16, "B"), _dev(tok_adapter, torch.int32, "tok_adapter"),
                                float(scaling), T, K, N, r, n_ad, _dev(workspace, torch.float32, "workspace"),
                                workspace.numel() * 4, _stream()))
    return y


def gather_mm_static(y, x, A, B, tok_adapter, scaling: float):
    """gather_mm through the entry point that allocates nothing: the kernels' scratch is a buffer built into the
    library (raises for shapes whose scratch exceeds it).  Calls that overlap on one GPU share that buffer and race."""
    xptr, xlay, T, K = _x_arg(x)
    n_ad, r, K2 = A.shape
    N = B.shape[1]
    if K2 != K or B.shape != (n_ad, N, r) or y.shape != (T, N) or tok_adapter.shape != (T,):
        raise ValueError("gather_mm_static: inconsistent shapes")
    if T == 0:
        return y
    if not y.is_cuda or y.stride(1) != 1:
        raise ValueError("gather_mm_static: y must be a GPU tensor with unit inner stride")
    ldy = y.stride(0) if T > 1 else max(N, y.stride(0))
    check(lib().mlora_gather_mm_static(y.data_ptr(), _dt(y), ldy, xptr, xlay, _dev(A, torch.float16, "A"),
                                       _dev(B, torch.float16, "B"), _dev(tok_adapter, torch.int32, "tok_adapter"),
                                       float(scaling), T, K, N, r, n_ad, _stream()))
    return y


def gather_mm_multi(y, x, buckets, tok_bucket, tok_adapter, workspace=None):
    """Adapters of several ranks in one batch: buckets = [(A [n_ad,r,K], B [n_ad,N,r], scaling) | None, ...]; token t uses
    adapter tok_adapter[t] of bucket tok_bucket[t] (-1 = none).  y is updated in place."""
    xptr, xlay, T, K = _x_arg(x)
    N = y.shape[1]
    if y.shape[0] != T or tok_bucket.shape != (T,) or tok_adapter.shape != (T,):
        raise ValueError("gather_mm_multi: inconsistent shapes")
    arr = b""
    rmax = 8
    for i, bk in enumerate(buckets):
        if bk is None:                      # the bucket's adapters do not target this projection
            arr += _bucket(0, 0, 0, 0, 0.0)
            continue
        A, B, scaling = bk
        n_ad, r, K2 = A.shape
        if K2 != K or B.shape != (n_ad, N, r):
            raise ValueError(f"gather_mm_multi: bucket {i} has A{tuple(A.shape)} B{tuple(B.shape)} for K={K} N={N}")
        arr += _bucket(_dev(A, torch.float16, "A"), _dev(B, torch.float16, "B"), r, n_ad, scaling)
        rmax = max(rmax, r)
    if workspace is None:
        workspace = gather_mm_workspace(T, K, rmax, x.device)
    if not y.is_cuda or y.stride(1) != 1:
        raise ValueError("gather_mm_multi: y must be a GPU tensor with unit inner stride")
    ldy = y.stride(0) if T > 1 else max(N, y.stride(0))
    check(lib().mlora_gather_mm_multi(y.data_ptr(), _dt(y), ldy, xptr, xlay, arr, len(buckets),
                                      _dev(tok_bucket, torch.int32, "tok_bucket"), _dev(tok_adapter, torch.int32, "tok_adapter"),
                                      T, K, N, _dev(workspace, torch.float32, "workspace"), workspace.numel() * 4, _stream()))
    return y


def gather_mm_multi_proj(y, x, proj_buckets, col_offsets, n_cols, tok_bucket, tok_adapter, workspace=None):
    """gather_mm_multi for several projections that read the same x and own disjoint column ranges of y (q, k, v in the
    fused qkv row; gate and up): proj_buckets[p] is the bucket list of projection p (as for gather_mm_multi, all of the
    same length), whose delta goes to y[:, col_offsets[p] : col_offsets[p] + n_cols[p]].  One launch at decode sizes."""
    xptr, xlay, T, K = _x_arg(x)
    n_proj = len(proj_buckets)
    n_buckets = len(proj_buckets[0])
    if y.shape[0] != T or tok_bucket.shape != (T,) or tok_adapter.shape != (T,) or len(col_offsets) != n_proj or len(n_cols) != n_proj \
            or any(len(b) != n_buckets for b in proj_buckets):
        raise ValueError("gather_mm_multi_proj: inconsistent shapes")
    if T == 0:
        return y
    arr = b""
    rmax = 8
    for p, buckets in enumerate(proj_buckets):
        for i, bk in enumerate(buckets):
            if bk is None:                      # the bucket's adapters do not target this projection
                arr += _bucket(0, 0, 0, 0, 0.0)
                continue
            A, B, scaling = bk
            n_ad, r, K2 = A.shape
            if K2 != K or B.shape != (n_ad, n_cols[p], r):
                raise ValueError(f"gather_mm_multi_proj: projection {p} bucket {i} has A{tuple(A.shape)} B{tuple(B.shape)} "
                                 f"for K={K} N={n_cols[p]}")
            arr += _bucket(_dev(A, torch.float16, "A"), _dev(B, torch.float16, "B"), r, n_ad, scaling)
            rmax = max(rmax, r)
    if workspace is None:
        one = gather_mm_workspace(T, K, rmax, x.device).numel()
        workspace = torch.empty(3 * one, dtype=torch.float32, device=x.device)     # a slice per projection sharing a launch
    if not y.is_cuda or y.stride(1) != 1:
        raise ValueError("gather_mm_multi_proj: y must be a GPU tensor with unit inner stride")
    ldy = y.stride(0) if T > 1 else max(y.shape[1], y.stride(0))
    co, nc = (struct.pack(f"{n_proj}i", *(int(c) for c in v)) for v in (col_offsets, n_cols))
    check(lib().mlora_gather_mm_multi_proj(y.data_ptr(), _dt(y), ldy, xptr, xlay, arr, n_buckets, n_proj, co, nc,
                                           _dev(tok_bucket, torch.int32, "tok_bucket"), _dev(tok_adapter, torch.int32, "tok_adapter"),
                                           T, K, _dev(workspace, torch.float32, "workspace"), workspace.numel() * 4, _stream()))
    return y


def gather_mm_segments(y, x, tables, col_offsets, n_cols, tok_adapter, scaling: float, workspace):
    """gather_mm for one to three projections ((A, B) in `tables`, of one rank and table size) that read the same x and own column ranges
    of y, where the tokens come in adapter segments: a prompt, or several behind each other.  On the matrix cores whatever T is."""
    xptr, xlay, T, K = _x_arg(x)
    n_ad, r, _ = tables[0][0].shape
    if y.shape[0] != T or tok_adapter.shape != (T,) or len(col_offsets) != len(tables) or len(n_cols) != len(tables) \
            or any(A.shape != (n_ad, r, K) or B.shape != (n_ad, n, r) for (A, B), n in zip(tables, n_cols)):
        raise ValueError("gather_mm_segments: inconsistent shapes")
    if not y.is_cuda or y.stride(1) != 1:
        raise ValueError("gather_mm_segments: y must be a GPU tensor with unit inner stride")
    if T == 0:
        return y
    arr = b"".join(_bucket(_dev(A, torch.float16, "A"), _dev(B, torch.float16, "B"), r, n_ad, scaling) for A, B in tables)
    ldy = y.stride(0) if T > 1 else max(y.shape[1], y.stride(0))
    co, nc = (struct.pack(f"{len(tables)}i", *v) for v in (col_offsets, n_cols))
    check(lib().mlora_gather_mm_segments(y.data_ptr(), _dt(y), ldy, xptr, xlay, arr, len(tables), co, nc, _dev(tok_adapter, torch.int32, "tok_adapter"),
                                         T, K, _dev(workspace, torch.float32, "workspace"), workspace.numel() * 4, _stream()))
    return y


class GatherMMBatch:
    """Several gather-matmul problems of one shape and one token->adapter table, issued as one launch.
    sets: list of (y, x, A, B) as for gather_mm (x row-major); the tensors are kept alive by this object."""

    def __init__(self, sets, tok_adapter, scaling: float, stream_passes: bool = True):
        """stream_passes: give the call a workspace, which lets it run eight or more sets as a shrink pass and an
        expand pass over all of them (same result bits as the single launch it uses otherwise)."""
        y0, x0, A0, B0 = sets[0]
        self.T, self.K = x0.shape
        self.n_ad, self.r, _ = A0.shape
        self.N = B0.shape[1]
        self.ldy = y0.stride(0) if self.T > 1 else max(self.N, y0.stride(0))
        self.ydt = _dt(y0)
        ptrs = []
        for y, x, A, B in sets:
            if (x.shape != (self.T, self.K) or A.shape != (self.n_ad, self.r, self.K) or B.shape != (self.n_ad, self.N, self.r)
                    or y.shape != (self.T, self.N) or _dt(y) != self.ydt or y.stride(1) != 1
                    or (self.T > 1 and y.stride(0) != self.ldy)):
                raise ValueError("GatherMMBatch: all sets must share shape, dtype and row stride")
            ptrs += [y.data_ptr(), _dev(x, torch.float16, "x"), _dev(A, torch.float16, "A"), _dev(B, torch.float16, "B")]
        self.sets = list(sets)
        self.ids = tok_adapter
        _dev(tok_adapter, torch.int32, "tok_adapter")
        self.scaling = float(scaling)
        self.table = torch.tensor(ptrs, dtype=torch.int64, device=x0.device)
        self.ws = None
        if stream_passes:
            n = len(sets) * lib().mlora_gather_mm_workspace_bytes(self.T, self.K, self.r)
            self.ws = torch.empty(max(n, 16) // 4, dtype=torch.float32, device=x0.device)

    def run(self):
        ws, nb = (self.ws.data_ptr(), self.ws.numel() * 4) if self.ws is not None else (None, 0)
        check(lib().mlora_gather_mm_batch(self.table.data_ptr(), len(self.sets), self.ydt, self.ldy, ROWMAJOR,
                                          self.ids.data_ptr(), self.scaling, self.T, self.K, self.N, self.r, self.n_ad,
                                          ws, nb, _stream()))


def lora_shrink(v_part, x, A, tok_adapter):
    xptr, xlay, T, K = _x_arg(x)
    n_ad, r, _ = A.shape
    check(lib().mlora_lora_shrink(_dev(v_part, torch.float32), xptr, xlay, _dev(A, torch.float16),
                                  _dev(tok_adapter, torch.int32), T, K, r, n_ad, _stream()))
    return v_part


def lora_expand(y, v_part, B, tok_adapter, scaling: float, K: int):
    T, N = y.shape
    n_ad, _, r = B.shape
    check(lib().mlora_lora_expand(_dev(y), _dt(y), N, _dev(v_part, torch.float32), _dev(B, torch.float16),
                                  _dev(tok_adapter, torch.int32), float(scaling), T, K, N, r, n_ad, _stream()))
    return y


def write_tensor_part(X, Y, ids, out=None):
    """Z = X; Z[ids[a]] = Y[a] over the leading dimension."""
    Z = torch.empty_like(X) if out is None else out
    B, A = X.shape[0], Y.shape[0]
    PH = X[0].numel() if B else (Y[0].numel() if A else 8)
    check(lib().mlora_write_tensor_part(_dev(Z, torch.float16), _dev(X, torch.float16), _dev(Y, torch.float16),
                                        _dev(ids, torch.int32), B, A, PH, _stream()))
    return Z


class PackedWeight:
    """A [N, K] 16-bit weight stored in matrix-core fragment order (see mlora_pack_weight)."""

    def __init__(self, W: torch.Tensor):
        N, K = W.shape
        self.N, self.K = N, K
        L = lib_of(W.dtype)
        n = L.mlora_packed_weight_elems(N, K)
        self.data = torch.empty(n, dtype=W.dtype, device=W.device)
        check(L.mlora_pack_weight(_dev(self.data), _dev(W, name="W"), N, K, _stream()), W.dtype)

    @property
    def shape(self):
        return (self.N, self.K)

    @property
    def dtype(self):
        return self.data.dtype

    def rows(self, n0: int, n: int) -> "PackedWeight":
        """Rows n0 .. n0 + n - 1 (n0 a multiple of 16) as a weight of their own: a view."""
        if n0 % 16 or n0 + n > self.N:
            raise ValueError("PackedWeight.rows: whole tiles of 16 rows")
        w = PackedWeight.__new__(PackedWeight)
        w.N, w.K, w.data = n, self.K, self.data[n0 * self.K: (n0 + -(-n // 16) * 16) * self.K]
        return w

    def unpack(self) -> torch.Tensor:
        """Back to row-major [N, K] (index arithmetic on the device tensor)."""
        nt = (self.N + 15) // 16
        v = self.data[: nt * 16 * self.K].view(nt, self.K // 32, 4, 16, 8)
        return v.permute(0, 3, 1, 2, 4).reshape(nt * 16, self.K)[: self.N].contiguous()


class QuantWeight:
    """A [N, K] weight scale * (q - zero) of 4-bit q, one fp16 scale and one 4-bit zero per `group` (32, 64 or 128) neighbours along K, in
    the layout of mlora_linear4."""

    dtype = torch.float16

    def __init__(self, q, scale, zero):
        """q [N, K] and zero [N, K / group] uint8 of 0 .. 15, scale [N, K / group] fp16."""
        N, K = q.shape
        n, G = scale.shape
        if n != N or zero.shape != scale.shape or G == 0 or K % G or K // G not in (32, 64, 128):
            raise ValueError(f"QuantWeight: q{tuple(q.shape)} scale{tuple(scale.shape)} zero{tuple(zero.shape)}: one scale and zero per 32, 64 or 128 columns")
        if q.dtype != torch.uint8 or zero.dtype != torch.uint8 or scale.dtype != torch.float16:
            raise TypeError("QuantWeight: q and zero are uint8, scale is float16")
        _here(q.device, "QuantWeight")
        if q.device != scale.device or q.device != zero.device:
            raise ValueError("QuantWeight: q, scale and zero on one device")
        if N and bool((q.amax() > 15) | (zero.amax() > 15)):
            raise ValueError("QuantWeight: q and zero of 4 bits")
        self.N, self.K, self.group = N, K, K // G
        tiles, blocks, gb = -(-N // 16), -(-K // 128), 128 // self.group
        if (tiles * 16, blocks * 128) != (N, K):
            q, full = torch.zeros((tiles * 16, blocks * 128), dtype=torch.uint8, device=q.device), q
            q[:N, :K] = full
            scale, zero = (torch.nn.functional.pad(t, (0, blocks * gb - G, 0, tiles * 16 - N)) for t in (scale, zero))
        # [tile][row][block][step][kg][p][2] -> [tile][block][kg][row][step] words of nibbles (p, 4 + p)
        v = q.view(tiles, 16, blocks, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
        low, high = ((v[..., h].contiguous().view(-1, 4) << torch.tensor([0, 4, 0, 4], device=q.device, dtype=torch.uint8)) for h in (0, 1))
        self.q = torch.stack([low[:, 0] | low[:, 1], low[:, 2] | low[:, 3], high[:, 0] | high[:, 1], high[:, 2] | high[:, 3]], 1).reshape(-1)
        scale, zero = (t.reshape(tiles, 16, blocks, gb).permute(0, 2, 1, 3).reshape(tiles, blocks, 16 * gb) for t in (scale, zero))
        self.meta = torch.cat([scale.contiguous().view(torch.uint8), zero], 2).reshape(-1)

    @property
    def shape(self):
        return (self.N, self.K)

    @property
    def device(self):
        return self.q.device

    def dequantize(self) -> torch.Tensor:
        """The weight [N, K] in fp32 (for inspection)."""
        tiles, blocks = -(-self.N // 16), -(-self.K // 128)
        b = self.q.view(-1, 4)
        nib = torch.stack([torch.stack([b[:, h * 2 + p // 2] >> (4 * (p % 2)) & 15 for h in (0, 1)], 1) for p in range(4)], 1)       # [words][p][2]
        q = nib.view(tiles, blocks, 4, 16, 4, 4, 2).permute(0, 3, 1, 4, 2, 5, 6).reshape(tiles * 16, blocks, 128 // self.group, self.group)
        meta = self.meta.view(tiles, blocks, -1)
        cut = meta.shape[2] // 3 * 2
        s, z = (t.reshape(tiles, blocks, 16, -1).permute(0, 2, 1, 3).reshape(tiles * 16, blocks, -1, 1).float()
                for t in (meta[:, :, :cut].contiguous().view(torch.float16), meta[:, :, cut:]))
        return ((q.float() - z) * s).reshape(tiles * 16, blocks * 128)[: self.N, : self.K].contiguous()


def quantize(W: torch.Tensor, group: int = 128) -> QuantWeight:
    """W [N, K] rounded to 4 bits: per group the 16 steps between its least and its greatest value, 0 among them."""
    N, K = W.shape
    if K % group or group not in (32, 64, 128):
        raise ValueError(f"quantize: groups of {group} for K={K}")
    w = W.float().view(N, K // group, group)
    lo, hi = w.amin(2).clamp_max(0.0), w.amax(2).clamp_min(0.0)
    scale = ((hi - lo) / 15).clamp_min(2.0 ** -24).to(torch.float16)
    s = scale.float()
    zero = (-lo / s).round().clamp_(0, 15)
    q = ((w / s[:, :, None]).round() + zero[:, :, None]).clamp_(0, 15)
    return QuantWeight(q.view(N, K).to(torch.uint8), scale, zero.to(torch.uint8))


def _linear4(x, W, out, out_dtype, accumulate):
    T, K = x.shape
    N, dev = W.N, W.q.device
    if W.K != K or x.dtype != torch.float16 or x.device != dev:
        raise ValueError(f"linear: x{tuple(x.shape)} {x.dtype} on {x.device} vs a 4-bit weight {W.shape} on {dev} (fp16 activations)")
    _here(dev, "linear")
    if out is None:
        if accumulate:
            raise ValueError("linear: accumulate needs out")
    elif out.shape != (T, N) or out.device != dev:
        raise ValueError(f"linear: out{tuple(out.shape)} on {out.device}, expected {(T, N)} on {dev}")
    else:
        out_dtype = out.dtype
    if out_dtype is not torch.float16 and out_dtype is not torch.float32:
        raise TypeError(f"linear: a 4-bit weight gives float16 or float32, not {out_dtype}")
    if out is None:
        out = _empty_strided_cuda((T, N), (N, 1), out_dtype)
    if T == 0:
        return out
    if isinstance(x, FragActivation):
        xp, lay, ldx = x.data.data_ptr(), FRAG, 0
    else:
        ldx, inner = x.stride()
        xp, lay = x.data_ptr(), ROWMAJOR
        if T == 1:
            ldx = K
        if inner != 1 or ldx < K or ldx % 8 or xp % 16:
            x = x.clone(memory_format=torch.contiguous_format)            # rows on 16 bytes
            xp, ldx = x.data_ptr(), K
    nb = _size(torch.float16, "mlora_linear4_workspace_bytes_of", T, K, N, lay)
    ws = _empty_strided_cuda((nb // 4,), (1,), torch.float32) if nb else None
    code = lib().mlora_linear4(_dev(out, name="out"), F16 if out_dtype is torch.float16 else F32, ACCUMULATE if accumulate else STORE, xp, lay, ldx, W.q.data_ptr(),
                               W.meta.data_ptr(), W.group, T, K, N, None if ws is None else ws.data_ptr(), nb, _stream())
    if code:
        check(code)
    return out


def linear(x, W, out=None, out_dtype=None, accumulate=False, kernel="auto"):
    """y (=|+=) x @ W.T.  x [T,K] (row stride may exceed K) or a FragActivation, W [N,K] of the same type or a
    PackedWeight, or a QuantWeight (f16 x); f16, bf16 (fragment order or packed) or f32 (plain); y has their type unless out_dtype says f32.  accumulate=True adds into the fp32 tensor `out`.  kernel: "auto" | "gemv" | "gemm"."""
    out_dtype = out_dtype or W.dtype
    if isinstance(W, QuantWeight):
        if kernel != "auto":
            raise ValueError(f"linear: a 4-bit weight has one kernel family, not {kernel!r}")
        return _linear4(x, W, out, out_dtype, accumulate)
    if isinstance(x, FragActivation):
        return _linear_frag(x, W, out, out_dtype, accumulate)
    T, K = x.shape
    packed = isinstance(W, PackedWeight)
    N, K2 = W.shape
    if K2 != K:
        raise ValueError(f"linear: x{tuple(x.shape)} vs W{tuple(W.shape)}")
    if T == 0:                                     # an empty batch
        if out is None:
            out = torch.empty((0, N), dtype=torch.float32 if accumulate else out_dtype, device=x.device)
        return out
    if not x.is_cuda or x.dtype != W.dtype or x.stride(1) != 1:
        raise ValueError("linear: x must be a GPU tensor of the weight's type with unit inner stride")
    ldx = x.stride(0) if T > 1 else max(K, x.stride(0))
    if out is None:
        if accumulate:
            raise ValueError("linear: accumulate needs out")
        out = torch.empty((T, N), dtype=out_dtype, device=x.device)
    if out.shape != (T, N):
        raise ValueError(f"linear: out{tuple(out.shape)} expected {(T, N)}")
    if packed:
        fn = getattr(lib_of(W.dtype), {"auto": "mlora_linear_packed", "gemv": "mlora_gemv_packed", "gemm": "mlora_gemm_packed"}[kernel])
        wptr = W.data.data_ptr()
    else:
        fn = getattr(lib_of(W.dtype), {"auto": "mlora_linear", "gemv": "mlora_gemv", "gemm": "mlora_gemm"}[kernel])
        wptr = _dev(W, name="W")
    check(fn(_dev(out), _dt(out), ACCUMULATE if accumulate else STORE, x.data_ptr(), ldx, wptr, T, K, N, _stream()), W.dtype)
    return out


def _linear_frag(x, W, out, out_dtype, accumulate):
    if not isinstance(W, PackedWeight) or W.dtype != x.dtype:
        raise TypeError("a fragment-ordered activation needs a PackedWeight of its type")
    T, K = x.shape
    N, K2 = W.shape
    if K2 != K:
        raise ValueError(f"linear: x{x.shape} vs W{W.shape}")
    if out is None:
        if accumulate:
            raise ValueError("linear: accumulate needs out")
        out = torch.empty((T, N), dtype=out_dtype, device=x.device)
    if out.shape != (T, N):
        raise ValueError(f"linear: out{tuple(out.shape)} expected {(T, N)}")
    check(lib_of(W.dtype).mlora_linear_frag(_dev(out), _dt(out), ACCUMULATE if accumulate else STORE, x.data.data_ptr(),
                                            W.data.data_ptr(), T, K, N, _stream()), W.dtype)
    return out


def gemm_frag_preferred(T: int, K: int, N: int) -> bool:
    """Whether a [T, K] x [N, K]^T product of this size runs best with its activations in fragment order."""
    return bool(_size(torch.float16, "mlora_gemm_frag_preferred", T, K, N))


def lora_block_adapters(tok_adapter: torch.Tensor, n_ad: int):
    """ids [T] int32 -> (blk_adapter [ceil(T / 256)]: the adapter a 256-token block agrees on or -1,
    tok_rest [T]: -1 where the block's delta can ride in the GEMM, else the token's id)."""
    T = tok_adapter.shape[0]
    blk = torch.empty((max(-(-T // 256), 1),), dtype=torch.int32, device=tok_adapter.device)
    rest = torch.empty((max(T, 1),), dtype=torch.int32, device=tok_adapter.device)[:T]
    check(lib().mlora_lora_block_adapters(blk.data_ptr(), rest.data_ptr(), _dev(tok_adapter, torch.int32), T, n_ad, _stream()))
    return blk, rest


def lora_shrink_split(x, A_list, tok_adapter, scaling: float, workspace, out=None):
    """The matrix-core shrink of up to three projections that read x (A [n_ad, r, K] each), as fp16 hi + lo halves:
    -> [(v_hi [T, r], v_lo [T, r]), ...]."""
    import ctypes as C
    xp, lay, T, K = _x_arg(x)
    n_ad, r, _ = A_list[0].shape
    dev = tok_adapter.device
    if out is None:
        out = [(torch.empty((T, r), dtype=torch.float16, device=dev), torch.empty((T, r), dtype=torch.float16, device=dev)) for _ in A_list]
    n = len(A_list)
    hi = (C.c_void_p * n)(*[o[0].data_ptr() for o in out])
    lo = (C.c_void_p * n)(*[o[1].data_ptr() for o in out])
    Ap = (C.c_void_p * n)(*[_dev(a, torch.float16, "A") for a in A_list])
    check(lib().mlora_lora_shrink_split(C.cast(hi, C.c_void_p), C.cast(lo, C.c_void_p), xp, lay, C.cast(Ap, C.c_void_p), n,
                                        _dev(tok_adapter, torch.int32), float(scaling), T, K, r, n_ad, _dev(workspace, torch.float32),
                                        workspace.numel() * 4, _stream()))
    return out


def linear_frag_lora(x: FragActivation, W: PackedWeight, projs, blk_adapter, r: int, out=None, out_dtype=torch.float16, accumulate=False):
    """`linear(x, W)` with the LoRA deltas of `projs` = [(B [n_ad, rows, r], v_hi, v_lo, first row, rows), ...] carried as
    extra k-steps of the GEMM for the token blocks that `blk_adapter` gives an adapter (shapes of the persistent GEMM)."""
    import ctypes as C
    from ._lib import FusedLora
    T, K = x.shape
    N, K2 = W.shape
    if K2 != K:
        raise ValueError(f"linear_frag_lora: x{x.shape} vs W{W.shape}")
    if out is None:
        if accumulate:
            raise ValueError("linear_frag_lora: accumulate needs out")
        out = torch.empty((T, N), dtype=out_dtype, device=x.device)
    if out.shape != (T, N):
        raise ValueError(f"linear_frag_lora: out{tuple(out.shape)} expected {(T, N)}")
    arr = (FusedLora * len(projs))()
    for e, (B, vh, vl, n0, rows) in zip(arr, projs):
        if B.shape[1] != rows or B.shape[2] != r or vh.shape != (T, r) or vl.shape != (T, r):
            raise ValueError("linear_frag_lora: table or v shape")
        e.B, e.v_hi, e.v_lo, e.n_begin, e.n_rows = _dev(B, torch.float16, "B"), _dev(vh, torch.float16, "v_hi"), _dev(vl, torch.float16, "v_lo"), n0, rows
    check(lib().mlora_linear_frag_lora(_dev(out), _dt(out), ACCUMULATE if accumulate else STORE, x.data.data_ptr(), W.data.data_ptr(),
                                       T, K, N, C.cast(arr, C.c_void_p), len(projs), _dev(blk_adapter, torch.int32), r, _stream()))
    return out


def linear_frag_deltas_pay(T: int, K: int, N: int, accumulate: bool, r: int, n_distinct: int) -> bool:
    """Whether `linear_frag_deltas` serves a shape and is the faster form for tokens that name n_distinct adapters."""
    return bool(lib().mlora_linear_frag_deltas_pay(T, K, N, int(accumulate), r, n_distinct))


def _delta_args(who, x, W, projs, tok_adapter, workspace):
    import ctypes as C
    from ._lib import LoraBucket
    T, K = x.shape
    N, K2 = W.shape
    n_ad, r, _ = projs[0][0].shape
    n = len(projs)
    b, c, nc = (LoraBucket * n)(), (C.c_int32 * n)(), (C.c_int32 * n)()
    if K2 != K or tok_adapter.shape != (T,):
        raise ValueError(f"{who}: x{x.shape} vs W{W.shape}, {tuple(tok_adapter.shape)} token ids")
    for i, (A, B, scaling, n0, rows) in enumerate(projs):
        if A.shape != (n_ad, r, K) or B.shape != (n_ad, rows, r):
            raise ValueError(f"{who}: A{tuple(A.shape)} B{tuple(B.shape)} for {rows} rows of K={K}")
        b[i].A, b[i].B, b[i].r, b[i].n_ad, b[i].scaling, c[i], nc[i] = _dev(A, torch.float16, "A"), _dev(B, torch.float16, "B"), r, n_ad, float(scaling), n0, rows
    return (C.cast(b, C.c_void_p), n, C.cast(c, C.c_void_p), C.cast(nc, C.c_void_p), _dev(tok_adapter, torch.int32), _dev(workspace, torch.float32),
            workspace.numel() * 4, _stream())


def linear_frag_deltas(x: FragActivation, W: PackedWeight, projs, tok_adapter, workspace, out=None, out_dtype=torch.float16, accumulate=False, ks_ws=None):
    """`linear(x, W)` with the LoRA deltas of `projs` = [(A [n_ad, r, K], B [n_ad, rows, r], scaling, first row, rows), ...] of tokens that name any
    adapters, inside the GEMM (up to 64 tokens, and shapes of the mid-size kernel).  accumulate: into `out`; with fp32 scratch `ks_ws` K may be split as in
    `linear_acc_ksplit`.  Returns (out, KSplitParts or None)."""
    T, K = x.shape
    N = W.shape[0]
    if out is None and not accumulate:
        out = torch.empty((T, N), dtype=out_dtype, device=x.device)
    if out is None or out.shape != (T, N):
        raise ValueError(f"linear_frag_deltas: out for {(T, N)}")
    args = _delta_args("linear_frag_deltas", x, W, projs, tok_adapter, workspace)
    ks = _size(W.dtype, "mlora_gemv_ksplit", T, K, N) if ks_ws is not None else 1
    if ks > 1 and ks_ws.numel() * 4 < _size(W.dtype, "mlora_gemv_ksplit_bytes", T, N, ks):
        ks = 1
    check(lib().mlora_linear_frag_deltas(_dev(out), _dt(out), ACCUMULATE if accumulate else STORE, _dev(ks_ws, torch.float32) if ks > 1 else None, ks,
                                         x.data.data_ptr(), W.data.data_ptr(), T, K, N, *args))
    return out, KSplitParts(ks_ws, ks, N) if ks > 1 else None


def linear_frag_silu_deltas(x: FragActivation, W: PackedWeight, projs, tok_adapter, workspace) -> FragActivation:
    """silu(gate) * up of the fused gate/up projection with the deltas of gate and / or up rows, as `linear_frag_deltas`; in fragment order."""
    T, K = x.shape
    N = W.shape[0]
    if N % 2:
        raise ValueError(f"linear_frag_silu_deltas: W{W.shape}")
    args = _delta_args("linear_frag_silu_deltas", x, W, projs, tok_adapter, workspace)
    out = FragActivation(T, N // 2, x.device)
    check(lib().mlora_linear_frag_silu_deltas(out.data.data_ptr(), x.data.data_ptr(), W.data.data_ptr(), T, K, N // 2, *args))
    return out


def linear_frag_silu(x: FragActivation, W: PackedWeight, projs=(), blk_adapter=None, r: int = 0, out: FragActivation = None) -> FragActivation:
    """silu(gate) * up of the fused gate/up projection `W` [2I, K] in the epilogue of the persistent GEMM, in fragment
    order.  `projs` as for linear_frag_lora, over the gate rows (first row 0) and / or the up rows (first row I); every
    256-token block must agree on one adapter (lora_block_adapters leaves no rest)."""
    import ctypes as C
    from ._lib import FusedLora
    T, K = x.shape
    N, K2 = W.shape
    I = N // 2
    if K2 != K or N % 2:
        raise ValueError(f"linear_frag_silu: x{x.shape} vs W{W.shape}")
    if out is None:
        out = FragActivation(T, I, x.device)
    if out.shape != (T, I):
        raise ValueError(f"linear_frag_silu: out{tuple(out.shape)} expected {(T, I)}")
    arr = (FusedLora * max(len(projs), 1))()
    for e, (B, vh, vl, n0, rows) in zip(arr, projs):
        if B.shape[1] != rows or B.shape[2] != r or vh.shape != (T, r) or vl.shape != (T, r):
            raise ValueError("linear_frag_silu: table or v shape")
        e.B, e.v_hi, e.v_lo, e.n_begin, e.n_rows = _dev(B, torch.float16, "B"), _dev(vh, torch.float16, "v_hi"), _dev(vl, torch.float16, "v_lo"), n0, rows
    check(lib().mlora_linear_frag_silu(out.data.data_ptr(), x.data.data_ptr(), W.data.data_ptr(), T, K, I,
                                       C.cast(arr, C.c_void_p) if projs else None, len(projs),
                                       _dev(blk_adapter, torch.int32) if projs else None, r, _stream()))
    return out


def linear_frag_glu(x: FragActivation, W: PackedWeight) -> FragActivation:
    """silu(gate) * up of the fused gate/up projection `W` [2I, K] for more than 64 tokens, in fragment order: the product leaves whichever
    kernel `linear(x, W)` takes (same bits as that and `silu_mul`)."""
    T, K = x.shape
    N, K2 = W.shape
    if K2 != K or N % 2:
        raise ValueError(f"linear_frag_glu: x{x.shape} vs W{W.shape}")
    out = FragActivation(T, N // 2, x.device, dtype=x.dtype)
    check(lib_of(W.dtype).mlora_linear_frag_glu(out.data.data_ptr(), x.data.data_ptr(), W.data.data_ptr(), T, K, N // 2, GLU_SILU, 0.0, 0.0, 0.0, _stream()),
          W.dtype)
    return out


def interleave_gate_up(gate_up: torch.Tensor) -> PackedWeight:
    """[2I, K] (gate rows, then up rows) -> PackedWeight whose 16-row tiles alternate gate and up."""
    I2, K = gate_up.shape
    I = I2 // 2
    if I % 16:
        raise ValueError("interleave_gate_up: intermediate size must be a multiple of 16")
    return PackedWeight(gate_up.view(2, I // 16, 16, K).permute(1, 0, 2, 3).reshape(I2, K).contiguous())


def gate_up_silu(x: FragActivation, W_il: PackedWeight, out: FragActivation = None) -> FragActivation:
    """silu(x @ Wgate.T) * (x @ Wup.T) in one launch; W_il from interleave_gate_up.  T <= 64."""
    T, K = x.shape
    I2, K2 = W_il.shape
    if K2 != K:
        raise ValueError(f"gate_up_silu: x{x.shape} vs W{W_il.shape}")
    out = FragActivation(T, I2 // 2, x.device) if out is None else out
    check(lib().mlora_gemv_frag_silu(out.data.data_ptr(), x.data.data_ptr(), W_il.data.data_ptr(), T, K, I2 // 2, _stream()))
    return out


def _out_arg(out, T, H, frag, device):
    """Output buffer of a producer: row-major tensor or FragActivation."""
    if frag:
        out = FragActivation(T, H, device) if out is None else out
        return out, out.data.data_ptr(), FRAG
    if out is None:
        out = torch.empty((T, H), dtype=torch.float16, device=device)
    return out, _dev(out, torch.float16, "out"), ROWMAJOR


class KSplitParts:
    """Partial results of a K-split accumulating GEMV (slices 1..ks-1), to be added by the next RMSNorm of the row."""

    def __init__(self, part: torch.Tensor, ks: int, ld: int):
        self.part, self.ks, self.ld = part, ks, ld


def linear_acc_ksplit(x: FragActivation, W: PackedWeight, resid: torch.Tensor, ws: torch.Tensor = None, riding_rows: int = 0):
    """resid [T, N] fp32 += x @ W.T as `linear(..., accumulate=True)`, with K split over several workgroups when the
    library recommends it for this shape and `ws` (fp32 scratch) is large enough: slice 0 lands in resid, the other
    slices in the returned KSplitParts, which the caller hands to the next `rmsnorm(resid, ..., parts=...)`.
    Returns None when the GEMV ran unsplit.  riding_rows: what the native decode step's launch of this linear carries
    besides the weight rows (`mlora_gemv_shrink_rows` for the shrink units of an adapted projection) - the slice count
    follows the same rule here, so that both paths add the same partial sums."""
    T, K = x.shape
    N, K2 = W.shape
    if K2 != K or resid.shape != (T, N) or resid.dtype != torch.float32:
        raise ValueError(f"linear_acc_ksplit: x{x.shape} W{W.shape} resid{tuple(resid.shape)}")
    L = lib_of(W.dtype)
    ks = _size(W.dtype, "mlora_gemv_ksplit", T, K, N + riding_rows) if ws is not None else 1
    if ks > 1 and ws.numel() * 4 < _size(W.dtype, "mlora_gemv_ksplit_bytes", T, N, ks):
        ks = 1
    check(L.mlora_gemv_frag_acc_ksplit(_dev(resid, torch.float32), None, _dev(ws, torch.float32) if ks > 1 else None, ks,
                                       x.data.data_ptr(), W.data.data_ptr(), T, K, N, 0, None, None, 0, None, 0, 0, _stream()), W.dtype)
    return KSplitParts(ws, ks, N) if ks > 1 else None


def linear_acc_ksplit_delta(x: FragActivation, W: PackedWeight, resid: torch.Tensor, ws: torch.Tensor, vpart, B, tok_adapter, scaling: float):
    """resid [T, N] fp32 += x @ W.T over K slices, with the LoRA expand scaling * B[id] @ sum_h vpart[h, t] of every token
    done by workgroups riding in the same launch (vpart [n_shares, T, r] fp32: the shrink results as shares that are
    added in order): returns the KSplitParts (slice partials, then the delta rows) that the next
    `rmsnorm(resid, ..., parts=...)` adds - or None when the library does not serve the shape this way (nothing is
    launched then)."""
    T, K = x.shape
    N, K2 = W.shape
    n_ad, N2, r = B.shape
    if K2 != K or N2 != N or vpart.dim() != 3 or tuple(vpart.shape[1:]) != (T, r) or resid.shape != (T, N) or resid.dtype != torch.float32:
        raise ValueError(f"linear_acc_ksplit_delta: x{x.shape} W{W.shape} vpart{tuple(vpart.shape)} B{tuple(B.shape)} resid{tuple(resid.shape)}")
    ks = lib().mlora_gemv_delta_ride_ksplit(T, K, N, r)
    if ks <= 0:
        return None
    if ws.numel() * 4 < lib().mlora_gemv_ksplit_bytes(T, N, ks + 1):
        raise ValueError("linear_acc_ksplit_delta: workspace too small")
    check(lib().mlora_gemv_frag_acc_ksplit_delta(_dev(resid, torch.float32), _dev(ws, torch.float32), ks, x.data.data_ptr(), W.data.data_ptr(),
                                                 T, K, N, _dev(vpart, torch.float32), vpart.shape[0], _dev(B, torch.float16, "B"),
                                                 _dev(tok_adapter, torch.int32), float(scaling), r, n_ad, _stream()))
    return KSplitParts(ws, ks + 1, N)


def rmsnorm(x, w, eps: float, out=None, frag=False, parts: KSplitParts = None):
    """Row-wise RMSNorm of x [T, H] (f16 | f32); frag=True writes a FragActivation.  With `parts` (x fp32) the K-split
    partials are first added to x in place."""
    T, H = x.shape
    if T == 0 and not frag:
        return torch.empty((0, H), dtype=torch.float16, device=x.device) if out is None else out
    out, optr, lay = _out_arg(out, T, H, frag, x.device)
    if parts is not None:
        check(lib().mlora_rmsnorm_ksplit(optr, lay, _dev(x, torch.float32), _dev(parts.part, torch.float32), parts.ks, parts.ld,
                                         _dev(w, torch.float16), float(eps), T, H, None, 0, None, None, 0.0, 0, 0, 0, _stream()))
        return out
    check(lib().mlora_rmsnorm(optr, lay, _dev(x), _dt(x), _dev(w, torch.float16), float(eps), T, H, _stream()))
    return out


def silu_mul(gate_up, out=None, frag=False):
    """gate_up [T, 2I] (gate columns first) -> silu(gate) * up [T, I]."""
    T, I2 = gate_up.shape
    I = I2 // 2
    if T == 0 and not frag:
        return torch.empty((0, I), dtype=torch.float16, device=gate_up.device) if out is None else out
    out, optr, lay = _out_arg(out, T, I, frag, gate_up.device)
    p = _dev(gate_up, torch.float16)
    check(lib().mlora_silu_mul(optr, lay, p, p + I * 2, I2, T, I, _stream()))
    return out


def silu_mul_split(gate, up, out=None):
    T, I = gate.shape
    if out is None:
        out = torch.empty((T, I), dtype=torch.float16, device=gate.device)
    check(lib().mlora_silu_mul(_dev(out, torch.float16), ROWMAJOR, _dev(gate, torch.float16), _dev(up, torch.float16), I, T, I, _stream()))
    return out


def embed(table, ids, out_dtype=torch.float32, out=None):
    T = ids.numel()
    V, H = table.shape
    if out is None:
        out = torch.empty((T, H), dtype=out_dtype, device=table.device)
    if T == 0:
        return out
    check(lib_of(table.dtype).mlora_embed(_dev(out), _dt(out), _dev(table), _dev(ids, torch.int32), T, H, V, _stream()), table.dtype)
    return out


def argmax(logits, out=None):
    B, V = logits.shape
    if out is None:
        out = torch.empty((B,), dtype=torch.int32, device=logits.device)
    if B == 0:
        return out
    check(_lib.loaded().mlora_argmax(_dev(out, torch.int32), _dev(logits, torch.float32), B, V, _stream()))
    return out


class LogitRules:
    """What the rows of a batch may answer with, for `constrained_argmax` (formulas at mlora_constrained_argmax in include/mlora.h).
    history [B, cap] int32: a row's prompt and generated tokens, lengths [B] of them, from gen_start [B] on the generated ones;
    repetition, presence, frequency [B] fp32; bias_ids [B, n] int32 (outside the vocabulary: none) and bias [B, n] fp32; masks
    [m, ceil(V / 32)] int32, bit v % 32 of word v / 32 for token v, and mask_row [B] int32 (outside 0..m-1: no mask).  append: a
    chosen token goes behind its row's history.  The tensors are the caller's, contiguous and on one device; what a call reads
    of them is what they hold when it runs."""

    def __init__(self, history=None, lengths=None, gen_start=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
                 masks=None, mask_row=None, append=False):
        i32, f32 = torch.int32, torch.float32
        given = {"history": (history, i32, 2), "lengths": (lengths, i32, 1), "gen_start": (gen_start, i32, 1), "repetition": (repetition, f32, 1),
                 "presence": (presence, f32, 1), "frequency": (frequency, f32, 1), "bias_ids": (bias_ids, i32, 2), "bias": (bias, f32, 2),
                 "masks": (masks, i32, 2), "mask_row": (mask_row, i32, 1)}
        given = {n: g for n, g in given.items() if g[0] is not None}
        self.rows, self.device = None, None
        self._args = _lib.LogitRulesArgs(append=int(bool(append)))
        for n, (t, dt, dims) in given.items():
            if t.dim() != dims:
                raise ValueError(f"LogitRules: {n}{tuple(t.shape)} needs {dims} dimensions")
            if n != "masks":
                if self.rows not in (None, t.shape[0]):
                    raise ValueError(f"LogitRules: {n} has {t.shape[0]} rows, others {self.rows}")
                self.rows = t.shape[0]
            if self.device not in (None, t.device):
                raise ValueError(f"LogitRules: {n} lies on {t.device}, others on {self.device}")
            self.device = t.device
            p = _dev(t, dt, n)
            setattr(self, n, t)
            setattr(self._args, n, p if t.numel() else None)
        for a, b in (("history", "lengths"), ("bias_ids", "bias"), ("masks", "mask_row")):
            if (a in given) != (b in given):
                raise ValueError(f"LogitRules: {a} and {b} come together")
        if "history" not in given and (append or any(n in given for n in ("gen_start", "repetition", "presence", "frequency"))):
            raise ValueError("LogitRules: penalties and append need a history")
        if "bias" in given:
            if bias.shape != bias_ids.shape:
                raise ValueError(f"LogitRules: bias{tuple(bias.shape)} for bias_ids{tuple(bias_ids.shape)}")
            self._args.n_bias = bias.shape[1] if bias.numel() else 0
        if "masks" in given:
            self._args.n_masks = masks.shape[0] if masks.numel() else 0
        if "history" in given:
            self._args.cap = history.shape[1]
            if not history.numel() and self.rows:
                raise ValueError("LogitRules: a history without room")
        self._words, self._ref = masks.shape[1] if self._args.n_masks else 0, ctypes.byref(self._args)


def constrained_argmax(logits, rules: LogitRules, out=None, ids=None):
    """The greedy token [B] int32 of logits [B, V] fp32 (any row stride) under `rules`, -1 for a row that has none left; out [B, V]
    fp32 (or None; may be `logits`) takes the logits after penalties, biases and masks."""
    B, V = logits.shape
    dev = _here(logits.device, "constrained_argmax")
    if rules.device is not None and (rules.rows != B and rules.rows is not None or rules.device != dev):
        raise ValueError(f"constrained_argmax: rules of {rules.rows} rows on {rules.device} for {B} on {dev}")
    if rules._words and rules._words != -(-V // 32):
        raise ValueError(f"constrained_argmax: masks of {rules._words} words for {V} tokens")
    ld, ld_out, p, p_out = _rows_of(logits, B, V, dev, "logits"), 0, logits.data_ptr(), None
    if out is not None:
        ld_out, p_out = _rows_of(out, B, V, dev, "out"), out.data_ptr()
        if p != p_out or ld != ld_out:
            apart = 4 * (B - 1)
            if p < p_out + apart * ld_out + 4 * V and p_out < p + apart * ld + 4 * V:
                raise ValueError("constrained_argmax: out overlaps the logits without being them")
    if ids is None:
        ids = _empty_strided_cuda((B,), (1,), torch.int32)
        p_ids = ids.data_ptr()
    elif ids.shape != (B,) or ids.device != dev:
        raise ValueError(f"constrained_argmax: ids{tuple(ids.shape)} on {ids.device} for {B} rows on {dev}")
    else:
        p_ids = _dev(ids, torch.int32, "ids")
    if B == 0:
        return ids
    L = _lib.loaded()
    nb = _rules_bytes(B, V)
    ws = _empty_strided_cuda((nb // 8,), (1,), torch.int64) if nb else None
    code = L.mlora_constrained_argmax(p_ids, p_out, ld_out, p, ld, rules._ref, B, V, None if ws is None else ws.data_ptr(), nb, _stream())
    if code:
        raise _lib.MloraError(code, L.mlora_last_error().decode())
    return ids


@functools.lru_cache(maxsize=256)
def _rules_bytes(B, V):
    return _lib.loaded().mlora_constrained_argmax_workspace_bytes(B, V)


def _rows_of(t, B, V, dev, name):
    """Row stride of fp32 rows [B, V] with unit inner stride."""
    ld, inner = t.stride()
    if t.dtype != torch.float32 or t.shape != (B, V) or (inner != 1 and V > 1) or (ld < V and B > 1) or t.device != dev:
        raise ValueError(f"constrained_argmax: {name} must be fp32 [{B}, {V}] on {dev} with unit inner stride")
    return ld if B > 1 else V if ld < V else ld


def rope_kv_append(qkv, k_cache, v_cache, block_table, tok_seq, tok_pos, rope_cos, rope_sin, Hq, Hkv, D):
    """qkv [T, Hq+2Hkv, D] f16 (q rotated in place); k_cache [n_pages,Hkv,D/32,4,16,8] (fragment order),
    v_cache [n_pages,Hkv,D,16]."""
    T = qkv.shape[0]
    n_pages = k_cache.shape[0]
    n_seq, max_blocks = block_table.shape
    max_pos = rope_cos.shape[0]
    check(lib().mlora_rope_kv_append(_dev(qkv, torch.float16), _dev(k_cache, torch.float16), _dev(v_cache, torch.float16),
                                     _dev(block_table, torch.int32), max_blocks, _dev(tok_seq, torch.int32),
                                     _dev(tok_pos, torch.int32), _dev(rope_cos, torch.float32), _dev(rope_sin, torch.float32),
                                     max_pos, T, Hq, Hkv, D, n_pages, n_seq, _stream()))


def o_shrink_served(B: int, Hq: int, Hkv: int, D: int, N: int, r: int) -> bool:
    """Whether a decode step of B sequences can take the o projection's adapter delta as head shares off the attention
    launch plus a launch of expand workgroups (the rule the native step applies for more than 64 sequences)."""
    return bool(lib().mlora_rope_attn_oshrink_ok(B, Hq, Hkv, D, r)) and bool(lib().mlora_lora_expand_shares_ok(N, r))


def lora_expand_shares(y, vpart, B, tok_adapter, scaling: float):
    """y [T, N] fp32 += scaling * B[id] @ sum_h vpart[h, t] for the tokens that name an adapter (vpart [shares, T, r] fp32)."""
    T, N = y.shape
    n_ad, N2, r = B.shape
    if N2 != N or y.dtype != torch.float32 or vpart.dim() != 3 or tuple(vpart.shape[1:]) != (T, r):
        raise ValueError(f"lora_expand_shares: y{tuple(y.shape)} vpart{tuple(vpart.shape)} B{tuple(B.shape)}")
    check(lib().mlora_lora_expand_shares(_dev(y, torch.float32), _dev(vpart, torch.float32), vpart.shape[0], _dev(B, torch.float16, "B"),
                                         _dev(tok_adapter, torch.int32), float(scaling), T, N, r, n_ad, _stream()))
    return y


def paged_attn_decode(qkv, k_cache, v_cache, block_table, seq_ids, ctx_len, Hq, Hkv, D, out=None, frag=False, o_shrink=None):
    """o_shrink = (A [n_ad, r, Hq * D] f16, tok_adapter [B] int32): the launch also writes the o projection's shrink as one
    share per query head and the call returns (out, vpart [Hq, B, r] fp32; rows of tokens without adapter are not written)."""
    B = qkv.shape[0]
    n_seq, max_blocks = block_table.shape
    out, optr, lay = _out_arg(out, B, Hq * D, frag, qkv.device)
    if o_shrink is not None:
        A, ids = o_shrink
        n_ad, r, Kq = A.shape
        if Kq != Hq * D or not lib().mlora_rope_attn_oshrink_ok(B, Hq, Hkv, D, r):
            raise ValueError(f"paged_attn_decode: o shrink A{tuple(A.shape)} not served for B={B} Hq={Hq} Hkv={Hkv} D={D}")
        vpart = torch.empty((Hq, B, r), dtype=torch.float32, device=qkv.device)
        check(lib().mlora_paged_attn_decode_oshrink(optr, lay, _dev(qkv, torch.float16), _dev(k_cache, torch.float16),
                                                    _dev(v_cache, torch.float16), _dev(block_table, torch.int32), max_blocks,
                                                    _dev(seq_ids, torch.int32), _dev(ctx_len, torch.int32), B, Hq, Hkv, D,
                                                    k_cache.shape[0], n_seq, _dev(ids, torch.int32), r, n_ad,
                                                    _dev(A, torch.float16, "A"), vpart.data_ptr(), _stream()))
        return out, vpart
    check(lib().mlora_paged_attn_decode(optr, lay, _dev(qkv, torch.float16), _dev(k_cache, torch.float16),
                                        _dev(v_cache, torch.float16), _dev(block_table, torch.int32), max_blocks,
                                        _dev(seq_ids, torch.int32), _dev(ctx_len, torch.int32), B, Hq, Hkv, D,
                                        k_cache.shape[0], n_seq, _stream()))
    return out


class SharedPrefixPlan:
    """Which rows of a decode batch share their first pages, for `paged_attn_decode_shared`: made once for a batch, good for all its
    layers and steps while its rows stay.  groups: (rows, pages) - batch rows whose block tables begin with the same `pages` pages, all
    within their contexts; a row is in one group at most.  lens: the rows' context lengths now, which choose how the work is cut: a plan
    that its rows have `outgrown` still gives their results, but slowly."""

    def __init__(self, groups, lens, Hq, Hkv, D, device):
        B, G = len(lens), Hq // Hkv
        if Hq % Hkv or not 1 <= G <= 16:
            raise ValueError(f"SharedPrefixPlan: {Hq} query heads over {Hkv}")
        groups = [([int(r) for r in rows], int(pages)) for rows, pages in groups]
        members = [r for rows, _ in groups for r in rows]
        if len(set(members)) != len(members) or any(not 0 <= r < B for r in members):
            raise ValueError(f"SharedPrefixPlan: rows {members} of {B}, each in one group at most")
        if any(not rows or pages <= 0 for rows, pages in groups) or any(16 * pages > lens[r] for rows, pages in groups for r in rows):
            raise ValueError("SharedPrefixPlan: a group has rows and pages, and its pages lie within their contexts")
        self.B, self.Hq, self.Hkv, self.D = B, Hq, Hkv, D
        self.earlier = None                                              # a plan that this one replaces, as long as recorded steps may read it
        row_pages, row_slots = [0] * B, [0] * B
        for rows, pages in groups:
            for r in rows:
                row_pages[r] = pages
        own = [-(-n // 16) - p for n, p in zip(lens, row_pages)]
        # more than eight query rows are a block's (us as units of single waves / of blocks: 16 rows of 32 heads over 32 behind 256 pages 27.0 / 24.4, behind 64
        # 14.9 / 13.4; 4 rows of 32 heads over 8 behind 64 pages 10.6 / 9.6, behind 1024 22.7 / 22.9; 4 of 16 over 16 behind 32 7.5 / 8.1, 2 of 32 over 32
        # behind 64 10.5 / 11.7)
        in_block = lambda rows: len(rows) * G > 8
        large, small = [g for g in groups if in_block(g[0])], [g for g in groups if not in_block(g[0])]
        most = lib().mlora_shared_attn_unit_rows() // G                  # rows of a block unit
        # pages of a unit: block units for two workgroups on each compute unit (16 rows behind 32752 tokens, 32 heads of 128 over 8, for one / two /
        # three: 50 / 46 / 46.5 us, three services of 20 rows behind 4096 tokens 44 / 44 / 49), units of single waves for four (the three
        # services, for two / four / eight / sixteen: 47 / 42 / 44.5 / 46, 32 rows behind 1024 tokens 22.7 / 22.7 / 22.7 / 26) - but no shorter than some pages
        # (own ones two / four / eight: the first 46.4 / 46.2 / 45.2), and no more units of a row than its second launch joins cheaply
        per_block = max(8, -(-sum(-(-len(rows) // most) * pages for rows, pages in large) * Hkv // 512))
        per_wave = max(4, -(-sum(pages for _, pages in small) * Hkv // 1024))
        self.groups = groups
        self.own_splits = self._shares(max(own, default=0))
        units = []
        for rows, pages in large + small:
            block = in_block(rows)
            n = min(-(-pages // (per_block if block else per_wave)), 64)
            cut = [pages * i // n for i in range(n + 1)]
            parts = -(-len(rows) // most) if block else 1
            edge = [len(rows) * i // parts for i in range(parts + 1)]
            for r in rows:
                row_slots[r] = n
            units += [(not block, lo - hi, rows[a:b], lo, j) for a, b in zip(edge, edge[1:]) for j, (lo, hi) in enumerate(zip(cut, cut[1:]))]
        units.sort(key=lambda u: u[:2])                                  # block units first, the longest first
        self.n_block = sum(not u[0] for u in units)
        self.n_units, self.slots = len(units), max(row_slots, default=0) + self.own_splits
        size = lib().mlora_shared_attn_record_ints()
        records = [x for _, less, rows, lo, j in units for x in (len(rows), lo, -less, j, 0, 0, 0, 0, *rows, *([rows[0]] * (size - 8 - len(rows))))]
        self.data = upload(torch.tensor(records + row_pages + row_slots, dtype=torch.int32), device)
        self.workspace_bytes = lib().mlora_shared_attn_workspace_bytes(B, Hq, D, self.slots)
        self._heads, self._page = (Hq, Hkv, D), ((Hkv, D // 32, 4, 16, 8), (Hkv, D, 16))
        self._bind()

    def _shares(self, pages):
        """How many units share the pages that a row has for itself."""
        return max(1, min(-(-pages // 8), 1024 // max(self.B * self.Hkv, 1), 64))

    def outgrown(self, lens) -> bool:
        """Whether a plan made for these contexts would cut the rows' own pages into twice as many shares.  us, a plan of 20 own tokens / a new one / no
        sharing, 8 rows behind 2048 tokens, 32 heads over 8: 200 own tokens 15.3 / 12.8 / 19.3, 400 20.6 / 13.1 / 20.5, 2000 65 / 19.5 / 31.8."""
        own = [-(-n // 16) for n in lens]
        for rows, pages in self.groups:
            for r in rows:
                own[r] -= pages
        return self._shares(max(own, default=0)) >= 2 * self.own_splits

    def _bind(self):
        """The plan's arrays as parts of `data`, and what the C call takes of them: addresses that hold while the plan lives."""
        n = self.data.numel() - 2 * self.B
        self.units, self.row_pages, self.row_slots = self.data[:n], self.data[n:n + self.B], self.data[n + self.B:]
        self._args = (self.units.data_ptr(), self.n_block, self.n_units, self.row_pages.data_ptr(), self.row_slots.data_ptr(), self.own_splits, self.slots)

    def __getstate__(self):
        return {n: v for n, v in self.__dict__.items() if n not in ("units", "row_pages", "row_slots", "_args", "earlier")}

    def __setstate__(self, state):
        """A copy has arrays of its own, and their addresses; no recorded step reads them."""
        self.__dict__.update(state, earlier=None)
        self._bind()


def paged_attn_decode_shared(qkv, k_cache, v_cache, block_table, seq_ids, ctx_len, plan: SharedPrefixPlan, Hq, Hkv, D, out=None, frag=False):
    """`paged_attn_decode` for a batch whose rows share prefixes as `plan` says: shared pages are read once for all their rows."""
    B, (n_seq, max_blocks), (n_pages, *page_k), (pages_v, *page_v) = qkv.shape[0], block_table.shape, k_cache.shape, v_cache.shape
    dev = _here(qkv.device, "paged_attn_decode_shared")
    if plan.B != B or plan._heads != (Hq, Hkv, D) or plan.data.device != dev:
        raise ValueError(f"paged_attn_decode_shared: a plan of {(plan.B, plan.Hq, plan.Hkv, plan.D)} on {plan.data.device} for {(B, Hq, Hkv, D)} on {dev}")
    if qkv.numel() != B * (Hq + 2 * Hkv) * D or seq_ids.shape != (B,) or ctx_len.shape != (B,) or pages_v != n_pages or (tuple(page_k), tuple(page_v)) != plan._page:
        raise ValueError(f"paged_attn_decode_shared: qkv{tuple(qkv.shape)} rows{tuple(seq_ids.shape)} contexts{tuple(ctx_len.shape)} k{tuple(k_cache.shape)} "
                         f"v{tuple(v_cache.shape)}")
    if out is not None and (tuple(out.shape) != (B, Hq * D) or isinstance(out, FragActivation) != frag):
        raise ValueError(f"paged_attn_decode_shared: out{tuple(out.shape)}")
    if k_cache.device != dev or v_cache.device != dev or block_table.device != dev or seq_ids.device != dev or ctx_len.device != dev \
            or out is not None and out.device != dev:
        raise ValueError(f"paged_attn_decode_shared: all tensors on {dev}")
    f16, i32 = torch.float16, torch.int32
    if not (qkv.dtype is f16 and k_cache.dtype is f16 and v_cache.dtype is f16 and block_table.dtype is i32 and seq_ids.dtype is i32 and ctx_len.dtype is i32
            and qkv.is_contiguous() and k_cache.is_contiguous() and v_cache.is_contiguous() and block_table.is_contiguous() and seq_ids.is_contiguous()
            and ctx_len.is_contiguous()):                                  # (says which)
        for t, dt, name in ((qkv, f16, "qkv"), (k_cache, f16, "k_cache"), (v_cache, f16, "v_cache"), (block_table, i32, "block_table"), (seq_ids, i32, "seq_ids"),
                            (ctx_len, i32, "ctx_len")):
            _dev(t, dt, name)
    if out is None and not frag:
        out, lay = _empty_strided_cuda((B, Hq * D), (Hq * D, 1), f16), ROWMAJOR
        optr = out.data_ptr()
    else:
        out, optr, lay = _out_arg(out, B, Hq * D, frag, dev)
    if B == 0:
        return out
    nb = plan.workspace_bytes
    ws = _empty_strided_cuda((nb // 4,), (1,), torch.float32)
    code = lib().mlora_paged_attn_decode_shared(optr, lay, qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), max_blocks,
                                                seq_ids.data_ptr(), ctx_len.data_ptr(), *plan._args, B, Hq, Hkv, D, n_pages, n_seq, ws.data_ptr(), nb, _stream())
    if code:
        check(code)
    return out


def rope_attn_decode(qkv, k_cache, v_cache, block_table, seq_ids, tok_pos, ctx_len, rope_cos, rope_sin, Hq, Hkv, D,
                     out=None, frag=False, o_shrink=None):
    """rope_kv_append + paged_attn_decode of one decode step in one launch (no LoRA on q, k, v); qkv is left unrotated.
    o_shrink = (A [n_ad, r, Hq * D] f16, tok_adapter [B] int32): the launch also writes the o projection's shrink as
    one share per query head and the call returns (out, vpart [Hq, B, r] fp32; rows of tokens without adapter are NaN)."""
    B = qkv.shape[0]
    n_seq, max_blocks = block_table.shape
    out, optr, lay = _out_arg(out, B, Hq * D, frag, qkv.device)
    if o_shrink is not None:
        A, ids = o_shrink
        n_ad, r, Kq = A.shape
        if Kq != Hq * D or not lib().mlora_rope_attn_oshrink_ok(B, Hq, Hkv, D, r):
            raise ValueError(f"rope_attn_decode: o shrink A{tuple(A.shape)} not served for B={B} Hq={Hq} Hkv={Hkv} D={D}")
        vpart = torch.full((Hq, B, r), float("nan"), dtype=torch.float32, device=qkv.device)
        check(lib().mlora_rope_attn_decode_oshrink(optr, lay, _dev(qkv, torch.float16), _dev(k_cache, torch.float16),
                                                   _dev(v_cache, torch.float16), _dev(block_table, torch.int32), max_blocks,
                                                   _dev(seq_ids, torch.int32), _dev(tok_pos, torch.int32), _dev(ctx_len, torch.int32),
                                                   _dev(rope_cos, torch.float32), _dev(rope_sin, torch.float32), rope_cos.shape[0],
                                                   B, Hq, Hkv, D, k_cache.shape[0], n_seq, None, 0, None, _dev(ids, torch.int32), 0.0,
                                                   0, r, n_ad, _dev(A, torch.float16, "A"), vpart.data_ptr(), _stream()))
        return out, vpart
    check(lib().mlora_rope_attn_decode(optr, lay, _dev(qkv, torch.float16), _dev(k_cache, torch.float16),
                                       _dev(v_cache, torch.float16), _dev(block_table, torch.int32), max_blocks,
                                       _dev(seq_ids, torch.int32), _dev(tok_pos, torch.int32), _dev(ctx_len, torch.int32),
                                       _dev(rope_cos, torch.float32), _dev(rope_sin, torch.float32), rope_cos.shape[0],
                                       B, Hq, Hkv, D, k_cache.shape[0], n_seq, None, 0, None, None, 0.0, 0, 0, 0, _stream()))
    return out


def paged_attn_prefill(qkv, k_cache, v_cache, block_table, tok_seq, tok_pos, Hq, Hkv, D, out=None, frag=False):
    T = qkv.shape[0]
    n_seq, max_blocks = block_table.shape
    out, optr, lay = _out_arg(out, T, Hq * D, frag, qkv.device)
    check(lib().mlora_paged_attn_prefill(optr, lay, _dev(qkv, torch.float16), _dev(k_cache, torch.float16),
                                         _dev(v_cache, torch.float16), _dev(block_table, torch.int32), max_blocks,
                                         _dev(tok_seq, torch.int32), _dev(tok_pos, torch.int32), T, Hq, Hkv, D,
                                         k_cache.shape[0], n_seq, _stream()))
    return out


class QuantPages:
    """A layer's pages of a paged cache in 8 bits, a step per page and head for keys and for values, with every sequence's last page unrounded (layouts and
    rounding: mlora_page_attn in include/mlora.h).  k [n_pages, Hkv, D / 64, 4, 16, 2, 8] and v [n_pages, Hkv, D / 64, 4, 16, 4, 4] int8, step [n_pages, Hkv, 2] fp32,
    tail_k [slots, Hkv, D / 32, 4, 16, 8] and tail_v [slots, Hkv, D, 16] fp16: a slot for every row of the block table.  The tensors are the caller's."""

    def __init__(self, k, v, step, tail_k, tail_v):
        if k.dim() != 7 or tail_v.dim() != 4:
            raise ValueError(f"QuantPages: k{tuple(k.shape)} tail_v{tuple(tail_v.shape)}")
        self.n_pages, self.Hkv, self.D, self.slots = k.shape[0], k.shape[1], 64 * k.shape[2], tail_v.shape[0]
        n, H, J, S = self.n_pages, self.Hkv, k.shape[2], self.slots
        given = {"k": (k, torch.int8, (n, H, J, 4, 16, 2, 8)), "v": (v, torch.int8, (n, H, J, 4, 16, 4, 4)), "step": (step, torch.float32, (n, H, 2)),
                 "tail_k": (tail_k, torch.float16, (S, H, 2 * J, 4, 16, 8)), "tail_v": (tail_v, torch.float16, (S, H, 64 * J, 16))}
        self.device = k.device
        for name, (t, dt, shape) in given.items():
            if t.dtype is not dt:
                raise TypeError(f"QuantPages: {name} must be {dt}, got {t.dtype}")
            if t.shape != shape or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"QuantPages: {name}{tuple(t.shape)} on {t.device}, expected {shape} on {self.device}, contiguous")
            setattr(self, name, t)

    @classmethod
    def empty(cls, n_pages, slots, Hkv, D, device):
        """Pages that hold nothing yet."""
        if D % 64:
            raise ValueError(f"QuantPages: head_dim {D} is not a multiple of 64")
        z = lambda shape, dt: torch.zeros(shape, dtype=dt, device=device)                                          # noqa: E731
        return cls(z((n_pages, Hkv, D // 64, 4, 16, 2, 8), torch.int8), z((n_pages, Hkv, D // 64, 4, 16, 4, 4), torch.int8), z((n_pages, Hkv, 2), torch.float32),
                   z((slots, Hkv, D // 32, 4, 16, 8), torch.float16), z((slots, Hkv, D, 16), torch.float16))

    def values(self, ids):
        """(keys, values) [n, Hkv, 16, D] fp16: what pages ids [n] int32 stand for (an id that is no page leaves its rows as they come)."""
        dev = _here(self.device, "QuantPages.values")
        if ids.dim() != 1 or ids.device != dev:
            raise ValueError(f"QuantPages.values: ids{tuple(ids.shape)} on {ids.device}")
        n, p = ids.shape[0], _dev(ids, torch.int32, "ids")
        shape, stride = (n, self.Hkv, 16, self.D), (self.Hkv * 16 * self.D, 16 * self.D, self.D, 1)
        keys, values = (_empty_strided_cuda(shape, stride, torch.float16) for _ in range(2))
        for i in range(0, n, 65535):                                     # (a launch's)
            m = min(n - i, 65535)
            check(lib().mlora_page_values(keys[i:].data_ptr(), values[i:].data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.step.data_ptr(), p + 4 * i, m, self.Hkv,
                                          self.D, self.n_pages, _stream()))
        return keys, values


def _window(who, window, sinks):
    if window is None and not sinks:
        return 0, 0
    if window is None or not 1 <= window <= 0x7fffffff or not 0 <= sinks <= 0x7fffffff:
        raise ValueError(f"{who}: a window of {window} tokens with {sinks} sinks")
    return int(window), int(sinks)


_NO_ROPE = (None, None)


def _page_attn(who, fn, qkv, k, v, quant, block_table, tok_seq, tok_pos, rope, Hq, Hkv, D, window, sinks, out, frag, longest):
    """The call behind attention over pages that k and v name."""
    T, (n_seq, max_blocks), dev = qkv.shape[0], block_table.shape, _here(qkv.device, who)
    window, sinks = _window(who, window, sinks)
    n_pages = k.shape[0]
    if qkv.numel() != T * (Hq + 2 * Hkv) * D or tok_seq.shape != (T,) or tok_pos.shape != (T,):
        raise ValueError(f"{who}: qkv{tuple(qkv.shape)} for {T} x {Hq + 2 * Hkv} x {D}, rows{tuple(tok_seq.shape)} positions{tuple(tok_pos.shape)}")
    cos, sin = rope
    f16, i32, max_pos = torch.float16, torch.int32, 0x7fffffff
    tensors = [(qkv, f16, "qkv"), (block_table, i32, "block_table"), (tok_seq, i32, "rows"), (tok_pos, i32, "positions")]
    if cos is not None:
        max_pos = cos.shape[0]
        if cos.shape != (max_pos, D // 2) or sin.shape != cos.shape:
            raise ValueError(f"{who}: rotation tables {tuple(cos.shape)} and {tuple(sin.shape)} for head_dim {D}")
        tensors += [(cos, torch.float32, "rope_cos"), (sin, torch.float32, "rope_sin")]
    if quant is not None:
        if (quant.Hkv, quant.D) != (Hkv, D) or quant.slots < n_seq or quant.device != dev:
            raise ValueError(f"{who}: pages of {quant.Hkv} heads of {quant.D} with {quant.slots} slots on {quant.device} for {Hkv} of {D}, {n_seq} rows of the table, on {dev}")
        step, tail_k, tail_v = quant.step.data_ptr(), quant.tail_k.data_ptr(), quant.tail_v.data_ptr()
    else:
        if D % 32 or k.shape != (n_pages, Hkv, D // 32, 4, 16, 8) or v.shape != (n_pages, Hkv, D, 16):
            raise ValueError(f"{who}: k{tuple(k.shape)} v{tuple(v.shape)} for {Hkv} heads of {D}")
        tensors += [(k, f16, "k_cache"), (v, f16, "v_cache")]
        step = tail_k = tail_v = 0
    for t, dt, name in tensors:
        if t.dtype is not dt or t.device != dev or not t.is_contiguous():
            _dev(t, dt, name)                                            # (says which)
            raise ValueError(f"{who}: {name} on {t.device}, others on {dev}")
    if out is None and not frag:
        out, lay = _empty_strided_cuda((T, Hq * D), (Hq * D, 1), f16), ROWMAJOR
        optr = out.data_ptr()
    else:
        if out is not None and (tuple(out.shape) != (T, Hq * D) or isinstance(out, FragActivation) != frag or out.device != dev):
            raise ValueError(f"{who}: out{tuple(out.shape)} on {out.device}")
        out, optr, lay = _out_arg(out, T, Hq * D, frag, dev)
    if T == 0:
        return out
    pages, ws, nb, prompt = max_blocks if longest is None else min(-(-longest // 16), max_blocks), 0, 0, int(fn == "mlora_page_attn_prefill")
    if window:
        pages = min(pages, (window + (T if prompt else 0) + 30) // 16 + (sinks + 15) // 16)
    splits = _size(f16, "mlora_page_attn_splits", prompt, T, Hq, Hkv, pages)
    if splits > 1:
        nb = _size(f16, "mlora_page_attn_workspace_bytes", T, Hq, D, splits)
        w = _empty_strided_cuda((nb // 4,), (1,), torch.float32)
        ws = w.data_ptr()
    args = _PAGE_ATTN.pack(optr, qkv.data_ptr(), k.data_ptr(), v.data_ptr(), step, tail_k, tail_v, block_table.data_ptr(), tok_seq.data_ptr(), tok_pos.data_ptr(),
                           0 if cos is None else cos.data_ptr(), 0 if cos is None else sin.data_ptr(), ws, nb, lay, max_blocks, max_pos, T, Hq, Hkv, D, n_pages, n_seq,
                           window, sinks, splits)
    code = getattr(lib(), fn)(args, _stream())
    if code:
        check(code)
    return out


def rope_attn_decode_q8(qkv, pages: QuantPages, block_table, seq_ids, tok_pos, rope_cos, rope_sin, Hq, Hkv, D, window=None, sinks=0, longest=None, out=None, frag=False):
    """One token of each of T different sequences on pages of 8 bits: q and k are rotated, the token's k and v stored (its page rounded to 8 bits, where it completes it),
    and the token attends to its own page unrounded and to those ahead of it.  qkv is left as it is.  window: only the last so many tokens are seen, the
    token itself among them, and the first `sinks`.  longest: most tokens of a row, its new ones among them; it chooses how the work is cut (None: as many as the table holds)."""
    return _page_attn("rope_attn_decode_q8", "mlora_page_attn_decode", qkv, pages.k, pages.v, pages, block_table, seq_ids, tok_pos, (rope_cos, rope_sin), Hq, Hkv, D, window,
                      sinks, out, frag, longest)


def rope_attn_prefill_q8(qkv, pages: QuantPages, block_table, tok_seq, tok_pos, rope_cos, rope_sin, Hq, Hkv, D, window=None, sinks=0, longest=None, out=None, frag=False):
    """`rope_attn_decode_q8` for the tokens of a pass, those of a sequence consecutive with increasing positions: the same results however a prompt is cut into passes, up to
    the order of sums."""
    return _page_attn("rope_attn_prefill_q8", "mlora_page_attn_prefill", qkv, pages.k, pages.v, pages, block_table, tok_seq, tok_pos, (rope_cos, rope_sin), Hq, Hkv, D, window,
                      sinks, out, frag, longest)


def rope_attn_decode_window(qkv, k_cache, v_cache, block_table, seq_ids, tok_pos, rope_cos, rope_sin, Hq, Hkv, D, window=None, sinks=0, longest=None, out=None, frag=False):
    """`rope_attn_decode` under a sliding window with sinks, and with long contexts shared out over the device (arguments as for `rope_attn_decode_q8`)."""
    return _page_attn("rope_attn_decode_window", "mlora_page_attn_decode", qkv, k_cache, v_cache, None, block_table, seq_ids, tok_pos, (rope_cos, rope_sin), Hq, Hkv, D, window,
                      sinks, out, frag, longest)


def paged_attn_prefill_window(qkv, k_cache, v_cache, block_table, tok_seq, tok_pos, Hq, Hkv, D, window=None, sinks=0, longest=None, out=None, frag=False):
    """`paged_attn_prefill` under a sliding window with sinks: behind `rope_kv_append` of the same tokens."""
    return _page_attn("paged_attn_prefill_window", "mlora_page_attn_prefill", qkv, k_cache, v_cache, None, block_table, tok_seq, tok_pos, _NO_ROPE, Hq, Hkv, D, window, sinks,
                      out, frag, longest)


def copy_pages(pools, src, dst):
    """Rows src [n] int32 of pools [layers, rows, ...] (contiguous tensors of any type, up to 8) go to rows dst [n], in every layer, in one launch.  A row that is written is in
    no other pair; indices that are no row copy nothing."""
    pools = list(pools)
    if not 1 <= len(pools) <= 8 or any(p.dim() < 2 for p in pools):
        raise ValueError(f"copy_pages: {[tuple(p.shape) for p in pools]}: one to eight pools of [layers, rows, ...]")
    dev = _here(pools[0].device, "copy_pages")
    if src.dim() != 1 or src.shape != dst.shape or src.device != dev or dst.device != dev:
        raise ValueError(f"copy_pages: src{tuple(src.shape)} on {src.device}, dst{tuple(dst.shape)} on {dst.device}, pools on {dev}")
    n, ps, pd, args = src.shape[0], _dev(src, torch.int32, "src"), _dev(dst, torch.int32, "dst"), b""
    for p in pools:
        if p.device != dev:
            raise ValueError(f"copy_pages: a pool on {p.device}, others on {dev}")
        at, (layers, rows), size = _dev(p, None, "pool"), p.shape[:2], p.element_size()
        if not p.numel():
            raise ValueError(f"copy_pages: a pool{tuple(p.shape)} without elements")
        args += _PAGE_POOL.pack(at, p.stride(1) * size if rows > 1 else p.numel() // layers * size, layers, rows)
    if n:
        L = _lib.loaded()
        code = L.mlora_copy_pages(args, len(pools), ps, pd, n, _stream())
        if code:
            raise _lib.MloraError(code, L.mlora_last_error().decode())


def beam_select(logits, scores, ended=None, eos=None, k=None):
    """The k (None: as many as beams) best continuations of R requests of W beams each: of beam b by token v with value scores[b] + logits[b, v] - logsumexp(logits[b]).
    logits [R * W, V] fp32 (any row stride), scores [R, W] fp32 (-inf: no beam there).  ended [R, W] int32: such a beam goes on with `eos` alone, at its score.
    -> scores [R, k] fp32, tokens [R, k], parents [R, k] int32 (the beam within its request), the best first - a beam's in the order of their logits,
    the lower token of equal ones first, and the lower beam of equal values -; -inf, -1, -1 where candidates run out."""
    (N, V), (R, W) = logits.shape, scores.shape
    dev = _here(logits.device, "beam_select")
    k = W if k is None else k
    ld, inner = logits.stride()
    if logits.dtype is not torch.float32 or (inner != 1 and V > 1) or (ld < V and N > 1):
        raise ValueError("beam_select: logits must be fp32 rows with unit inner stride")
    if N != R * W or scores.device != dev or ended is not None and (ended.shape != (R, W) or ended.device != dev or eos is None):
        raise ValueError(f"beam_select: logits{tuple(logits.shape)} scores{tuple(scores.shape)} ended{None if ended is None else tuple(ended.shape)} eos={eos}")
    if ended is not None and not 0 <= eos < V:
        raise ValueError(f"beam_select: eos={eos} of {V} tokens")
    p_scores, p_ended = _dev(scores, torch.float32, "scores"), None if ended is None else _dev(ended, torch.int32, "ended")
    best = _empty_strided_cuda((R, k), (k, 1), torch.float32)
    tokens, parents = _empty_strided_cuda((R, k), (k, 1), torch.int32), _empty_strided_cuda((R, k), (k, 1), torch.int32)
    if R == 0:
        return best, tokens, parents
    L = _lib.loaded()
    nb = _beam_bytes(R, W, V, k)
    ws = _empty_strided_cuda((nb // 8,), (1,), torch.int64)
    code = L.mlora_beam_select(best.data_ptr(), tokens.data_ptr(), parents.data_ptr(), logits.data_ptr(), ld if N > 1 else max(V, ld), p_scores, p_ended,
                               -1 if eos is None else eos, R, W, V, k, ws.data_ptr(), nb, _stream())
    if code:
        raise _lib.MloraError(code, L.mlora_last_error().decode())
    return best, tokens, parents


@functools.lru_cache(maxsize=256)
def _beam_bytes(R, W, V, k):
    return _lib.loaded().mlora_beam_select_workspace_bytes(R, W, V, k)


class BeamMoves(typing.NamedTuple):
    """What is to be copied behind a reordering, [R * W] int32 each, -1 for nothing: the contents of slots, and of last pages (for `copy_pages`)."""
    src_slot: torch.Tensor
    dst_slot: torch.Tensor
    src_page: torch.Tensor
    dst_page: torch.Tensor


def beam_reorder(parents, slots, block_table, tok_pos):
    """Where beams go on whose parents [R, W] int32 `beam_select` has chosen: slots [R * W] int32, the rows of block_table that the beams have, become those returned: a
    parent's first child keeps its slot, further children take those of beams without any, whose rows of the table are changed to the parent's pages up to
    that of the token appended last (tok_pos [R * W] int32; positions of the next tokens: a page that is complete is taken over as well, not copied).  -> (slots, BeamMoves): the last pages, and what else a slot holds, are to be copied by the moves."""
    dev = _here(parents.device, "beam_reorder")
    if parents.dim() != 2 or block_table.dim() != 2 or slots.shape != (parents.numel(),) or tok_pos.shape != slots.shape:
        raise ValueError(f"beam_reorder: parents{tuple(parents.shape)} slots{tuple(slots.shape)} table{tuple(block_table.shape)} positions{tuple(tok_pos.shape)}")
    ptrs = []
    for t, name in ((parents, "parents"), (slots, "slots"), (block_table, "block_table"), (tok_pos, "tok_pos")):
        if t.device != dev:
            raise ValueError(f"beam_reorder: {name} on {t.device}, others on {dev}")
        ptrs.append(_dev(t, torch.int32, name))
    R, W = parents.shape
    N = R * W
    new = _empty_strided_cuda((5, N), (N, 1), torch.int32)
    if N:
        at, L = new.data_ptr(), _lib.loaded()
        code = L.mlora_beam_reorder(at, at + 4 * N, at + 8 * N, at + 12 * N, at + 16 * N, *ptrs, R, W, *block_table.shape, _stream())
        if code:
            raise _lib.MloraError(code, L.mlora_last_error().decode())
    return new[0], BeamMoves(new[1], new[2], new[3], new[4])
