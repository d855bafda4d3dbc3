// Linear with 4-bit weights and group scales:
//   y[t, n] (=|+=) sum over groups g of K:  s[n, g] sum_{k in g} x[t, k] (q[n, k] - z[n, g]),   q, z = 0 .. 15
//
// The matrix cores multiply fp16 activations with the integers q - z, which fp16 holds exactly, and a group's sum is scaled in fp32: no
// rounding but those of fp32 sums and the result's.  For up to 64 tokens the weight stream from HBM is the bound (N K / 2 bytes and 3
// N K / group of scales and zeros).
//
// Layout (mlora_linear4_bytes; K in blocks of 128, N in tiles of 16 rows, both padded with zeros):
//   q     [tile][block][lane 64][k-step 4] words: lane (kg, row) = lane / 16, lane % 16 holds k = 32 step + 8 kg + e of its row in word
//         `step`, e = 2 p in bits 4 p .., e = 2 p + 1 in bits 16 + 4 p ..: a tile's block is 1 KiB that a wave reads with one load a
//         lane, and pairs of neighbouring k come out of a word with one mask-and-or each
//   scale [tile][block][row 16][128 / group] fp16,  zero likewise in bytes
#include "lora_device.h"

namespace {

constexpr int L4_WAVES = 8;
constexpr int L4_BLOCK = 128;
enum { L4_F16 = 0, L4_F32 = 1, L4_ACC = 2 };

struct Linear4 {
  void* y;
  const f16* x;
  const uint32_t* q;
  const f16* scale;
  const uint8_t* zero;
  int ldx, frag_tt, T, K, N;       // frag_tt: token tiles of a fragment-ordered x, 0: rows of ldx
  bool wide;                       // rows of y take four columns at a time
};

// The eight weights of a word as fp16 integers q - z; zz = 1024 + z twice.  An fp16 of 1024 .. 2047 holds an integer in its low bits, so
// 1024 + q is the nibble with an exponent put above it, and 1024 + 16 q the one four bits higher.
__device__ __forceinline__ f16x8 l4_weights(uint32_t w, f16x2 zz, f16x2 zs) {
  const uint32_t ex = 0x64006400u, lo = 0x000f000fu, hi = 0x00f000f0u;
  union { uint32_t u; f16x2 h; } a, b, c, d;
  a.u = (w & lo) | ex;
  b.u = (w & hi) | ex;
  w >>= 8;
  c.u = (w & lo) | ex;
  d.u = (w & hi) | ex;
  const f16x2 s = f16x2{(f16)0.0625f, (f16)0.0625f};
  a.h = a.h - zz;
  b.h = __builtin_elementwise_fma(b.h, s, zs);               // (1024 + 16 q) / 16 - (64 + z)
  c.h = c.h - zz;
  d.h = __builtin_elementwise_fma(d.h, s, zs);
  return f16x8{a.h[0], a.h[1], b.h[0], b.h[1], c.h[0], c.h[1], d.h[0], d.h[1]};
}

// Workgroup: NT tiles of rows and up to 16 TT tokens; its waves take every eighth block of K and their sums meet in LDS, in wave order.
template <int NT, int TT, int GB, int OUT>      // GB: groups per block
__global__ __launch_bounds__(L4_WAVES * WAVE) void linear4_kernel(Linear4 a) {
  constexpr int TILES = NT * TT;
  constexpr int HT = TILES > 8 ? 8 : TILES;     // tiles summed per pass through LDS
  __shared__ f32x4 red[L4_WAVES][HT][WAVE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, kg = lane >> 4;
  const int nb = (a.K + L4_BLOCK - 1) / L4_BLOCK, KB = a.K / 32, tiles = (a.N + 15) / 16;
  const int tile0 = blockIdx.x * NT, t0 = blockIdx.y * (16 * TT);
  size_t row_block[NT];                         // first block of a tile
#pragma unroll
  for (int i = 0; i < NT; ++i) row_block[i] = (size_t)(tile0 + i < tiles ? tile0 + i : tiles - 1) * nb;
  const f16* xp[TT];
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    if (a.frag_tt) {
      const int tt = t0 / 16 + j;
      xp[j] = a.x + (size_t)(tt < a.frag_tt ? tt : a.frag_tt - 1) * 512 + lane * 8;
    } else {
      const int t = t0 + j * 16 + r16;
      xp[j] = a.x + (size_t)(t < a.T ? t : a.T - 1) * a.ldx + kg * 8;
    }
  }
  const size_t xstep = a.frag_tt ? (size_t)a.frag_tt * 512 : 32;
  f32x4 acc[NT][TT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    uint4 q[NT];
    f16 s[NT][4 * GB];
    uint8_t z[NT][GB];
  };
  auto load = [&](Stage& st, int b) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const size_t rb = row_block[i] + b;
      st.q[i] = *reinterpret_cast<const uint4*>(a.q + rb * 256 + lane * 4);
      __builtin_memcpy(st.s[i], __builtin_assume_aligned(a.scale + (rb * 16 + kg * 4) * GB, 8), sizeof(st.s[i]));
      __builtin_memcpy(st.z[i], __builtin_assume_aligned(a.zero + (rb * 16 + r16) * GB, GB), sizeof(st.z[i]));
    }
  };
  Stage st;
  for (int b = wave; b < nb; b += L4_WAVES) {
    load(st, b);
    f16x8 x[4][TT];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        const int ks = b * 4 + k;
        x[k][j] = ks < KB ? ld8(xp[j] + (size_t)ks * xstep) : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
      }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t w[4] = {st.q[i].x, st.q[i].y, st.q[i].z, st.q[i].w};
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        const f16 z = (f16)(float)st.z[i][g];
        const f16x2 zz = f16x2{(f16)1024.f + z, (f16)1024.f + z}, zs = f16x2{-((f16)64.f + z), -((f16)64.f + z)};
        f32x4 sum[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = g * (4 / GB); k < (g + 1) * (4 / GB); ++k) {
          const f16x8 wf = l4_weights(w[k], zz, zs);
#pragma unroll
          for (int j = 0; j < TT; ++j) sum[j] = mfma_16x16x32(wf, x[k][j], sum[j]);
        }
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sum[j][e], (float)st.s[i][e * GB + g], acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < TILES / HT; ++h) {
    if (h) __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j)
        if ((i * TT + j) / HT == h) red[wave][(i * TT + j) % HT][lane] = acc[i][j];
    __syncthreads();
    for (int o = threadIdx.x; o < HT * WAVE; o += L4_WAVES * WAVE) {
      const int tile = h * HT + o / WAVE, sl = o % WAVE;
      f32x4 s = red[0][o / WAVE][sl];
#pragma unroll
      for (int w = 1; w < L4_WAVES; ++w) s += red[w][o / WAVE][sl];
      const int n = (tile0 + tile / TT) * 16 + (sl >> 4) * 4, t = t0 + (tile % TT) * 16 + (sl & 15);
      if (t >= a.T || n >= a.N) continue;
      const size_t at = (size_t)t * a.N + n;
      if (a.wide) {
        if constexpr (OUT == L4_F16) *reinterpret_cast<f16x4*>((f16*)a.y + at) = f16x4{(f16)s[0], (f16)s[1], (f16)s[2], (f16)s[3]};
        else if constexpr (OUT == L4_F32) *reinterpret_cast<f32x4*>((float*)a.y + at) = s;
        else *reinterpret_cast<f32x4*>((float*)a.y + at) += s;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) {
            if constexpr (OUT == L4_F16) ((f16*)a.y)[at + e] = (f16)s[e];
            else if constexpr (OUT == L4_F32) ((float*)a.y)[at + e] = s[e];
            else ((float*)a.y)[at + e] += s[e];
          }
      }
    }
  }
}

template <int NT, int TT, int GB>
void launch(const Linear4& a, int out, hipStream_t s) {
  const dim3 grid(ceil_div(ceil_div(a.N, 16), NT), ceil_div(a.T, 16 * TT)), block(L4_WAVES * WAVE);
  if (out == L4_F16) hipLaunchKernelGGL((linear4_kernel<NT, TT, GB, L4_F16>), grid, block, 0, s, a);
  else if (out == L4_F32) hipLaunchKernelGGL((linear4_kernel<NT, TT, GB, L4_F32>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((linear4_kernel<NT, TT, GB, L4_ACC>), grid, block, 0, s, a);
}

template <int GB>
void launch_shape(const Linear4& a, int out, hipStream_t s) {
  const int tiles = ceil_div(a.N, 16);
  if (a.T <= 16) {
    if (tiles <= 512) launch<1, 1, GB>(a, out, s);
    else launch<2, 1, GB>(a, out, s);
  } else if (a.T <= 32) launch<1, 2, GB>(a, out, s);
  else launch<1, 4, GB>(a, out, s);
}

}  // namespace

extern "C" int mlora_linear4_sizes(int N, int K, int group, size_t* q_bytes, size_t* scale_bytes, size_t* zero_bytes) {
  MLORA_CHECK(N > 0 && K > 0 && K % 32 == 0 && (group == 32 || group == 64 || group == 128) && K % group == 0, MLORA_ERR_UNSUPPORTED,
              "linear4: N=%d K=%d in groups of %d (K a multiple of the group: 32, 64 or 128)", N, K, group);
  const size_t blocks = (size_t)ceil_div(N, 16) * ceil_div(K, L4_BLOCK);
  if (q_bytes) *q_bytes = blocks * 1024;
  if (scale_bytes) *scale_bytes = blocks * 16 * (L4_BLOCK / group) * 2;
  if (zero_bytes) *zero_bytes = blocks * 16 * (L4_BLOCK / group);
  return MLORA_OK;
}

extern "C" int mlora_linear4(void* y, int y_dtype, int mode, const void* x, int x_layout, int ldx, const void* q, const void* scale, const void* zero, int group,
                             int T, int K, int N, void* stream) {
  MLORA_CHECK(y && x && q && scale && zero, MLORA_ERR_INVALID, "linear4: null pointer");
  if (int e = mlora_linear4_sizes(N, K, group, nullptr, nullptr, nullptr)) return e;
  MLORA_CHECK(T >= 0 && T <= 65535 * 16, MLORA_ERR_INVALID, "linear4: bad T=%d", T);
  MLORA_CHECK(y_dtype == MLORA_F16 || y_dtype == MLORA_F32, MLORA_ERR_INVALID, "linear4: bad y_dtype %d", y_dtype);
  MLORA_CHECK(mode == MLORA_STORE || (mode == MLORA_ACCUMULATE && y_dtype == MLORA_F32), MLORA_ERR_UNSUPPORTED, "linear4: results are added to fp32 alone (mode=%d)", mode);
  MLORA_CHECK(x_layout == MLORA_FRAG || (x_layout == MLORA_ROWMAJOR && ldx >= K && ldx % 8 == 0), MLORA_ERR_INVALID, "linear4: bad x (layout=%d ldx=%d K=%d)", x_layout,
              ldx, K);
  MLORA_CHECK((((uintptr_t)x | (uintptr_t)q | (uintptr_t)scale | (uintptr_t)zero) & 15) == 0, MLORA_ERR_INVALID, "linear4: operands not 16-byte aligned");
  MLORA_CHECK(((uintptr_t)y & (y_dtype == MLORA_F32 ? 3 : 1)) == 0, MLORA_ERR_INVALID, "linear4: y not aligned to its elements");
  if (T == 0) return MLORA_OK;
  Linear4 a = {y, (const f16*)x, (const uint32_t*)q, (const f16*)scale, (const uint8_t*)zero, ldx, x_layout == MLORA_FRAG ? mlora_frag_tiles(T) : 0, T, K, N, N % 4 == 0 && ((uintptr_t)y & 15) == 0};
  const int out = mode == MLORA_ACCUMULATE ? L4_ACC : y_dtype == MLORA_F32 ? L4_F32 : L4_F16;
  hipStream_t s = (hipStream_t)stream;
  if (group == 128) launch_shape<1>(a, out, s);
  else if (group == 64) launch_shape<2>(a, out, s);
  else launch_shape<4>(a, out, s);
  return mlora_launch_status("linear4");
}
