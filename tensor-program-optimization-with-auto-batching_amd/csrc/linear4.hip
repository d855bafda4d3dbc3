// Linear with 4-bit weights and group scales:
//   y[t, n] (=|+=) sum over groups g of K:  s[n, g] sum_{k in g} x[t, k] (q[n, k] - z[n, g]),   q, z = 0 .. 15
//
// The matrix cores multiply fp16 activations with the integers q - z, which fp16 holds exactly, and a group's sum is scaled in fp32: no
// rounding but those of fp32 sums and the result's.  Up to 16 tokens the weight stream from HBM is the bound (N K / 2 bytes and 3 N K /
// group of scales and zeros): 8 tokens, 32003 x 4096, groups of 128: 17.5 us, 4.0 TB/s (the fp16 products of this library stream 5.5); 16 tokens, 22016 x 4096:
// 13.3 us, 3.6 TB/s; one token, 4096 x 4096: 5.0 us, a launch and two rounds to memory.  With more tokens it is the
// unpacking and scaling on the vector units beside the products and the reads of LDS: 200 tokens, 12288 x 4096, groups of 64: 38 us, 530 TFLOP/s
// (a plain fp16 product of 8192^3: 1.17 PFLOP/s).
//
// Layout (sizes: mlora_linear4_sizes; K in blocks of 128, N in tiles of 16 rows, both padded with zeros):
//   q     [tile][block][lane 64][k-step 4] words: lane (kg, row) = lane / 16, lane % 16 holds k = 32 step + 8 kg + e of its row in word
//         `step`, e = 2 p in bits 4 p .., e = 2 p + 1 in bits 16 + 4 p ..: a tile's block is 1 KiB that a wave reads with one load a
//         lane, and pairs of neighbouring k come out of a word with one mask-and-or each
//   meta  [tile][block] {scale [row 16][128 / group] fp16, zero likewise in bytes}: 48 bytes a group and tile
#include <type_traits>

#include "lora_device.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int L4_WAVES = 8;
constexpr int L4_BLOCK = 128;
enum { L4_F16 = 0, L4_F32 = 1, L4_ACC = 2 };

struct Linear4 {
  void* y;
  const f16* x;
  const uint32_t* q;
  const char* meta;
  int ldx, frag_tt, T, K, N;       // frag_tt: token tiles of a fragment-ordered x, 0: rows of ldx
  bool wide;                       // rows of y take four columns at a time
};

// The eight weights of a word as fp16 integers q - z; zz = 1024 + z, zs = -(64 + z), twice.  An fp16 of 1024 .. 2047 holds an integer in its low
// bits, so 1024 + q is the nibble with an exponent put above it, and 1024 + 16 q the one four bits higher.  Mask and exponent come in
// registers (nibble_consts): as literals each pair of and / or would be two instructions, 13 a word instead of 9.
struct NibbleConsts {
  uint32_t lo, hi, ex;
};
__device__ __forceinline__ NibbleConsts nibble_consts() {
  NibbleConsts c = {0x000f000fu, 0x00f000f0u, 0x64006400u};
  asm("" : "+s"(c.lo), "+s"(c.hi), "+v"(c.ex));
  return c;
}
__device__ __forceinline__ f16x8 l4_weights(uint32_t w, const NibbleConsts& k, f16x2 zz, f16x2 zs) {
  union { uint32_t u; f16x2 h; } a, b, c, d;
  a.u = (w & k.lo) | k.ex;
  b.u = (w & k.hi) | k.ex;
  w >>= 8;
  c.u = (w & k.lo) | k.ex;
  d.u = (w & k.hi) | k.ex;
  const f16x2 s = f16x2{(f16)0.0625f, (f16)0.0625f};
  a.h = a.h - zz;
  b.h = __builtin_elementwise_fma(b.h, s, zs);               // (1024 + 16 q) / 16 - (64 + z)
  c.h = c.h - zz;
  d.h = __builtin_elementwise_fma(d.h, s, zs);
  return f16x8{a.h[0], a.h[1], b.h[0], b.h[1], c.h[0], c.h[1], d.h[0], d.h[1]};
}

// A uniform address that stays in scalar registers: lanes then add a 32-bit offset to it, where the compiler would carry 64 bits a lane for every
// pointer of a loop.  It costs scalar instructions ahead of each load (16 tokens, 22016 x 4096: 12.9 to 13.5 us), and pays where the vector
// registers would run out (the same in groups of 32: 32 to 17.7 us).
__device__ __forceinline__ const char* uniform(const char* p) {
  asm("" : "+s"(p));
  return p;
}

// Four columns n .. of a token's result
template <int OUT>
__device__ __forceinline__ void l4_store(const Linear4& a, int t, int n, f32x4 s) {
  const size_t at = (size_t)t * a.N + n;
  if (a.wide) {
    if constexpr (OUT == L4_F16) *reinterpret_cast<f16x4*>((f16*)a.y + at) = f16x4{(f16)s[0], (f16)s[1], (f16)s[2], (f16)s[3]};
    else if constexpr (OUT == L4_F32) *reinterpret_cast<f32x4*>((float*)a.y + at) = s;
    else *reinterpret_cast<f32x4*>((float*)a.y + at) += s;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) {
      if constexpr (OUT == L4_F16) ((f16*)a.y)[at + e] = (f16)s[e];
      else if constexpr (OUT == L4_F32) ((float*)a.y)[at + e] = s[e];
      else ((float*)a.y)[at + e] += s[e];
    }
}

__device__ __forceinline__ void l4_store(const Linear4& a, int out, int t, int n, f32x4 s) {
  if (out == L4_F16) l4_store<L4_F16>(a, t, n, s);                          // uniform
  else if (out == L4_F32) l4_store<L4_F32>(a, t, n, s);
  else l4_store<L4_ACC>(a, t, n, s);
}

// Up to 16 TT tokens: a workgroup has NT tiles of rows, its waves take every eighth block of K and their sums meet in LDS, in wave order.
template <int TT, int NT, int GB, int DEPTH, bool XFRAG>      // GB: groups per block; DEPTH: blocks of a wave on their way
__global__ __launch_bounds__(L4_WAVES * WAVE, NT > 3 || TT > 1 ? 2 : 4) void linear4_kernel(Linear4 a, int out) {
  __shared__ f32x4 red[L4_WAVES][NT][WAVE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, kg = lane >> 4;
  const int nb = (a.K + L4_BLOCK - 1) / L4_BLOCK, KB = a.K / 32, tiles = (a.N + 15) / 16;
  const NibbleConsts nc = nibble_consts();
  const int tile0 = blockIdx.x * NT;
  size_t row_block[NT];                         // first block of a tile
#pragma unroll
  for (int i = 0; i < NT; ++i) row_block[i] = (size_t)(tile0 + i < tiles ? tile0 + i : tiles - 1) * nb;
  // (rows behind the last token: the last one again, whose results are dropped)
  const bool frag = TT == 1 ? a.frag_tt > 0 : XFRAG;            // (one token tile: the same code for either order)
  const f16* xp[TT];
#pragma unroll
  for (int j = 0; j < TT; ++j)
    xp[j] = a.x + (frag ? (size_t)lane * 8 : (size_t)(j * 16 + r16 < a.T ? j * 16 + r16 : a.T - 1) * a.ldx + kg * 8);
  const size_t xstep = frag ? (size_t)a.frag_tt * 512 : 32;
  const uint32_t qoff = lane * 16, soff = kg * 8 * GB, zoff = 32 * GB + r16 * GB;
  f32x4 acc[NT][TT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    u32x4 q[NT];
    f16 s[NT][4 * GB];
    uint8_t z[NT][GB];
    f16x8 x[4][TT];
  };
  auto load = [&](Stage& st, int b, auto WHOLE) {          // (no branch where four k-steps are sure: behind one, a block on its way is waited for)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const size_t rb = row_block[i] + b;
      const char *m = a.meta + rb * (48 * GB), *q = (const char*)a.q + rb * 1024;
      if constexpr (GB >= 2 && (NT == 3 || NT * GB >= 16) || TT > 1 && NT * GB >= 12) m = uniform(m), q = uniform(q);
      st.q[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(q + qoff));
      __builtin_memcpy(st.s[i], __builtin_assume_aligned(m + soff, 8), sizeof(st.s[i]));
      __builtin_memcpy(st.z[i], __builtin_assume_aligned(m + zoff, GB), sizeof(st.z[i]));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ks = b * 4 + k;
#pragma unroll
      for (int j = 0; j < TT; ++j)
        st.x[k][j] = decltype(WHOLE)::value || ks < KB ? ld8(xp[XFRAG ? 0 : j] + (size_t)ks * xstep + (XFRAG ? j * 512 : 0)) : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  };
  auto multiply = [&](const Stage& st) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        const f16 z = (f16)(float)st.z[i][g];
        const f16x2 zz = f16x2{(f16)1024.f + z, (f16)1024.f + z}, zs = f16x2{-((f16)64.f + z), -((f16)64.f + z)};
        f32x4 sum[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = g * (4 / GB); k < (g + 1) * (4 / GB); ++k) {
          const f16x8 w = l4_weights(st.q[i][k], nc, zz, zs);
#pragma unroll
          for (int j = 0; j < TT; ++j) sum[j] = mfma_16x16x32(w, st.x[k][j], sum[j]);
        }
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sum[j][e], (float)st.s[i][e * GB + g], acc[i][j][e]);
      }
  };
  const int whole = KB / 4, own = (whole - wave + L4_WAVES - 1) / L4_WAVES;      // whole blocks, those of this wave
  Stage st[DEPTH];
  if (own > 0) {                                // uniform
    auto at = [&](int i) { return wave + i * L4_WAVES; };
    constexpr std::true_type sure;
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load(st[u], at(u < own ? u : own - 1), sure);
    int i = 0;
    for (; i + 2 * DEPTH <= own; i += DEPTH)
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        multiply(st[u]);
        load(st[u], at(i + DEPTH + u), sure);
      }
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      if (i + u < own) multiply(st[u]);
      if (i + DEPTH + u < own) load(st[u], at(i + DEPTH + u), sure);
    }
#pragma unroll
    for (int u = 0; u < DEPTH - 1; ++u)
      if (i + DEPTH + u < own) multiply(st[u]);
  }
  if (whole < nb && whole % L4_WAVES == wave) { // the end of K
    load(st[0], whole, std::false_type());
    multiply(st[0]);
  }
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    if (j > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) red[wave][i][lane] = acc[i][j];
    __syncthreads();
    for (int o = threadIdx.x; o < NT * WAVE; o += L4_WAVES * WAVE) {
      const int sl = o % WAVE, n = (tile0 + o / WAVE) * 16 + (sl >> 4) * 4, t = j * 16 + (sl & 15);
      f32x4 s = red[0][o / WAVE][sl];
#pragma unroll
      for (int w = 1; w < L4_WAVES; ++w) s += red[w][o / WAVE][sl];
      if (t < a.T && n < a.N) l4_store(a, out, t, n, s);
    }
  }
}

// More tokens: two groups of four waves take every second block of a slice of K each; a group's waves split the workgroup's rows (NT tiles each)
// and share the token block, which comes block of K by block of K straight into the group's LDS ring together with the weights and
// their scales; a wave's share of a stage is the same number of requests for all, so that a counted wait leaves the later stages in
// flight.  The groups take turns: one reads its next block from LDS into registers, the other multiplies.  (Both at a time, as four
// waves a group or eight, took 5% longer; LDS, the matrix cores and what unpacks and scales the weights each need a third of the time.)
// Rows of x lie in LDS as 256 bytes each, their sixteen 16-byte pieces exchanged by the row's number: the lanes that fetch a fragment of
// 16 rows then touch every bank once.  The groups' sums meet in LDS; more slices of K leave fp32 partial sums for a second launch.
constexpr int MID_WAVES = 4, MID_GROUPS = 2, MID_THREADS = MID_GROUPS * MID_WAVES * WAVE;
constexpr int MID_WBYTES = 1024 + 256;          // a tile's block: words, then scales and zeros (padded to a request of 4 bytes a lane)
constexpr int mid_stage_bytes(int TT, int NT) { return TT * 4096 + MID_WAVES * NT * MID_WBYTES; }
constexpr int mid_ring(int TT, int NT) { return MID_GROUPS * 3 * mid_stage_bytes(TT, NT) <= 160 * 1024 ? 3 : 2; }      // stages

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

__device__ __forceinline__ void to_lds16(const void* g, char* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void* g, char* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 4, 0, 0);
}

template <int TT, int NT, int GB, bool XFRAG>
__global__ __launch_bounds__(MID_THREADS, 2) void linear4_mid_kernel(Linear4 a, int out, float* __restrict__ part) {
  constexpr int RING = mid_ring(TT, NT), STAGE = mid_stage_bytes(TT, NT), XQ = TT * 4 / MID_WAVES, LOADS = XQ + 2 * NT;   // requests of a wave per stage
  constexpr int HELD = NT * TT > 8 ? GB < 4 ? 3 : 2 : 4;     // k-steps whose x waits in registers: all, where they are enough
  using zeros_t = std::conditional_t<GB == 1, uint8_t, std::conditional_t<GB == 2, uint16_t, uint32_t>>;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % MID_WAVES;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / MID_WAVES;
  char* ring = lds + group * (RING * STAGE);
  const int r16 = lane & 15, kg = lane >> 4;
  const int nb = (a.K + L4_BLOCK - 1) / L4_BLOCK, KB = a.K / 32, tiles = (a.N + 15) / 16;
  const NibbleConsts nc = nibble_consts();
  const int tile0 = (blockIdx.x * MID_WAVES + wave) * NT, t0 = blockIdx.z * (16 * TT);
  const int b0 = (int)((long)nb * blockIdx.y / gridDim.y), b1 = (int)((long)nb * (blockIdx.y + 1) / gridDim.y);

  // uniform bases, and 32-bit offsets of the lanes
  const char* wsrc[NT];
  const char* msrc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const size_t rb = (size_t)(tile0 + i < tiles ? tile0 + i : tiles - 1) * nb;
    wsrc[i] = (const char*)a.q + rb * 1024;
    msrc[i] = a.meta + rb * (48 * GB);
  }
  const uint32_t woff = lane * 16, moff = (lane < 12 * GB ? lane : 12 * GB - 1) * 4;
  uint32_t xoff[XQ], xend[XQ];                  // of a whole block, and of a last one of fewer than four k-steps
  const char* xbase = (const char*)a.x + (XFRAG ? 0 : (size_t)t0 * a.ldx * 2);
  const size_t xblock = XFRAG ? (size_t)a.frag_tt * 4096 : 256;        // bytes from a block to the next
#pragma unroll
  for (int q = 0; q < XQ; ++q) {
    const int f = wave + MID_WAVES * q;
    if constexpr (XFRAG) {
      const int tt = t0 / 16 + f % TT, ks = f / TT, last = (KB - 1) & 3;
      const uint32_t o = (uint32_t)(tt < a.frag_tt ? tt : a.frag_tt - 1) * 1024 + lane * 16;
      xoff[q] = o + (uint32_t)ks * a.frag_tt * 1024;
      xend[q] = o + (uint32_t)(ks < last ? ks : last) * a.frag_tt * 1024;
    } else {
      const int row = 4 * f + kg, k = (r16 ^ (row & 15)) * 8, last = (a.K - 8) & 127;
      const uint32_t o = (uint32_t)(t0 + row < a.T ? row : a.T - 1 - t0) * a.ldx * 2;
      xoff[q] = o + k * 2;
      xend[q] = o + (k < last ? k : last) * 2;
    }
  }
  const int whole = KB / 4;                     // blocks of four k-steps
  // Workgroups begin at different blocks of their slice, so that they do not all ask for the same lines of x at a time.
  const int n_own = (b1 - b0 + MID_GROUPS - 1) / MID_GROUPS;            // of a group: block i is b0 + group + 2 i; the second's last may be none
  int next = blockIdx.x % n_own;
  auto issue = [&](int slot) {
    char* st = ring + slot * STAGE;
    int b = b0 + group + MID_GROUPS * next;     // past the slice: once more from the front, and not multiplied
    b = b < b1 ? b : b0;
    next = next + 1 == n_own ? 0 : next + 1;
    const char* xb = uniform(xbase + b * xblock);
    if (b < whole) {                            // uniform
#pragma unroll
      for (int q = 0; q < XQ; ++q) to_lds16(xb + xoff[q], st + (wave + MID_WAVES * q) * 1024);
    } else {
#pragma unroll
      for (int q = 0; q < XQ; ++q) to_lds16(xb + xend[q], st + (wave + MID_WAVES * q) * 1024);
    }
    char* w = st + TT * 4096 + wave * (NT * MID_WBYTES);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      to_lds16(uniform(wsrc[i] + (size_t)b * 1024) + woff, w + i * MID_WBYTES);
      to_lds4(uniform(msrc[i] + (size_t)b * (48 * GB)) + moff, w + i * MID_WBYTES + 1024);
    }
  };
  f32x4 acc[NT][TT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < RING - 1; ++u) issue(u);
  int rd = 0, wr = RING - 1, at = blockIdx.x % n_own;
  wait_loads<(RING - 2) * LOADS>();
  bare_barrier();
  if (group == 1) bare_barrier();               // one group reads LDS while the other multiplies
  for (int n = 0; n < n_own; ++n) {
    const int b = b0 + group + MID_GROUPS * at;
    at = at + 1 == n_own ? 0 : at + 1;
    issue(wr);
    const char* st = ring + rd * STAGE;
    const char* w = st + TT * 4096 + wave * (NT * MID_WBYTES);
    rd = rd + 1 == RING ? 0 : rd + 1;
    wr = wr + 1 == RING ? 0 : wr + 1;
    u32x4 q[NT];
    f16 sc[NT][4 * GB];
    zeros_t zr[NT];
    f16x8 x[HELD][TT];
    auto fetch = [&](int k) {                   // the fragments of k-step k
#pragma unroll
      for (int j = 0; j < TT; ++j)
        x[k % HELD][j] = *reinterpret_cast<const f16x8*>(XFRAG ? st + (k * TT + j) * 1024 + lane * 16 : st + (j * 16 + r16) * 256 + (((k * 4 + kg) ^ r16) * 16));
    };
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      q[i] = *reinterpret_cast<const u32x4*>(w + i * MID_WBYTES + lane * 16);
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        const f16x4 v = *reinterpret_cast<const f16x4*>(w + i * MID_WBYTES + 1024 + kg * 8 * GB + g * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[i][g * 4 + e] = v[e];
      }
      zr[i] = *reinterpret_cast<const zeros_t*>(w + i * MID_WBYTES + 1024 + 32 * GB + r16 * GB);
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) fetch(k);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bare_barrier();
    const int nks = b < b1 ? KB - b * 4 : 0;    // k-steps of the block: 4, or fewer at the end of K
    auto block = [&](auto WHOLE) {
      constexpr int PER = 4 / GB;
      constexpr bool LATE = HELD == 4;       // a group's sums are scaled between the next one's products, where registers hold both
      f32x4 sum[NT][TT];
      f16x8 wf[2][NT];
      auto weights = [&](int k) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const f16 z = (f16)(float)(zr[i] >> 8 * (k / PER) & 0xff);
          wf[k & 1][i] = l4_weights(q[i][k], nc, f16x2{(f16)1024.f + z, (f16)1024.f + z}, f16x2{-((f16)64.f + z), -((f16)64.f + z)});
        }
      };
      auto multiply = [&](int k, int j) {
#pragma unroll
        for (int i = 0; i < NT; ++i) sum[i][j] = mfma_16x16x32(wf[k & 1][i], x[k % HELD][j], k % PER == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[i][j]);
      };
      auto scale = [&](int g, int j) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sum[i][j][e], (float)sc[i][e * GB + g], acc[i][j][e]);
      };
      weights(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!decltype(WHOLE)::value && k >= nks) break;       // uniform
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          if (LATE && k % PER == 0 && k > 0) scale(k / PER - 1, j);
          multiply(k, j);
        }
        if (k + HELD < 4) {
          __builtin_amdgcn_sched_barrier(0);
          fetch(k + HELD);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (k < 3) weights(k + 1);
        // a product occupies the matrix cores for the time of four other instructions
#pragma unroll
        for (int j = 0; j < NT * TT; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!LATE && k % PER == PER - 1) {
#pragma unroll
          for (int j = 0; j < TT; ++j) scale(k / PER, j);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int k = PER; k <= 4; k += PER)
        if (LATE && k == (decltype(WHOLE)::value ? 4 : nks)) {
#pragma unroll
          for (int j = 0; j < TT; ++j) scale(k / PER - 1, j);
        }
    };
    if (nks >= 4) block(std::true_type());
    else if (nks > 0) block(std::false_type());
    wait_loads<(RING - 2) * LOADS>();           // this wave's pieces of the next block have landed
    bare_barrier();
  }
  if (group == 0) bare_barrier();
  wait_loads<0>();                              // nothing is in flight into LDS that is used otherwise now
  bare_barrier();
  f32x4* meet = reinterpret_cast<f32x4*>(lds) + wave * (NT * TT * WAVE) + lane;
  constexpr int GROUP = MID_WAVES * NT * TT * WAVE;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) meet[group * GROUP + (i * TT + j) * WAVE] = acc[i][j];
  __syncthreads();
#pragma unroll 1
  for (int o = group; o < NT * TT; o += MID_GROUPS) {
    const f32x4 sum = meet[o * WAVE] + meet[GROUP + o * WAVE];
    const int tile = tile0 + o / TT, j = o % TT, n = tile * 16 + kg * 4, t = t0 + j * 16 + r16;
    if (part) {                                 // whole tiles in the lanes' order: 1 KiB a store, where rows of y would be 16 pieces of 64 bytes
      if (tile < tiles && t0 + j * 16 < a.T)
        reinterpret_cast<f32x4*>(part)[(((size_t)blockIdx.y * tiles + tile) * ((a.T + 15) / 16) + t0 / 16 + j) * WAVE + lane] = sum;
    } else if (t < a.T && n < a.N) {
      l4_store(a, out, t, n, sum);
    }
  }
}

// y from the slices' partial sums, in slice order
__global__ __launch_bounds__(256) void linear4_join_kernel(Linear4 a, int out, const float* __restrict__ part, int slices) {
  const int tts = (a.T + 15) / 16, tiles = (a.N + 15) / 16;
  const size_t i = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6), n_tiles = (size_t)tiles * tts;
  if (i >= n_tiles) return;
  const int lane = threadIdx.x & 63, n = (int)(i / tts) * 16 + (lane >> 4) * 4, t = (int)(i % tts) * 16 + (lane & 15);
  const f32x4* __restrict__ p = reinterpret_cast<const f32x4*>(part) + i * WAVE + lane;
  f32x4 s = p[0];
#pragma unroll 4
  for (int k = 1; k < slices; ++k) s += p[k * n_tiles * WAVE];
  if (t < a.T && n < a.N) l4_store(a, out, t, n, s);
}

// Blocks of a wave on their way: two of one tile (one token, 4096 x 11008, one, two, three: 11.7, 9.4, 10.2 us); with more tiles they cost the registers of
// a second workgroup on the compute unit (16 tokens, 12288 x 4096: 8.9 to 14.8 us).
constexpr int depth_of(int NT) { return NT == 1 ? 2 : 1; }

template <int TT, int NT, int GB>
int launch(const Linear4& a, int out, hipStream_t s) {
  const dim3 grid(ceil_div(ceil_div(a.N, 16), NT)), block(L4_WAVES * WAVE);
  if (TT > 1 && a.frag_tt) hipLaunchKernelGGL((linear4_kernel<TT, NT, GB, depth_of(NT), (TT > 1)>), grid, block, 0, s, a, out);
  else hipLaunchKernelGGL((linear4_kernel<TT, NT, GB, depth_of(NT), false>), grid, block, 0, s, a, out);
  return mlora_launch_status("linear4");
}

// How a product of more tokens is cut: row tiles of a wave, and slices of K (0 slices: the kernel for few tokens).
struct MidCut {
  int tiles, slices;
};

int mid_tt(int T) { return T <= 32 ? 2 : 4; }

// Whether the kernel for few tokens takes a product: up to 16 tokens; up to 32, where K is short and a compute unit has at most six tiles of rows, always with
// x in fragment order, of which a wave's load touches eight lines.  In rows it touches one a token, which costs the more the more tokens and the
// longer K, and is hidden the better the more rows of the weight a compute unit has.  us with 32 tokens in fragment order (17; 24; 32 in rows), that kernel / two groups
// of waves, N x K, groups of 64 and 128:
//   1024 x 1024   4.2 / 5.5 ( 4.7 /  5.5;  5.3 /  5.8;  6.3 /  5.6)     1024 x 2048  4.6 / 7.4 (5.1 /  7.6;  5.9 / 7.6;  6.5 /  7.6)
//   1024 x 4096   7.0 / 8.2 ( 7.7 /  8.3;  9.3 /  8.4; 10.2 /  8.3)     4096 x 4096  7.3 / 10.3 (7.9 / 10.4;  9.3 / 10.4; 10.5 / 10.3)
//   8192 x 4096   8.4 / 12.0 (8.7 / 13.8; 10.1 / 13.8; 11.5 / 12.0)    24576 x 4096 16.4 / 20.5 (15.0 / 20.0; 17.8 / 21.3; 17.5 / 20.8)
//   1024 x 6144   9.1 / 8.8 (10.2 /  9.0; 12.7 /  9.0; 15.0 /  9.0)     8192 x 6144 11.7 / 14.6 (12.2 / 15.3; 14.0 / 15.1; 16.0 / 14.9)
// and beyond, in fragment order: 32003 x 4096 22.3 / 21.0, 4096 x 11008 15.4 / 14.2.  In rows the rule took the side that was slower by 3 to 5 % in six of 188
// such products, by more in none.
bool few_tokens(int T, int K, int N, bool frag) {
  if (T <= 16) return true;
  if (T > 32 || K > 6144 || N > 6 * 256 * 16) return false;
  if (frag) return true;
  if (K <= 2048) return T <= 24 || N > 4096 || K <= 512 || K > 1024;
  return K <= 4096 ? (T - 16) * K <= 12 * N : N >= 4096 && (T - 16) * K <= 6 * N;
}

// The cut of the least estimated time: rounds of the 256 compute units, which hold one workgroup each, times 3 us and what a step costs - a block
// for either group, (1 + tiles) / 2 us for 64 tokens and a third less for 32 -, and for more than one slice the partial sums' write and read
// and the second launch.  Measured, us with 1, 2 and 3 tiles, then 1 tile in 2 and in 4 slices and 2 in 4 (N x K,
// groups of 64; the choice in brackets, which was the best of these in all of 27 such products):
//   64 tokens, 4096 x 4096      17.7  25.3  31.8  14.3  [12.9]  15.2      200 tokens, 12288 x 4096    52.5  50.6  [36.6]  66.0  82.6  66.2
//   64 tokens, 12288 x 4096    [18.6]  26.1  32.7  24.8  26.0  25.5      32 tokens, 4096 x 11008     29.6  43.5  56.8  19.5  [14.2]  17.7
//   128 tokens, 16384 x 4096    36.2  [28.5]  34.4  46.8  60.2  51.4      64 tokens, 4096 x 11008     39.2  59.0  75.8  25.1  [17.4]  22.6
MidCut mid_cut(int T, int K, int N, bool frag) {
  if (few_tokens(T, K, N, frag)) return {0, 0};
  const int nb = ceil_div(K, L4_BLOCK), tt = mid_tt(T);
  MidCut best = {1, 1};
  double least = 0;
  for (int tiles = 1; tiles <= 3; ++tiles)
    for (int slices = 1; slices <= 16 && (slices == 1 || 4 * slices <= nb); ++slices) {
      const long wgs = (long)ceil_div(N, 16 * MID_WAVES * tiles) * ceil_div(T, 16 * tt) * slices;
      const int steps = ceil_div(ceil_div(nb, slices), MID_GROUPS);
      const double us = (double)((wgs + 255) / 256) * (3 + steps * (tt == 4 ? 0.5 : 0.33) * (1 + tiles)) + (slices > 1 ? 2.5 + 3e-6 * slices * T * N : 0);
      if (least == 0 || us < least) {
        best = {tiles, slices};
        least = us;
      }
    }
  return best;
}

template <int TT, int NT, int GB, bool XFRAG>
int launch_mid_as(const Linear4& a, int out, int slices, float* part, hipStream_t s) {
  constexpr int ring = MID_GROUPS * mid_ring(TT, NT) * mid_stage_bytes(TT, NT), meet = MID_THREADS * NT * TT * 16, lds = ring > meet ? ring : meet;
  static const hipError_t configured = hipFuncSetAttribute((const void*)linear4_mid_kernel<TT, NT, GB, XFRAG>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (configured != hipSuccess) return mlora_set_error(MLORA_ERR_LAUNCH, "linear4: cannot reserve %d bytes of LDS: %s", lds, hipGetErrorString(configured));
  hipLaunchKernelGGL((linear4_mid_kernel<TT, NT, GB, XFRAG>), dim3(ceil_div(a.N, 16 * MID_WAVES * NT), slices, ceil_div(a.T, 16 * TT)), dim3(MID_THREADS), lds, s, a,
                     out, slices > 1 ? part : nullptr);
  if (int e = mlora_launch_status("linear4")) return e;
  if (slices > 1)
    hipLaunchKernelGGL(linear4_join_kernel, dim3((unsigned)(((long)ceil_div(a.T, 16) * ceil_div(a.N, 16) + 3) / 4)), dim3(256), 0, s, a, out, (const float*)part, slices);
  return mlora_launch_status("linear4");
}

template <int TT, int GB, bool XFRAG>
int launch_mid(const Linear4& a, int out, MidCut cut, float* part, hipStream_t s) {
  if (cut.tiles == 1) return launch_mid_as<TT, 1, GB, XFRAG>(a, out, cut.slices, part, s);
  if (cut.tiles == 2) return launch_mid_as<TT, 2, GB, XFRAG>(a, out, cut.slices, part, s);
  return launch_mid_as<TT, 3, GB, XFRAG>(a, out, cut.slices, part, s);
}

// Tiles of a workgroup up to 16 tokens: as many as leave the most loaded compute unit the fewest; of equal counts the larger, whose fewer
// workgroups read x less often.  Measured, us with 1, 2, 3, 4, 6 and 8 tiles (groups of 128; the choice in brackets):
//   1 token, 4096 x 4096    [4.7]  5.8   7.1   8.1  10.3  12.3      16 tokens, 22016 x 4096   27.7  17.4  15.1  16.2  [12.3]  14.5
//   8 tokens, 8192 x 4096    8.3  [6.4]  7.4   8.6  10.7  12.7      8 tokens, 32003 x 4096    26.1  18.6  17.9  17.1  21.0  [17.7]
//   16 tokens, 12288 x 4096 15.6  12.3  [8.6]  9.1  11.3  13.3      16 tokens, 128256 x 4096   133  81.5  69.8  66.2  63.5  [60.6]
int row_tiles(int tiles) {
  int best = 1;
  long least = 0;
  for (int nt : {1, 2, 3, 4, 6, 8}) {
    const long most = (long)nt * ceil_div(ceil_div(tiles, nt), 256);
    if (nt == 1 || most <= least) {
      best = nt;
      least = most;
    }
  }
  return best;
}

template <int TT, int GB>
int launch_rows(const Linear4& a, int out, hipStream_t s) {
  switch (row_tiles(ceil_div(a.N, 16))) {
    case 1: return launch<TT, 1, GB>(a, out, s);
    case 2: return launch<TT, 2, GB>(a, out, s);
    case 3: return launch<TT, 3, GB>(a, out, s);
    case 4: return launch<TT, 4, GB>(a, out, s);
    case 6: return launch<TT, 6, GB>(a, out, s);
    default: return launch<TT, (TT > 1 ? 4 : 8), GB>(a, out, s);
  }
}

template <int GB>
int launch_shape(const Linear4& a, int out, MidCut cut, float* part, hipStream_t s) {
  if (cut.slices == 0) return a.T <= 16 ? launch_rows<1, GB>(a, out, s) : launch_rows<2, GB>(a, out, s);
  if (a.T <= 32) return a.frag_tt ? launch_mid<2, GB, true>(a, out, cut, part, s) : launch_mid<2, GB, false>(a, out, cut, part, s);
  return a.frag_tt ? launch_mid<4, GB, true>(a, out, cut, part, s) : launch_mid<4, GB, false>(a, out, cut, part, s);
}

}  // namespace

extern "C" int mlora_linear4_sizes(int N, int K, int group, size_t* q_bytes, size_t* meta_bytes) {
  MLORA_CHECK(N > 0 && K > 0 && K % 32 == 0 && (group == 32 || group == 64 || group == 128) && K % group == 0, MLORA_ERR_UNSUPPORTED,
              "linear4: N=%d K=%d in groups of %d (K a multiple of the group: 32, 64 or 128)", N, K, group);
  const size_t blocks = (size_t)ceil_div(N, 16) * ceil_div(K, L4_BLOCK);
  if (q_bytes) *q_bytes = blocks * 1024;
  if (meta_bytes) *meta_bytes = blocks * 48 * (L4_BLOCK / group);
  return MLORA_OK;
}

static size_t partial_bytes(int slices, int T, int N) { return slices > 1 ? (size_t)slices * ceil_div(T, 16) * ceil_div(N, 16) * 256 * sizeof(float) : 0; }

extern "C" size_t mlora_linear4_workspace_bytes_of(int T, int K, int N, int x_layout) {
  return T > 0 && K > 0 && N > 0 ? partial_bytes(mid_cut(T, K, N, x_layout == MLORA_FRAG).slices, T, N) : 0;
}

extern "C" size_t mlora_linear4_workspace_bytes(int T, int K, int N) {
  const size_t rows = mlora_linear4_workspace_bytes_of(T, K, N, MLORA_ROWMAJOR), frag = mlora_linear4_workspace_bytes_of(T, K, N, MLORA_FRAG);
  return rows > frag ? rows : frag;
}

extern "C" int mlora_linear4(void* y, int y_dtype, int mode, const void* x, int x_layout, int ldx, const void* q, const void* meta, int group,
                             int T, int K, int N, void* workspace, size_t workspace_bytes, void* stream) {
  MLORA_CHECK(y && x && q && meta, MLORA_ERR_INVALID, "linear4: null pointer");
  if (int e = mlora_linear4_sizes(N, K, group, nullptr, nullptr)) return e;
  MLORA_CHECK(T >= 0 && T <= 65535 * 16 && N <= 1 << 30, MLORA_ERR_INVALID, "linear4: bad T=%d", T);
  MLORA_CHECK(y_dtype == MLORA_F16 || y_dtype == MLORA_F32, MLORA_ERR_INVALID, "linear4: bad y_dtype %d", y_dtype);
  MLORA_CHECK(mode == MLORA_STORE || (mode == MLORA_ACCUMULATE && y_dtype == MLORA_F32), MLORA_ERR_UNSUPPORTED, "linear4: results are added to fp32 alone (mode=%d)", mode);
  MLORA_CHECK(x_layout == MLORA_FRAG || (x_layout == MLORA_ROWMAJOR && ldx >= K && ldx % 8 == 0 && ldx <= 1 << 24), MLORA_ERR_INVALID, "linear4: bad x (layout=%d ldx=%d K=%d)", x_layout,
              ldx, K);
  MLORA_CHECK((((uintptr_t)x | (uintptr_t)q | (uintptr_t)meta) & 15) == 0, MLORA_ERR_INVALID, "linear4: operands not 16-byte aligned");
  MLORA_CHECK(((uintptr_t)y & (y_dtype == MLORA_F32 ? 3 : 1)) == 0, MLORA_ERR_INVALID, "linear4: y not aligned to its elements");
  if (T == 0) return MLORA_OK;
  Linear4 a = {y, (const f16*)x, (const uint32_t*)q, (const char*)meta, ldx, x_layout == MLORA_FRAG ? mlora_frag_tiles(T) : 0, T, K, N, N % 4 == 0 && ((uintptr_t)y & 15) == 0};
  const int out = mode == MLORA_ACCUMULATE ? L4_ACC : y_dtype == MLORA_F32 ? L4_F32 : L4_F16;
  hipStream_t s = (hipStream_t)stream;
  const MidCut cut = mid_cut(T, K, N, a.frag_tt > 0);
  const size_t need = partial_bytes(cut.slices, T, N);
  MLORA_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), MLORA_ERR_WORKSPACE,
              "linear4: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (group == 128) return launch_shape<1>(a, out, cut, (float*)workspace, s);
  if (group == 64) return launch_shape<2>(a, out, cut, (float*)workspace, s);
  return launch_shape<4>(a, out, cut, (float*)workspace, s);
}
