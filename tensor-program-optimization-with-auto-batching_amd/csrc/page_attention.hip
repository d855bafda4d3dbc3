// Attention over paged caches that hold more: pages of 8 bits, and sliding windows with sinks over those or over fp16 pages.
//
//   out[t, h] = softmax(scale q[t, h] . K) V  over the tokens that position p sees: j <= p and (j > p - window or j < sinks)
//
// Pages of 8 bits: once the 16 tokens of a page are there, its keys and its values are rounded per kv head to code * step, step = fp32(a / 127),
// a = max |x|, code = rint(127 x / a).  That can be had exactly from fp32: x and a are fp16 numbers, so 127 x / a, where it is below 2^(8 - d), is a ratio whose
// denominator is below 2^(11 + d): it is half-way between two integers or at least 2^(-12 - d) off.
// A page with an infinity or NaN has a step that is NaN.  The tokens of a sequence's last page lie unrounded in its tail.  A query sees its
// own page unrounded and the pages ahead of it in 8 bits, so results do not depend on how a prompt is cut into passes.
//
// Codes enter the matrix cores as fp16 integers (exact), steps multiply scores and a page's weighted values in fp32.
#include "common.h"

int mlora_check_attn(const char* who, int Hq, int Hkv, int D, int n_pages, int n_seq, int max_blocks);

namespace {

constexpr int PAGE = MLORA_PAGE_SIZE;
constexpr float LOG2E = 1.4426950408889634f;
// Weights enter the matrix cores as two fp16 halves, the greatest as 2^14 (2^15 with a page's factor): 22 bits, and none of them is off by more than 2^-39 of the greatest, where
// fp16 numbers end.  (With 1 for the greatest it is 2^-25: too much where small weights meet values that are 2^25 times those of the others.)
constexpr float TOP = 14.f;
constexpr float NOTHING = -1e30f;             // the maximum of no scores: below every score but -inf, whose weight stays 0

struct PageAttn {
  f16* out;
  const f16* qkv;
  void *k, *v;                 // fp16 pages as in attention.hip, or codes [n_pages][Hkv][D / 64][4][16][2][8] and [n_pages][Hkv][D / 64][4][16][4][4]
  float* step;                 // [n_pages][Hkv][2] of keys and values (8 bits)
  f16 *tail_k, *tail_v;        // [n_seq] pages in the layouts of fp16 pages (8 bits)
  const int32_t *block_table, *tok_seq, *tok_pos;
  const float *rope_cos, *rope_sin;
  float *acc, *ml;             // [T][Hq][splits][D], [T][Hq][splits][2]
  int max_blocks, max_pos, T, Hq, Hkv, n_pages, n_seq, window, sinks, splits, frag_tt;
  float scale;                 // of scores, with log2 e: weights are powers of two
};

// the maximum over the lanes of a column, i.e. over the four rows of 16 lanes
__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Eight codes as fp16 integers: a byte under the exponent of 1024 is 1024 + byte
__device__ __forceinline__ f16x8 from_codes(uint32_t a, uint32_t b) {
  union { uint32_t u[4]; f16x8 h; } x;
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  x.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x07010700u);
  x.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x07030702u);
  x.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x07010700u);
  x.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x07030702u);
  const f16 c = (f16)1152.f;
  return x.h - f16x8{c, c, c, c, c, c, c, c};
}

__device__ __forceinline__ f16x4 from_codes(uint32_t a) {
  union { uint32_t u[2]; f16x4 h; } x;
  a ^= 0x80808080u;
  x.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x07010700u);
  x.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x07030702u);
  const f16 c = (f16)1152.f;
  return x.h - f16x4{c, c, c, c};
}

// Eight pairs (x, y) of a head row, rotated.  Separately rounded products, as in attention.hip: the keys are those of the fp16 cache bit for bit.
__device__ __forceinline__ void rotate8(f16x8& x, f16x8& y, const float* __restrict__ c, const float* __restrict__ s) {
  const f32x4 c0 = *reinterpret_cast<const f32x4*>(c), c1 = *reinterpret_cast<const f32x4*>(c + 4);
  const f32x4 s0 = *reinterpret_cast<const f32x4*>(s), s1 = *reinterpret_cast<const f32x4*>(s + 4);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float cc = e < 4 ? c0[e & 3] : c1[e & 3], ss = e < 4 ? s0[e & 3] : s1[e & 3], a = (float)x[e], b = (float)y[e];
    float r1, r2;
    {
#pragma clang fp contract(off)
      r1 = a * cc - b * ss;
      r2 = b * cc + a * ss;
    }
    asm volatile("" : "+v"(r1), "+v"(r2));                 // the fp32 result exists before the conversion
    x[e] = (f16)r1;
    y[e] = (f16)r2;
  }
}

// A head row of a token as the lane (group g) of an operand holds it - dims 32 kb + 8 g .. + 7 -, rotated: both elements of a pair are the lane's own
template <int D>
__device__ __forceinline__ void load_rotated(f16x8 (&x)[D / 32], const f16* __restrict__ row, const float* __restrict__ c, const float* __restrict__ s, int g) {
  constexpr int H = D / 64;
#pragma unroll
  for (int kb = 0; kb < D / 32; ++kb) x[kb] = ld8(row + kb * 32 + g * 8);
#pragma unroll
  for (int kb = 0; kb < H; ++kb) rotate8(x[kb], x[kb + H], c + kb * 32 + g * 8, s + kb * 32 + g * 8);
}

__device__ __forceinline__ bool token_ok(const PageAttn& a, int seq, int pos) {
  return seq >= 0 && seq < a.n_seq && pos >= 0 && pos < a.max_pos && pos / PAGE < a.max_blocks;
}

// How a page's keys or values are rounded, of which a wave holds all
struct Rounding {
  float by, step;                                          // 127 / a, 0 for a page of zeros
  uint32_t keep;                                           // 0: codes are 0
  // A code in the low byte, behind others' bits.  The product by 127 / a is less than 2^-23 of itself off (two roundings).  Rounded to 21 bits it is what the quotient would be, rounded so: a quotient below
  // 2^(8 - d) is half-way between two integers or 2^(-12 - d) off at least, steps of 21 bits are 2^(-13 - d), and half-way points are among them.  Behind the sum with 1.5 2^23 the whole
  // number, ties to even, is the last bits.  (Divisions took 15 instructions a code, this takes 5: 8 prompts of 456 tokens, 32 heads, 33 us to 27.)
  __device__ __forceinline__ uint32_t bits(float x) const {
    const uint32_t y = (__float_as_uint(x * by) + 4) & ~7u;
    return __float_as_uint(__fadd_rn(__uint_as_float(y), 12582912.f)) & keep;
  }
};

// Four codes of bits() as bytes
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
}

// Of a wave's whole page: magnitudes of fp16 numbers are in the order of their bits, infinities and NaN last
template <class T, int N>
__device__ __forceinline__ Rounding rounding_of(const T (&x)[N]) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    union { T h; uint32_t u[sizeof(T) / 4]; } y = {x[i]};
#pragma unroll
    for (int e = 0; e < (int)(sizeof(T) / 4); ++e) {
      union { uint32_t u; u16x2 h; } z = {y.u[e] & 0x7fff7fffu};
      most = __builtin_elementwise_max(most, z.h);
    }
  }
  const uint32_t m = (uint32_t)wave_max((float)max(most[0], most[1]));
  union { uint16_t u; f16 h; } a = {(uint16_t)m};
  const bool bad = m >= 0x7c00, none = m == 0;
  return Rounding{bad || none ? 0.f : 127.f / (float)a.h, bad ? NAN : (float)a.h / 127.f, bad ? 0u : ~0u};
}

// A whole page of a head from a wave's operands - keys: lane (g, token) dims 32 kb + 8 g ..; values: lane (g, col) tokens 4 g .. of dims 16 db + col -
// in 8 bits
template <int D>
__device__ __forceinline__ void store_codes(const PageAttn& a, int page, int kh, const f16x8 (&k)[D / 32], const f16x4 (&v)[D / 16]) {
  const int lane = threadIdx.x & 63;
  const Rounding rk = rounding_of(k), rv = rounding_of(v);
  uint8_t* kp = (uint8_t*)a.k + ((size_t)page * a.Hkv + kh) * PAGE * D + lane * 16;
  uint8_t* vp = (uint8_t*)a.v + ((size_t)page * a.Hkv + kh) * PAGE * D + lane * 16;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    uint32_t x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x8& h = k[2 * j + e / 2];
      const f16x4& w = v[4 * j + e];
      const int at = 4 * (e % 2);
      x[e] = bytes_of(rk.bits(h[at]), rk.bits(h[at + 1]), rk.bits(h[at + 2]), rk.bits(h[at + 3]));
      y[e] = bytes_of(rv.bits(w[0]), rv.bits(w[1]), rv.bits(w[2]), rv.bits(w[3]));
    }
    *reinterpret_cast<uint4*>(kp + j * 1024) = uint4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<uint4*>(vp + j * 1024) = uint4{y[0], y[1], y[2], y[3]};
  }
  if (lane == 0) *reinterpret_cast<f32x2*>(a.step + 2 * ((size_t)page * a.Hkv + kh)) = f32x2{rk.step, rv.step};
}

// ---------------------------------------------------------------------------------------------
// One token a sequence: rotation, the new token's place in the cache, and attention.  A workgroup has a kv head of a sequence, or a share of
// its pages; its waves take them in turn, in the matrix-core layouts of the decode kernel in attention.hip.  A wave keeps two pages on their way in registers.
//
// Bound by the memory: 256 rows of 128 to 2048 tokens, 8 kv heads of 128, 579 MB in 8 bits, take 139 us (4.2 TB/s), 4 rows of 31000 55 (4.7) and 5 for the join, 48 rows that
// see 2052 tokens of fp16 pages 78 (5.2).  Equal rows (256 of 1080) take 125, only read 107: what is left are the tokens' own pages, which are dirtied in lines of 64 bytes for
// 2 or 16 of them, and a workgroup's first reads, which wait for one another.  Three or four pages on their way, loads past the caches, several kv heads a workgroup and an order
// of workgroups by chiplet: no faster, or slower.
// ---------------------------------------------------------------------------------------------
template <int D, bool Q8>
struct PageRegs {
  uint4 k[Q8 ? D / 64 : D / 32];
  uint4 v[Q8 ? D / 64 : D / 32];     // fp16: tokens 4 g .. of dims 16 (2 j) + col, then 16 (2 j + 1) + col
  f32x2 step;
  int page;                          // < 0: none
};

template <int D, bool Q8, int NW>
__global__ __launch_bounds__(NW* WAVE, 4) void page_decode_kernel(PageAttn a) {
  constexpr int NKB = D / 32, NDB = D / 16, RING = 2, NL = Q8 ? D / 64 : D / 32;
  __shared__ float sm[NW][16], sl[NW][16];
  extern __shared__ float sacc[];                           // [NW][G][D]
  const int kh = blockIdx.x, split = blockIdx.y, b = blockIdx.z, G = a.Hq / a.Hkv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int seq = a.tok_seq[b], pos = a.tok_pos[b];
  const bool ok = token_ok(a, seq, pos);                    // uniform; otherwise no token is seen
  float m = NOTHING, l = 0.f;
  f32x4 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (ok) {
    const int32_t* __restrict__ bt = a.block_table + (size_t)seq * a.max_blocks;
    const int own = pos / PAGE, slot = pos % PAGE;
    // the pages ahead of the own one: those of the sinks, then those of the window
    const int least = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, from = least / PAGE;
    const int heads = a.sinks > 0 ? min((a.sinks - 1) / PAGE + 1, from) : 0;
    const int n = heads + own - from, per = (n + a.splits - 1) / a.splits;
    const int i0 = min(split * per, n), i1 = min(i0 + per, n);
    const bool mine = split == a.splits - 1 && wave == (i1 - i0) % NW;       // the wave that has the own page
    auto page_of = [&](int i) { return i < heads ? i : from + i - heads; };
    const float* rc = a.rope_cos + (size_t)pos * (D / 2);
    const float* rs = a.rope_sin + (size_t)pos * (D / 2);
    f16x8 q[NKB];
    if (col < G) load_rotated<D>(q, a.qkv + ((size_t)b * (a.Hq + 2 * a.Hkv) + kh * G + col) * D, rc, rs, g);
    else
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) q[kb] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};

    // the scores of a page become weights: st, by `scale`, of which a lane has tokens first .. first + 3; EDGE: some may not be seen
    auto weights = [&](f32x4 st, float scale, int first, int end, f16x8& p, bool edge) {
      float pm = NOTHING;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[e] *= scale;
        if (edge && (first + e >= end || (first + e < least && first + e >= a.sinks))) st[e] = -INFINITY;
        pm = fmaxf(pm, st[e]);
      }
      if (__any(pm > m + 1.9f)) {                           // (seldom behind the first pages: m may be so far below the greatest, whose weight is below 2^15.9 then)
        const float mn = fmaxf(m, groups_max(pm)), alpha = __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
        m = mn;
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] *= alpha;
      }
      const float base = m - TOP;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = __builtin_amdgcn_exp2f(st[e] - base);
        l += w;
        p[e] = (f16)w;
        p[4 + e] = (f16)(w - (float)p[e]);
      }
    };

    if (mine) {
      int id = bt[own];
      if (id < 0 || id >= a.n_pages) id = -1;
      const bool there = Q8 || id >= 0;                     // uniform
      const f16* kp = Q8 ? a.tail_k + ((size_t)seq * a.Hkv + kh) * PAGE * D : (const f16*)a.k + ((size_t)(there ? id : 0) * a.Hkv + kh) * PAGE * D;
      const f16* vp = Q8 ? a.tail_v + ((size_t)seq * a.Hkv + kh) * PAGE * D : (const f16*)a.v + ((size_t)(there ? id : 0) * a.Hkv + kh) * PAGE * D;
      if (there) {
        f16x8 k[NKB], kn[NKB];
        f16x4 v[NDB];
        const f16* vn = a.qkv + ((size_t)b * (a.Hq + 2 * a.Hkv) + a.Hq + a.Hkv + kh) * D + col;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) k[kb] = ld8(kp + kb * 512 + lane * 8);
#pragma unroll
        for (int db = 0; db < NDB; ++db) v[db] = *reinterpret_cast<const f16x4*>(vp + (db * 16 + col) * PAGE + g * 4);
        load_rotated<D>(kn, a.qkv + ((size_t)b * (a.Hq + 2 * a.Hkv) + a.Hq + kh) * D, rc, rs, g);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
          if (col == slot) k[kb] = kn[kb];
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const f16 x = vn[db * 16];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * g + e == slot) v[db][e] = x;
        }
        if constexpr (Q8) {
          if (slot == PAGE - 1 && id >= 0) store_codes<D>(a, id, kh, k, v);
        }
        f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) st = mfma_16x16x32(k[kb], q[kb], st);
        const int first = own * PAGE + 4 * g;
        f16x8 p;
        weights(st, a.scale, first, pos + 1, p, true);
        bool see[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) see[e] = first + e <= pos && (first + e >= least || first + e < a.sinks);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          f16x4 x;                                          // (slots behind the token hold anything)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = see[e] ? v[db][e] : (f16)0.f;
          o[db] = mfma_16x16x32(f16x8{x[0], x[1], x[2], x[3], x[0], x[1], x[2], x[3]}, p, o[db]);
        }
      }
    }

    PageRegs<D, Q8> r[RING];
    // 64 pages of the wave at a time, whose ids a lane each holds
    for (int k0 = i0 + wave; k0 < i1; k0 += 64 * NW) {
      const int i = k0 + lane * NW, count = min((i1 - k0 + NW - 1) / NW, 64);
      int ids = i < i1 ? bt[page_of(i)] : -1;
      if (ids >= a.n_pages) ids = -1;
      auto load = [&](PageRegs<D, Q8>& r, int c) {
        const int id = __builtin_amdgcn_readlane(ids, c < count ? c : count - 1);
        r.page = c < count && id >= 0 ? page_of(k0 + c * NW) : -1;
        const size_t at = ((size_t)(id < 0 ? 0 : id) * a.Hkv + kh);
        if constexpr (Q8) {
          const uint8_t* kp = (const uint8_t*)a.k + at * (PAGE * D) + lane * 16;
          const uint8_t* vp = (const uint8_t*)a.v + at * (PAGE * D) + lane * 16;
#pragma unroll
          for (int j = 0; j < NL; ++j) r.k[j] = *reinterpret_cast<const uint4*>(kp + j * 1024);
#pragma unroll
          for (int j = 0; j < NL; ++j) r.v[j] = *reinterpret_cast<const uint4*>(vp + j * 1024);
          r.step = *reinterpret_cast<const f32x2*>(a.step + 2 * at);
        } else {
          const f16* kp = (const f16*)a.k + at * (PAGE * D) + lane * 8;
          const f16* vp = (const f16*)a.v + at * (PAGE * D) + col * PAGE + g * 4;
#pragma unroll
          for (int j = 0; j < NL; ++j) r.k[j] = *reinterpret_cast<const uint4*>(kp + j * 512);
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            const uint2 lo = *reinterpret_cast<const uint2*>(vp + (2 * j) * 16 * PAGE), hi = *reinterpret_cast<const uint2*>(vp + (2 * j + 1) * 16 * PAGE);
            r.v[j] = uint4{lo.x, lo.y, hi.x, hi.y};
          }
        }
      };
      auto work = [&](PageRegs<D, Q8>& r) {
        if (r.page < 0) return;                             // uniform
        f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            st = mfma_16x16x32(from_codes(r.k[j].x, r.k[j].y), q[2 * j], st);
            st = mfma_16x16x32(from_codes(r.k[j].z, r.k[j].w), q[2 * j + 1], st);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            union { uint4 u; f16x8 h; } x = {r.k[j]};
            st = mfma_16x16x32(x.h, q[j], st);
          }
        }
        const int first = r.page * PAGE + 4 * g;
        const bool edge = r.page * PAGE < least;            // uniform
        f16x8 p;
        weights(st, Q8 ? a.scale * r.step[0] : a.scale, first, 0x7fffffff, p, edge);
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            const uint32_t u[4] = {r.v[j].x, r.v[j].y, r.v[j].z, r.v[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f16x4 x = from_codes(u[i]);
              const f32x4 t = mfma_16x16x32(f16x8{x[0], x[1], x[2], x[3], x[0], x[1], x[2], x[3]}, p, f32x4{0.f, 0.f, 0.f, 0.f});
              o[4 * j + i] += t * r.step[1];
            }
          }
        } else {
          uint32_t keep[2] = {~0u, ~0u};                    // of a lane's four tokens (those that are not seen may be infinite)
          if (edge) {
            const int t0 = first, s = a.sinks;
            const auto see = [&](int t) { return t >= least || t < s; };
            keep[0] = (see(t0) ? 0xffffu : 0u) | (see(t0 + 1) ? 0xffff0000u : 0u);
            keep[1] = (see(t0 + 2) ? 0xffffu : 0u) | (see(t0 + 3) ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            union { uint32_t u[4]; f16x8 h; } x = {{r.v[j].x & keep[0], r.v[j].y & keep[1], r.v[j].x & keep[0], r.v[j].y & keep[1]}},
                                              y = {{r.v[j].z & keep[0], r.v[j].w & keep[1], r.v[j].z & keep[0], r.v[j].w & keep[1]}};
            o[2 * j] = mfma_16x16x32(x.h, p, o[2 * j]);
            o[2 * j + 1] = mfma_16x16x32(y.h, p, o[2 * j + 1]);
          }
        }
      };
#pragma unroll
      for (int u = 0; u < RING; ++u) load(r[u], u);
      for (int c = 0; c < count; c += RING) {
#pragma unroll
        for (int u = 0; u < RING; ++u) {
          work(r[u]);
          load(r[u], c + u + RING);
        }
      }
    }
    // The token is appended last, by stores that go past the caches: a wave's loads are waited for behind its stores, and 256 rows of 1080 tokens under
    // 32 / 8 heads take 125 us so, 131 with the stores ahead of the pages (114 with none: they touch 48 lines of a page for a token's two).
    if (mine) {
      const int id = bt[own];
      if (Q8 || (id >= 0 && id < a.n_pages)) {
        const size_t at = ((size_t)(Q8 ? seq : id) * a.Hkv + kh) * PAGE * D;
        f16* kp = Q8 ? a.tail_k + at : (f16*)a.k + at;
        f16* vp = Q8 ? a.tail_v + at : (f16*)a.v + at;
        const f16* row = a.qkv + ((size_t)b * (a.Hq + 2 * a.Hkv) + a.Hq + kh) * D;
        f16x8 k[NKB];
        load_rotated<D>(k, row, rc, rs, g);
        if (col == slot)
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) __builtin_nontemporal_store(k[kb], reinterpret_cast<f16x8*>(kp + kb * 512 + lane * 8));
#pragma unroll
        for (int d = lane; d < D; d += WAVE) __builtin_nontemporal_store(row[a.Hkv * D + d], vp + d * PAGE + slot);
      }
    }
  }
  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);
  if (col < G) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(&sacc[((size_t)wave * G + col) * D + db * 16 + 4 * g]) = o[db];
    if (g == 0) {
      sm[wave][col] = m;
      sl[wave][col] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * D; e += NW * WAVE) {
    const int qh = e / D, d = e % D, h = kh * G + qh;
    float M = sm[0][qh];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, sm[w][qh]);
    float L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][qh] - M);
      L += sl[w][qh] * f;
      x += sacc[((size_t)w * G + qh) * D + d] * f;
    }
    if (a.splits == 1) {
      const size_t at = a.frag_tt ? frag_offset(b, h * D + d, a.frag_tt) : ((size_t)b * a.Hq + h) * D + d;
      a.out[at] = (f16)(L == 0.f ? 0.f : x / L);            // no token: 0; a sum that is NaN stays so
    } else {
      const size_t at = ((size_t)b * a.Hq + h) * a.splits + split;
      a.acc[at * D + d] = x;
      if (d == 0) *reinterpret_cast<f32x2*>(a.ml + 2 * at) = f32x2{M, L};
    }
  }
}

// The shares of a row and head, joined by a wave
template <int D>
__global__ __launch_bounds__(4 * WAVE) void page_join_kernel(PageAttn a) {
  constexpr int PER = D / WAVE;
  const int lane = threadIdx.x & 63, h = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y;
  if (h >= a.Hq) return;
  const size_t at = ((size_t)b * a.Hq + h) * a.splits;
  float M = -INFINITY, L = 0.f, o[PER] = {};
  for (int s0 = 0; s0 < a.splits; s0 += 4) {                // four at a time, requested together
    f32x2 ml[4];
    float x[4][PER];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u;
      ml[u] = s < a.splits ? *reinterpret_cast<const f32x2*>(a.ml + 2 * (at + s)) : f32x2{-INFINITY, 0.f};
#pragma unroll
      for (int e = 0; e < PER; ++e) x[u][e] = s < a.splits ? a.acc[(at + s) * D + lane * PER + e] : 0.f;
    }
    float m = M;
#pragma unroll
    for (int u = 0; u < 4; ++u) m = fmaxf(m, ml[u][0]);
    const float f = __builtin_amdgcn_exp2f(M - m);             // (m is NOTHING at least)
    M = m;
    L *= f;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float fu = __builtin_amdgcn_exp2f(ml[u][0] - m);
      L += ml[u][1] * fu;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += x[u][e] * fu;
    }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int d = lane * PER + e;
    const size_t oo = a.frag_tt ? frag_offset(b, h * D + d, a.frag_tt) : ((size_t)b * a.Hq + h) * D + d;
    a.out[oo] = (f16)(L == 0.f ? 0.f : o[e] / L);
  }
}

// ---------------------------------------------------------------------------------------------
// Prompts.  A workgroup has 16 NW rows, each a token of the pass under one of a kv head's query heads, tokens consecutive, a wave 16 of them; the
// tokens' runs (consecutive positions of one sequence) are worked one behind the other, each over the pages that it sees, four at a time.  The waves bring
// their pieces of the next four from the cache into LDS as fp16 operands while the workgroup multiplies four.  Tokens' own pages of 8-bit caches come first, unrounded.
//
// Bound by what a SIMD's four waves issue and wait for in turn, over the same phases between two barriers (per cent of the time of 4096 tokens under a window of 1024: vector
// instructions 50, of them products 36, LDS reads 25; taken out one by one, loads, LDS reads, the softmax and the weights' second halves were 15 to 24 % each).  Those 4096 tokens,
// 32 heads over 8, take 128 us, 470 TFLOP/s; 8 prompts of 456 on 8-bit pages, 32 heads, 97, with 27 + 6 for rounding and storing; 777 tokens behind 3500, 32 heads over 8, 126
// (350 TFLOP/s) with 20 for storing and joining.  No faster: keys ahead by four or six fragments, values by four; slower: two tiles a wave (below).
// The form for 8 bits and heads of 128 keeps 17 of its values in scratch memory, which are read back for an own page, ahead of a run's blocks and behind them, not among them.
//
// Of a page's step 2^e f (1 <= f < 2), the power of two goes into the values' operand, relative to the largest so far, where it is exact, and f into the
// weights, so that two pages with steps of their own fill one matrix instruction.
// ---------------------------------------------------------------------------------------------
constexpr int NO_EXP = -1000;                 // exponent of a step that is zero or NaN

// Where a token of the pass lies: the row of position p of sequence seq, of which row t has position pos; -1: it is not in the pass
__device__ __forceinline__ int row_of(const PageAttn& a, int t, int pos, int seq, int p) {
  const long r = (long)t + p - pos;
  return r >= 0 && r < a.T && p < a.max_pos && a.tok_seq[r] == seq && a.tok_pos[r] == p ? (int)r : -1;
}

// The rows of an unrounded page (tokens p0 .. p0 + 15 of seq, of which the pass has position pos), keys or values, lane (g, token) with dims 32 kb + 8 g .. + 7 of its token:
// from the pass's row `mine` of the token, and from the tail what stands ahead of those.  Tokens that are in neither are zero.
template <int D>
__device__ __forceinline__ void load_own(const PageAttn& a, int seq, int kh, int mine, int pos, bool values, f16x8 (&x)[D / 32]) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, p0 = pos / PAGE * PAGE, HH = a.Hq + 2 * a.Hkv;
  const size_t at = ((size_t)seq * a.Hkv + kh) * PAGE * D, p = (size_t)(p0 + col) * (D / 2);
  const f16* row = a.qkv + ((size_t)(mine < 0 ? 0 : mine) * HH + a.Hq + (values ? a.Hkv : 0) + kh) * D;
  if (mine >= 0) {
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) x[kb] = ld8(row + kb * 32 + g * 8);
    if (!values)
#pragma unroll
      for (int kb = 0; kb < D / 64; ++kb) rotate8(x[kb], x[kb + D / 64], a.rope_cos + p + kb * 32 + g * 8, a.rope_sin + p + kb * 32 + g * 8);
  } else if (p0 + col < pos) {
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) {
      if (!values) x[kb] = ld8(a.tail_k + at + kb * 512 + lane * 8);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) x[kb][e] = a.tail_v[at + (size_t)(kb * 32 + g * 8 + e) * PAGE + col];
    }
  } else {
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) x[kb] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // -126 <= e <= 127

// What a tile's column does not see, of P times four tokens that begin with first[p]: those from lim on, and those ahead of lo (0 <= lo, or 0 where nothing is
// seen) but for the sinks, if there are any.  Of what it sees, the tokens of `bad` (a bit for each of the four) are NaN.
template <int P>
__device__ __forceinline__ void tile_mask(f32x4 (&st)[P], const int (&first)[P], int lim, int lo, int sinks, const uint32_t (&bad)[P], bool any_bad) {
  if (any_bad) {                                           // uniform, seldom
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (bad[p] >> e & 1) st[p][e] = NAN;
  }
  const uint32_t reach = (uint32_t)max(lim - lo, 0), few = (uint32_t)min(sinks, lim);
  if (sinks > 0) {                                         // uniform
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((uint32_t)(first[p] + e - lo) >= reach && (uint32_t)(first[p] + e) >= few) st[p][e] = -INFINITY;
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((uint32_t)(first[p] + e - lo) >= reach) st[p][e] = -INFINITY;
  }
}

// w - h, of an fp16 number in the lower or upper half of a register (the compiler converts it first)
template <int HALF>
__device__ __forceinline__ float rest_of(float w, f16x2 h) {
  union { f16x2 h; uint32_t u; } x = {h};
  float r;
  if constexpr (HALF) asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(x.u), "v"(w));
  else asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(x.u), "v"(w));
  return r;
}

// Scores of P pages under a tile's column, in units by[p] > 0, become weights, as pairs of fp16 halves, and the column's maximum and sum go on.  A page's weights
// come times 2^up[p] = 1 / share[p].
//
// m is a score that was the greatest when it was taken, and is up to SLACK below the greatest: weights are below 2^15.9, which fp16 holds, and seldom behind the first blocks is the
// greatest looked for over a column's lanes and are the accumulators rescaled (4096 tokens under a window of 1024: 129 us, 132 with a rescaling for every greater score).
template <int D, int P, bool UP>
__device__ __forceinline__ void tile_weights(const f32x4 (&st)[P], const float (&by)[P], const float (&up)[P], const float (&share)[P], float& m, float& l, f32x4 (&o)[D / 16],
                                             f16x2 (&hi)[2 * P], f16x2 (&low)[2 * P]) {
  float pm = NOTHING;
#pragma unroll
  for (int p = 0; p < P; ++p) pm = fmaxf(pm, fmaxf(fmaxf(st[p][0], st[p][1]), fmaxf(st[p][2], st[p][3])) * by[p]);
  constexpr float SLACK = UP ? 0.9f : 1.9f;
  if (__any(pm > m + SLACK)) {
    const float mn = fmaxf(m, groups_max(pm)), alpha = __builtin_amdgcn_exp2f(m - mn);
    l *= alpha;
    m = mn;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[db] *= alpha;
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const float b = UP ? up[p] - (m - TOP) : TOP - m;
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[p][e], by[p], b));
    const float sum = (w[0] + w[1]) + (w[2] + w[3]);
    l = UP ? __builtin_fmaf(sum, share[p], l) : l + sum;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f16x2 h = __builtin_convertvector((f32x2{w[2 * i], w[2 * i + 1]}), f16x2);
      hi[2 * p + i] = h;
      low[2 * p + i] = __builtin_convertvector((f32x2{rest_of<0>(w[2 * i], h), rest_of<1>(w[2 * i + 1], h)}), f16x2);
    }
  }
}

__device__ __forceinline__ f16x8 join(f16x2 a, f16x2 b, f16x2 c, f16x2 d) { return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

template <int D, bool Q8, int NW>
__global__ __launch_bounds__(NW* WAVE, 4) void page_prefill_kernel(PageAttn a) {
  constexpr int NKB = D / 32, NDB = D / 16, PE = PAGE * D, QB = 16 * NW, KLD = QB + 1, VLD = D + 8;
  constexpr int NL = Q8 ? D / 64 : D / 32, NU = 8 * NL / NW;          // KiB of a page's keys or values; pieces of 1 KiB that a wave brings of four pages
  static_assert(NU * NW == 8 * NL, "a wave's pieces are as many as another's");
  // two buffers of four pages: keys [page][kb][lane][8]; values of 8-bit pages [pair of pages][db][lane][page of the pair][4 tokens], of fp16 pages
  // [pair][32 dims][page][half of the tokens][dim][8].  Before that, of pages of 8 bits, the tokens' own keys [kb][g][token][8] and values [token][d]
  // (fp16: keys of odd pages 64 bytes on, for a read that goes over a pair of pages meets a bank once: of the 37 % of the time that LDS reads, a third less)
  constexpr int KP = Q8 ? 0 : 32, KB = 4 * PE + 2 * KP, VB = 2 * KB;         // a buffer of keys; where the values begin
  constexpr int RING = VB + 8 * PE, OWN = Q8 ? 4 * NKB * KLD * 8 + QB * VLD : 0;
  __shared__ __align__(16) f16 lds[RING > OWN ? RING : OWN];
  __shared__ uint32_t odd[2][4 * NL];                                 // tokens of a page whose values are not all finite, by piece
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int kh = blockIdx.x, split = blockIdx.z, G = a.Hq / a.Hkv, HH = a.Hq + 2 * a.Hkv;
  const int TB = QB / G, t0 = (gridDim.y - 1 - blockIdx.y) * TB, nt = min(TB, a.T - t0);       // tokens; a row of a tile is one of them under one of the kv head's heads
  // where runs begin
  constexpr int NB = QB / 64;
  unsigned long long begins[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int r = j * 64 + lane, t = t0 + r;
    bool b = false;
    if (r < nt) b = r == 0 || a.tok_seq[t] != a.tok_seq[t - 1] || a.tok_pos[t] != a.tok_pos[t - 1] + 1 || a.tok_pos[t] == 0;      // (0 behind -1, which is none)
    begins[j] = __ballot(b);
  }
  // 8 bits: the tokens' own keys and values, on their way to LDS: a thread's pairs of 8 dims of keys, and 8 dims of values
  constexpr int KI = Q8 ? QB * (D / 16) / (NW * WAVE) : 1, VI = Q8 ? 2 * KI : 1;
  f16x8 kx[KI], ky[KI], vx[VI];
  int kpos[KI];
  if (Q8 && __builtin_expect(split == 0, 1)) {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int e = threadIdx.x + i * NW * WAVE, rr = e / (D / 16), c = e % (D / 16), tt = t0 + min(rr, nt - 1);
      const f16* row = a.qkv + ((size_t)tt * HH + a.Hq + kh) * D + (c >> 2) * 32 + (c & 3) * 8;
      kx[i] = ld8(row);
      ky[i] = ld8(row + D / 2);
      const int pos = a.tok_pos[tt];
      kpos[i] = rr < nt && token_ok(a, a.tok_seq[tt], pos) ? pos : -1;
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int e = threadIdx.x + i * NW * WAVE, rr = e / (D / 8), c = e % (D / 8);
      vx[i] = ld8(a.qkv + ((size_t)(t0 + min(rr, nt - 1)) * HH + a.Hq + a.Hkv + kh) * D + c * 8);
    }
  }
  f16x8 q[NKB];
  f32x4 o[NDB];
  float m = NOTHING, l = 0.f;
  int ctok, cpos;                                                     // the column's token, nt: none, and its position, -1: none
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  {
    const int r = wave * 16 + col;
    ctok = min(r / G, nt);
    const int t = t0 + (ctok < nt ? ctok : 0), pos = a.tok_pos[t];
    cpos = ctok < nt && token_ok(a, a.tok_seq[t], pos) ? pos : -1;
    const f16* qp = a.qkv + ((size_t)t * HH + kh * G + r % G) * D;
    if (cpos < 0) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) q[kb] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
    } else if constexpr (Q8) {
      load_rotated<D>(q, qp, a.rope_cos + (size_t)pos * (D / 2), a.rope_sin + (size_t)pos * (D / 2), g);
    } else {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) q[kb] = ld8(qp + kb * 32 + g * 8);
    }
  }

  if (Q8 && __builtin_expect(split == 0, 1)) {
    // The own pages, unrounded: the tokens' keys and values by way of LDS.  (Expected, or the compiler puts this behind the loop: 8 prompts of 456 tokens, all launches, 149 us for 147)
    f16* ok = lds;
    f16* ov = lds + 4 * NKB * KLD * 8;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int e = threadIdx.x + i * NW * WAVE, rr = e / (D / 16), c = e % (D / 16), gg = c & 3, kb = c >> 2;
      if (kpos[i] < 0) continue;
      const size_t at = (size_t)kpos[i] * (D / 2) + kb * 32 + gg * 8;
      rotate8(kx[i], ky[i], a.rope_cos + at, a.rope_sin + at);
      st8(ok + ((kb * 4 + gg) * KLD + rr) * 8, kx[i]);
      st8(ok + (((kb + NKB / 2) * 4 + gg) * KLD + rr) * 8, ky[i]);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int e = threadIdx.x + i * NW * WAVE, rr = e / (D / 8), c = e % (D / 8);
      if (rr < nt) st8(ov + rr * VLD + c * 8, vx[i]);
    }
    __syncthreads();
    const int t = t0 + (ctok < nt ? ctok : 0);
    const int seq = a.tok_seq[t], own = cpos >= 0 ? cpos / PAGE : -1;
    unsigned todo = (unsigned)(__ballot(cpos >= 0) & 0xffff);
    while (todo) {                                                    // the pages of a tile's columns one behind the other
      const int c = __builtin_ctz(todo);
      const int s = __builtin_amdgcn_readlane(seq, c), p = __builtin_amdgcn_readlane(own, c), ps = __builtin_amdgcn_readlane(cpos, c);
      const int row = __builtin_amdgcn_readlane(t, c), r0 = row - t0 - (ps - p * PAGE);       // where the page would begin among the workgroup's tokens
      const bool in = own == p && seq == s && t - row == cpos - ps;        // (of the same run)
      todo &= ~(unsigned)(__ballot(in) & 0xffff);
      f32x4 st[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
      f16x4 v[NDB];
      bool whole = r0 >= 0;                                           // uniform: no run begins behind its first token
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int from = max(r0 + 1 - 64 * j, 0), to = row - t0 - 64 * j;     // of begins[j], bits from .. to
        if (from <= to && from < 64 && (begins[j] >> from << from) & (to < 63 ? (2ull << to) - 1 : ~0ull)) whole = false;
      }
      if (whole) {
        const int rk = min(r0 + col, QB - 1);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) st[0] = mfma_16x16x32(ld8(ok + ((kb * 4 + g) * KLD + rk) * 8), q[kb], st[0]);
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[db][e] = ov[min(r0 + 4 * g + e, QB - 1) * VLD + db * 16 + col];
      } else {                                                        // tokens ahead of the workgroup's, of the pass or of the tail
        f16x8 vr[NKB];
        const int mine = row_of(a, row, ps, s, p * PAGE + col);
        load_own<D>(a, s, kh, mine, ps, false, vr);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) st[0] = mfma_16x16x32(vr[kb], q[kb], st[0]);
        load_own<D>(a, s, kh, mine, ps, true, vr);
        // rows to columns: the lane of (dim 16 db + col, token 4 g + e) asks lane (dim % 32 / 8, token)
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int from = (((db & 1) * 2 + (col >> 3)) << 4) + 4 * g + e;
            union { f16x8 h; uint32_t u[4]; } x = {vr[db >> 1]};
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __shfl(x.u[j], from, WAVE);
            const uint32_t w = col & 4 ? (col & 2 ? y[3] : y[2]) : (col & 2 ? y[1] : y[0]);
            union { uint16_t u; f16 h; } z = {(uint16_t)(col & 1 ? w >> 16 : w)};
            v[db][e] = z.h;
          }
      }
      uint32_t bad[1] = {0};                                          // tokens whose values are not finite: their scores are NaN where they are seen
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bool not_finite = false;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const bool y = !(fabsf((float)v[db][e]) <= 65504.f);
          not_finite = not_finite || y;
          if (y) v[db][e] = (f16)0.f;
        }
        const unsigned long long b = __ballot(not_finite);
        if (b >> (16 * g) & 0xffff) bad[0] |= 1u << e;
      }
      const float by[1] = {a.scale}, one[1] = {1.f};
      const int first[1] = {p * PAGE + 4 * g};
      f16x2 hi[2], low[2];
      tile_mask<1>(st, first, in ? cpos + 1 : 0, in && a.window > 0 ? max(cpos - a.window + 1, 0) : 0, a.sinks, bad, __any(bad[0]));
      tile_weights<D, 1, false>(st, by, one, one, m, l, o, hi, low);
      const f16x8 w = join(hi[0], hi[1], low[0], low[1]);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        o[db] = mfma_16x16x32(f16x8{v[db][0], v[db][1], v[db][2], v[db][3], v[db][0], v[db][1], v[db][2], v[db][3]}, w, o[db]);
    }
    __syncthreads();                                                  // (the ring begins)
  }
  int unit = 0;                                                       // o is in units of 2^unit
  const uint32_t page_elems = (uint32_t)a.Hkv * PE;
  const f16* k_of = (const f16*)a.k + (size_t)kh * PE;
  const f16* v_of = (const f16*)a.v + (size_t)kh * PE;

  for (int c = 0; c < nt;) {
    int next = nt;                                                    // where the run ends
#pragma unroll
    for (int j = NB - 1; j >= 0; --j) {
      const int from = c + 1 - 64 * j;
      const unsigned long long rest = from >= 64 ? 0ull : from > 0 ? begins[j] >> from << from : begins[j];
      if (rest) next = min(next, 64 * j + __builtin_ctzll(rest));
    }
    const int seq = __builtin_amdgcn_readfirstlane(a.tok_seq[t0 + c]), pc = __builtin_amdgcn_readfirstlane(a.tok_pos[t0 + c]);
    const int c0 = c;
    c = next;
    if (!token_ok(a, seq, pc)) continue;
    const int pe = min(pc + next - c0 - 1, min(a.max_pos, a.max_blocks * PAGE) - 1);
    const int32_t* __restrict__ bt = a.block_table + (size_t)seq * a.max_blocks;
    // Blocks of four of the pages that the run sees: those of the sinks, then those of the window.  fp16: in one row (4096 tokens under a window of 1024 with 4 sinks:
    // 133 us, 142 with blocks of their own for the sinks).  8 bits: blocks of their own; one row takes registers that are not there (8 prompts of 456 tokens, no window: 170 us for 165)
    const int end = Q8 ? pe / PAGE : pe / PAGE + 1;
    const int from = min(a.window > 0 && pc >= a.window ? (pc - a.window + 1) / PAGE : 0, end);
    const int heads = a.sinks > 0 ? min((a.sinks - 1) / PAGE + 1, from) : 0;
    const int head_blocks = Q8 ? (heads + 3) / 4 : 0, blocks = Q8 ? head_blocks + (end - from + 3) / 4 : (heads + end - from + 3) / 4;
    const int blk0 = (int)((long)blocks * split / a.splits), blk1 = (int)((long)blocks * (split + 1) / a.splits);
    auto page_of = [&](int blk, int p) {
      const int i = 4 * blk + p;
      if constexpr (Q8) return (blk < head_blocks ? 4 * blk : from + 4 * (blk - head_blocks)) + p;
      else return i < heads ? i : from + i - heads;
    };
    auto end_of = [&](int blk) { return Q8 && blk < head_blocks ? heads : end; };                               // where a block's pages end, at most four on
    const bool in_run = ctok >= c0 && ctok < next && cpos >= 0;
    const int lim = !in_run ? 0 : Q8 ? cpos / PAGE * PAGE : cpos + 1, lo = in_run && a.window > 0 ? max(cpos - a.window + 1, 0) : 0;
    int ends[4] = {lim, lim, in_run ? lo : 0x7fffffff, lo};
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) {
      ends[0] = min(ends[0], __shfl_xor(ends[0], s, WAVE));
      ends[1] = max(ends[1], __shfl_xor(ends[1], s, WAVE));
      ends[2] = min(ends[2], __shfl_xor(ends[2], s, WAVE));
      ends[3] = max(ends[3], __shfl_xor(ends[3], s, WAVE));
    }
    const int least_lim = __builtin_amdgcn_readfirstlane(ends[0]), most_lim = __builtin_amdgcn_readfirstlane(ends[1]);
    const int least_lo = __builtin_amdgcn_readfirstlane(ends[2]), most_lo = __builtin_amdgcn_readfirstlane(ends[3]);
    const int run_lim = Q8 ? pc / PAGE * PAGE : pc + 1, run_lo = a.window > 0 ? pe - a.window + 1 : 0;

    // of the four pages on their way: a lane's id (of page lane % 4), this wave's operands; then what the block needs beside its operands
    auto id_of = [&](int blk) {
      const int i = page_of(blk, lane & 3);
      const int id = blk < blk1 && i < end_of(blk) ? bt[i] : -1;
      return id < a.n_pages ? id : -1;
    };
    // (piece u of a block: page u / (2 NL), its keys, then its values)
    uint4 piece[Q8 ? NU : 1];
    f32x2 rstep;
    auto fetch = [&](int buf, int ids) {
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int u = wave + i * NW, p = u / (2 * NL), j = u % NL;
        const bool values = u / NL & 1;
        const int id = __builtin_amdgcn_readlane(ids, p);
        if constexpr (Q8) {
          const size_t at = ((size_t)(id < 0 ? 0 : id) * a.Hkv + kh) * PE;
          piece[i] = *reinterpret_cast<const uint4*>((const uint8_t*)(values ? a.v : a.k) + at + j * 1024 + lane * 16);
        } else {                                                      // straight into the ring
          const f16* from = (values ? v_of + (lane & 31) * PAGE + (lane >> 5) * 8 : k_of + lane * 8) + (size_t)(uint32_t)max(id, 0) * page_elems + j * 512;
          f16* to = lds + (values ? VB + buf * 4 * PE + (p >> 1) * 2 * PE + (p & 1) * 512 + j * 1024 : buf * KB + p * PE + (p + 1) / 2 * KP + j * 512);
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        }
      }
      if constexpr (Q8) rstep = *reinterpret_cast<const f32x2*>(a.step + 2 * ((size_t)(ids < 0 ? 0 : ids) * a.Hkv + kh));
    };
    int there = 0;
    // fp16: whether somebody may not see all of a block, so that its values are looked at
    auto checked = [&](int blk) {
      const int first = page_of(blk, 0) * PAGE;
      return there != 15 || first + 4 * PAGE > run_lim || (first < run_lo && first + 4 * PAGE > a.sinks);
    };
    float by[4] = {a.scale, a.scale, a.scale, a.scale}, up[4] = {0.f, 0.f, 0.f, 0.f}, share[4] = {1.f, 1.f, 1.f, 1.f};       // of the block in LDS (uniform)
    int unit_next = unit;
    uint32_t nans = 0;                                                // pages of 8 bits that are NaN
    auto stage = [&](int buf, int blk, int ids) {
      there = (int)(__ballot(ids >= 0) & 15);
      if constexpr (Q8) {
        // a lane for page lane % 4
        const int ek = (int)(__float_as_uint(rstep[0]) >> 23 & 255), ev = (int)(__float_as_uint(rstep[1]) >> 23 & 255);
        nans = (uint32_t)(__ballot(ids >= 0 && (ek == 255 || ev == 255)) & 15);
        const int ex = ids >= 0 && ev > 0 && ev < 255 ? ev - 127 : NO_EXP;
        int most = max(ex, __builtin_amdgcn_update_dpp(0, ex, 0xb1, 0xf, 0xf, false));       // over the four: lanes 1 0 3 2, then 2 3 0 1
        most = max(most, __builtin_amdgcn_update_dpp(0, most, 0x4e, 0xf, 0xf, false));
        unit_next = max(unit_next, __builtin_amdgcn_readfirstlane(most));
        const int k = ex == NO_EXP ? 0 : max(ex - unit_next, -24);    // (exact: codes have seven bits, fp16 numbers multiples of 2^-24)
        const float f = ex == NO_EXP ? 1.f : rstep[1] * power(-(unit_next + k));
        const float lane_by = ek == 255 ? 1.f : fmaxf(a.scale * rstep[0], 0x1p-126f);        // (a page of zeros: scores of zero, and -inf stays what it is)
        const float lane_up = __builtin_amdgcn_logf(f), lane_share = __builtin_amdgcn_rcpf(f);
        const float mult = ex == NO_EXP ? 0.f : power(k);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          by[p] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_by), p));
          up[p] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_up), p));
          share[p] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_share), p));
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          const int u = wave + i * NW, p = u / (2 * NL), j = u % NL;
            if (u / NL & 1) {                                         // uniform
            const f16 x = (f16)__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mult), p));
            f16* to = lds + VB + buf * 4 * PE + ((p >> 1) * NDB * 64 + lane) * 8 + (p & 1) * 4 + 4 * j * 512;
            const uint32_t y[4] = {piece[i].x, piece[i].y, piece[i].z, piece[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<f16x4*>(to + e * 512) = from_codes(y[e]) * f16x4{x, x, x, x};
          } else {
            f16* to = lds + buf * KB + p * PE + 2 * j * 512 + lane * 8;
            st8(to, from_codes(piece[i].x, piece[i].y));
            st8(to + 512, from_codes(piece[i].z, piece[i].w));
          }
        }
      } else {
        // Where somebody may not see all of a page, values that are not finite would reach those columns as well, by 0 * inf: the wave looks at what it has brought
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          const int u = wave + i * NW, p = u / (2 * NL), j = u % NL;
          if (!(u / NL & 1)) continue;
          uint32_t bad = 0;
          const int first = page_of(blk, p) * PAGE;
          if (!checked(blk)) break;                                   // uniform
          if (!(there >> p & 1) || first + PAGE > run_lim || (first < run_lo && first + PAGE > a.sinks)) {        // uniform
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            f16* at = lds + VB + buf * 4 * PE + (p >> 1) * 2 * PE + (p & 1) * 512 + j * 1024 + lane * 8;
            f16x8 x = ld8(at);
#pragma unroll
            for (int e = 0; e < 8; ++e) {                             // tokens 8 (lane / 32) + e
              const bool not_finite = !(fabsf((float)x[e]) <= 65504.f);
              if (not_finite) x[e] = (f16)0.f;
              const unsigned long long b = __ballot(not_finite);
              bad |= (uint32_t)((b & 0xffffffffull) != 0) << e | (uint32_t)(b >> 32 != 0) << (8 + e);
            }
            st8(at, x);
          }
          if (lane == 0) odd[buf][p * NL + j] = bad;
        }
      }
    };

    if (blk0 == blk1) continue;                                        // uniform over the workgroup
    int ids = id_of(blk0);
    fetch(0, ids);
    int ids_next = id_of(blk0 + 1);
    stage(0, blk0, ids);                                                 // (everybody is done with the ring: a barrier ends every block)
    __syncthreads();
    for (int blk = blk0; blk < blk1; ++blk) {
      const int buf = (blk - blk0) & 1;
      const int ids_then = id_of(blk + 2);
      if (blk + 1 < blk1) fetch(buf ^ 1, ids_next);
      if constexpr (Q8) {
        if (unit_next != unit) {                                      // uniform
          const float f = power(max(unit - unit_next, -126));
#pragma unroll
          for (int db = 0; db < NDB; ++db) o[db] *= f;
          unit = unit_next;
        }
      }
      const int first0 = page_of(blk, 0) * PAGE;                      // (of a block that has pages of both, with others between them, nobody sees all by these comparisons)
      const bool sees = first0 < most_lim && (first0 + 4 * PAGE > least_lo || first0 < a.sinks);
      bool whole = there == 15 && first0 + 4 * PAGE <= least_lim && (first0 >= most_lo || first0 + 4 * PAGE <= a.sinks);
      if (sees) {                                                     // uniform over the wave
        uint32_t bad[4];                                              // of the pages
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          bad[p] = Q8 && (nans >> p & 1) ? 0xffffu : 0u;
        }
        if (!Q8 && checked(blk)) {                                    // (148 us for 153, 4096 tokens under a window of 1024: otherwise nothing waits for these)
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            uint32_t x = 0;
#pragma unroll
            for (int j = 0; j < NL; ++j) x |= odd[buf][p * NL + j];
            bad[p] = __builtin_amdgcn_readfirstlane(x);
          }
        }
        if (bad[0] | bad[1] | bad[2] | bad[3]) whole = false;
        // Four products of scores.  8 bits: of a page each; a lane has tokens 4 g .. + 3, as its values lie.  fp16: two of a pair of pages, so that over both a lane has the
        // eight tokens that are 16 bytes of the values as they come, half g % 2 of page g / 2
        f32x4 st[4];
        const f16* kl = lds + buf * KB + (Q8 ? lane * 8 : (col >> 3) * (PE + KP) + (g * 16 + (col >> 2 & 1) * 8 + (col & 3)) * 8);
        auto keys = [&](int p, int kb) { return ld8(kl + (Q8 ? p * PE : (p >> 1) * (2 * PE + KP) + (p & 1) * 32) + kb * 512); };
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          f16x8 k[NKB];
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) k[kb] = keys(p, kb);
          st[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) st[p] = mfma_16x16x32(k[kb], q[kb], st[p]);
        }
        f16x2 hi[8], low[8];
        if (!whole) {                                                 // uniform
          int first[4], gm = g, lim_ = lim, lo_ = lo;
          asm volatile("" : "+v"(gm), "+v"(lim_), "+v"(lo_));         // (or the comparisons are made ahead of the branch that seldom leads here)
          uint32_t four[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const int page = Q8 ? p : (p & 2) + (gm >> 1), in = Q8 ? 4 * gm : 8 * (gm & 1) + 4 * (p & 1);
            first[p] = there >> page & 1 ? (Q8 ? first0 + page * PAGE : page_of(blk, page) * PAGE) + in : 0x3fffffff;
            four[p] = (Q8 ? bad[p] : gm >> 1 ? bad[p | 1] : bad[p & 2]) >> in & 15;
          }
          tile_mask<4>(st, first, lim_, lo_, first0 < a.sinks ? a.sinks : 0, four, (bad[0] | bad[1] | bad[2] | bad[3]) != 0);
        }
        tile_weights<D, 4, Q8>(st, by, up, share, m, l, o, hi, low);
        const f16* vl = lds + VB + buf * 4 * PE + (Q8 ? lane * 8 : (g >> 1) * 512 + (g & 1) * 256 + col * 8);
        auto values = [&](int j) {                                    // of pair j / NDB, dims 16 (j % NDB) ..
          const int pair = j / NDB, db = j % NDB;
          return ld8(vl + (Q8 ? (pair * NDB + db) * 512 : pair * 2 * PE + (db >> 1) * 1024 + (db & 1) * 128));
        };
        constexpr int AHEAD = 2;
        f16x8 v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) v[j] = values(j);
#pragma unroll
        for (int j = 0; j < 2 * NDB; ++j) {
          const int pair = j / NDB, db = j % NDB;
          const f16x8 x = v[j % AHEAD];
          if (j + AHEAD < 2 * NDB) v[j % AHEAD] = values(j + AHEAD);
          o[db] = mfma_16x16x32(x, join(hi[4 * pair], hi[4 * pair + 1], hi[4 * pair + 2], hi[4 * pair + 3]), o[db]);
          o[db] = mfma_16x16x32(x, join(low[4 * pair], low[4 * pair + 1], low[4 * pair + 2], low[4 * pair + 3]), o[db]);
        }
      }
      if (blk + 1 < blk1) stage(buf ^ 1, blk + 1, ids_next);
      ids_next = ids_then;
      __syncthreads();
    }
  }

  // Results go by way of LDS, a wave's tile, so that lines are written whole (everybody is done with the ring: a barrier ends every block)
  constexpr int OLD = D + 8;
  static_assert(NW * 16 * OLD <= (RING > OWN ? RING : OWN), "the tiles fit the ring");
  f16* mine = lds + wave * 16 * OLD;
  const float scale_up = power(unit);
  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);
  if (a.splits > 1) {                                                 // uniform
    if (ctok >= nt) return;
    const int t = t0 + ctok, h = kh * G + (wave * 16 + col) % G;
    const size_t at = ((size_t)t * a.Hq + h) * a.splits + split;
#pragma unroll
    for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(a.acc + at * D + db * 16 + 4 * g) = o[db] * scale_up;
    if (g == 0) *reinterpret_cast<f32x2*>(a.ml + 2 * at) = f32x2{m, l};
    return;
  }
  const float f = l == 0.f ? 0.f : scale_up / l;
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    f16x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (f16)(l == 0.f ? 0.f : o[db][e] * f);
    *reinterpret_cast<f16x4*>(mine + col * OLD + db * 16 + 4 * g) = x;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const int e = j * WAVE + lane, rr = e / (D / 8), c = e % (D / 8), row = wave * 16 + rr, tok = row / G, d = (kh * G + row % G) * D + c * 8;
    const f16x8 x = ld8(mine + rr * OLD + c * 8);
    if (tok < nt) st8(a.out + (a.frag_tt ? frag_offset(t0 + tok, d, a.frag_tt) : (size_t)(t0 + tok) * a.Hq * D + d), x);
  }
}

// Pages that a pass completes, in 8 bits: a wave has the keys or the values of 16 tokens of the pass under a kv head, and of the tokens those that are the first of their page
// in the pass.  D / 16 lanes take a token's row, so that a load's lines are whole; the codes go by way of LDS into their order.  8 prompts of 456 tokens, 32 heads of 128, 90 MB:
// 27 us, 3.3 TB/s; a page's steps (its 16 rows, the largest, codes, LDS, the store) wait for one another.  More waves a SIMD than the five of 97 registers: spills (80 registers: 37).
template <int D>
__global__ __launch_bounds__(4 * WAVE) void page_store_kernel(PageAttn a) {
  constexpr int LD = 20, NCH = D / 16, PER = WAVE / NCH, NP = 16 / PER;       // bytes of a dim's tokens in LDS, apart for the banks; lanes of a row; rows of a load; loads
  __shared__ __align__(16) uint8_t turn[4][D * LD];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, kh = blockIdx.y * 2 + (wave >> 1), t0 = blockIdx.x * 16;
  const int ch = lane % NCH, HH = a.Hq + 2 * a.Hkv;
  const bool values = wave & 1;                                       // uniform
  if (kh >= a.Hkv) return;
  // a lane knows token t0 - 16 + lane: all that the pages of the wave's tokens can reach
  const int t = t0 - 16 + lane;
  int seq = -1, pos = -1;
  if (t >= 0 && t < a.T) {
    seq = a.tok_seq[t];
    pos = a.tok_pos[t];
    if (!token_ok(a, seq, pos)) seq = -1;
  }
  const int before_seq = __shfl(seq, lane - 1, WAVE), before_pos = __shfl(pos, lane - 1, WAVE);
  const int last = (lane + PAGE - 1 - pos % PAGE) & 63, last_seq = __shfl(seq, last, WAVE), last_pos = __shfl(pos, last, WAVE);      // of its page's last token
  bool lead = lane >= 16 && lane < 32 && seq >= 0 && (pos % PAGE == 0 || before_seq != seq || before_pos != pos - 1);
  lead = lead && last_seq == seq && last_pos == pos / PAGE * PAGE + PAGE - 1;
  int page = -1;
  if (lead) page = a.block_table[(size_t)seq * a.max_blocks + pos / PAGE];
  unsigned todo = (unsigned)__ballot(lead);
  while (todo) {
    const int c = __builtin_ctz(todo);
    todo &= todo - 1;
    const int s = __builtin_amdgcn_readlane(seq, c), p = __builtin_amdgcn_readlane(pos, c), p0 = p / PAGE * PAGE;
    f16x8 x[2 * NP];                                                  // dims 8 ch .. + 7 of a token, then those half a row on
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int token = lane / NCH + PER * i, from = c + token - (p - p0);                  // the lane that knows the token
      const int from_seq = __shfl(seq, from, WAVE), from_pos = __shfl(pos, from, WAVE);
      if (from_seq == s && from_pos == p0 + token) {
        const f16* row = a.qkv + ((size_t)(t0 - 16 + from) * HH + a.Hq + (values ? a.Hkv : 0) + kh) * D + ch * 8;
        x[2 * i] = ld8(row);
        x[2 * i + 1] = ld8(row + D / 2);
        if (!values) {
          const size_t at = (size_t)(p0 + token) * (D / 2) + ch * 8;
          rotate8(x[2 * i], x[2 * i + 1], a.rope_cos + at, a.rope_sin + at);
        }
      } else {                                                        // (a page that the pass completes has its other tokens in the tail)
        const size_t at = ((size_t)s * a.Hkv + kh) * PAGE * D;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k8 = ch + h * NCH;                                // dims 8 k8 ..
          if (!values) x[2 * i + h] = ld8(a.tail_k + at + ((size_t)k8 * 16 + token) * 8);
          else
#pragma unroll
            for (int e = 0; e < 8; ++e) x[2 * i + h][e] = a.tail_v[at + (size_t)(k8 * 8 + e) * PAGE + token];
        }
      }
    }
    const int id = __builtin_amdgcn_readlane(page, c);
    if (id < 0 || id >= a.n_pages) continue;                          // uniform
    const Rounding r = rounding_of(x);
    uint8_t* at = turn[wave];
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) {
      const int token = lane / NCH + PER * (i / 2), k8 = ch + (i % 2) * NCH;
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = r.bits(x[i][e]);
      if (!values) *reinterpret_cast<uint2*>(at + (((k8 / 8) * 4 + k8 % 4) * 16 + token) * 16 + (k8 / 4 % 2) * 8) = uint2{bytes_of(y[0], y[1], y[2], y[3]), bytes_of(y[4], y[5], y[6], y[7])};
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) at[(k8 * 8 + e) * LD + token] = (uint8_t)y[e];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    uint8_t* to = (uint8_t*)(values ? a.v : a.k) + ((size_t)id * a.Hkv + kh) * PAGE * D + lane * 16;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      uint4 y;
      if (!values) y = *reinterpret_cast<const uint4*>(at + j * 1024 + lane * 16);
      else {
        const uint8_t* from = at + (64 * j + col) * LD + 4 * g;
        y = uint4{*reinterpret_cast<const uint32_t*>(from), *reinterpret_cast<const uint32_t*>(from + 16 * LD), *reinterpret_cast<const uint32_t*>(from + 32 * LD),
                  *reinterpret_cast<const uint32_t*>(from + 48 * LD)};
      }
      *reinterpret_cast<uint4*>(to + j * 1024) = y;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (lane == 0) a.step[2 * ((size_t)id * a.Hkv + kh) + values] = r.step;
  }
}

// The tokens of the pass that lie in their sequence's last page, into its tail: behind the launches that read what stands there
template <int D>
__global__ __launch_bounds__(4 * WAVE) void page_tail_kernel(PageAttn a) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, kh = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x * 16 + col;
  if (kh >= a.Hkv || t >= a.T) return;
  const int seq = a.tok_seq[t], pos = a.tok_pos[t];
  if (!token_ok(a, seq, pos) || row_of(a, t, pos, seq, pos / PAGE * PAGE + PAGE) >= 0) return;
  const f16* row = a.qkv + ((size_t)t * (a.Hq + 2 * a.Hkv) + a.Hq + kh) * D;
  f16x8 k[D / 32];
  load_rotated<D>(k, row, a.rope_cos + (size_t)pos * (D / 2), a.rope_sin + (size_t)pos * (D / 2), g);
  const size_t at = ((size_t)seq * a.Hkv + kh) * PAGE * D;
  const int slot = pos % PAGE;
#pragma unroll
  for (int kb = 0; kb < D / 32; ++kb) st8(a.tail_k + at + kb * 512 + (g * 16 + slot) * 8, k[kb]);
  const f16* vr = row + (size_t)a.Hkv * D;
#pragma unroll
  for (int kb = 0; kb < D / 32; ++kb) {
    const f16x8 v = ld8(vr + kb * 32 + g * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) a.tail_v[at + (size_t)(kb * 32 + g * 8 + e) * PAGE + slot] = v[e];
  }
}

// What pages of 8 bits stand for, as rows: a thread has eight dims of a token
template <int D>
__global__ __launch_bounds__(256) void page_values_kernel(f16* __restrict__ keys, f16* __restrict__ values, const uint8_t* __restrict__ k, const uint8_t* __restrict__ v,
                                                          const float* __restrict__ step, const int32_t* __restrict__ ids, int Hkv, int n_pages) {
  const int n = blockIdx.y, kh = blockIdx.x, id = ids[n];
  if (id < 0 || id >= n_pages) return;
  const size_t at = ((size_t)id * Hkv + kh), to = ((size_t)n * Hkv + kh) * PAGE * D;
  const float sk = step[2 * at], sv = step[2 * at + 1];
  for (int i = threadIdx.x; i < PAGE * D / 8; i += 256) {
    const int token = i / (D / 8), d = i % (D / 8) * 8, j = d / 64;
    const uint2 kc = *reinterpret_cast<const uint2*>(k + at * PAGE * D + j * 1024 + ((d % 32 / 8) * 16 + token) * 16 + (d % 64 / 32) * 8);
    const f16x8 x = from_codes(kc.x, kc.y);
    f16x8 a, b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = (f16)((float)x[e] * sk);
      b[e] = (f16)((float)(int8_t)v[at * PAGE * D + j * 1024 + ((token / 4) * 16 + d % 16 + e) * 16 + (d % 64 / 16) * 4 + token % 4] * sv);
    }
    st8(keys + to + (size_t)token * D + d, a);
    st8(values + to + (size_t)token * D + d, b);
  }
}

int check(const char* who, const mlora_page_attn& p, bool rotates) {
  if (int e = mlora_check_attn(who, p.Hq, p.Hkv, p.D, p.n_pages, p.n_seq, p.max_blocks)) return e;
  MLORA_CHECK(p.out && p.qkv && p.k && p.v && p.block_table && p.tok_seq && p.tok_pos, MLORA_ERR_INVALID, "%s: null pointer", who);
  MLORA_CHECK(!p.step || (p.tail_k && p.tail_v), MLORA_ERR_INVALID, "%s: pages of 8 bits without tails", who);
  MLORA_CHECK(!rotates || (p.rope_cos && p.rope_sin), MLORA_ERR_INVALID, "%s: null pointer", who);
  MLORA_CHECK(!rotates || (((uintptr_t)p.rope_cos | (uintptr_t)p.rope_sin) & 15) == 0, MLORA_ERR_INVALID, "%s: rotation tables not on 16 bytes", who);
  MLORA_CHECK((((uintptr_t)p.out | (uintptr_t)p.qkv | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.tail_k | (uintptr_t)p.tail_v) & 15) == 0 && ((uintptr_t)p.step & 7) == 0,
              MLORA_ERR_INVALID, "%s: tensors not on 16 bytes", who);
  MLORA_CHECK(p.T >= 0 && p.max_pos > 0 && p.max_blocks <= 1 << 26, MLORA_ERR_INVALID, "%s: bad T=%d max_pos=%d max_blocks=%d", who, p.T, p.max_pos, p.max_blocks);
  MLORA_CHECK(p.window >= 0 && p.sinks >= 0, MLORA_ERR_INVALID, "%s: a window of %d with %d sinks", who, p.window, p.sinks);
  MLORA_CHECK(p.out_layout == MLORA_ROWMAJOR || p.out_layout == MLORA_FRAG, MLORA_ERR_INVALID, "%s: bad out_layout %d", who, p.out_layout);
  MLORA_CHECK(p.splits >= 1 && p.splits <= 64 && (p.splits == 1 || p.T <= 65535), MLORA_ERR_INVALID, "%s: %d tokens in %d shares", who, p.T, p.splits);
  const size_t need = mlora_page_attn_workspace_bytes(p.T, p.Hq, p.D, p.splits);
  MLORA_CHECK(need == 0 || (p.workspace && ((uintptr_t)p.workspace & 15) == 0 && p.workspace_bytes >= need), MLORA_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, %zu needed", who, p.workspace_bytes, need);
  return MLORA_OK;
}

PageAttn args_of(const mlora_page_attn& p) {
  return PageAttn{(f16*)p.out, (const f16*)p.qkv, p.k, p.v, p.step, (f16*)p.tail_k, (f16*)p.tail_v, p.block_table, p.tok_seq, p.tok_pos, p.rope_cos, p.rope_sin,
                  (float*)p.workspace, p.workspace ? (float*)p.workspace + (size_t)p.T * p.Hq * p.splits * p.D : nullptr, p.max_blocks, p.max_pos, p.T, p.Hq, p.Hkv, p.n_pages,
                  p.n_seq, p.window, p.sinks, p.splits, p.out_layout == MLORA_FRAG ? mlora_frag_tiles(p.T) : 0, LOG2E / sqrtf((float)p.D)};
}

template <int D, bool Q8, int NW>
int launch_decode(const PageAttn& a, hipStream_t s) {
  const int G = a.Hq / a.Hkv;
  const size_t lds = (size_t)NW * G * D * sizeof(float);
  if constexpr (NW * 16 * D * 4 > 60 * 1024) {
    static const hipError_t configured = hipFuncSetAttribute((const void*)page_decode_kernel<D, Q8, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, NW * 16 * D * 4);
    if (configured != hipSuccess) return mlora_set_error(MLORA_ERR_LAUNCH, "page_attn_decode: cannot reserve LDS: %s", hipGetErrorString(configured));
  }
  hipLaunchKernelGGL((page_decode_kernel<D, Q8, NW>), dim3(a.Hkv, a.splits, a.T), dim3(NW * WAVE), lds, s, a);
  return mlora_launch_status("page_attn_decode");
}

// Few workgroups have eight waves, more than fill the device twice four: us with 8 / 4, 1 row of 300 tokens, 16 heads of 64, 5.8 / 7.1; 256 rows of 1080 tokens, 8 kv heads of 128
// (2048 workgroups), 127 / 125; 128 rows of 570, 32 heads, 149 / 141; 1024 of 1080, 8 heads, 478 / 464.
template <int D, bool Q8>
int decode(const PageAttn& a, hipStream_t s) {
  const long wgs = (long)a.T * a.Hkv * a.splits;
  const int e = wgs > 2048 ? launch_decode<D, Q8, 4>(a, s) : launch_decode<D, Q8, 8>(a, s);
  if (e || a.splits == 1) return e;
  hipLaunchKernelGGL(page_join_kernel<D>, dim3(ceil_div(a.Hq, 4), a.T), dim3(4 * WAVE), 0, s, a);
  return mlora_launch_status("page_attn_decode");
}

// Eight waves of one tile: four waves on a SIMD.  (Us at the time, so / four waves of two tiles, whose registers leave two: 8 prompts of 456 115 / 128, 777 tokens behind 3500
// 136 / 165, 4096 tokens under a window of 1024 in fp16 185 / 179)
constexpr int PREFILL_WAVES = 8, PREFILL_ROWS = 16 * PREFILL_WAVES;

template <int D, bool Q8>
int launch_prefill(const PageAttn& a, hipStream_t s) {
  const int G = a.Hq / a.Hkv;
  hipLaunchKernelGGL((page_prefill_kernel<D, Q8, PREFILL_WAVES>), dim3(a.Hkv, ceil_div(a.T, PREFILL_ROWS / G), a.splits), dim3(PREFILL_WAVES * WAVE), 0, s, a);
  if (int e = mlora_launch_status("page_attn_prefill")) return e;
  if (a.splits == 1) return MLORA_OK;
  hipLaunchKernelGGL(page_join_kernel<D>, dim3(ceil_div(a.Hq, 4), a.T), dim3(4 * WAVE), 0, s, a);
  return mlora_launch_status("page_attn_prefill");
}

template <int D>
int prefill(const PageAttn& a, hipStream_t s) {
  if (!a.step) return launch_prefill<D, false>(a, s);
  const dim3 tiles(ceil_div(a.T, 16), ceil_div(a.Hkv, 4));
  hipLaunchKernelGGL(page_store_kernel<D>, dim3(ceil_div(a.T, 16), ceil_div(a.Hkv, 2)), dim3(4 * WAVE), 0, s, a);
  if (int e = mlora_launch_status("page_attn_prefill")) return e;
  if (int e = launch_prefill<D, true>(a, s)) return e;
  hipLaunchKernelGGL(page_tail_kernel<D>, tiles, dim3(4 * WAVE), 0, s, a);
  return mlora_launch_status("page_attn_prefill");
}

}  // namespace

extern "C" int mlora_page_attn_splits(int prompt, int T, int Hq, int Hkv, int pages) {
  if (T <= 0 || Hkv <= 0 || Hq < Hkv || T > 65535) return 1;
  const int G = Hq / Hkv;
  if (prompt) {
    if (G > PREFILL_ROWS) return 1;
    // as many as run at once, two a compute unit: a round that is not full costs less than partial results do (777 tokens of 32 heads: 13 MB a share, written and read)
    const long wgs = (long)Hkv * ceil_div(T, PREFILL_ROWS / G);
    long n = 512 / wgs;
    n = n < pages / 32 ? n : pages / 32;
    return n < 1 ? 1 : n > 64 ? 64 : (int)n;
  }
  // Two workgroups a compute unit, and shares of 16 pages at least.  (us with so many / twice: 4 rows of 31000 tokens 64 / 67, 64 of 4345 116 / 121, 48 under a window of 2048
  // 86 / 93, 64 of 128 to 8192 149 / 133, 16 of 1280 to 20480 105 / 101; shares of 8 pages, one row of 4345: 17 for 14)
  const long wgs = (long)T * Hkv;
  long n = (512 + wgs - 1) / wgs;
  n = n < pages / 16 ? n : pages / 16;
  return n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

extern "C" size_t mlora_page_attn_workspace_bytes(int T, int Hq, int D, int splits) {
  return T <= 0 || Hq <= 0 || D <= 0 || splits <= 1 ? 0 : (size_t)T * Hq * splits * (D + 2) * sizeof(float);
}

extern "C" int mlora_page_attn_decode(const mlora_page_attn* args, void* stream) {
  MLORA_CHECK(args, MLORA_ERR_INVALID, "page_attn_decode: null pointer");
  const mlora_page_attn& p = *args;
  if (int e = check("page_attn_decode", p, true)) return e;
  MLORA_CHECK(p.T <= 65535, MLORA_ERR_INVALID, "page_attn_decode: %d sequences", p.T);
  MLORA_CHECK(p.Hq / p.Hkv <= 16, MLORA_ERR_UNSUPPORTED, "page_attn_decode: more than 16 query heads per kv head (%d)", p.Hq / p.Hkv);
  if (p.T == 0) return MLORA_OK;
  const PageAttn a = args_of(p);
  hipStream_t s = (hipStream_t)stream;
  if (p.D == 128) return p.step ? decode<128, true>(a, s) : decode<128, false>(a, s);
  return p.step ? decode<64, true>(a, s) : decode<64, false>(a, s);
}

extern "C" int mlora_page_attn_prefill(const mlora_page_attn* args, void* stream) {
  MLORA_CHECK(args, MLORA_ERR_INVALID, "page_attn_prefill: null pointer");
  const mlora_page_attn& p = *args;
  if (int e = check("page_attn_prefill", p, p.step != nullptr)) return e;
  MLORA_CHECK(p.Hq / p.Hkv <= 64, MLORA_ERR_UNSUPPORTED, "page_attn_prefill: more than 64 query heads per kv head (%d)", p.Hq / p.Hkv);
  MLORA_CHECK(ceil_div(p.T, PREFILL_ROWS / (p.Hq / p.Hkv)) <= 65535 && p.Hkv <= 65535, MLORA_ERR_UNSUPPORTED, "page_attn_prefill: %d tokens under %d heads", p.T, p.Hq);
  if (p.T == 0) return MLORA_OK;
  const PageAttn a = args_of(p);
  return p.D == 128 ? prefill<128>(a, (hipStream_t)stream) : prefill<64>(a, (hipStream_t)stream);
}

extern "C" int mlora_page_values(void* keys, void* values, const void* k, const void* v, const float* step, const int32_t* ids, int n, int Hkv, int D, int n_pages,
                                 void* stream) {
  MLORA_CHECK(D == 64 || D == 128, MLORA_ERR_UNSUPPORTED, "page_values: head_dim %d not in {64, 128}", D);
  MLORA_CHECK(keys && values && k && v && step && (ids || n == 0), MLORA_ERR_INVALID, "page_values: null pointer");
  MLORA_CHECK(n >= 0 && n <= 65535 && Hkv > 0 && n_pages > 0, MLORA_ERR_INVALID, "page_values: %d pages of %d under %d heads", n, n_pages, Hkv);
  if (n == 0) return MLORA_OK;
  const dim3 grid(Hkv, n);
  if (D == 128) hipLaunchKernelGGL(page_values_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, (f16*)keys, (f16*)values, (const uint8_t*)k, (const uint8_t*)v, step, ids, Hkv, n_pages);
  else hipLaunchKernelGGL(page_values_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, (f16*)keys, (f16*)values, (const uint8_t*)k, (const uint8_t*)v, step, ids, Hkv, n_pages);
  return mlora_launch_status("page_values");
}
