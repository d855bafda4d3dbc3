// Decode attention for a batch whose rows share long prefixes: the pages of a prefix are read once for all the rows behind it.
//
//   out[b, h] = softmax(scale q[b, h] . K) V  over the ctx[b] cached tokens of row b
//
// A softmax over a union of ranges of tokens joins from each range's maximum m, sum l = sum exp(s - m) and o = sum exp(s - m) v:
//   M = max m_i,   out = sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.
// So the work is cut into units - (query rows, range of pages, kv head) - and a second launch joins a row's units.  Bound by the pages
// read, 4 D bytes a token and kv head: 16 rows behind 32752 tokens, 32 heads of 128 over 8: 45 us, 3.2 TB/s (39 for the units, of which 23 are
// the loads and 20 the products, half of them at a time, and the rest partial results; 6 for the join); 32 rows behind 1024 tokens, 32 heads
// over 32: 24 us, 3.1 TB/s; four rows of 16 heads of 64 behind 512: 9 us, two launches.
//
// Everywhere a wave holds a tile of 16 query rows (the G = Hq / Hkv heads of one or more requests) in the matrix-core layouts of the decode
// kernel in attention.hip: S^T = K . Q^T, then O^T += V^T . P^T, where a lane's probabilities are already the operand that it must supply
// - as two fp16 halves, so that they enter with 22 bits - and the keys of two pages fill a k-step.
//   block units  up to 64 query rows of a group: four waves share pages that come straight into an LDS ring
//   wave units   up to 16 query rows - a small group, or the pages of a single request behind its prefix: a wave for itself, the next
//                page on its way to registers
#include "lora_device.h"

namespace {

constexpr int PAGE = MLORA_PAGE_SIZE;
constexpr int SA_WAVES = 4;
constexpr int SA_ROWS = 16 * SA_WAVES;        // query rows of a block unit
constexpr int SA_RING = 3;                    // stages of two pages
constexpr int SA_RECORD = 8 + SA_ROWS;
constexpr float LOG2E = 1.4426950408889634f;

struct SharedAttn {
  f16* out;
  const f16* qkv;
  const f16* k_cache;
  const f16* v_cache;
  const int32_t* block_table;
  const int32_t* seq_ids;
  const int32_t* ctx_len;
  const int32_t* units;        // [n_units][SA_RECORD] {rows, first page, pages, slot, 0 .., then up to SA_ROWS batch rows}, the n_block block units first
  const int32_t* row_pages;    // [B] shared pages ahead of a row's own
  const int32_t* row_slots;    // [B] units over those
  float* acc;                  // [B][Hq][slots][D]
  float* ml;                   // [B][Hq][slots][2]
  int max_blocks, B, Hq, Hkv, n_pages, n_seq, n_block, n_units, own_splits, slots, frag_tt;
  float scale;                 // of scores, with log2 e: weights are powers of two
};

__device__ __forceinline__ int context_of(const SharedAttn& a, int row, int& seq) {
  seq = a.seq_ids[row];
  if (seq < 0 || seq >= a.n_seq) {
    seq = 0;
    return 0;
  }
  const int c = a.ctx_len[row];
  return c < 0 ? 0 : c > a.max_blocks * PAGE ? a.max_blocks * PAGE : c;
}

// the sequence whose table names the pages of a unit's rows (a lane each): the first that is one
__device__ __forceinline__ int sequence_of(const SharedAttn& a, const int32_t* __restrict__ d) {
  const int lane = threadIdx.x & 63;
  const int row = d[8 + lane], seq = lane < d[0] && (uint32_t)row < (uint32_t)a.B ? a.seq_ids[row] : -1;
  const unsigned long long ok = __ballot(seq >= 0 && seq < a.n_seq);
  return ok ? __builtin_amdgcn_readlane(seq, __builtin_ctzll(ok)) : 0;
}

// the maximum over the lanes of a column, i.e. over the four rows of 16 lanes: each swap exchanges rows (halves) of two copies, which then hold one
// partner each.  (Through LDS, as a shuffle goes, it is 300 cycles on the way from the scores to the weights.)
__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// a tile of 16 query rows: lane (g, col) has row col, its dims 16 db + 4 g .. + 3 of the output and a quarter of its sum
template <int D>
struct Tile {
  f16x8 q[D / 32];
  f32x4 o[D / 16];
  float m, l;
  int row, head, ctx, least, most;     // batch row and head (row < 0: no query row), context; shortest and longest context of the tile
};

template <int D>
__device__ __forceinline__ void tile_begin(Tile<D>& t, const SharedAttn& a, int row, int head) {
  const int g = (threadIdx.x & 63) >> 4;
  if (row >= a.B) row = -1;
  t.row = row;
  t.head = head;
  int unused;
  t.ctx = row >= 0 ? context_of(a, row, unused) : 0;
  t.least = row >= 0 ? t.ctx : 0x7fffffff;
  t.most = t.ctx;
  const f16* qp = a.qkv + ((size_t)(row >= 0 ? row : 0) * (a.Hq + 2 * a.Hkv) + head) * D + g * 8;
#pragma unroll
  for (int kb = 0; kb < D / 32; ++kb) t.q[kb] = row >= 0 ? ld8(qp + kb * 32) : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const int lo = __shfl_xor(t.least, o, WAVE), hi = __shfl_xor(t.most, o, WAVE);
    t.least = lo < t.least ? lo : t.least;
    t.most = hi > t.most ? hi : t.most;
  }
  t.least = __builtin_amdgcn_readfirstlane(t.least);
  t.most = __builtin_amdgcn_readfirstlane(t.most);
  t.m = -INFINITY;
  t.l = 0.f;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) t.o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// P pages pg, pg + 1, ..: keys k(p, kb) in fragment order, values v(p, db) of tokens 4 g .. + 3.  EDGE: some row may end within them, or one of
// them may be none (pages: bit p).  What then does not count is masked without branches - inside one, every value's operand would wait for
// its own read.
template <int D, int P, bool EDGE, class K, class V>
__device__ __forceinline__ void tile_step(Tile<D>& t, float scale, int pg, int pages, K k, V v) {
  f32x4 st[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    st[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) st[p] = mfma_16x16x32(k(p, kb), t.q[kb], st[p]);
  }
  uint32_t keep[P][2];                                      // of a lane's four tokens: slots behind every context hold anything
  float pm = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int first = (pg + p) * PAGE + 4 * ((int)(threadIdx.x & 63) >> 4), here = pages >> p & 1;
    if constexpr (EDGE) {
      const int n = here ? t.most - first : 0;
      keep[p][0] = n > 1 ? ~0u : n > 0 ? 0xffffu : 0u;
      keep[p][1] = n > 3 ? ~0u : n > 2 ? 0xffffu : 0u;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      st[p][e] *= scale;
      if (EDGE && (first + e >= t.ctx || !here)) st[p][e] = -INFINITY;
      pm = fmaxf(pm, st[p][e]);
    }
  }
  pm = groups_max(pm);
  if (__any(pm > t.m)) {                                    // (after the first pages seldom)
    const float m = fmaxf(t.m, pm), alpha = __builtin_amdgcn_exp2f(t.m - (EDGE && m == -INFINITY ? 0.f : m));
    t.l *= alpha;
    t.m = m;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) t.o[db] *= alpha;
  }
  const float base = t.m == -INFINITY ? 0.f : t.m;          // a row with no token yet, or none above -inf
  f16 hi[P * 4], lo[P * 4];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float w = __builtin_amdgcn_exp2f(st[p][e] - base);
      t.l += w;
      hi[p * 4 + e] = (f16)w;
      lo[p * 4 + e] = (f16)(w - (float)hi[p * 4 + e]);
    }
#pragma unroll
  for (int db = 0; db < D / 16; ++db) {
    union { f16x4 h; uint32_t u[2]; } x[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      x[p].h = v(p, db);
      if constexpr (EDGE) {
        x[p].u[0] &= keep[p][0];
        x[p].u[1] &= keep[p][1];
      }
    }
    const f16x4 x0 = x[0].h, x1 = x[P - 1].h;               // (one page: its values twice, for both halves of the weights)
    const f16x8 both = f16x8{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    if constexpr (P == 1) {
      t.o[db] = mfma_16x16x32(both, f16x8{hi[0], hi[1], hi[2], hi[3], lo[0], lo[1], lo[2], lo[3]}, t.o[db]);
    } else {
      t.o[db] = mfma_16x16x32(both, f16x8{hi[0], hi[1], hi[2], hi[3], hi[4], hi[5], hi[6], hi[7]}, t.o[db]);
      t.o[db] = mfma_16x16x32(both, f16x8{lo[0], lo[1], lo[2], lo[3], lo[4], lo[5], lo[6], lo[7]}, t.o[db]);
    }
  }
}

template <int D>
__device__ __forceinline__ void tile_end(Tile<D>& t) {
  t.l += __shfl_xor(t.l, 16, WAVE);
  t.l += __shfl_xor(t.l, 32, WAVE);
}

template <int D>
__device__ __forceinline__ void tile_store(const Tile<D>& t, const SharedAttn& a, int slot) {
  if (t.row < 0 || (uint32_t)slot >= (uint32_t)a.slots) return;
  const int g = (threadIdx.x & 63) >> 4;
  const size_t at = ((size_t)t.row * a.Hq + t.head) * a.slots + slot;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f32x4*>(a.acc + at * D + db * 16 + 4 * g) = t.o[db];
  if (g == 0) *reinterpret_cast<f32x2*>(a.ml + 2 * at) = f32x2{t.m, t.l};
}

// A page's id; -1 where the table names none
__device__ __forceinline__ int page_id(const SharedAttn& a, int id) { return id >= 0 && id < a.n_pages ? id : -1; }

template <int D>
__device__ __forceinline__ void wave_unit(const SharedAttn& a, int u, int kh) {
  constexpr int NKB = D / 32, NDB = D / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, G = a.Hq / a.Hkv;
  int seq, page0, page1, slot, row;
  if (u < a.n_units) {
    const int32_t* __restrict__ d = a.units + (size_t)SA_RECORD * u;
    page0 = d[1];
    page1 = d[1] + d[2];
    slot = d[3];
    row = col < d[0] * G ? d[8 + col / G] : -1;
    seq = sequence_of(a, d);
  } else {
    const int i = u - a.n_units, part = i % a.own_splits, b = i / a.own_splits;
    const int have = (context_of(a, b, seq) + PAGE - 1) / PAGE, from = a.row_pages[b] > 0 ? a.row_pages[b] : 0;
    const int n = have > from ? have - from : 0, per = (n + a.own_splits - 1) / a.own_splits;
    page0 = from + part * per;
    page1 = page0 + per < from + n ? page0 + per : from + n;
    slot = a.row_slots[b] + part;
    row = col < G ? b : -1;
  }
  if (page0 < 0) page0 = 0;
  if (page1 > a.max_blocks) page1 = a.max_blocks;
  const int32_t* __restrict__ bt = a.block_table + (size_t)seq * a.max_blocks;
  f16x8 k[2][NKB];
  f16x4 v[2][NDB];
  bool live[2];
  int own = -1, from = page0, to = page0;                   // the ids of up to 64 pages from .. to - 1, one a lane
  // page pg into set s; behind the last that one again, for a page that is none the first: loads without a branch, behind which the next page
  // would be waited for as well
  auto load = [&](int s, int pg) {
    int id = page_id(a, __builtin_amdgcn_readlane(own, (pg < to ? pg : to - 1) - from));
    live[s] = pg < to && id >= 0;
    id = id < 0 ? 0 : id;
    const f16* kp = a.k_cache + ((size_t)id * a.Hkv + kh) * (PAGE * D) + lane * 8;
    const f16* vp = a.v_cache + (((size_t)id * a.Hkv + kh) * D + col) * PAGE + g * 4;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) k[s][kb] = ld8(kp + kb * 512);
#pragma unroll
    for (int db = 0; db < NDB; ++db) v[s][db] = *reinterpret_cast<const f16x4*>(vp + db * 16 * PAGE);
  };
  Tile<D> t;
  tile_begin(t, a, row, kh * G + (row >= 0 ? col % G : 0));
  auto work = [&](int s, int pg) {
    if (live[s]) tile_step<D, 1, true>(t, a.scale, pg, 1, [&](int, int kb) { return k[s][kb]; }, [&](int, int db) { return v[s][db]; });   // uniform
  };
  // 64 pages at a time: the wait for ids loaded inside the loop would be one for every page on its way
  while (from < page1) {
    to = from + 64 < page1 ? from + 64 : page1;
    own = from + lane < to ? bt[from + lane] : -1;
    load(0, from);
    load(1, from + 1);
    for (int pg = from; pg < to; pg += 2) {
      work(0, pg);
      load(0, pg + 2);
      work(1, pg + 1);
      load(1, pg + 3);
    }
    from = to;
  }
  tile_end(t);
  tile_store(t, a, slot);
}

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// A wave has 16 of the query rows (of up to 32 rows two waves with half of the pages each were no faster: 5 rows of 4 heads behind 16384 tokens 25.0 us, this
// way 24.6) and fetches the keys or the values of one page of a stage, which is two.
template <int D>
__device__ __forceinline__ void block_unit(const SharedAttn& a, const int32_t* __restrict__ d, int kh, f16* ring) {
  constexpr int KP = D / 32, PE = PAGE * D, STAGE = 4 * PE;       // pieces of 1 KiB a wave fetches; elements of a page's keys; of a stage
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int G = a.Hq / a.Hkv, rows = d[0] * G, page0 = d[1] > 0 ? d[1] : 0, slot = d[3];
  const int page1 = d[1] + d[2] < a.max_blocks ? d[1] + d[2] : a.max_blocks;
  const int seq = sequence_of(a, d);
  const int32_t* __restrict__ bt = a.block_table + (size_t)seq * a.max_blocks;
  const f16* src = (wave & 1 ? a.v_cache : a.k_cache) + (size_t)kh * PE + lane * 8;
  const int r = wave * 16 + col;
  Tile<D> t;                                                // (ahead of the first pages: loads return in order)
  tile_begin(t, a, r < rows ? d[8 + r / G] : -1, kh * G + (r < rows ? r % G : 0));
  // 64 pages at a time: the wait for ids loaded inside the loop would be one for the whole ring
  for (int from = page0; from < page1; from += 64) {
    const int to = from + 64 < page1 ? from + 64 : page1;
    int own = from + lane < to ? bt[from + lane] : -1;
    asm volatile("" : "+v"(own));                           // (waited for here, not again with each of the first stages)
    int next = from;
    auto issue = [&](int slot_) {
      const int pg = next + (wave >> 1);
      int id = page_id(a, __builtin_amdgcn_readlane(own, (pg < to ? pg : to - 1) - from));
      id = id < 0 ? 0 : id;                                 // a page that is none, or behind the last: a valid address, and not multiplied
      const f16* p = src + (size_t)id * a.Hkv * PE;
      f16* l = ring + slot_ * STAGE + wave * PE;
#pragma unroll
      for (int j = 0; j < KP; ++j)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p + j * 512), (__attribute__((address_space(3))) void*)(l + j * 512), 16, 0, 0);
      next += 2;
    };
    if (from > page0) bare_barrier();                       // (everybody is done with the ring)
#pragma unroll
    for (int i = 0; i < SA_RING - 1; ++i) issue(i);
    int rd = 0, wr = SA_RING - 1;
    for (int pg = from; pg < to; pg += 2) {
      wait_loads<KP*(SA_RING - 2)>();                       // this wave's part of the stage has landed, its reads of the one before are done
      bare_barrier();
      issue(wr);
      const f16* st = ring + rd * STAGE;
      rd = rd + 1 == SA_RING ? 0 : rd + 1;
      wr = wr + 1 == SA_RING ? 0 : wr + 1;
      if (wave * 16 >= rows) continue;                      // uniform: no row of this wave exists; it takes its part in the loads
      const bool one = page_id(a, __builtin_amdgcn_readlane(own, pg - from)) >= 0;
      const bool two = pg + 1 < to && page_id(a, __builtin_amdgcn_readlane(own, pg + 1 - from)) >= 0;
      const int pages = one | two << 1;
      auto kf = [=](int p, int kb) { return ld8(st + p * 2 * PE + kb * 512 + lane * 8); };
      auto vf = [=](int p, int db) { return *reinterpret_cast<const f16x4*>(st + p * 2 * PE + PE + (db * 16 + col) * PAGE + g * 4); };
      if (pages == 3 && (pg + 2) * PAGE <= t.least) tile_step<D, 2, false>(t, a.scale, pg, pages, kf, vf);       // uniform
      else if (pages) tile_step<D, 2, true>(t, a.scale, pg, pages, kf, vf);
    }
    wait_loads<0>();                                        // the requests past the end, too, ahead of the end or of what the ring holds next
  }
  tile_end(t);
  tile_store(t, a, slot);
}

template <int D>
__global__ __launch_bounds__(SA_WAVES * WAVE, 3) void shared_attn_kernel(SharedAttn a) {
  __shared__ __align__(16) f16 ring[SA_RING * 4 * PAGE * D];
  int i = blockIdx.x;
  if (i < a.n_block * a.Hkv) {
    block_unit<D>(a, a.units + (size_t)SA_RECORD * (i / a.Hkv), i % a.Hkv, ring);
    return;
  }
  i -= a.n_block * a.Hkv;
  const int per = (a.Hkv + SA_WAVES - 1) / SA_WAVES;
  const int kh = i % per * SA_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (kh < a.Hkv) wave_unit<D>(a, a.n_block + i / per, kh);
}

// A row's units joined: W waves for a (row, head), each taking every W-th unit
template <int D, int W>
__global__ __launch_bounds__(4 * WAVE) void shared_attn_join_kernel(SharedAttn a) {
  constexpr int PER = D / WAVE;
  __shared__ float so[W > 1 ? W : 1][D], sm[W], sl[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b = blockIdx.y;
  const int h = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave, w0 = W > 1 ? wave : 0;
  if (h >= a.Hq) return;                                    // (whole workgroups where waves meet)
  const int n = a.row_slots[b] + a.own_splits < a.slots ? a.row_slots[b] + a.own_splits : a.slots;
  const size_t at = ((size_t)b * a.Hq + h) * a.slots;
  float M = -INFINITY, L = 0.f, o[PER] = {};
  for (int s0 = w0; s0 < n; s0 += 4 * W) {                  // four units at a time, requested together
    f32x2 ml[4];
    float x[4][PER];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * W;
      ml[u] = s < n ? *reinterpret_cast<const f32x2*>(a.ml + 2 * (at + s)) : f32x2{-INFINITY, 0.f};
#pragma unroll
      for (int e = 0; e < PER; ++e) x[u][e] = s < n ? a.acc[(at + s) * D + lane * PER + e] : 0.f;
    }
    float m = M;
#pragma unroll
    for (int u = 0; u < 4; ++u) m = fmaxf(m, ml[u][0]);
    const float base = m == -INFINITY ? 0.f : m, f = __builtin_amdgcn_exp2f(M - base);
    M = m;
    L *= f;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float fu = __builtin_amdgcn_exp2f(ml[u][0] - base);
      L += ml[u][1] * fu;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += x[u][e] * fu;
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < PER; ++e) so[wave][lane * PER + e] = o[e];
    if (lane == 0) {
      sm[wave] = M;
      sl[wave] = L;
    }
    __syncthreads();
    if (wave > 0) return;
    float m = sm[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, sm[w]);
    const float base = m == -INFINITY ? 0.f : m;
    L = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w] - base);
      L += sl[w] * f;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += so[w][lane * PER + e] * f;
    }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int d = lane * PER + e;
    const size_t oo = a.frag_tt ? frag_offset(b, h * D + d, a.frag_tt) : ((size_t)b * a.Hq + h) * D + d;
    a.out[oo] = (f16)(L == 0.f ? 0.f : o[e] / L);           // no token: 0; a sum that is NaN stays so
  }
}

}  // namespace

int mlora_check_attn(const char* who, int Hq, int Hkv, int D, int n_pages, int n_seq, int max_blocks);

extern "C" int mlora_shared_attn_unit_rows(void) { return SA_ROWS; }
extern "C" int mlora_shared_attn_record_ints(void) { return SA_RECORD; }

extern "C" size_t mlora_shared_attn_workspace_bytes(int B, int Hq, int D, int slots) {
  return B <= 0 || Hq <= 0 || D <= 0 || slots <= 0 ? 0 : (size_t)B * Hq * slots * (D + 2) * sizeof(float);
}

extern "C" int mlora_paged_attn_decode_shared(void* out, int out_layout, const void* qkv, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                              int max_blocks, const int32_t* seq_ids, const int32_t* ctx_len, const int32_t* units, int n_block,
                                              int n_units, const int32_t* row_pages, const int32_t* row_slots, int own_splits,
                                              int slots, int B, int Hq, int Hkv, int D, int n_pages, int n_seq, void* workspace, size_t workspace_bytes,
                                              void* stream) {
  if (int e = mlora_check_attn("paged_attn_decode_shared", Hq, Hkv, D, n_pages, n_seq, max_blocks)) return e;
  MLORA_CHECK(out && qkv && k_cache && v_cache && block_table && seq_ids && ctx_len && row_pages && row_slots, MLORA_ERR_INVALID, "paged_attn_decode_shared: null pointer");
  MLORA_CHECK(n_block >= 0 && n_units >= n_block && (n_units == 0 || units), MLORA_ERR_INVALID, "paged_attn_decode_shared: bad plan");
  MLORA_CHECK(B >= 0 && B <= 65535 && own_splits > 0 && slots >= own_splits && ((long)B * own_splits + n_units) * Hkv <= 0x7fffffff, MLORA_ERR_INVALID,
              "paged_attn_decode_shared: B=%d with %d units and %d shares of a row's own pages", B, n_units, own_splits);
  MLORA_CHECK(Hq / Hkv <= 16, MLORA_ERR_UNSUPPORTED, "paged_attn_decode_shared: more than 16 query heads per kv head (%d)", Hq / Hkv);
  MLORA_CHECK(out_layout == MLORA_ROWMAJOR || out_layout == MLORA_FRAG, MLORA_ERR_INVALID, "paged_attn_decode_shared: bad out_layout %d", out_layout);
  if (B == 0) return MLORA_OK;
  MLORA_CHECK(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= mlora_shared_attn_workspace_bytes(B, Hq, D, slots), MLORA_ERR_WORKSPACE,
              "paged_attn_decode_shared: workspace of %zu bytes, %zu needed", workspace_bytes, mlora_shared_attn_workspace_bytes(B, Hq, D, slots));
  SharedAttn a = {(f16*)out, (const f16*)qkv, (const f16*)k_cache, (const f16*)v_cache, block_table, seq_ids, ctx_len, units, row_pages, row_slots,
                  (float*)workspace, (float*)workspace + (size_t)B * Hq * slots * D, max_blocks, B, Hq, Hkv, n_pages, n_seq, n_block, n_units, own_splits, slots,
                  out_layout == MLORA_FRAG ? mlora_frag_tiles(B) : 0, LOG2E / sqrtf((float)D)};
  hipStream_t s = (hipStream_t)stream;
  const unsigned grid = (unsigned)(n_block * Hkv + ((long)B * own_splits + n_units - n_block) * ceil_div(Hkv, SA_WAVES));
  const bool many = slots > 8;                              // units of a row: a wave joins up to eight in two rounds (us, a wave / four: 2 and 3 units
                                                            // 12.3 / 12.8, 8.7 / 8.9; 9 units 8.0 / 7.5, 65 units 32.7 / 25.1)
#define MLORA_SHARED(DD)                                                                                                                          \
  do {                                                                                                                                            \
    hipLaunchKernelGGL(shared_attn_kernel<DD>, dim3(grid), dim3(SA_WAVES * WAVE), 0, s, a);                                                       \
    if (int e = mlora_launch_status("paged_attn_decode_shared")) return e;                                                                        \
    if (many) hipLaunchKernelGGL((shared_attn_join_kernel<DD, 4>), dim3(Hq, B), dim3(4 * WAVE), 0, s, a);                                         \
    else hipLaunchKernelGGL((shared_attn_join_kernel<DD, 1>), dim3(ceil_div(Hq, 4), B), dim3(4 * WAVE), 0, s, a);                                 \
  } while (0)
  if (D == 128) MLORA_SHARED(128);
  else MLORA_SHARED(64);
#undef MLORA_SHARED
  return mlora_launch_status("paged_attn_decode_shared");
}
