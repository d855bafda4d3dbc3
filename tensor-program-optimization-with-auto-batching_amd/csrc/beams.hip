// A step of a beam search: the best continuations of a request's beams, the places in which they go on, and the copies that this needs.
//
//   value(b, v) = score[b] + z[b, v] - log sum_u exp z[b, u]        candidates of a request: its beams x the vocabulary
//
// The k greatest.  Within a beam the order is that of the logits, exactly, the lower token of equal ones first; between beams values are compared in 64 bits, the lower beam of
// equal ones first, of sums of exponentials that were taken in 32 (values closer than those are exact may change places).
#include "common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_BEAMS = 16, MAX_BEST = 32;
constexpr int TILE = 1024;                    // columns that a wave holds at once

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }

// over all lanes: rotations within the rows of 16, then exchanges of rows and halves
template <class F>
__device__ __forceinline__ uint32_t wave_all(uint32_t v, F f) {
  v = f(v, dpp<0x128>(v));
  v = f(v, dpp<0x124>(v));
  v = f(v, dpp<0x122>(v));
  v = f(v, dpp<0x121>(v));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(r[0], r[1]);
}

__device__ __forceinline__ float all_max(float v) {
  return __uint_as_float(wave_all(__float_as_uint(v), [](uint32_t x, uint32_t y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); }));
}
__device__ __forceinline__ uint32_t all_min(uint32_t v) { return wave_all(v, [](uint32_t x, uint32_t y) { return x < y ? x : y; }); }

// A wave's best logits in order, one a lane: lane i < k has the i-th
struct Best {
  float z;
  int v;
};

// (z, v) takes its place behind those that are greater, or equal and of lower columns
__device__ __forceinline__ void insert(Best& b, int k, float z, int v) {
  const int lane = threadIdx.x & 63;
  const int at = __popcll(__ballot(lane < k && (b.z > z || (b.z == z && b.v < v))));
  const float uz = __uint_as_float(dpp<0x138>(__float_as_uint(b.z)));           // the lane's before
  const int uv = (int)dpp<0x138>((uint32_t)b.v);
  if (lane == at) b = Best{z, v};
  else if (lane > at) b = Best{uz, uv};
}

__device__ __forceinline__ float last(const Best& b, int k) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(b.z), k - 1)); }

// Wave (part, row): the row's tiles part * per .. of 1024 columns, of which it has one in registers and the next on its way.  64 requests of 8 beams over
// 128256 columns take 50 us, 5.3 TB/s: the rate of the memory.  4 beams over 32000: 5 us, most of it the launch and one read's latency.
__global__ __launch_bounds__(4 * WAVE) void beam_scan_kernel(Best* __restrict__ best, f32x2* __restrict__ sums, const float* __restrict__ logits, long ld,
                                                             const float* __restrict__ scores, const int32_t* __restrict__ ended, int V, int k, int parts, int per) {
  constexpr int E = TILE / (4 * WAVE);
  const int lane = threadIdx.x & 63, part = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.y;
  if (part >= parts) return;
  if ((ended && ended[row]) || !(scores[row] > -INFINITY)) return;              // uniform: the second launch does not look here
  const float* __restrict__ zr = logits + (size_t)row * ld;
  const int lead = (int)(((uintptr_t)zr >> 2) & 3);                             // tiles begin on 16 bytes
  Best b = {-INFINITY, 0x7fffffff};
  float m = -INFINITY, s = 0.f;
  f32x4 z[E], nz[E];
  auto load = [&](f32x4 (&z)[E], int tile) {
    const int c0 = tile * TILE - lead;
    if (c0 >= 0 && c0 + TILE <= V) {                                            // uniform
#pragma unroll
      for (int u = 0; u < E; ++u) z[u] = *reinterpret_cast<const f32x4*>(zr + c0 + (u * WAVE + lane) * 4);
    } else {
#pragma unroll
      for (int u = 0; u < E; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = c0 + (u * WAVE + lane) * 4 + e;
          z[u][e] = c >= 0 && c < V ? zr[c] : -INFINITY;
        }
    }
  };
  const int from = part * per, tiles = (V + lead + TILE - 1) / TILE, to = min(from + per, tiles);
  if (from < to) load(z, from);
  for (int tile = from; tile < to; ++tile) {
    if (tile + 1 < to) load(nz, tile + 1);
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < E; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, z[u][e]);
    if (top > m) {
      s *= __builtin_amdgcn_exp2f((m - top) * LOG2E);
      m = top;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < E; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((z[u][e] - base) * LOG2E);       // (the difference is exact where it counts)
    // What beats the last of the best goes in.  When more than k lanes have such a logit, the k-th of the lanes' greatest is a bound that no less one passes,
    // found by taking the greatest away k - 1 times: the columns are looked through once (50 us, above; 72 where they are for each logit that is taken).
    const float least = last(b, k);
    if (__any(top > least)) {
      float bound = least;
      if (__popcll(__ballot(top > least)) > k) {
        float t = top;
        for (int i = 1; i < k; ++i) {
          const unsigned long long first = __ballot(t == all_max(t));
          if (lane == __builtin_ctzll(first)) t = -INFINITY;
        }
        bound = all_max(t);                                                     // > least, and taken itself
      }
#pragma unroll
      for (int u = 0; u < E; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unsigned long long in = __ballot(z[u][e] > least && z[u][e] >= bound);
          while (in) {                                                          // uniform
            const int l = __builtin_ctzll(in);
            in &= in - 1;
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(z[u][e]), l));
            insert(b, k, w, tile * TILE - lead + (u * WAVE + l) * 4 + e);       // (one that is behind all of them falls off the end)
          }
        }
    }
#pragma unroll
    for (int u = 0; u < E; ++u) z[u] = nz[u];
  }
  const float M = all_max(m);
  s = wave_sum(m == -INFINITY && s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f((m - M) * LOG2E));
  const size_t at = (size_t)row * parts + part;
  if (lane < k) best[at * k + lane] = b;
  if (lane == 0) sums[at] = f32x2{M, s};
}

// A request, of which a wave each merges a beam's parts.  A candidate's place is then the number of those ahead of it: in its own beam the lanes before, for they
// are in order, and in the others, whose values fall, by halving.  8.5 us for 64 requests of 8 beams, 5.6 for one of 4 (17 and 9 with four waves a request that take out the
// greatest k times): bound by steps that wait for one another, most of them the merge's.
__global__ __launch_bounds__(MAX_BEAMS* WAVE) void beam_join_kernel(float* __restrict__ out_scores, int32_t* __restrict__ tokens, int32_t* __restrict__ parents,
                                                                    const Best* __restrict__ best, const f32x2* __restrict__ sums, const float* __restrict__ scores,
                                                                    const int32_t* __restrict__ ended, int eos, int W, int k, int parts) {
  __shared__ double value[MAX_BEAMS * MAX_BEST];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = blockIdx.x, row = r * W + w;
  const int n = parts * k;
  const float score = scores[row];
  const bool over = ended && ended[row];
  // (requested together; of a row that the first launch passed over they hold anything, and are not looked at)
  const f32x2 none = {-INFINITY, 0.f}, first = lane < parts ? sums[(size_t)row * parts + lane] : none;
  Best c = lane < n ? best[(size_t)row * n + lane] : Best{-INFINITY, 0x7fffffff};
  Best b = {-INFINITY, 0x7fffffff};
  double val = -INFINITY;
  if (!(score > -INFINITY)) {                                                   // uniform
  } else if (over) {
    if (lane == 0) b.v = eos, val = score;
  } else {
    float M = first[0];
    for (int i = lane + WAVE; i < parts; i += WAVE) M = fmaxf(M, sums[(size_t)row * parts + i][0]);
    M = all_max(M);
    double s = 0;
    for (int i = lane; i < parts; i += WAVE) {
      const f32x2 x = i == lane ? first : sums[(size_t)row * parts + i];
      s += x[0] == -INFINITY && x[1] == 0.f ? 0. : (double)x[1] * exp2(((double)x[0] - M) * 1.4426950408889634);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, WAVE);
    const double lse = M + log(s);
    for (int i0 = 0; i0 < n; i0 += WAVE) {
      if (i0 > 0) c = i0 + lane < n ? best[(size_t)row * n + i0 + lane] : Best{-INFINITY, 0x7fffffff};
      while (__any(c.z > last(b, k))) {                                         // (parts are in the order of their columns)
        const float z = all_max(c.z);
        const int v = (int)all_min(c.z == z ? (uint32_t)c.v : 0x7fffffffu);
        insert(b, k, z, v);
        if (c.v == v) c.z = -INFINITY;
      }
    }
    if (b.z > -INFINITY) val = (double)score + ((double)b.z - lse);
    if (!(val > -INFINITY)) val = -INFINITY;                                    // NaN is no candidate
  }
  if (lane < k) value[w * k + lane] = val;
  __syncthreads();
  int place = lane;                                                             // (values may be equal in 64 bits where logits are not)
  for (int o = 0; o < W; ++o) {
    if (o == w) continue;
    int n = 0;                                                                  // equal ones of an earlier beam are ahead
#pragma unroll
    for (int step = MAX_BEST; step > 0; step >>= 1)
      if (n + step <= k) {
        const double x = value[o * k + n + step - 1];
        if (x > val || (x == val && o < w)) n += step;
      }
    place += n;
  }
  const bool in = lane < k && val > -INFINITY;
  if (in && place < k) {
    out_scores[(size_t)r * k + place] = (float)val;
    tokens[(size_t)r * k + place] = b.v;
    parents[(size_t)r * k + place] = w;
  }
  const int all = __syncthreads_count(in);                                      // fewer than k candidates: none behind them
  if (w == 0 && lane >= all && lane < k) {
    out_scores[(size_t)r * k + lane] = -INFINITY;
    tokens[(size_t)r * k + lane] = parents[(size_t)r * k + lane] = -1;
  }
}

// Where a request's beams go on: a parent's first child in the parent's slot, further children in those of beams without any, whose rows of the block
// table become the parent's up to the page of the last token; that page's contents are to be copied.  A wave has a request, a lane a beam.
__global__ __launch_bounds__(WAVE) void beam_reorder_kernel(int32_t* __restrict__ new_slots, int32_t* __restrict__ src_slot, int32_t* __restrict__ dst_slot,
                                                            int32_t* __restrict__ src_page, int32_t* __restrict__ dst_page, const int32_t* __restrict__ parents,
                                                            const int32_t* __restrict__ slots, int32_t* table, const int32_t* __restrict__ pos, int W, int n_rows, int max_blocks) {
  const int lane = threadIdx.x, r = blockIdx.x, at = r * W + lane;
  const bool in = lane < W;
  int p = in ? parents[at] : -1;
  if (p >= W) p = -1;
  const int slot = in ? slots[at] : -1, ps = in ? pos[at] : -1;
  bool first = p >= 0;
  unsigned long long taken = 0;
  for (int c = 0; c < W; ++c) {
    const int q = __builtin_amdgcn_readlane(p, c);
    if (q < 0) continue;
    if (c < lane && q == p) first = false;
    taken |= 1ull << q;
  }
  // the n-th beam that does not go on in its parent's slot takes the n-th that has no child
  const unsigned long long others = __ballot(in && !first);
  int left = __popcll(others & ((1ull << lane) - 1)), dead = 0;
  for (int c = 0; c < W; ++c)
    if (!(taken >> c & 1) && left-- == 0) dead = c;
  const int from = __shfl(slot, p < 0 ? 0 : p, WAVE), block = __shfl(ps, p < 0 ? 0 : p, WAVE) >> 4;
  const int to = __shfl(slot, first ? (p < 0 ? 0 : p) : dead, WAVE);
  const bool copy = in && p >= 0 && !first && from >= 0 && from < n_rows && to >= 0 && to < n_rows && from != to;
  int sp = -1, dp = -1;
  if (copy && block >= 0 && block < max_blocks) {
    sp = table[(size_t)from * max_blocks + block];
    dp = table[(size_t)to * max_blocks + block];
    if (sp < 0 || dp < 0 || sp == dp) sp = dp = -1;
  }
  if (in) {
    new_slots[at] = to;
    src_slot[at] = copy ? from : -1;
    dst_slot[at] = copy ? to : -1;
    src_page[at] = sp;
    dst_page[at] = dp;
  }
  for (int c = 0; c < W; ++c) {
    if (!__builtin_amdgcn_readlane((int)copy, c)) continue;
    const int f = __builtin_amdgcn_readlane(from, c), t = __builtin_amdgcn_readlane(to, c), n = min(__builtin_amdgcn_readlane(block, c), max_blocks);
    for (int j = lane; j < n; j += WAVE) table[(size_t)t * max_blocks + j] = table[(size_t)f * max_blocks + j];
  }
}

// Rows copied within pools [layers][n][bytes]: a workgroup has a piece of a row, each thread 64 bytes of it on their way at once.  600 pages of 32 KiB in two
// pools of 16 layers, 1.26 GB read and written: 260 us, 4.8 TB/s, near the 5.2 of one large copy.  A step of 16 requests of 4 beams, in 32 layers: 19 us.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int MAX_POOLS = 8, PIECE = 16384;
struct Pool {
  uint8_t* p;
  size_t layer;                // bytes of a layer
  int bytes, pieces, rows;     // of a row; pieces of a row; rows
  int begin;                   // the first unit
};
struct Pools {
  Pool at[MAX_POOLS];
};

template <class T>
__device__ __forceinline__ void copy_piece(uint8_t* __restrict__ to, const uint8_t* __restrict__ from, int bytes) {
  const int n = bytes / (int)sizeof(T);
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * 4) {
    T x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < n) x[u] = reinterpret_cast<const T*>(from)[i0 + u * 256];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < n) reinterpret_cast<T*>(to)[i0 + u * 256] = x[u];
  }
}

__global__ __launch_bounds__(256) void copy_pages_kernel(Pools a, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int pairs) {
  const int unit = blockIdx.x;
  int i = 0;
#pragma unroll
  for (int k = 1; k < MAX_POOLS; ++k) i += unit >= a.at[k].begin;
  const Pool p = a.at[i];                                                       // uniform: read from the arguments
  const int u = unit - p.begin, layer = u / p.pieces, off = (u - layer * p.pieces) * PIECE, bytes = min(PIECE, p.bytes - off);
  uint8_t* base = p.p + p.layer * layer + off;
  for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
    const int s = src[pair], d = dst[pair];
    if (s < 0 || s >= p.rows || d < 0 || d >= p.rows || s == d) continue;               // uniform
    uint8_t* to = base + (size_t)d * p.bytes;
    const uint8_t* from = base + (size_t)s * p.bytes;
    const size_t all = (uintptr_t)to | (uintptr_t)from | (size_t)bytes;                 // uniform
    if ((all & 15) == 0) copy_piece<u32x4>(to, from, bytes);
    else if ((all & 3) == 0) copy_piece<uint32_t>(to, from, bytes);
    else copy_piece<uint8_t>(to, from, bytes);
  }
}

struct ScanCut {
  int parts, per;
};

// Waves of a row, and tiles of a wave
ScanCut scan_cut(int rows, int V) {
  const int tiles = (V + 3 + TILE - 1) / TILE;
  long waves = 4096 / (rows > 0 ? rows : 1);
  if (waves < 1) waves = 1;
  const int per = (int)((tiles + waves - 1) / waves);
  return {ceil_div(tiles, per), per};
}

}  // namespace

extern "C" size_t mlora_beam_select_workspace_bytes(int R, int W, int V, int k) {
  if (R <= 0 || W <= 0 || V <= 0 || k <= 0) return 0;
  return (size_t)R * W * scan_cut(R * W, V).parts * (k + 1) * sizeof(Best);
}

extern "C" int mlora_beam_select(float* out_scores, int32_t* tokens, int32_t* parents, const float* logits, long ld, const float* scores, const int32_t* ended, int eos, int R,
                                 int W, int V, int k, void* workspace, size_t workspace_bytes, void* stream) {
  MLORA_CHECK(out_scores && tokens && parents && logits && scores, MLORA_ERR_INVALID, "beam_select: null pointer");
  MLORA_CHECK(R >= 0 && V > 0 && V <= 1 << 30 && ld >= V, MLORA_ERR_INVALID, "beam_select: %d requests, rows of %ld columns for V=%d", R, ld, V);
  MLORA_CHECK(W >= 1 && W <= MAX_BEAMS && k >= 1 && k <= MAX_BEST, MLORA_ERR_UNSUPPORTED, "beam_select: %d of %d beams, at most %d of %d", k, W, MAX_BEST, MAX_BEAMS);
  MLORA_CHECK((long)R * W <= 65535, MLORA_ERR_UNSUPPORTED, "beam_select: %d requests of %d beams", R, W);
  MLORA_CHECK(!ended || (eos >= 0 && eos < V), MLORA_ERR_INVALID, "beam_select: eos=%d of %d", eos, V);
  MLORA_CHECK(((uintptr_t)logits & 3) == 0, MLORA_ERR_INVALID, "beam_select: rows not aligned to an element");
  if (R == 0) return MLORA_OK;
  const size_t need = mlora_beam_select_workspace_bytes(R, W, V, k);
  MLORA_CHECK(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need, MLORA_ERR_WORKSPACE, "beam_select: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const ScanCut cut = scan_cut(R * W, V);
  f32x2* sums = (f32x2*)workspace;
  Best* best = (Best*)(sums + (size_t)R * W * cut.parts);
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(beam_scan_kernel, dim3(ceil_div(cut.parts, 4), R * W), dim3(4 * WAVE), 0, s, best, sums, logits, ld, scores, ended, V, k, cut.parts, cut.per);
  if (int e = mlora_launch_status("beam_select")) return e;
  hipLaunchKernelGGL(beam_join_kernel, dim3(R), dim3(W * WAVE), 0, s, out_scores, tokens, parents, (const Best*)best, (const f32x2*)sums, scores, ended, eos, W, k, cut.parts);
  return mlora_launch_status("beam_select");
}

extern "C" int mlora_beam_reorder(int32_t* new_slots, int32_t* src_slot, int32_t* dst_slot, int32_t* src_page, int32_t* dst_page, const int32_t* parents, const int32_t* slots,
                                  int32_t* block_table, const int32_t* pos, int R, int W, int n_rows, int max_blocks, void* stream) {
  MLORA_CHECK(new_slots && src_slot && dst_slot && src_page && dst_page && parents && slots && block_table && pos, MLORA_ERR_INVALID, "beam_reorder: null pointer");
  MLORA_CHECK(R >= 0 && n_rows > 0 && max_blocks > 0, MLORA_ERR_INVALID, "beam_reorder: %d requests on a table of %d x %d", R, n_rows, max_blocks);
  MLORA_CHECK(W >= 1 && W <= MAX_BEAMS, MLORA_ERR_UNSUPPORTED, "beam_reorder: %d beams, at most %d", W, MAX_BEAMS);
  if (R == 0) return MLORA_OK;
  hipLaunchKernelGGL(beam_reorder_kernel, dim3(R), dim3(WAVE), 0, (hipStream_t)stream, new_slots, src_slot, dst_slot, src_page, dst_page, parents, slots, block_table, pos, W, n_rows,
                     max_blocks);
  return mlora_launch_status("beam_reorder");
}

extern "C" int mlora_copy_pages(const mlora_page_pool* pools, int n_pools, const int32_t* src, const int32_t* dst, int n, void* stream) {
  MLORA_CHECK(pools && (n == 0 || (src && dst)), MLORA_ERR_INVALID, "copy_pages: null pointer");
  MLORA_CHECK(n_pools >= 1 && n_pools <= MAX_POOLS && n >= 0, MLORA_ERR_INVALID, "copy_pages: %d rows of %d pools, at most %d", n, n_pools, MAX_POOLS);
  Pools a = {};
  long units = 0;
  for (int i = 0; i < n_pools; ++i) {
    const mlora_page_pool& p = pools[i];
    MLORA_CHECK(p.data && p.layers > 0 && p.rows > 0 && p.row_bytes > 0 && p.row_bytes <= 1l << 30, MLORA_ERR_INVALID, "copy_pages: pool %d of %d x %d rows of %ld bytes", i,
                p.layers, p.rows, p.row_bytes);
    const int pieces = (int)((p.row_bytes + PIECE - 1) / PIECE);
    a.at[i] = Pool{(uint8_t*)p.data, (size_t)p.rows * p.row_bytes, (int)p.row_bytes, pieces, p.rows, (int)units};
    units += (long)p.layers * pieces;
    MLORA_CHECK(units < 1 << 30, MLORA_ERR_UNSUPPORTED, "copy_pages: too many pieces");
  }
  for (int i = n_pools; i < MAX_POOLS; ++i) a.at[i].begin = 0x7fffffff;
  if (n == 0) return MLORA_OK;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)units, n < 65535 ? n : 65535), dim3(256), 0, (hipStream_t)stream, a, src, dst, n);
  return mlora_launch_status("copy_pages");
}
