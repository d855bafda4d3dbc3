// The greedy token of every row under its request's rules: penalties for tokens it has seen, biases, a grammar mask.
//
//   c[v] = times token v was generated, seen[v] = v stands in the prompt or was generated
//   z'   = (seen[v] ? (z > 0 ? z / rep : z rep) : z) - (freq c + pres [c > 0]) + the sum of the row's biases of v
//   z'   = -inf where the row's mask has no bit v;   id = lowest index of the maximum, -1 where no token is above -inf
//
// Every step is a separately rounded IEEE fp32 operation in this order, so the results are those of a plain evaluation bit for bit.
// Bound by the logits (4 V bytes read a row, 4 V more where they are asked for): 256 rows of 128256 with histories of 4096, the logits asked
// for: 61 us, 4.4 TB/s; for few rows by latency: one row of 32000 6 us, 32 rows 11 us, two launches.  The counts are made from the
// row's token history in LDS: a table of counts per row kept in memory would add half as much traffic again to a row of 128256
// tokens, while a history of 4096 is 16 KiB.  They come from integer atomics, whose order does not matter.  A workgroup's logits and
// mask words are requested ahead of that and wait in registers.
#include "common.h"

namespace {

constexpr uint32_t IN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30, GENERATED = HAS_BIAS - 1;

struct Best {
  float v;
  int i;
};

// the greater value, the lower index of equal ones; NaN never wins
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

// A wave's maximum and the lowest index that has it: rotations within the rows of 16 lanes, then exchanges of rows and halves (through LDS, as
// shuffles go, the two reductions of a chunk were a third of its time)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }

template <class F>
__device__ __forceinline__ uint32_t wave_all(uint32_t v, F f) {
  v = f(v, dpp<0x128>(v));                                   // row_ror:8, 4, 2, 1
  v = f(v, dpp<0x124>(v));
  v = f(v, dpp<0x122>(v));
  v = f(v, dpp<0x121>(v));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(r[0], r[1]);
}

__device__ __forceinline__ Best wave_best(Best a) {
  const float v = __uint_as_float(wave_all(__float_as_uint(a.v), [](uint32_t x, uint32_t y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); }));
  const uint32_t i = wave_all(a.v == v ? (uint32_t)a.i : 0x7fffffffu, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
  return Best{v, (int)i};
}

__device__ __forceinline__ int history_of(const mlora_logit_rules& r, int row) {
  if (!r.history) return 0;
  const int n = r.lengths[row];
  return n < 0 ? 0 : n > r.cap ? r.cap : n;
}

// a row's token, and its place in the history
__device__ __forceinline__ void finish(int32_t* ids, const mlora_logit_rules& r, int row, Best b, int n) {
  const int id = b.v > -INFINITY ? b.i : -1;
  ids[row] = id;
  if (r.append && id >= 0 && n < r.cap) {
    r.history[(size_t)row * r.cap + n] = id;
    r.lengths[row] = n + 1;
  }
}

// Workgroup (chunk, row): the row's columns first .. first + C - 1, counted from the 16-byte boundary at or before its start, so that
// every full quadruple is one aligned load.  One chunk: the whole row, and no second launch.
template <int NTH, int E>
__global__ __launch_bounds__(NTH) void token_rules_kernel(int32_t* __restrict__ ids, float* out, long ld_out, const float* logits, long ld,
                                                          mlora_logit_rules r, int V, Best* __restrict__ part) {
#pragma clang fp contract(off)
  constexpr int C = NTH * 4 * E;
  extern __shared__ __align__(16) uint32_t lds[];           // counts [C], ids and values of the row's biases
  __shared__ Best wbest[NTH / WAVE];
  const int row = blockIdx.y, tid = threadIdx.x;
  const float* z_in = logits + (size_t)row * ld;
  float* z_out = out ? out + (size_t)row * ld_out : nullptr;
  const int lead = (int)(((uintptr_t)z_in >> 2) & 3);        // columns in front of the row in its first quadruple
  const int first = blockIdx.x * C - lead;                   // column of count 0
  f32x4 z[E];
#pragma unroll
  for (int u = 0; u < E; ++u) {
    const int c = first + (u * NTH + tid) * 4;
    if (c >= 0 && c + 3 < V) z[u] = *reinterpret_cast<const f32x4*>(z_in + c);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e) z[u][e] = c + e >= 0 && c + e < V ? z_in[c + e] : -INFINITY;
  }
  const int mrow = r.masks ? r.mask_row[row] : -1;
  const bool masked = mrow >= 0 && mrow < r.n_masks;         // uniform
  uint32_t w0[E], w1[E];                                     // mask words of a quadruple's first and last column
#pragma unroll
  for (int u = 0; u < E; ++u) w0[u] = w1[u] = ~0u;
  if (masked) {
    const int W = (V + 31) >> 5;
    const uint32_t* __restrict__ words = (const uint32_t*)r.masks + (size_t)mrow * W;
#pragma unroll
    for (int u = 0; u < E; ++u) {
      const int c = first + (u * NTH + tid) * 4;
      if (c + 3 >= 0 && c < V) {
        w0[u] = words[c < 0 ? 0 : c >> 5];
        w1[u] = words[c + 3 < V ? (c + 3) >> 5 : W - 1];
      }
    }
  }
  const int n = history_of(r, row);
  const bool counted = n > 0 || r.n_bias > 0;                // uniform
  float rep = 1.f, pres = 0.f, freq = 0.f;
  uint32_t* bias_ids = lds + C;
  float* bias = reinterpret_cast<float*>(lds + C + r.n_bias);
  if (counted) {
    if (r.repetition) rep = r.repetition[row];
    if (r.presence) pres = r.presence[row];
    if (r.frequency) freq = r.frequency[row];
    const int gen = r.gen_start ? r.gen_start[row] : 0;
#pragma unroll
    for (int u = 0; u < E; ++u) *reinterpret_cast<uint4*>(lds + (u * NTH + tid) * 4) = uint4{0, 0, 0, 0};
    __syncthreads();
    for (int j = tid; j < r.n_bias; j += NTH) {
      const int v = r.bias_ids[(size_t)row * r.n_bias + j];
      bias_ids[j] = (uint32_t)v;
      bias[j] = r.bias[(size_t)row * r.n_bias + j];
      if (v >= 0 && v < V && v >= first && v < first + C) atomicOr(&lds[v - first], HAS_BIAS);
    }
    const int32_t* __restrict__ h = r.history + (size_t)row * r.cap;
    for (int j0 = tid; j0 < n; j0 += 4 * NTH) {
      int v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = j0 + u * NTH < n ? h[j0 + u * NTH] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v[u] >= 0 && v[u] < V && v[u] >= first && v[u] < first + C) {
          if (j0 + u * NTH < gen) atomicOr(&lds[v[u] - first], IN_PROMPT);
          else atomicAdd(&lds[v[u] - first], 1u);
        }
    }
    __syncthreads();
  }
  const bool wide = z_out && (((uintptr_t)z_out >> 2) & 3) == (unsigned)lead;
  Best best = {-INFINITY, 0x7fffffff};
#pragma unroll
  for (int u = 0; u < E; ++u) {
    const int c = first + (u * NTH + tid) * 4;
    if (counted) {
      const uint4 q = *reinterpret_cast<const uint4*>(lds + (u * NTH + tid) * 4);
      const uint32_t k4[4] = {q.x, q.y, q.z, q.w};
      if (q.x | q.y | q.z | q.w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = k4[e];
          if (!k) continue;
          float v = z[u][e];
          const uint32_t times = k & GENERATED;
          if (k & ~HAS_BIAS) {
            v = v > 0.f ? v / rep : v * rep;
            v = v - (freq * (float)times + (times ? pres : 0.f));
          }
          if (k & HAS_BIAS) {                                 // all entries of the token, in their order
            float sum = 0.f;
            for (int j = 0; j < r.n_bias; ++j)
              if (bias_ids[j] == (uint32_t)(c + e)) sum = sum + bias[j];
            v = v + sum;
          }
          z[u][e] = v;
        }
      }
    }
    if (masked) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = (c + e) >> 5 == c >> 5 ? w0[u] : w1[u];
        if (!((w >> ((c + e) & 31)) & 1)) z[u][e] = -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e >= 0 && c + e < V) best = better(best, Best{z[u][e], c + e});
    if (z_out) {
      if (wide && c >= 0 && c + 3 < V) *reinterpret_cast<f32x4*>(z_out + c) = z[u];
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e >= 0 && c + e < V) z_out[c + e] = z[u][e];
    }
  }
  best = wave_best(best);
  if ((tid & 63) == 0) wbest[tid >> 6] = best;
  __syncthreads();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < NTH / WAVE; ++w) best = better(best, wbest[w]);
  if (part) part[(size_t)row * gridDim.x + blockIdx.x] = best;
  else finish(ids, r, row, best, n);
}

// the chunks of a row, a wave each
__global__ __launch_bounds__(WAVE) void token_rules_join_kernel(int32_t* __restrict__ ids, mlora_logit_rules r, const Best* __restrict__ part, int chunks) {
  const int row = blockIdx.x;
  Best best = {-INFINITY, 0x7fffffff};
  for (int c = threadIdx.x; c < chunks; c += WAVE) best = better(best, part[(size_t)row * chunks + c]);
  best = wave_best(best);
  if (threadIdx.x == 0) finish(ids, r, row, best, history_of(r, row));
}

constexpr int CHUNK_THREADS = 256, ROW_THREADS = 1024;
constexpr int MAX_BIAS = 1024;

// How rows are cut: threads of a workgroup, quadruples of a thread, workgroups of a row.
struct RowCut {
  int threads, quads, chunks;
};

// A row that 16384 columns hold is one workgroup's, and needs no second launch; so is one of up to 32768 where rows are many; us of GPU time (of an eager
// call) in chunks / whole: 8 rows of 8000 7.6 / 6.0 (10.8 / 7.8), of 16000 7.4 / 8.1 (11.1 / 7.8), of 32000 7.3 / 12.1; 128 rows of 16000 9.6 / 9.5 (10.6 /
// 9.0), of 32000 13.2 / 15.4; 256 rows of 32000 21.1 / 18.4.  Chunks: four quadruples a thread while that leaves the device eight workgroups a
// compute unit or more, two below (one row of 32000: 7.5 to 6.3 us; 256 rows of 128256 with two: 62 to 73 us, each chunk reading the row's history anew).
RowCut row_cut(int B, int V) {
  auto chunks = [&](int threads, int quads) { return (int)(((long)V + 3 + threads * 4 * quads - 1) / (threads * 4 * quads)); };
  if (chunks(CHUNK_THREADS, 2) == 1) return {CHUNK_THREADS, 2, 1};
  for (int quads : {2, 4, 8})
    if (chunks(ROW_THREADS, quads) == 1 && (quads < 8 || B >= 192)) return {ROW_THREADS, quads, 1};
  const int quads = (long)B * V >= 2048l * CHUNK_THREADS * 16 ? 4 : 2;
  return {CHUNK_THREADS, quads, chunks(CHUNK_THREADS, quads)};
}

template <int NTH, int E>
int launch(dim3 grid, hipStream_t s, int32_t* ids, float* out, long ld_out, const float* logits, long ld, const mlora_logit_rules& r, int V, Best* part) {
  constexpr int counts = NTH * 4 * E * 4, most = counts + 2 * MAX_BIAS * 4;
  if constexpr (most > 64 * 1024) {
    static const hipError_t configured = hipFuncSetAttribute((const void*)token_rules_kernel<NTH, E>, hipFuncAttributeMaxDynamicSharedMemorySize, most);
    if (configured != hipSuccess) return mlora_set_error(MLORA_ERR_LAUNCH, "constrained_argmax: cannot reserve %d bytes of LDS: %s", most, hipGetErrorString(configured));
  }
  hipLaunchKernelGGL((token_rules_kernel<NTH, E>), grid, dim3(NTH), counts + 8 * (size_t)r.n_bias, s, ids, out, ld_out, logits, ld, r, V, part);
  return mlora_launch_status("constrained_argmax");
}

}  // namespace

extern "C" size_t mlora_constrained_argmax_workspace_bytes(int B, int V) {
  const int chunks = B > 0 && V > 0 ? row_cut(B, V).chunks : 0;
  return chunks > 1 ? (size_t)B * chunks * sizeof(Best) : 0;
}

extern "C" int mlora_constrained_argmax(int32_t* ids, float* out, long ld_out, const float* logits, long ld, const mlora_logit_rules* rules, int B, int V,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  MLORA_CHECK(ids && logits && rules, MLORA_ERR_INVALID, "constrained_argmax: null pointer");
  MLORA_CHECK(B >= 0 && B <= 65535 && V > 0 && V <= 1 << 30, MLORA_ERR_INVALID, "constrained_argmax: bad shape B=%d V=%d", B, V);
  MLORA_CHECK(ld >= V && (!out || ld_out >= V), MLORA_ERR_INVALID, "constrained_argmax: rows of %ld and %ld columns for V=%d", ld, ld_out, V);
  MLORA_CHECK(((uintptr_t)logits & 3) == 0 && ((uintptr_t)out & 3) == 0, MLORA_ERR_INVALID, "constrained_argmax: rows not aligned to an element");
  const mlora_logit_rules& r = *rules;
  MLORA_CHECK(!r.history || (r.lengths && r.cap > 0), MLORA_ERR_INVALID, "constrained_argmax: a history needs lengths and room (cap=%d)", r.cap);
  MLORA_CHECK(r.history || (!r.append && !r.repetition && !r.presence && !r.frequency), MLORA_ERR_INVALID, "constrained_argmax: penalties without a history");
  MLORA_CHECK(r.n_bias >= 0 && r.n_bias <= MAX_BIAS, MLORA_ERR_UNSUPPORTED, "constrained_argmax: %d biases a row, at most %d", r.n_bias, MAX_BIAS);
  MLORA_CHECK(r.n_bias == 0 || (r.bias_ids && r.bias), MLORA_ERR_INVALID, "constrained_argmax: null biases");
  MLORA_CHECK(!r.masks || (r.mask_row && r.n_masks > 0), MLORA_ERR_INVALID, "constrained_argmax: masks without their rows");
  if (B == 0) return MLORA_OK;
  hipStream_t s = (hipStream_t)stream;
  const RowCut cut = row_cut(B, V);
  const size_t need = cut.chunks > 1 ? (size_t)B * cut.chunks * sizeof(Best) : 0;
  MLORA_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 7) == 0), MLORA_ERR_WORKSPACE,
              "constrained_argmax: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const dim3 grid(cut.chunks, B);
  Best* part = need ? (Best*)workspace : nullptr;
  int e;
  if (cut.threads == CHUNK_THREADS) {
    e = cut.quads == 4 ? launch<CHUNK_THREADS, 4>(grid, s, ids, out, ld_out, logits, ld, r, V, part) : launch<CHUNK_THREADS, 2>(grid, s, ids, out, ld_out, logits, ld, r, V, part);
  } else {
    e = cut.quads == 2 ? launch<ROW_THREADS, 2>(grid, s, ids, out, ld_out, logits, ld, r, V, part)
      : cut.quads == 4 ? launch<ROW_THREADS, 4>(grid, s, ids, out, ld_out, logits, ld, r, V, part)
                       : launch<ROW_THREADS, 8>(grid, s, ids, out, ld_out, logits, ld, r, V, part);
  }
  if (e || cut.chunks == 1) return e;
  hipLaunchKernelGGL(token_rules_join_kernel, dim3(B), dim3(WAVE), 0, s, ids, r, (const Best*)workspace, cut.chunks);
  return mlora_launch_status("constrained_argmax");
}
