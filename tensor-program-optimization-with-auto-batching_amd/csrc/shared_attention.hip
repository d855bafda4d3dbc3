// Decode attention for a batch whose rows share long prefixes: the pages of a prefix are read once for all the rows behind it.
//
//   out[b, h] = softmax(scale q[b, h] . K) V  over the ctx[b] cached tokens of row b
//
// A softmax over a union of ranges of tokens joins from each range's maximum m, sum l = sum exp(s - m) and o = sum exp(s - m) v:
//   M = max m_i,   out = sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.
// So the work is cut into units - (rows, range of pages, kv head) - that a workgroup each attends over, and a second launch joins a row's units.
// A unit of a prefix has up to 128 query rows (the G = Hq / Hkv heads of every request of the group), one of the pages behind it the G
// of a single request.  Bound by the pages read, 4 D bytes a token and kv head, as long as a page serves no more than some hundred query rows.
//
// A wave holds a tile of 16 query rows and the matrix-core layouts are those of the decode kernel in attention.hip: S^T = K . Q^T, with a
// lane's four probabilities as the operand of O^T += V^T . P^T (as two fp16 halves, so that they enter with 22 bits).  The waves of a
// workgroup are R row tiles times 8 / R shares of the unit's pages.
#include "lora_device.h"

namespace {

constexpr int PAGE = MLORA_PAGE_SIZE;
constexpr int SA_WAVES = 8;
constexpr int SA_ROWS = 16 * SA_WAVES;        // query rows of a unit

struct SharedAttn {
  f16* out;
  const f16* qkv;
  const f16* k_cache;
  const f16* v_cache;
  const int32_t* block_table;
  const int32_t* seq_ids;
  const int32_t* ctx_len;
  const int32_t* units;        // [n_units][8] {first member, members, first page, pages, slot}
  const int32_t* members;      // batch rows, group after group
  const int32_t* row_pages;    // [B] shared pages ahead of a row's own
  const int32_t* row_slots;    // [B] units over those
  float* acc;                  // [B][Hq][slots][D]
  float* ml;                   // [B][Hq][slots][2]
  int max_blocks, B, Hq, Hkv, n_pages, n_seq, n_units, n_members, own_splits, slots, frag_tt;
  float scale;
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

template <int D>
__global__ __launch_bounds__(SA_WAVES * WAVE, 4) void shared_attn_kernel(SharedAttn a) {
  constexpr int NKB = D / 32, NDB = D / 16;
  __shared__ float sm[SA_WAVES][16], sl[SA_WAVES][16];
  extern __shared__ __align__(16) float sacc[];             // [SA_WAVES][16][D]
  const int kh = blockIdx.x, G = a.Hq / a.Hkv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, g = lane >> 4;
  int rows, first_member = -1, own_row = 0, page0, page1, slot, seq;
  if ((int)blockIdx.y < a.n_units) {
    const int32_t* u = a.units + 8 * blockIdx.y;
    first_member = u[0];
    rows = u[1] * G;
    page0 = u[2];
    page1 = u[2] + u[3];
    slot = u[4];
    context_of(a, a.members[first_member], seq);
  } else {
    const int i = blockIdx.y - a.n_units, part = i % a.own_splits;
    own_row = i / a.own_splits;
    rows = G;
    const int have = (context_of(a, own_row, seq) + PAGE - 1) / PAGE, from = a.row_pages[own_row];
    const int n = have > from ? have - from : 0, per = (n + a.own_splits - 1) / a.own_splits;
    page0 = from + part * per;
    page1 = page0 + per < from + n ? page0 + per : from + n;
    slot = a.row_slots[own_row] + part;
  }
  const int tiles = (rows + 15) / 16;
  const int R = tiles <= 1 ? 1 : tiles <= 2 ? 2 : tiles <= 4 ? 4 : 8;
  const int tile = wave & (R - 1), share = wave / R, shares = SA_WAVES / R;
  const int32_t* __restrict__ bt = a.block_table + (size_t)seq * a.max_blocks;
  if (page1 > a.max_blocks) page1 = a.max_blocks;

  // the lane's query row
  const int r = tile * 16 + col;
  const bool live = r < rows;
  const int row = first_member < 0 ? own_row : a.members[first_member + (live ? r / G : 0)];
  const int head = kh * G + (live ? r % G : 0);
  int unused;
  const int ctx = live ? context_of(a, row, unused) : 0;
  f16x8 qf[NKB];
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) qf[kb] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  if (live) {
    const f16* qp = a.qkv + ((size_t)row * (a.Hq + 2 * a.Hkv) + head) * D + g * 8;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) qf[kb] = ld8(qp + kb * 32);
  }
  int most = ctx;                                           // the longest context of the tile
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const int other = __shfl_xor(most, o, WAVE);
    most = other > most ? other : most;
  }

  float m = -INFINITY, l = 0.f;
  f32x4 O[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) O[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tile < tiles) {
    for (int pg = page0 + share; pg < page1; pg += shares) {
      const int page = bt[pg];
      if (page < 0 || page >= a.n_pages) continue;          // uniform
      const f16* kp = a.k_cache + ((size_t)page * a.Hkv + kh) * PAGE * D + lane * 8;
      const f16* vp = a.v_cache + (((size_t)page * a.Hkv + kh) * D + col) * PAGE + g * 4;
      f16x8 kf[NKB];
      f16x4 vf[NDB];
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) kf[kb] = ld8(kp + kb * 512);
#pragma unroll
      for (int db = 0; db < NDB; ++db) vf[db] = *reinterpret_cast<const f16x4*>(vp + db * 16 * PAGE);
      f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kb], qf[kb], st, 0, 0, 0);
      const int tok = pg * PAGE + 4 * g;
      if (pg * PAGE + PAGE > most) {                        // slots behind every context hold anything
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tok + e >= most)
#pragma unroll
            for (int db = 0; db < NDB; ++db) vf[db][e] = (f16)0.f;
      }
      float pm = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[e] = tok + e >= ctx ? -INFINITY : st[e] * a.scale;
        pm = fmaxf(pm, st[e]);
      }
      pm = fmaxf(pm, __shfl_xor(pm, 16, WAVE));
      pm = fmaxf(pm, __shfl_xor(pm, 32, WAVE));
      const float m_new = fmaxf(m, pm);
      const float base = m_new == -INFINITY ? 0.f : m_new;  // a row with no token yet
      const float alpha = __expf(m - base);
      f16x8 pa;
      float ps = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __expf(st[e] - base);
        ps += p;
        const f16 hi = (f16)p;
        pa[e] = hi;
        pa[4 + e] = (f16)(p - (float)hi);
      }
      l = l * alpha + ps;
      m = m_new;
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        O[db] *= alpha;
        const f16x8 vv = f16x8{vf[db][0], vf[db][1], vf[db][2], vf[db][3], vf[db][0], vf[db][1], vf[db][2], vf[db][3]};
        O[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pa, O[db], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);
  if (shares == 1) {                                        // uniform
    if (live) {
      const size_t at = ((size_t)row * a.Hq + head) * a.slots + slot;
#pragma unroll
      for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(a.acc + at * D + db * 16 + 4 * g) = O[db];
      if (g == 0) {
        a.ml[2 * at] = m;
        a.ml[2 * at + 1] = l;
      }
    }
    return;
  }
  if (live) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(&sacc[(wave * 16 + col) * D + db * 16 + 4 * g]) = O[db];
    if (g == 0) {
      sm[wave][col] = m;
      sl[wave][col] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 4); e += SA_WAVES * WAVE) {
    const int rr = e / (D / 4), d = e % (D / 4) * 4, c = rr & 15, w0 = rr >> 4;
    float M = -INFINITY;
    for (int w = w0; w < SA_WAVES; w += R) M = fmaxf(M, sm[w][c]);
    float L = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = w0; w < SA_WAVES; w += R) {
      const float f = sm[w][c] == -INFINITY ? 0.f : __expf(sm[w][c] - M);
      L += sl[w][c] * f;
      o += *reinterpret_cast<const f32x4*>(&sacc[(w * 16 + c) * D + d]) * f;
    }
    const int orow = first_member < 0 ? own_row : a.members[first_member + rr / G];
    const size_t at = ((size_t)orow * a.Hq + kh * G + rr % G) * a.slots + slot;
    *reinterpret_cast<f32x4*>(a.acc + at * D + d) = o;
    if (d == 0) {
      a.ml[2 * at] = M;
      a.ml[2 * at + 1] = L;
    }
  }
}

// a row's units joined: four heads a workgroup, a wave each
template <int D>
__global__ __launch_bounds__(4 * WAVE) void shared_attn_join_kernel(SharedAttn a) {
  const int h = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, b = blockIdx.y;
  if (h >= a.Hq) return;
  const int n = a.row_slots[b] + a.own_splits;
  const size_t at = ((size_t)b * a.Hq + h) * a.slots;
  constexpr int PER = D / WAVE;
  float M = -INFINITY, L = 0.f, o[PER] = {};
  for (int s = 0; s < n; ++s) M = fmaxf(M, a.ml[2 * (at + s)]);
  for (int s = 0; s < n; ++s) {
    const float m = a.ml[2 * (at + s)], f = m == -INFINITY ? 0.f : __expf(m - M);
    L += a.ml[2 * (at + s) + 1] * f;
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] += a.acc[(at + s) * D + lane * PER + e] * f;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int d = lane * PER + e;
    const size_t oo = a.frag_tt ? frag_offset(b, h * D + d, a.frag_tt) : ((size_t)b * a.Hq + h) * D + d;
    a.out[oo] = (f16)(L > 0.f ? o[e] / L : 0.f);
  }
}

}  // namespace

int mlora_check_attn(const char* who, int Hq, int Hkv, int D, int n_pages, int n_seq, int max_blocks);

extern "C" int mlora_shared_attn_unit_rows(void) { return SA_ROWS; }

extern "C" size_t mlora_shared_attn_workspace_bytes(int B, int Hq, int D, int slots) {
  return B <= 0 || Hq <= 0 || D <= 0 || slots <= 0 ? 0 : (size_t)B * Hq * slots * (D + 2) * sizeof(float);
}

extern "C" int mlora_paged_attn_decode_shared(void* out, int out_layout, const void* qkv, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                              int max_blocks, const int32_t* seq_ids, const int32_t* ctx_len, const int32_t* units, int n_units,
                                              const int32_t* members, int n_members, const int32_t* row_pages, const int32_t* row_slots, int own_splits,
                                              int slots, int B, int Hq, int Hkv, int D, int n_pages, int n_seq, void* workspace, size_t workspace_bytes,
                                              void* stream) {
  if (int e = mlora_check_attn("paged_attn_decode_shared", Hq, Hkv, D, n_pages, n_seq, max_blocks)) return e;
  MLORA_CHECK(out && qkv && k_cache && v_cache && block_table && seq_ids && ctx_len && row_pages && row_slots, MLORA_ERR_INVALID, "paged_attn_decode_shared: null pointer");
  MLORA_CHECK(n_units >= 0 && n_members >= 0 && (n_units == 0 || (units && members && n_members > 0)), MLORA_ERR_INVALID, "paged_attn_decode_shared: bad plan");
  MLORA_CHECK(B >= 0 && own_splits > 0 && slots >= own_splits && (long)B * own_splits + n_units <= 65535, MLORA_ERR_INVALID,
              "paged_attn_decode_shared: B=%d with %d units and %d shares of a row's own pages", B, n_units, own_splits);
  MLORA_CHECK(Hq / Hkv <= 16, MLORA_ERR_UNSUPPORTED, "paged_attn_decode_shared: more than 16 query heads per kv head (%d)", Hq / Hkv);
  MLORA_CHECK(out_layout == MLORA_ROWMAJOR || out_layout == MLORA_FRAG, MLORA_ERR_INVALID, "paged_attn_decode_shared: bad out_layout %d", out_layout);
  if (B == 0) return MLORA_OK;
  MLORA_CHECK(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= mlora_shared_attn_workspace_bytes(B, Hq, D, slots), MLORA_ERR_WORKSPACE,
              "paged_attn_decode_shared: workspace of %zu bytes, %zu needed", workspace_bytes, mlora_shared_attn_workspace_bytes(B, Hq, D, slots));
  SharedAttn a = {(f16*)out, (const f16*)qkv, (const f16*)k_cache, (const f16*)v_cache, block_table, seq_ids, ctx_len, units, members, row_pages, row_slots,
                  (float*)workspace, (float*)workspace + (size_t)B * Hq * slots * D, max_blocks, B, Hq, Hkv, n_pages, n_seq, n_units, n_members, own_splits, slots,
                  out_layout == MLORA_FRAG ? mlora_frag_tiles(B) : 0, 1.f / sqrtf((float)D)};
  hipStream_t s = (hipStream_t)stream;
#define MLORA_SHARED(DD)                                                                                                                         \
  do {                                                                                                                                           \
    constexpr size_t lds = (size_t)SA_WAVES * 16 * DD * sizeof(float);                                                                           \
    static const hipError_t configured =                                                                                                         \
        hipFuncSetAttribute((const void*)shared_attn_kernel<DD>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);                          \
    if (configured != hipSuccess)                                                                                                                \
      return mlora_set_error(MLORA_ERR_LAUNCH, "paged_attn_decode_shared: cannot reserve %zu bytes of LDS: %s", lds, hipGetErrorString(configured)); \
    hipLaunchKernelGGL(shared_attn_kernel<DD>, dim3(Hkv, n_units + B * own_splits), dim3(SA_WAVES * WAVE), lds, s, a);                           \
    if (int e = mlora_launch_status("paged_attn_decode_shared")) return e;                                                                       \
    hipLaunchKernelGGL(shared_attn_join_kernel<DD>, dim3(ceil_div(Hq, 4), B), dim3(4 * WAVE), 0, s, a);                                          \
  } while (0)
  if (D == 128) MLORA_SHARED(128);
  else MLORA_SHARED(64);
#undef MLORA_SHARED
  return mlora_launch_status("paged_attn_decode_shared");
}
