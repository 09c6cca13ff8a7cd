// Norm of the query and key heads, rotation, and the write of keys and values into the 4-bit paged cache, in one pass over the
// rows that the Q/K/V projection left (kv_q4.cuh has the page format):
//   q' = R(pos) (q / rms(q) * wq)          32 bits, to q_out or in place
//   k' = R(pos) (k / rms(k) * wk)          64 bits, rounded once, then quantised with one scale and minimum to a row
//   v                                       quantised likewise
// Bound by the bytes of the fp32 rows (read all, write the queries), and close behind it by instructions.  A warp takes several heads
// of one kind (query, key or value) of a row: their loads are all in flight before the first is worked on, and the lane's offsets,
// norm weights and angles are fetched once.  Few rows take one head to a warp, which is the shorter way through them.
// 8192 rows of 32 query and 8 kv heads of 128: 71 us, 4.9 TB/s.  What hides the loads' latency is the number of warps: with the 74
// registers that the compiler takes by itself (three blocks to an SM) it is 86 us, with 64 (four) 71, with 48 (five) 73; 4 query heads
// to a warp and five blocks 71, one key head 83.  32 query and 32 kv heads of 80: 185 us, 1.9 TB/s, by then 0.70 of the issue slots.
#include "kv_q4.cuh"
#include <atomic>

namespace rlz {

// 3405: a page id outside the cache (the row's K and V are not written)
__device__ int g_q4_append_error = 0;
static std::atomic<bool> q4_append_ran{false};       // until a launch there is no status to fetch, which takes a synchronous copy

struct QkAppendParams {
  const float* qkv;            // [rows, ld]: q heads | k heads | v heads
  float* q_out;                // [rows, ld_q]; may be qkv itself (rotation in place)
  uint8_t* k_cache;
  uint8_t* v_cache;            // [pages, n_kv_heads, 16, D / 2 + 4]
  const int32_t* positions;    // [rows]; < 0: the row is idle and nothing of it is written
  const int32_t* page_rows;    // [rows] physical page of the row's position
  const float* q_norm_w;       // [head_dim] or null
  const float* k_norm_w;
  const float2* rope_table;    // [rope_table_len, rope_dim / 2] (cos, sin) or null
  int64_t ld, ld_q;
  double eps;
  int32_t rows, n_heads, n_kv_heads, head_dim;
  int32_t rope_dim, rope_type, rope_table_len, num_pages;
  float rope_theta;
  int32_t _pad;
};

constexpr int QA_WARPS = 8;

// the lane's pairs of N heads, `step` floats apart; ADJACENT: the two values of a pair are neighbours
template <int D, int N, bool ADJACENT>
__device__ __forceinline__ void load_heads(const float* src, int n, const int2 (&at)[HeadPairs<D>::NP], int lane, float (&a)[N][HeadPairs<D>::NP],
                                           float (&b)[N][HeadPairs<D>::NP]) {
#pragma unroll
  for (int k = 0; k < HeadPairs<D>::NP; ++k) {
    const bool in = lane + 32 * k < D / 2;
    const float *pa = src + at[k].x, *pb = src + at[k].y;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      a[j][k] = b[j][k] = 0.f;
      if (in && j < n) {
        if constexpr (ADJACENT) { const float2 v = *(const float2*)(pa + j * D); a[j][k] = v.x; b[j][k] = v.y; }
        else { a[j][k] = pa[j * D]; b[j][k] = pb[j * D]; }
      }
    }
  }
}

// SPLIT: rotation of split halves, else pairs are neighbours throughout.  NQ query heads, or NK key or value heads, to a warp
template <int D, bool SPLIT, int NQ, int NK>
__global__ void __launch_bounds__(QA_WARPS * 32, NQ > 1 ? 4 : 1) qk_norm_rope_append_kernel(const __grid_constant__ QkAppendParams p) {
  constexpr int NP = HeadPairs<D>::NP;
  __shared__ __align__(16) uint8_t codes_s[QA_WARPS][NK][D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q_units = (p.n_heads + NQ - 1) / NQ, k_units = (p.n_kv_heads + NK - 1) / NK, units = q_units + 2 * k_units;
  const int64_t unit = (int64_t)blockIdx.x * QA_WARPS + warp;
  const int t = (int)(unit / units);
  int u = (int)(unit - (int64_t)t * units);
  if (t >= p.rows) return;
  const int pos = p.positions[t], page = p.page_rows[t], half = p.rope_dim >> 1, type = SPLIT ? 2 : 0;
  const float* row = p.qkv + (int64_t)t * p.ld;
  int2 at[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) at[k] = pair_dims(lane + 32 * k, half, type);
  const RopeArgs rope = {p.rope_table, p.rope_table_len, p.rope_dim, type, p.rope_theta};
  float2 cs[NP];

  if (u < q_units) {
    const int h0 = u * NQ, n = min(NQ, p.n_heads - h0);
    float a[NQ][NP], b[NQ][NP];
    load_heads<D, NQ, !SPLIT>(row + h0 * D, n, at, lane, a, b);
    if (pos < 0) return;
    load_rope<D>(rope, pos, lane, cs);
    float wa[NP], wb[NP];
    if (p.q_norm_w) {
#pragma unroll
      for (int k = 0; k < NP; ++k) { const bool in = lane + 32 * k < D / 2; wa[k] = in ? __ldg(p.q_norm_w + at[k].x) : 0.f; wb[k] = in ? __ldg(p.q_norm_w + at[k].y) : 0.f; }
    }
    float* out = p.q_out + (int64_t)t * p.ld_q + h0 * D;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      if (j >= n) break;
      if (p.q_norm_w) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < NP; ++k) ss += a[j][k] * a[j][k] + b[j][k] * b[j][k];
        const float rs = rsqrtf(warp_sum(ss) * (1.f / D) + (float)p.eps);
#pragma unroll
        for (int k = 0; k < NP; ++k) { a[j][k] *= rs * wa[k]; b[j][k] *= rs * wb[k]; }
      }
#pragma unroll
      for (int k = 0; k < NP; ++k) {                             // (pairs that are not rotated have the angle 0)
        const float x = a[j][k], y = b[j][k], c = cs[k].x, s = cs[k].y;
        a[j][k] = x * c - y * s; b[j][k] = x * s + y * c;
        if (lane + 32 * k < D / 2) {
          if constexpr (SPLIT) { out[j * D + at[k].x] = a[j][k]; out[j * D + at[k].y] = b[j][k]; }
          else *(float2*)(out + j * D + at[k].x) = make_float2(a[j][k], b[j][k]);
        }
      }
    }
    return;
  }
  u -= q_units;
  const bool is_v = u >= k_units;
  const int h0 = (is_v ? u - k_units : u) * NK, n = min(NK, p.n_kv_heads - h0);
  const float* src = row + (int64_t)(p.n_heads + (is_v ? p.n_kv_heads : 0) + h0) * D;
  float a[NK][NP], b[NK][NP];
  if (is_v) {
#pragma unroll
    for (int k = 0; k < NP; ++k) at[k] = pair_dims(lane + 32 * k, 0, 0);
    load_heads<D, NK, true>(src, n, at, lane, a, b);
  } else {
    load_heads<D, NK, !SPLIT>(src, n, at, lane, a, b);
  }
  if (pos < 0) return;
  if ((unsigned)page >= (unsigned)p.num_pages) { if (u == 0 && lane == 0) atomicExch(&g_q4_append_error, 3405); return; }
  if (!is_v) load_rope<D>(rope, pos, lane, cs);
  uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((int64_t)page * p.n_kv_heads + h0) * q4_page_bytes(D);
  // each stage for all heads of the warp (those behind the last are zeros), so that their chains of dependent steps overlap
  uint32_t meta[NK];
  if (!is_v) {
#pragma unroll
    for (int j = 0; j < NK; ++j) norm_rope_d<D>(a[j], b[j], p.k_norm_w, p.eps, rope, cs, lane);
  }
  const int slot = pos % Q4_PAGE;
  if (SPLIT && !is_v && (half & 1)) {                            // a byte's two dims lie in unrelated lanes: by way of shared memory
#pragma unroll
    for (int j = 0; j < NK; ++j) meta[j] = q4_quantise<D>(a[j], b[j], half, type, lane, codes_s[warp][j]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NK; ++j) if (j < n) q4_store_k<D>(dst + j * q4_page_bytes(D), slot, codes_s[warp][j], meta[j], lane);
    return;
  }
  uint32_t byte[NK][NP];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    uint32_t ca[NP], cb[NP];
    meta[j] = q4_codes<D>(a[j], b[j], lane, ca, cb);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      byte[j][k] = ca[k] | cb[k] << 4;
      if (SPLIT && !is_v) {
        // the neighbour has the other value of each of the two bytes: even lanes take the one of the first half, odd lanes the second
        const uint32_t v = byte[j][k], w = __shfl_xor_sync(0xFFFFFFFFu, v, 1);
        if (lane + 32 * k < half) byte[j][k] = lane & 1 ? w >> 4 | (v & 0xF0u) : (v & 15u) | (w & 15u) << 4;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int i = lane + 32 * k;
    if (i < D / 2) {
      const int bi = SPLIT && !is_v && i < half ? (lane & 1 ? i - 1 + half : i) >> 1 : i;      // my byte: dims 2 bi, 2 bi + 1
      uint8_t* at_byte = dst + (is_v ? q4_v_byte<D>(slot, bi) : q4_k_byte<D>(slot, bi));
#pragma unroll
      for (int j = 0; j < NK; ++j) if (j < n) at_byte[j * q4_page_bytes(D)] = (uint8_t)byte[j][k];
    }
  }
#pragma unroll
  for (int j = 0; j < NK; ++j) if (j < n && lane == 0) *(uint32_t*)(dst + j * q4_page_bytes(D) + 8 * D + 4 * slot) = meta[j];
}

template <int D, bool SPLIT, int NQ, int NK>
static int launch_qk_append_n(const QkAppendParams& p, cudaStream_t st) {
  const int64_t units = (p.n_heads + NQ - 1) / NQ + 2 * ((p.n_kv_heads + NK - 1) / NK);
  return (int)launch(qk_norm_rope_append_kernel<D, SPLIT, NQ, NK>, dim3((unsigned)((p.rows * units + QA_WARPS - 1) / QA_WARPS)), dim3(QA_WARPS * 32), 0, st, p);
}
template <int D>
static int launch_qk_append(const QkAppendParams& p, cudaStream_t st) {
  // one head to a warp while that makes at most about one wave of warps (148 SMs x 32)
  const bool few = (int64_t)p.rows * (p.n_heads + 2 * p.n_kv_heads) <= 148 * 32;
  if (p.rope_dim > 0 && p.rope_type == 2) return few ? launch_qk_append_n<D, true, 1, 1>(p, st) : launch_qk_append_n<D, true, 8, 2>(p, st);
  return few ? launch_qk_append_n<D, false, 1, 1>(p, st) : launch_qk_append_n<D, false, 8, 2>(p, st);
}

}  // namespace rlz

extern "C" {

int rlz_qk_norm_rope_append(const rlz::QkAppendParams* pp, void* stream) {
  using namespace rlz;
  const QkAppendParams& p = *pp;
  if (!q4_head_dim_ok(p.head_dim)) return -1;
  if (p.rows < 1 || p.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % p.n_kv_heads || p.num_pages < 1) return -2;
  if (p.rope_dim < 0 || p.rope_dim > p.head_dim || (p.rope_dim & 1)) return -3;
  if (((uintptr_t)p.k_cache & 15) || ((uintptr_t)p.v_cache & 15)) return -4;
  if (!p.q_norm_w != !p.k_norm_w) return -5;
  if (((uintptr_t)p.qkv & 7) || ((uintptr_t)p.q_out & 7) || (p.ld & 1) || (p.ld_q & 1)) return -6;       // pairs are moved as 8 bytes
  cudaStream_t st = (cudaStream_t)stream;
  q4_append_ran.store(true, std::memory_order_relaxed);
  switch (p.head_dim) {
    case 64: return launch_qk_append<64>(p, st);
    case 80: return launch_qk_append<80>(p, st);
    case 96: return launch_qk_append<96>(p, st);
    default: return launch_qk_append<128>(p, st);
  }
}

// 0 / 3405
int rlz_q4_append_error(int clear) {
  int v = 0;
  if (!rlz::q4_append_ran.load(std::memory_order_relaxed)) return 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_q4_append_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_q4_append_error, &z, sizeof(int)); }
  return v;
}

int rlz_sizeof_qk_append_params() { return (int)sizeof(rlz::QkAppendParams); }

}  // extern "C"
