// Norm of the query and key heads, rotation, and the write of keys and values into the 4-bit paged cache, in one pass over the
// rows that the Q/K/V projection left (kv_q4.cuh has the page format):
//   q' = R(pos) (q / rms(q) * wq)          32 bits, to q_out or in place
//   k' = R(pos) (k / rms(k) * wk)          64 bits, rounded once, then quantised with one scale and minimum to a row
//   v                                       quantised likewise
#include "kv_q4.cuh"

namespace rlz {

// 3405: a page id outside the cache (the row's K and V are not written)
__device__ int g_q4_append_error = 0;

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

template <int D>
__global__ void __launch_bounds__(QA_WARPS * 32) qk_norm_rope_append_kernel(const __grid_constant__ QkAppendParams p) {
  constexpr int NP = HeadPairs<D>::NP;
  __shared__ __align__(16) uint8_t codes_s[QA_WARPS][D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x;
  const int pos = p.positions[t];
  if (pos < 0) return;
  const int page = p.page_rows[t];
  const bool page_ok = (unsigned)page < (unsigned)p.num_pages;
  if (!page_ok && threadIdx.x == 0) atomicExch(&g_q4_append_error, 3405);
  const RopeArgs rope = {p.rope_table, p.rope_table_len, p.rope_dim, p.rope_type, p.rope_theta};
  const RopeArgs none = {nullptr, 0, 0, 0, 0.f};
  float2 cs[NP];
  load_rope<D>(rope, pos, lane, cs);
  const int njobs = p.n_heads + 2 * p.n_kv_heads, half = p.rope_dim >> 1;
  for (int job = blockIdx.y * QA_WARPS + warp; job < njobs; job += gridDim.y * QA_WARPS) {
    const float* src = p.qkv + (int64_t)t * p.ld + (int64_t)job * D;
    const bool is_v = job >= p.n_heads + p.n_kv_heads;
    const int hf = is_v ? 0 : half, type = is_v ? 0 : p.rope_type;
    float a[NP], b[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      a[k] = b[k] = 0.f;
      if (i < D / 2) { const int2 at = pair_dims(i, hf, type); a[k] = src[at.x]; b[k] = src[at.y]; }
    }
    if (job < p.n_heads) {
      norm_rope_f<D>(a, b, p.q_norm_w, (float)p.eps, rope, cs, lane);
      float* dst = p.q_out + (int64_t)t * p.ld_q + (int64_t)job * D;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int i = lane + 32 * k;
        if (i < D / 2) { const int2 at = pair_dims(i, hf, type); dst[at.x] = a[k]; dst[at.y] = b[k]; }
      }
      continue;
    }
    if (!page_ok) continue;
    const int h = job - p.n_heads - (is_v ? p.n_kv_heads : 0);
    if (!is_v) norm_rope_d<D>(a, b, p.k_norm_w, p.eps, rope, cs, lane);
    const uint32_t meta = q4_quantise<D>(a, b, hf, type, lane, codes_s[warp]);
    __syncwarp();
    uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((int64_t)page * p.n_kv_heads + h) * q4_page_bytes(D);
    if (is_v) q4_store_v<D>(dst, pos % Q4_PAGE, codes_s[warp], meta, lane);
    else q4_store_k<D>(dst, pos % Q4_PAGE, codes_s[warp], meta, lane);
    __syncwarp();
  }
}

template <int D>
static int launch_qk_append(const QkAppendParams& p, cudaStream_t st) {
  const int njobs = p.n_heads + 2 * p.n_kv_heads;
  return (int)launch(qk_norm_rope_append_kernel<D>, dim3(p.rows, (njobs + QA_WARPS - 1) / QA_WARPS), dim3(QA_WARPS * 32), 0, st, p);
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
  cudaStream_t st = (cudaStream_t)stream;
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
  if (cudaMemcpyFromSymbol(&v, rlz::g_q4_append_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_q4_append_error, &z, sizeof(int)); }
  return v;
}

int rlz_sizeof_qk_append_params() { return (int)sizeof(rlz::QkAppendParams); }

}  // extern "C"
