// Attention of the rows of a prompt chunk over the 4-bit paged cache (kv_q4.cuh).
#include "attention_q4.cuh"
#include "kv_q4.cuh"

namespace rlz {

// 3113: a page id outside the cache (read as page 0); 3114: a row beyond the page table (skipped)
__device__ int g_prefill_q4_error = 0;

__device__ __forceinline__ int q4_page_id(int raw, int num_pages) {
  if (num_pages > 0 && (unsigned)raw >= (unsigned)num_pages) { atomicExch(&g_prefill_q4_error, 3113); return 0; }
  return raw;
}

// One warp to a (chunk row, query head)
template <int D>
__global__ void __launch_bounds__(128) attn_prefill_q4_simple_kernel(const __grid_constant__ AttnPrefillParams p) {
  constexpr int NP = HeadPairs<D>::NP;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y, r = blockIdx.x * 4 + warp;
  if (r >= p.n_tokens) return;
  const int kvh = head / (p.n_heads / p.n_kv_heads);
  const int pos = (p.pos0_ptr ? *p.pos0_ptr : p.pos0) + r;
  if (pos < 0 || pos / Q4_PAGE >= p.pt_len) { atomicExch(&g_prefill_q4_error, 3114); return; }
  const int lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  const float* src = p.qkv + (int64_t)r * p.ld_qkv + p.q_off + (int64_t)head * D;
  float q[NP][2] = {}, m = -INFINITY;
  double l = 0.0, o[NP][2] = {};                      // a serial sum over tens of thousands of tokens
#pragma unroll
  for (int k = 0; k < NP; ++k) { const int i = lane + 32 * k; if (i < D / 2) { q[k][0] = src[2 * i] * p.scale; q[k][1] = src[2 * i + 1] * p.scale; } }
  for (int t = lo; t <= pos; ++t) {
    const int64_t at = ((int64_t)q4_page_id(p.page_table[t / Q4_PAGE], p.num_pages) * p.n_kv_heads + kvh) * q4_page_bytes(D);
    const uint8_t *kp = (const uint8_t*)p.k_cache + at, *vp = (const uint8_t*)p.v_cache + at;
    const int slot = t % Q4_PAGE;
    const uint32_t km = *(const uint32_t*)(kp + 8 * D + 4 * slot), vm = *(const uint32_t*)(vp + 8 * D + 4 * slot);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      if (i >= D / 2) continue;
      const int w = kp[q4_k_byte<D>(slot, i)];
      s += q[k][0] * ((float)(w & 15) * q4_scale(km) + q4_min(km)) + q[k][1] * ((float)(w >> 4) * q4_scale(km) + q4_min(km));
    }
    s = warp_sum(s);
    const float mn = fmaxf(m, s), corr = expf(m - mn), e = expf(s - mn);
    l = l * corr + e; m = mn;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      if (i >= D / 2) continue;
      const int w = vp[q4_v_byte<D>(slot, i)];
      o[k][0] = o[k][0] * corr + e * ((float)(w & 15) * q4_scale(vm) + q4_min(vm));
      o[k][1] = o[k][1] * corr + e * ((float)(w >> 4) * q4_scale(vm) + q4_min(vm));
    }
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int i = lane + 32 * k;
    if (i >= D / 2) continue;
    const int64_t at = (int64_t)r * p.ld_out + (int64_t)head * D + 2 * i;
    if (p.out_bf16) *(__nv_bfloat162*)((__nv_bfloat16*)p.out + at) = __floats2bfloat162_rn((float)(o[k][0] / l), (float)(o[k][1] / l));
    else { p.out[at] = (float)(o[k][0] / l); p.out[at + 1] = (float)(o[k][1] / l); }
  }
}

int attn_prefill_q4_dispatch(const AttnPrefillParams& p, cudaStream_t st) {
  dim3 grid((p.n_tokens + 3) / 4, p.n_heads);
  switch (p.head_dim) {
    case 64: return (int)launch(attn_prefill_q4_simple_kernel<64>, grid, dim3(128), 0, st, p);
    case 80: return (int)launch(attn_prefill_q4_simple_kernel<80>, grid, dim3(128), 0, st, p);
    case 96: return (int)launch(attn_prefill_q4_simple_kernel<96>, grid, dim3(128), 0, st, p);
    case 128: return (int)launch(attn_prefill_q4_simple_kernel<128>, grid, dim3(128), 0, st, p);
    default: return -1;
  }
}

}  // namespace rlz

extern "C" {

// floats of scratch that a chunk of up to n_tokens rows can use
long long rlz_attn_prefill_q4_scratch_floats(int n_tokens, int n_heads, int n_kv_heads, int head_dim) { return 1; }

// 0 / 3113 / 3114
int rlz_attn_prefill_q4_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_prefill_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_prefill_q4_error, &z, sizeof(int)); }
  return v;
}

}  // extern "C"
