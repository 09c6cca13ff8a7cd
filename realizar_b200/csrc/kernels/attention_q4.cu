// Attention over the 4-bit paged cache (kv_q4.cuh): one new token per sequence, with the norm and rotation of its heads and the
// write of its row in the same launch, and the rows of a prompt chunk.
#include "attention_q4.cuh"
#include "kv_q4.cuh"

namespace rlz {

// 3311: a position beyond the page-table row (the sequence is skipped); 3312: a page id outside the cache (read as page 0, not written)
__device__ int g_attn_q4_error = 0;

__device__ __forceinline__ int q4_page_id(int raw, int num_pages) {
  if (num_pages > 0 && (unsigned)raw >= (unsigned)num_pages) { atomicExch(&g_attn_q4_error, 3312); return 0; }
  return raw;
}

// One CTA to a (sequence, kv head): its warps take the query heads in turn and walk the tokens one by one, the lanes over the dims.
template <int D>
__global__ void __launch_bounds__(128) attn_q4_simple_kernel(const __grid_constant__ AttnDecodeParams p) {
  constexpr int NP = HeadPairs<D>::NP;
  __shared__ __align__(16) uint8_t page_s[2][q4_page_bytes(D)];       // slot 0 of each: the new token's row
  __shared__ __align__(16) uint8_t codes_s[4][D];
  __shared__ float q_s[4][D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.x, b = blockIdx.y, G = p.n_heads / p.n_kv_heads;
  const int pos = p.positions[b];
  if (pos < 0) return;
  if (pos / Q4_PAGE >= p.max_pages) { if (threadIdx.x == 0) atomicExch(&g_attn_q4_error, 3311); return; }
  const int32_t* pt = p.page_table + (int64_t)b * p.pt_stride;
  const float* row = p.qkv + (int64_t)b * p.ld_qkv;
  const RopeArgs rope = {p.rope_table, p.rope_table_len, p.rope_dim, p.rope_type, p.rope_theta};
  const int half = p.rope_dim >> 1;
  float2 cs[NP];
  load_rope<D>(rope, pos, lane, cs);
  float a[NP], c[NP];
  auto load = [&](const float* src, int hf, int type) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      a[k] = c[k] = 0.f;
      if (i < D / 2) { const int2 at = pair_dims(i, hf, type); a[k] = src[at.x]; c[k] = src[at.y]; }
    }
  };
  if (!p.no_append && warp < 2) {
    const bool v = warp == 1;
    load(row + (v ? p.v_off : p.k_off) + kvh * D, v ? 0 : half, v ? 0 : p.rope_type);
    if (!v) norm_rope_d<D>(a, c, p.q_norm_w ? p.k_norm_w : nullptr, (double)p.eps, rope, cs, lane);
    const uint32_t meta = q4_quantise<D>(a, c, v ? 0 : half, v ? 0 : p.rope_type, lane, codes_s[warp]);
    __syncwarp();
    const int raw = pt[pos / Q4_PAGE];
    const bool ok = p.num_pages <= 0 || (unsigned)raw < (unsigned)p.num_pages;
    uint8_t* dst = (uint8_t*)(v ? p.v_cache : p.k_cache) + ((int64_t)(ok ? raw : 0) * p.n_kv_heads + kvh) * q4_page_bytes(D);
    if (v) { q4_store_v<D>(page_s[1], 0, codes_s[warp], meta, lane); if (ok) q4_store_v<D>(dst, pos % Q4_PAGE, codes_s[warp], meta, lane); }
    else { q4_store_k<D>(page_s[0], 0, codes_s[warp], meta, lane); if (ok) q4_store_k<D>(dst, pos % Q4_PAGE, codes_s[warp], meta, lane); }
    if (!ok && lane == 0) atomicExch(&g_attn_q4_error, 3312);
  }
  __syncthreads();
  const int lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  for (int g = warp; g < G; g += 4) {
    load(row + p.q_off + (int64_t)(kvh * G + g) * D, half, p.rope_type);
    norm_rope_f<D>(a, c, p.q_norm_w, p.eps, rope, cs, lane);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      if (i < D / 2) { const int2 at = pair_dims(i, half, p.rope_type); q_s[warp][at.x] = a[k] * p.scale; q_s[warp][at.y] = c[k] * p.scale; }
    }
    __syncwarp();
    float m = -INFINITY;
    double l = 0.0, o[NP][2] = {};                    // a serial sum over tens of thousands of tokens
    for (int t = lo; t <= pos; ++t) {
      const bool fresh = t == pos && !p.no_append;
      const int64_t at = ((int64_t)q4_page_id(pt[t / Q4_PAGE], p.num_pages) * p.n_kv_heads + kvh) * q4_page_bytes(D);
      const uint8_t* kp = fresh ? page_s[0] : (const uint8_t*)p.k_cache + at;
      const uint8_t* vp = fresh ? page_s[1] : (const uint8_t*)p.v_cache + at;
      const int slot = fresh ? 0 : t % Q4_PAGE;
      const uint32_t km = *(const uint32_t*)(kp + 8 * D + 4 * slot), vm = *(const uint32_t*)(vp + 8 * D + 4 * slot);
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int i = lane + 32 * k;
        if (i >= D / 2) continue;
        const int w = kp[q4_k_byte<D>(slot, i)];
        s += q_s[warp][2 * i] * ((float)(w & 15) * q4_scale(km) + q4_min(km)) + q_s[warp][2 * i + 1] * ((float)(w >> 4) * q4_scale(km) + q4_min(km));
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
    float* dst = p.out + (int64_t)b * p.ld_out + (int64_t)(kvh * G + g) * D;
#pragma unroll
    for (int k = 0; k < NP; ++k) { const int i = lane + 32 * k; if (i < D / 2) { dst[2 * i] = (float)(o[k][0] / l); dst[2 * i + 1] = (float)(o[k][1] / l); } }
    __syncwarp();
  }
}

int attn_decode_q4_dispatch(const AttnDecodeParams& p, cudaStream_t st) {
  if (!q4_head_dim_ok(p.head_dim)) return -1;
  if (p.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % p.n_kv_heads || p.batch < 1 || p.max_pages < 1) return -2;
  if (p.rope_dim < 0 || p.rope_dim > p.head_dim || (p.rope_dim & 1)) return -3;
  if (((uintptr_t)p.k_cache & 15) || ((uintptr_t)p.v_cache & 15)) return -4;
  if (p.window < 0) return -5;
  dim3 grid(p.n_kv_heads, p.batch);
  switch (p.head_dim) {
    case 64: return (int)launch(attn_q4_simple_kernel<64>, grid, dim3(128), 0, st, p);
    case 80: return (int)launch(attn_q4_simple_kernel<80>, grid, dim3(128), 0, st, p);
    case 96: return (int)launch(attn_q4_simple_kernel<96>, grid, dim3(128), 0, st, p);
    default: return (int)launch(attn_q4_simple_kernel<128>, grid, dim3(128), 0, st, p);
  }
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
  const int pos = (p.pos0_ptr ? *p.pos0_ptr : p.pos0) + r, lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
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

// scratch sizes (floats)
long long rlz_attn_q4_partial_floats(int head_dim) { return head_dim + 2; }
long long rlz_attn_prefill_q4_scratch_floats(int n_tokens, int n_heads, int n_kv_heads, int head_dim) { return 1; }

// 0 / 3311 / 3312
int rlz_attn_q4_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_attn_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_attn_q4_error, &z, sizeof(int)); }
  return v;
}

}  // extern "C"
