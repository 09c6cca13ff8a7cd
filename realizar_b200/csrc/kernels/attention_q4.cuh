// Parameter block of the prompt attention, and the launchers of the kernels over 4-bit caches (attention_decode_q4.cu,
// attention_prefill_q4.cu) that the general entry points hand over to.
#pragma once
#include "attention_decode_body.cuh"

namespace rlz {

struct AttnPrefillParams {
  const float* qkv;            // [T, ld_qkv] fp32, q section already rotated
  float* out;                  // [T, ld_out] fp32, head-major
  const __nv_bfloat16* k_cache;
  const __nv_bfloat16* v_cache;
  const int32_t* page_table;   // [max_pages] of this sequence
  int64_t ld_qkv, ld_out;
  int32_t n_heads, n_kv_heads, head_dim, q_off;
  int32_t n_tokens, pos0;      // chunk rows are positions pos0 .. pos0 + n_tokens - 1
  int32_t window, kv_q8;       // kv_q8: 1 int8 cache rows of head_dim + 16 bytes (codes, then the fp32 row scale), 2 pages of 4-bit rows (kv_q4.cuh)
  float scale;
  int32_t out_bf16;            // 1: `out` is bf16 [T, ld_out] (the operand of the output projection GEMM), else fp32
  const int32_t* pos0_ptr;     // when set, the position of row 0 is read from here (a launch captured in a CUDA graph serves any chunk)
  int32_t num_pages, pt_len;   // 4-bit caches: pages in the cache and entries of the page table, which ids and positions are checked against
  float* scratch;              // 4-bit caches: workspace of the split over the keys, or null
  int64_t scratch_floats;
};

// -1 .. -7: refused arguments; else the launch's CUDA error
int attn_decode_q4_dispatch(const AttnDecodeParams& p, cudaStream_t st);
int attn_prefill_q4_dispatch(const AttnPrefillParams& p, cudaStream_t st);

}  // namespace rlz
