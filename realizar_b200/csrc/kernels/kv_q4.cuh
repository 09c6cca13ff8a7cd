// 4-bit KV pages: the format, and the warp-wide routines that build a row of it.
//
// A page holds 16 tokens of one kv head, 16 * (D / 2 + 4) bytes: 8 D bytes of codes, then for every token a bf16 scale and a
// bf16 minimum.  value = code * scale + minimum, code 0..15, with one scale and minimum to a (token, kv head) row:
//   minimum = bf16(min x), scale = bf16((max x - min x) / 15), code = the integer nearest to (x - minimum) / scale, 0..15
// (x limited to +-32768, a NaN counts as 0, a scale of 0 gives codes 0).
//
// The codes lie in the order in which mma.m16n8k16 takes its B operand, so that a lane fetches its fragments of a page with
// one or two wide loads and no shuffles (NG = D / 32; gq = lane / 4, tq = lane % 4):
//   keys    token rows of D / 2 bytes; the 32-bit word of dims 32 g + 8 tq .. + 7 is word tq * NG + g of the row.
//   values  word [half][gq][tq][g]: tokens 8 half + 2 tq (low 16 bits) and + 1 (high 16 bits), dims 32 g + 4 gq .. + 3 each.
// D % 32 == 16 leaves 16 dims: keys, the last two words of the row in their own order; values, byte words [gq][tq] of tokens
// 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9 with dims 32 NG + 2 gq and + 1.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

namespace rlz {

constexpr int Q4_PAGE = 16;
constexpr float Q4_LIMIT = 32768.f;      // |value| stays below 65504 after the roundings of scale and minimum: it fits fp16 wherever a kernel needs that

__host__ __device__ constexpr int q4_row_bytes(int d) { return d / 2 + 4; }
__host__ __device__ constexpr int q4_page_bytes(int d) { return Q4_PAGE * q4_row_bytes(d); }
__host__ __device__ constexpr bool q4_head_dim_ok(int d) { return d == 64 || d == 80 || d == 96 || d == 128; }

// byte of a page that holds dims (2 b, 2 b + 1) of token t (even dim in the low four bits)
template <int D> __device__ __forceinline__ int q4_k_byte(int t, int b) {
  constexpr int NG = D / 32;
  const int w = b >> 2;
  return t * (D / 2) + (w < 4 * NG ? (w & 3) * NG + (w >> 2) : w) * 4 + (b & 3);
}
template <int D> __device__ __forceinline__ int q4_v_byte(int t, int b) {
  constexpr int NG = D / 32;
  const int half = t >> 3, tq = (t & 7) >> 1, odd = t & 1, e = b >> 1;
  if (D % 32 == 0 || b < 16 * NG) return (((half * 8 + (e & 7)) * 4 + tq) * NG + (e >> 3)) * 4 + odd * 2 + (b & 1);
  return 256 * NG + ((b - 16 * NG) * 4 + tq) * 4 + half * 2 + odd;
}

// what a token's meta word stands for
__device__ __forceinline__ float q4_scale(uint32_t meta) { return __uint_as_float(meta << 16); }
__device__ __forceinline__ float q4_min(uint32_t meta) { return __uint_as_float(meta & 0xFFFF0000u); }

// ---- one head row spread over a warp: lane holds pairs i = lane + 32 k, each the two values that a rotation mixes ----------
// pair i < rope_dim / 2: dims (i, i + rope_dim / 2) for split halves (type 2), (2 i, 2 i + 1) for adjacent pairs; the pairs
// behind them, (2 i, 2 i + 1), are not rotated
template <int D> struct HeadPairs { static constexpr int NP = (D / 2 + 31) / 32; };

__device__ __forceinline__ int2 pair_dims(int i, int half, int rope_type) {
  return i < half && rope_type == 2 ? make_int2(i, i + half) : make_int2(2 * i, 2 * i + 1);
}

// cos and sin of a rotary pair beyond the table, in 64 bits (far positions lose their angle in 32)
static __device__ __noinline__ float2 rope_angle(int pos, int i, int rope_dim, float theta) {
  double sn, cs;
  sincos((double)pos * pow((double)theta, -2.0 * i / rope_dim), &sn, &cs);
  return make_float2((float)cs, (float)sn);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// smallest and largest of a value over the warp
__device__ __forceinline__ float redux_min(float v) { float r; asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float redux_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }

// 1 / sqrt(x) in 64 bits: two Newton steps y (3 - x y^2) / 2 on the 32-bit result (2^-22 -> 2^-43 -> below 2^-52), a third of the
// time of the square root and the division.  Where 32 bits do not hold x, those.
__device__ __forceinline__ double rsqrt_d(double x) {
  if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);
  double y = (double)rsqrtf((float)x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = y * fma(-0.5 * x * y, y, 1.5);
  return y;
}

struct RopeArgs {
  const float2* table;     // [table_len, rope_dim / 2] (cos, sin) or null
  int table_len, rope_dim, rope_type;
  float theta;
};

template <int D>
__device__ __forceinline__ void load_rope(const RopeArgs& r, int pos, int lane, float2 (&cs)[HeadPairs<D>::NP]) {
  const int half = r.rope_dim >> 1;
#pragma unroll
  for (int k = 0; k < HeadPairs<D>::NP; ++k) {
    const int i = lane + 32 * k;
    cs[k] = make_float2(1.f, 0.f);
    if (i < half) cs[k] = r.table && pos < r.table_len ? __ldg(r.table + (int64_t)pos * half + i) : rope_angle(pos, i, r.rope_dim, r.theta);
  }
}

// RMS norm (w may be null) and rotation of a head row in 32 bits; a / b: first and second value of the lane's pairs
template <int D>
__device__ __forceinline__ void norm_rope_f(float (&a)[HeadPairs<D>::NP], float (&b)[HeadPairs<D>::NP], const float* w, float eps, const RopeArgs& r,
                                            const float2 (&cs)[HeadPairs<D>::NP], int lane) {
  constexpr int NP = HeadPairs<D>::NP;
  const int half = r.rope_dim >> 1;
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NP; ++k) ss += a[k] * a[k] + b[k] * b[k];
    const float rs = rsqrtf(warp_sum(ss) / (float)D + eps);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int i = lane + 32 * k;
      if (i < D / 2) { const int2 at = pair_dims(i, half, r.rope_type); a[k] = a[k] * rs * __ldg(w + at.x); b[k] = b[k] * rs * __ldg(w + at.y); }
    }
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    if (lane + 32 * k < half) { const float x = a[k], y = b[k]; a[k] = x * cs[k].x - y * cs[k].y; b[k] = x * cs[k].y + y * cs[k].x; }
  }
}

// The same for a key row in 64 bits, rounded to 32 once at the end: 32-bit values of a row that two kernels (or two orders of
// the sum) compute differ in their last bit, and where such a value lies next to the border of two codes the cached row would
// differ by a whole step.  Only keys pay for it, and they are 1 / (group + 2) of the row.
template <int D>
__device__ __forceinline__ void norm_rope_d(float (&a)[HeadPairs<D>::NP], float (&b)[HeadPairs<D>::NP], const float* w, double eps, const RopeArgs& r,
                                            const float2 (&cs)[HeadPairs<D>::NP], int lane) {
  constexpr int NP = HeadPairs<D>::NP;
  const int half = r.rope_dim >> 1;
  double rs = 1.0;
  if (w) {
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < NP; ++k) ss += (double)a[k] * a[k] + (double)b[k] * b[k];
    rs = rsqrt_d(warp_sum_d(ss) * (1.0 / D) + eps);
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const int i = lane + 32 * k;
    if (i >= D / 2) continue;
    double x = a[k], y = b[k];
    if (w) { const int2 at = pair_dims(i, half, r.rope_type); x *= rs * (double)__ldg(w + at.x); y *= rs * (double)__ldg(w + at.y); }
    if (i < half) {
      const double c = cs[k].x, s = cs[k].y, t = x * c - y * s;
      y = x * s + y * c;
      x = t;
    }
    a[k] = (float)x; b[k] = (float)y;
  }
}

// the code of a value in 64 bits
static __device__ __noinline__ float q4_code_64(float x, float mn, float sc) {
  return sc > 0.f ? (float)fmin(fmax(rint(((double)x - (double)mn) / (double)sc), 0.0), 15.0) : 0.f;
}
// x / 15 rounded once: the product with 1 / 15 and one correction (checked for every 24-bit x; below 2^-100 the division itself)
__device__ __forceinline__ float div_15(float x) {
  if (x < 0x1p-100f) return __fdiv_rn(x, 15.f);
  const float q = x * (1.f / 15.f);
  return fmaf(fmaf(-15.f, q, x), 1.f / 15.f, q);
}

// Codes of the lane's pairs (low four bits of ca / cb); returns the row's meta word
template <int D>
__device__ __forceinline__ uint32_t q4_codes(const float (&a)[HeadPairs<D>::NP], const float (&b)[HeadPairs<D>::NP], int lane, uint32_t (&ca)[HeadPairs<D>::NP],
                                             uint32_t (&cb)[HeadPairs<D>::NP]) {
  constexpr int NP = HeadPairs<D>::NP;
  float lo = INFINITY, hi = -INFINITY;
  float x[NP][2];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    x[k][0] = a[k] == a[k] ? fminf(fmaxf(a[k], -Q4_LIMIT), Q4_LIMIT) : 0.f;
    x[k][1] = b[k] == b[k] ? fminf(fmaxf(b[k], -Q4_LIMIT), Q4_LIMIT) : 0.f;
    if (lane + 32 * k < D / 2) { lo = fminf(lo, fminf(x[k][0], x[k][1])); hi = fmaxf(hi, fmaxf(x[k][0], x[k][1])); }
  }
  lo = redux_min(lo); hi = redux_max(hi);
  const __nv_bfloat16 sb = __float2bfloat16_rn(div_15(hi - lo)), mb = __float2bfloat16_rn(lo);
  const float sc = __bfloat162float(sb), mn = __bfloat162float(mb);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sc));       // infinite for scales of 0 and below 2^-126
  // 32 bits settle a code unless the quotient lies within 2^-14 of a border (its error is below 16 x 2^-22: difference 2^-24,
  // reciprocal 2^-23, product 2^-24); those divide in 64.
  // y + 1.5 x 2^23 rounds y to an integer, ties to even, and leaves it in the low bits
  float t[NP][2];
  bool near = !(inv < 1e30f);
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float y = fminf(fmaxf((x[k][e] - mn) * inv, 0.f), 15.f);
      t[k][e] = y + 12582912.f;
      near |= fabsf(y - (t[k][e] - 12582912.f)) > 0.5f - 0x1p-14f;
    }
  if (near) {
#pragma unroll
    for (int k = 0; k < NP; ++k) { t[k][0] = q4_code_64(x[k][0], mn, sc) + 12582912.f; t[k][1] = q4_code_64(x[k][1], mn, sc) + 12582912.f; }
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) { ca[k] = __float_as_uint(t[k][0]) & 15u; cb[k] = __float_as_uint(t[k][1]) & 15u; }
  return (uint32_t)__bfloat16_as_ushort(sb) | (uint32_t)__bfloat16_as_ushort(mb) << 16;
}
// the same as bytes in `codes` [D], shared memory of this warp
template <int D>
__device__ __forceinline__ uint32_t q4_quantise(const float (&a)[HeadPairs<D>::NP], const float (&b)[HeadPairs<D>::NP], int half, int rope_type, int lane,
                                                uint8_t* codes) {
  uint32_t ca[HeadPairs<D>::NP], cb[HeadPairs<D>::NP];
  const uint32_t meta = q4_codes<D>(a, b, lane, ca, cb);
#pragma unroll
  for (int k = 0; k < HeadPairs<D>::NP; ++k) {
    if (lane + 32 * k < D / 2) { const int2 at = pair_dims(lane + 32 * k, half, rope_type); codes[at.x] = (uint8_t)ca[k]; codes[at.y] = (uint8_t)cb[k]; }
  }
  return meta;
}

// Write a row of codes and its meta word into a page (global or shared memory); the warp calls together
template <int D>
__device__ __forceinline__ void q4_store_k(uint8_t* page, int t, const uint8_t* codes, uint32_t meta, int lane) {
  if (lane < D / 8) {
    const uint2 c = *(const uint2*)(codes + 8 * lane);
    const uint32_t lo = c.x | c.x >> 4, hi = c.y | c.y >> 4;                   // bytes 0 and 2 of each hold two codes
    *(uint32_t*)(page + q4_k_byte<D>(t, 4 * lane)) = (lo & 0xFFu) | (lo >> 8 & 0xFF00u) | (hi & 0xFFu) << 16 | (hi >> 8 & 0xFF00u) << 16;
  }
  if (lane == 31) *(uint32_t*)(page + 8 * D + 4 * t) = meta;
}
template <int D>
__device__ __forceinline__ void q4_store_v(uint8_t* page, int t, const uint8_t* codes, uint32_t meta, int lane) {
  constexpr int NG = D / 32;
  if (lane < 8 * NG) {
    const uint32_t c = *(const uint32_t*)(codes + 4 * lane), p = c | c >> 4;
    *(uint16_t*)(page + q4_v_byte<D>(t, 2 * lane)) = (uint16_t)((p & 0xFFu) | (p >> 8 & 0xFF00u));
  }
  if (D % 32 && lane < 8) {
    const uint32_t c = *(const uint16_t*)(codes + 32 * NG + 2 * lane);
    page[q4_v_byte<D>(t, 16 * NG + lane)] = (uint8_t)(c | c >> 4);
  }
  if (lane == 31) *(uint32_t*)(page + 8 * D + 4 * t) = meta;
}

}  // namespace rlz
