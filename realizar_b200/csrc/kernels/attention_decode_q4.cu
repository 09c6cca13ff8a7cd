// Decode attention over the 4-bit paged cache (kv_q4.cuh): one new token per sequence, with the norm and rotation of its heads
// and the write of its row in the same launch.
//
//   s_t = q . k_t = scale_t (q . code_t) + min_t sum(q)        o = sum_t p_t v_t = sum_t (p_t scale'_t) code'_t + sum_t p_t min'_t
//
// Bound by the bytes of the cache.  What a page costs besides them:
//   * Codes are never turned into numbers.  A nibble moved to bits 6..9 of an fp16 is the subnormal code x 2^-18, and mma.sync
//     multiplies subnormals exactly: a shift and an AND to two codes instead of a conversion and a multiply-add each.  (The unit
//     lines products up by the exponent fields, so that a nibble left at the low bits, code x 2^-24 without the shift, costs the
//     sum as many bits as stand empty above it: 2e-5 of the result where this gives 3e-7.)
//   * The pages lie in fragment order, so a lane takes its operands with one wide shared-memory load and no shuffles.
//   * Keys (16 tokens) and values (16 dims) are the A operand and the heads the 8 columns of B: 4 heads, each as the fp16 head of
//     its value and what that leaves, also fp16.  22 bits of q and of p x scale' at the price of 11, and the two products of a
//     head meet in one lane.  Up to 4 heads take one such tile, up to 8 two, sharing the A operand.  (Heads as rows, 8 + 8 of
//     16, took twice the instructions and registers for 4 heads: 46 us for every 65536 pages of 128, this STEP2.)
//     q is scaled by a power of two so that its largest value lies in [2^13, 2^14), p x scale' by one that follows the scales.
//   * The running maximum moves only when a score passes it by 2^8, so that the accumulators are rarely rescaled.
// Each warp has a ring of whole pages (K and V) filled by bulk copies.
//
// Split: the pages of all (sequence, kv head, head group) tiles, in units of four, are divided evenly over one wave of CTAs,
// whatever the lengths are; positions are read on the device, so a captured launch serves growing sequences.  A CTA whose units
// do not cover a tile leaves its part in scratch, and the last of the tile's CTAs to arrive joins them in a fixed order.
#include "attention_q4.cuh"
#include "kv_q4.cuh"
#include <algorithm>

namespace rlz {

// 3211: a page never arrived (bounded wait ran out); 3311: a position beyond the page-table row (the sequence is skipped);
// 3312: a page id outside the cache (read as page 0, not written)
__device__ int g_attn_q4_error = 0;

constexpr int QD_WARPS = 4, QD_THREADS = 32 * QD_WARPS, QD_STAGES = 4;
constexpr int QD_MAX_PARTS = 64;              // CTAs that share a tile: bounds the time of the last one, which joins their parts
// query heads of a CTA (HN tiles of 4) and CTAs to an SM, by registers
constexpr int qd_heads(int hn) { return 4 * hn; }
constexpr int qd_occupancy(int hn) { return hn == 1 ? 4 : 3; }
constexpr int QD_MAX_SMS = 148;

template <int D, int HN> struct QdSmem {
  float q[4 * HN][D];
  float part[QD_WARPS][4 * HN][D + 4];         // per warp and head: sum, then maximum and weight
  float qc[4 * HN], qx[4 * HN];               // 2^18 / f of a head whose fragments hold q f, and the sum of q
  uint8_t codes[2][D];                        // the new token's rows
  uint32_t meta[2];
  int wsum[QD_WARPS];
  int plan_b, plan_rem, last;
  unsigned long long full[QD_WARPS][QD_STAGES];
};

__device__ __forceinline__ int q4_page_id(int raw, int num_pages) {
  if (num_pages > 0 && (unsigned)raw >= (unsigned)num_pages) { atomicExch(&g_attn_q4_error, 3312); return 0; }
  return raw;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// nibble J of both halves of a word as fp16 subnormals: code x 2^-18
template <int J> __device__ __forceinline__ uint32_t nib(uint32_t w) {
  return (J == 0 ? w << 6 : J == 1 ? w << 2 : J == 2 ? w >> 2 : w >> 6) & 0x03C003C0u;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// fp16 head of a value (low half) and of what the head leaves (high half)
__device__ __forceinline__ uint32_t split_f16(float x) {
  const __half h = __float2half_rn(x);
  const __half2 r = __halves2half2(h, __float2half_rn(x - __half2float(h)));
  return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {       // of 16-bit values, row = lane / 4
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 2^(e - exponent of x), at most 2^100; x > 0
__device__ __forceinline__ float pow2_for(float x, int e) {
  const int k = e + 254 - (int)(__float_as_uint(x) >> 23);
  return __uint_as_float((uint32_t)max(1, min(k, 227)) << 23);
}
template <int N> __device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&w)[N]) {
  if constexpr (N == 4) { const uint4 v = *(const uint4*)src; w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
  else if constexpr (N == 2) { const uint2 v = *(const uint2*)src; w[0] = v.x; w[1] = v.y; }
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = ((const uint32_t*)src)[i];
  }
}

struct QdSeq { int pos, lo, first_page, pages, units; };      // units of QD_WARPS pages; 0: nothing to do
__device__ __forceinline__ QdSeq qd_seq(const AttnDecodeParams& p, int b) {
  QdSeq s = {p.positions[b], 0, 0, 0, 0};
  if (s.pos < 0) return s;
  if (s.pos / Q4_PAGE >= p.max_pages) { atomicExch(&g_attn_q4_error, 3311); return s; }
  s.lo = p.window > 0 ? max(0, s.pos + 1 - p.window) : 0;
  s.first_page = s.lo / Q4_PAGE;
  s.pages = s.pos / Q4_PAGE + 1;
  s.units = (s.pages - s.first_page + QD_WARPS - 1) / QD_WARPS;
  return s;
}

template <int D, int HN>
__global__ void __launch_bounds__(QD_THREADS, qd_occupancy(HN)) attn_decode_q4_kernel(const __grid_constant__ AttnDecodeParams p) {
  constexpr int QD_ROWS = 4 * HN;
  constexpr int NG = D / 32, TAIL = D % 32 ? 1 : 0, KS = 2 * NG + TAIL, NT = 2 * NG + TAIL, PB = q4_page_bytes(D), NP = HeadPairs<D>::NP;
  extern __shared__ __align__(128) uint8_t qd_ring[];
  __shared__ __align__(16) QdSmem<D, HN> sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  if (tid < QD_WARPS * QD_STAGES) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(att_smem_u32(&sm.full[0][0] + tid)));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();

  // ---- my share of the units: [u, uend) of the sequence of all tiles' units -------------------------------------------------
  const int G = p.n_heads / p.n_kv_heads, hgroups = (G + QD_ROWS - 1) / QD_ROWS, tiles = p.n_kv_heads * hgroups;
  const int per = (p.batch + QD_THREADS - 1) / QD_THREADS, b_lo = min(tid * per, p.batch), b_hi = min(b_lo + per, p.batch);
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += qd_seq(p, b).units * tiles;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o); if (lane >= o) incl += v; }
  if (lane == 31) sm.wsum[warp] = incl;
  __syncthreads();
  int total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < QD_WARPS; ++w) { if (w < warp) before += sm.wsum[w]; total += sm.wsum[w]; }
  const int ctas = min((int)gridDim.x, total), c = blockIdx.x;
  if (c >= ctas) return;
  const int u0 = (int)((int64_t)c * total / ctas), uend = (int)((int64_t)(c + 1) * total / ctas);
  if (mine > 0 && before <= u0 && u0 < before + mine) {
    int b = b_lo, at = before;
    for (;; ++b) { const int n = qd_seq(p, b).units * tiles; if (u0 < at + n) break; at += n; }
    sm.plan_b = b; sm.plan_rem = u0 - at;
  }
  __syncthreads();

  const RopeArgs rope = {p.rope_table, p.rope_table_len, p.rope_dim, p.rope_type, p.rope_theta};
  const int half = p.rope_dim >> 1;
  const float qscale = p.scale * 1.4426950408889634f;
  uint8_t* my_ring = qd_ring + (size_t)warp * QD_STAGES * 2 * PB;
  uint32_t taken = 0;                                          // pages this warp has been through: ring slot and parity
  bool ok = true;

  for (int u = u0, b = sm.plan_b, rem = sm.plan_rem; u < uend;) {
    const QdSeq s = qd_seq(p, b);
    if (s.units == 0) { ++b; rem = 0; continue; }
    const int tile = rem / s.units, ub = rem - tile * s.units, n_units = min(s.units - ub, uend - u);
    const int kvh = tile / hgroups, g0 = (tile - kvh * hgroups) * QD_ROWS, gn = min(QD_ROWS, G - g0);
    const int tile_u0 = u - ub;
    const int page0 = s.first_page + ub * QD_WARPS, page1 = min(s.pages, page0 + n_units * QD_WARPS);
    const bool owner = !p.no_append && page1 == s.pages;         // the new token's page is mine
    const int n_my = max(0, (page1 - page0 - warp + QD_WARPS - 1) / QD_WARPS);
    const int32_t* pt = p.page_table + (int64_t)b * p.pt_stride + page0 + warp;

    // ---- first pages under way; lane i keeps the id of my i-th page of a group of 32, and of the next group -------------------
    int ids = lane < n_my ? q4_page_id(pt[QD_WARPS * lane], p.num_pages) : 0, ids_next = 0;
    auto issue = [&](int i) {                                     // pages i and i + 1 (i even): lanes 0 and 1 take one each
      if ((i & 31) == 0) {
        if (i > 0) ids = ids_next;
        ids_next = i + 32 + lane < n_my ? q4_page_id(pt[QD_WARPS * (i + 32 + lane)], p.num_pages) : 0;
      }
      const int id = __shfl_sync(0xFFFFFFFFu, ids, (i + lane) & 31);
      if (lane < 2 && i + lane < n_my) {
        const uint32_t slot = (taken + i + lane) % QD_STAGES;
        unsigned long long* bar = &sm.full[warp][slot];
        uint8_t* dst = my_ring + slot * (2 * PB);
        const int64_t off = ((int64_t)id * p.n_kv_heads + kvh) * PB;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(att_smem_u32(bar)), "r"((uint32_t)(2 * PB)) : "memory");
        att_bulk_g2s(dst, (const uint8_t*)p.k_cache + off, PB, bar);
        att_bulk_g2s(dst + PB, (const uint8_t*)p.v_cache + off, PB, bar);
      }
    };
    for (int i = 0; i < min(QD_STAGES, n_my); i += 2) issue(i);

    // ---- the new token: queries of the group, and in the owner its key and value rows ------------------------------------------
    const float* row = p.qkv + (int64_t)b * p.ld_qkv;
    float2 cs[NP];
    load_rope<D>(rope, s.pos, lane, cs);
    float x0[NP], x1[NP];
    auto load = [&](const float* src, int hf, int type) {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int i = lane + 32 * k;
        x0[k] = x1[k] = 0.f;
        if (i < D / 2) { const int2 at = pair_dims(i, hf, type); x0[k] = src[at.x]; x1[k] = src[at.y]; }
      }
    };
    for (int g = warp; g < gn; g += QD_WARPS) {
      load(row + p.q_off + (int64_t)(kvh * G + g0 + g) * D, half, p.rope_type);
      norm_rope_f<D>(x0, x1, p.q_norm_w, p.eps, rope, cs, lane);
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        x0[k] *= qscale; x1[k] *= qscale;
        top = fmaxf(top, fmaxf(fabsf(x0[k]), fabsf(x1[k]))); sum += x0[k] + x1[k];
      }
      top = warp_max(top); sum = warp_sum(sum);
      const float f = top > 0.f ? pow2_for(top, 13) : 1.f;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int i = lane + 32 * k;
        if (i < D / 2) { const int2 at = pair_dims(i, half, p.rope_type); sm.q[g][at.x] = x0[k] * f; sm.q[g][at.y] = x1[k] * f; }
      }
      if (lane == 0) { sm.qc[g] = 262144.f / f; sm.qx[g] = sum; }
    }
    if (owner && warp >= 2) {
      const bool v = warp == 3;
      load(row + (v ? p.v_off : p.k_off) + kvh * D, v ? 0 : half, v ? 0 : p.rope_type);
      if (!v) norm_rope_d<D>(x0, x1, p.q_norm_w ? p.k_norm_w : nullptr, (double)p.eps, rope, cs, lane);
      const uint32_t meta = q4_quantise<D>(x0, x1, v ? 0 : half, v ? 0 : p.rope_type, lane, sm.codes[v]);
      __syncwarp();
      if (lane == 0) sm.meta[v] = meta;
      if (g0 == 0) {                                             // one head group writes the row
        const int raw = p.page_table[(int64_t)b * p.pt_stride + s.pos / Q4_PAGE];
        if (p.num_pages <= 0 || (unsigned)raw < (unsigned)p.num_pages) {
          uint8_t* dst = (uint8_t*)(v ? p.v_cache : p.k_cache) + ((int64_t)raw * p.n_kv_heads + kvh) * PB;
          if (v) q4_store_v<D>(dst, s.pos % Q4_PAGE, sm.codes[1], meta, lane);
          else q4_store_k<D>(dst, s.pos % Q4_PAGE, sm.codes[0], meta, lane);
        }
      }
    }
    __syncthreads();

    // ---- query fragments: column gq is head gq / 2 of a tile, its head (even) or what that leaves (odd).  Word tq of a group of 32
    // dims holds dims 8 tq .. + 7 and its nibbles pair as (0, 4), (1, 5), (2, 6), (3, 7) ----
    uint32_t qb[HN][KS][2];
    float qc[HN], qx[HN];
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      const int head = 4 * h + (gq >> 1);
      const bool has = head < gn;
      const float* qr = sm.q[has ? head : 0];
      const uint32_t sel = gq & 1 ? 0x7632u : 0x5410u;            // odd columns take the high halves of the two splits
      auto frag = [&](int d0, int d1) { return has ? __byte_perm(split_f16(qr[d0]), split_f16(qr[d1]), sel) : 0u; };
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int d = 32 * g + 8 * tq;
        qb[h][2 * g][0] = frag(d, d + 4); qb[h][2 * g][1] = frag(d + 1, d + 5);
        qb[h][2 * g + 1][0] = frag(d + 2, d + 6); qb[h][2 * g + 1][1] = frag(d + 3, d + 7);
      }
      if constexpr (TAIL) { const int d = 32 * NG + 4 * tq; qb[h][2 * NG][0] = frag(d, d + 1); qb[h][2 * NG][1] = frag(d + 2, d + 3); }
      const bool mine_is = 4 * h + tq < gn;                      // the head whose scores this lane holds
      qc[h] = mine_is ? sm.qc[4 * h + tq] : 0.f; qx[h] = mine_is ? sm.qx[4 * h + tq] : 0.f;
    }

    float o[HN][NT][4], m[HN], l[HN], om[HN];                    // om: sum of p x min'
#pragma unroll
    for (int h = 0; h < HN; ++h) {
#pragma unroll
      for (int n = 0; n < NT; ++n) o[h][n][0] = o[h][n][1] = o[h][n][2] = o[h][n][3] = 0.f;
      m[h] = -INFINITY; l[h] = om[h] = 0.f;
    }
    float vf = 0x1p100f;                                          // power of two that p x scale' carries

    for (int i = 0; i < n_my; i += 2) {                           // two pages at a time (of an odd number, the last comes with a masked one)
      uint8_t* kp[2];
      int t0[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t slot = (taken + i + j) % QD_STAGES, parity = ((taken + i + j) / QD_STAGES) & 1u;
        kp[j] = my_ring + slot * (2 * PB);
        const int page = page0 + warp + QD_WARPS * (i + j);
        t0[j] = page * Q4_PAGE;
        if (i + j < n_my) {
          bool arrived = false;
          const uint32_t limit = ok ? ATT_WAIT_LIMIT : 1024u;
          for (uint32_t spin = 0; spin < limit; ++spin) if (att_try_wait(&sm.full[warp][slot], parity)) { arrived = true; break; }
          if (!arrived) { ok = false; atomicExch(&g_attn_q4_error, 3211); }
          if (owner && page == s.pages - 1) {                    // the copy may have passed the write of the new row
            q4_store_k<D>(kp[j], s.pos % Q4_PAGE, sm.codes[0], sm.meta[0], lane);
            q4_store_v<D>(kp[j] + PB, s.pos % Q4_PAGE, sm.codes[1], sm.meta[1], lane);
            __syncwarp();
          }
        }
      }
      // ---- scores: lane has tokens gq and gq + 8 of head tq of a tile ----
      float acc[2][HN][4], sc[HN][2][2], sv[2][2], mv[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int h = 0; h < HN; ++h) acc[j][h][0] = acc[j][h][1] = acc[j][h][2] = acc[j][h][3] = 0.f;
        uint32_t wa[NG], wb[NG];
        load_words<NG>(kp[j] + gq * (D / 2) + tq * NG * 4, wa);
        load_words<NG>(kp[j] + (gq + 8) * (D / 2) + tq * NG * 4, wb);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t a0 = nib<0>(wa[g]), a1 = nib<0>(wb[g]), a2 = nib<1>(wa[g]), a3 = nib<1>(wb[g]);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(acc[j][h], a0, a1, a2, a3, qb[h][2 * g][0], qb[h][2 * g][1]);
          const uint32_t b0 = nib<2>(wa[g]), b1 = nib<2>(wb[g]), b2 = nib<3>(wa[g]), b3 = nib<3>(wb[g]);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(acc[j][h], b0, b1, b2, b3, qb[h][2 * g + 1][0], qb[h][2 * g + 1][1]);
        }
        if constexpr (TAIL) {
          const uint8_t* kt = kp[j] + 16 * NG + 2 * tq;
          const uint32_t ra = (uint32_t)*(const uint16_t*)(kt + gq * (D / 2)) * 0x10001u, rb = (uint32_t)*(const uint16_t*)(kt + (gq + 8) * (D / 2)) * 0x10001u;
          const uint32_t a0 = (nib<0>(ra) & 0xFFFFu) | (nib<1>(ra) & 0xFFFF0000u), a1 = (nib<0>(rb) & 0xFFFFu) | (nib<1>(rb) & 0xFFFF0000u);
          const uint32_t a2 = (nib<2>(ra) & 0xFFFFu) | (nib<3>(ra) & 0xFFFF0000u), a3 = (nib<2>(rb) & 0xFFFFu) | (nib<3>(rb) & 0xFFFF0000u);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(acc[j][h], a0, a1, a2, a3, qb[h][2 * NG][0], qb[h][2 * NG][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t km = *(const uint32_t*)(kp[j] + 8 * D + (gq + 8 * n) * 4), vm = *(const uint32_t*)(kp[j] + PB + 8 * D + (gq + 8 * n) * 4);
          sv[j][n] = q4_scale(vm); mv[j][n] = q4_min(vm);
#pragma unroll
          for (int h = 0; h < HN; ++h) sc[h][j][n] = fmaf((acc[j][h][2 * n] + acc[j][h][2 * n + 1]) * qc[h], q4_scale(km), q4_min(km) * qx[h]);
        }
        if (i + j >= n_my || t0[j] < s.lo || t0[j] + Q4_PAGE - 1 > s.pos) {      // rows outside the window or behind the last token hold anything
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int t = t0[j] + gq + 8 * n;
            if (i + j >= n_my || t < s.lo || t > s.pos) {
              sv[j][n] = mv[j][n] = 0.f;
#pragma unroll
              for (int h = 0; h < HN; ++h) sc[h][j][n] = -INFINITY;
            }
          }
        }
      }
      // ---- running maximum and scale: moved only where they fall behind by 2^8 and 2^2 ----
      float mx[HN], top = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
      bool behind = top * vf > 126.f;
#pragma unroll
      for (int h = 0; h < HN; ++h) {
        mx[h] = fmaxf(fmaxf(sc[h][0][0], sc[h][0][1]), fmaxf(sc[h][1][0], sc[h][1][1]));
        behind |= mx[h] > m[h] + 8.f;
      }
      if (__any_sync(0xFFFFFFFFu, behind)) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
#pragma unroll
          for (int h = 0; h < HN; ++h) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], k));
        }
        const float vn = top * vf > 126.f ? pow2_for(top, 5) : vf, vr = vn / vf;
        vf = vn;
#pragma unroll
        for (int h = 0; h < HN; ++h) {
          const float mn = fmaxf(m[h], mx[h]), corr = m[h] == -INFINITY ? 0.f : ex2(m[h] - mn), co = corr * vr;
#pragma unroll
          for (int n = 0; n < NT; ++n) { o[h][n][0] *= co; o[h][n][1] *= co; o[h][n][2] *= co; o[h][n][3] *= co; }
          l[h] *= corr; om[h] *= corr; m[h] = mn;
        }
      }
      // ---- O += P V: rows gq and gq + 8 of tile 2 g + k are dims 32 g + 4 gq + 2 k and + 1 ----
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t pb[HN][2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float f = sv[j][n] * vf;
#pragma unroll
          for (int h = 0; h < HN; ++h) {
            const float e = ex2(sc[h][j][n] - m[h]);
            l[h] += e;
            om[h] = fmaf(e, mv[j][n], om[h]);
            pb[h][n] = transpose_8x8(split_f16(e * f));
          }
        }
        const uint8_t* vp = kp[j] + PB;
        uint32_t w0[NG], w1[NG];
        load_words<NG>(vp + lane * NG * 4, w0);
        load_words<NG>(vp + 128 * NG + lane * NG * 4, w1);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t a0 = nib<0>(w0[g]), a1 = nib<1>(w0[g]), a2 = nib<0>(w1[g]), a3 = nib<1>(w1[g]);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(o[h][2 * g], a0, a1, a2, a3, pb[h][0], pb[h][1]);
          const uint32_t b0 = nib<2>(w0[g]), b1 = nib<3>(w0[g]), b2 = nib<2>(w1[g]), b3 = nib<3>(w1[g]);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(o[h][2 * g + 1], b0, b1, b2, b3, pb[h][0], pb[h][1]);
        }
        if constexpr (TAIL) {
          const uint32_t w = *(const uint32_t*)(vp + 256 * NG + lane * 4);
          const uint32_t r0 = __byte_perm(w, 0u, 0x4140), r1 = __byte_perm(w, 0u, 0x4342);
#pragma unroll
          for (int h = 0; h < HN; ++h) mma_f16(o[h][2 * NG], nib<0>(r0), nib<1>(r0), nib<0>(r1), nib<1>(r1), pb[h][0], pb[h][1]);
        }
      }
      if (i + QD_STAGES < n_my) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // this warp's reads of the slots come before the refill
        __syncwarp();
        issue(i + QD_STAGES);
      }
    }
    taken += n_my;

    // ---- join the warps -----------------------------------------------------------------------------------------------------
    const float e0 = 262144.f / vf;
#pragma unroll
    for (int h = 0; h < HN; ++h) {
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) { l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], k); om[h] += __shfl_xor_sync(0xFFFFFFFFu, om[h], k); }
      if (4 * h + tq < gn) {
        float* dst = sm.part[warp][4 * h + tq];
        auto val = [&](int n, int k) { return fmaf(o[h][n][2 * k] + o[h][n][2 * k + 1], e0, om[h]); };
#pragma unroll
        for (int g = 0; g < NG; ++g) *(float4*)(dst + 32 * g + 4 * gq) = make_float4(val(2 * g, 0), val(2 * g, 1), val(2 * g + 1, 0), val(2 * g + 1, 1));
        if constexpr (TAIL) *(float2*)(dst + 32 * NG + 2 * gq) = make_float2(val(2 * NG, 0), val(2 * NG, 1));
        if (gq == 0) { dst[D] = m[h]; dst[D + 1] = l[h]; }
      }
    }
    __syncthreads();
    const bool whole = n_units == s.units;
    float* out = p.out + (int64_t)b * p.ld_out + (int64_t)(kvh * G + g0) * D;
    // slots of a CTA in scratch: 0 the tile its units begin in, 1 the one they end in
    float* parts = p.partial + (int64_t)(2 * c + (u == u0 ? 0 : 1)) * QD_ROWS * (D + 4);
    for (int it = tid; it < gn * (D / 4); it += QD_THREADS) {
      const int g = it / (D / 4), j = 4 * (it - g * (D / 4));
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < QD_WARPS; ++w) mm = fmaxf(mm, sm.part[w][g][D]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < QD_WARPS; ++w) {
        const float mw = sm.part[w][g][D], e = mw == -INFINITY ? 0.f : ex2(mw - mm);
        const float4 v = *(const float4*)&sm.part[w][g][j];
        ll = fmaf(e, sm.part[w][g][D + 1], ll);
        a.x = fmaf(e, v.x, a.x); a.y = fmaf(e, v.y, a.y); a.z = fmaf(e, v.z, a.z); a.w = fmaf(e, v.w, a.w);
      }
      if (whole) {
        float* dst = out + g * D + j;
        dst[0] = a.x / ll; dst[1] = a.y / ll; dst[2] = a.z / ll; dst[3] = a.w / ll;
      } else {
        float* dst = parts + g * (D + 4);
        *(float4*)(dst + j) = a;
        if (j == 0) { dst[D] = mm; dst[D + 1] = ll; }
      }
    }
    if (!whole) {
      // CTA that holds unit x: the largest c with c total / ctas <= x
      const int c_lo = (int)(((int64_t)(tile_u0 + 1) * ctas - 1) / total), c_hi = (int)(((int64_t)(tile_u0 + s.units) * ctas - 1) / total);
      __threadfence();
      __syncthreads();
      int32_t* ctr = p.counters + (int64_t)b * tiles + tile;
      if (tid == 0) {
        sm.last = atomicAdd(ctr, 1) == c_hi - c_lo;
        if (sm.last) *ctr = 0;                                   // zero again for the next launch
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        const int lead = (int)((int64_t)c_lo * total / ctas) == tile_u0 ? 0 : 1;
        for (int it = tid; it < gn * (D / 4); it += QD_THREADS) {
          const int g = it / (D / 4), j = 4 * (it - g * (D / 4));
          float mm = -INFINITY, ll = 0.f;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = c_lo; k0 <= c_hi; k0 += 8) {
            float2 st[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int kc = min(k0 + k, c_hi);
              const float* src = p.partial + ((int64_t)(2 * kc + (kc == c_lo ? lead : 0)) * QD_ROWS + g) * (D + 4);
              st[k] = __ldcg((const float2*)(src + D));
              v[k] = __ldcg((const float4*)(src + j));
            }
            float mn = mm;
#pragma unroll
            for (int k = 0; k < 8; ++k) mn = fmaxf(mn, st[k].x);
            const float c0 = mm == -INFINITY ? 0.f : ex2(mm - mn);
            a.x *= c0; a.y *= c0; a.z *= c0; a.w *= c0; ll *= c0; mm = mn;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float e = k0 + k > c_hi || st[k].x == -INFINITY ? 0.f : ex2(st[k].x - mm);
              ll = fmaf(e, st[k].y, ll);
              a.x = fmaf(e, v[k].x, a.x); a.y = fmaf(e, v[k].y, a.y); a.z = fmaf(e, v[k].z, a.z); a.w = fmaf(e, v[k].w, a.w);
            }
          }
          float* dst = out + g * D + j;
          dst[0] = a.x / ll; dst[1] = a.y / ll; dst[2] = a.z / ll; dst[3] = a.w / ll;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();                                             // the staging areas and the rings are free for the next tile
    u += n_units; rem += n_units;
    if (rem == s.units * tiles) { ++b; rem = 0; }
  }
}

template <int D, int HN>
static int launch_decode_q4(const AttnDecodeParams& p, cudaStream_t st) {
  int dev = 0, sms = QD_MAX_SMS;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int hgroups = (p.n_heads / p.n_kv_heads + qd_heads(HN) - 1) / qd_heads(HN);
  const long long tiles = (long long)p.batch * p.n_kv_heads * hgroups;
  const int ctas = (int)std::min<long long>(std::min(sms, QD_MAX_SMS) * qd_occupancy(HN), tiles * QD_MAX_PARTS);
  const size_t ring = (size_t)QD_WARPS * QD_STAGES * 2 * q4_page_bytes(D);
  static SmemOptIn opt;
  if (cudaError_t e = opt.ensure(attn_decode_q4_kernel<D, HN>, ring, 0); e != cudaSuccess) return (int)e;
  return (int)launch(attn_decode_q4_kernel<D, HN>, dim3(ctas), dim3(QD_THREADS), ring, st, p);
}

int attn_decode_q4_dispatch(const AttnDecodeParams& p, cudaStream_t st) {
  if (!q4_head_dim_ok(p.head_dim)) return -1;
  if (p.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % p.n_kv_heads || p.batch < 1 || p.max_pages < 1) return -2;
  if (p.rope_dim < 0 || p.rope_dim > p.head_dim || (p.rope_dim & 1)) return -3;
  if (((uintptr_t)p.k_cache & 15) || ((uintptr_t)p.v_cache & 15) || ((uintptr_t)p.partial & 15)) return -4;
  if (p.window < 0) return -5;
  const bool narrow = p.n_heads / p.n_kv_heads <= qd_heads(1);
  switch (p.head_dim) {
    case 64: return narrow ? launch_decode_q4<64, 1>(p, st) : launch_decode_q4<64, 2>(p, st);
    case 80: return narrow ? launch_decode_q4<80, 1>(p, st) : launch_decode_q4<80, 2>(p, st);
    case 96: return narrow ? launch_decode_q4<96, 1>(p, st) : launch_decode_q4<96, 2>(p, st);
    default: return narrow ? launch_decode_q4<128, 1>(p, st) : launch_decode_q4<128, 2>(p, st);
  }
}

}  // namespace rlz

extern "C" {

// floats of scratch (`partial`) that any launch over a 4-bit cache needs
long long rlz_attn_q4_partial_floats(int head_dim) { 
  using namespace rlz;
  return 2LL * QD_MAX_SMS * std::max(qd_occupancy(1) * qd_heads(1), qd_occupancy(2) * qd_heads(2)) * (head_dim + 4);
}

// 0 / 3211 / 3311 / 3312
int rlz_attn_q4_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_attn_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_attn_q4_error, &z, sizeof(int)); }
  return v;
}

}  // extern "C"
