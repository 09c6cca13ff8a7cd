// Decode attention over the 4-bit paged cache (kv_q4.cuh): one new token per sequence, with the norm and rotation of its heads
// and the write of its row in the same launch.
//
//   s_t = q . k_t = scale_t (q . code_t) + min_t sum(q)        o = sum_t p_t v_t = sum_t (p_t scale'_t) code'_t + sum_t p_t min'_t
//
// Meant to be bound by the bytes of the cache, so the arithmetic of the codes has to be cheap (96 ragged sequences of up to 8192 tokens of
// 128 dims, 8 kv heads: 129 us, 4.5 TB/s of the 6.6 that a copy reaches; what is missing is latency, a warp's steps from a pair's keys to
// its values one after another, with 0.53 of the issue slots used):
//   * Keys: a masked word holds four codes as bytes, and the 8-bit integer product takes them as they are; q comes as three 8-bit
//     digits of a 24-bit integer (its largest value in [2^22, 2^23) x 127 / 128), so the sums over the dims are exact; sum(q) is that of
//     the integers.
//   * Values: a nibble under the exponent of 1024 is the fp16 1024 + code (or 1024 + 16 code), which one subtraction (or
//     multiply-add) turns into code - 8 exactly: 9 instructions to 8 codes.  The 8 goes into the minimum: without it, sum p scale code
//     and sum p min cancel, over 131072 tokens to 1 / 900, and so do the digits of the result (2e-4 of it instead of 1e-6).
//     p x scale' comes as its fp16 head and 2^11 times what that leaves, also fp16: 22 bits down to 2^-23 of the largest weight (and 1
//     less to each factor of 2 below), because where the largest belongs to a value near zero the result is the sum of the small ones
//     (32768 keys, one with 99.9% of the weight: 1.7e-3 off when the rest was not scaled).  Its power of two follows the scales.
//   * Tokens (keys) and dims (values) are the 16 rows of the instruction and 4 heads its 8 columns, two digits or halves each, so
//     the parts of a head's sum meet in one lane.  Up to 8 heads take two such tiles and share the other operand.
//   * The pages lie in fragment order: a lane takes its operands with one wide shared-memory load and no shuffles.
//   * The running maximum moves only when a score passes it by 4, a factor of 2^4, so that the accumulators are rarely rescaled (2, 6 and 8
//     take the same time).
//
// One CTA to an SM.  The main warps do nothing but pages: each has a ring of page pairs (K and V) that its lanes fill by 16-byte
// asynchronous copies, and its pages follow one another across tiles.  (Bulk copies need a dozen instructions each, and a warp that
// issued them for all was too slow.)  Four helper warps prepare the next tile's query fragments (and the new token's rows) and join
// and store the finished tile meanwhile, through two buffers each.
// (With every warp doing its share of that between two tiles, a batch of 64 x 2048 tokens spent 28 of its 60 us there.)
//
// Split, in pairs of pages: with more tiles (sequence, kv head, head group) than CTAs, the pairs of all tiles are divided evenly,
// whatever the lengths are; with fewer, every tile gets the same number of CTAs, unless that leaves one of them with much more
// than an even share.  Positions are read on the device, so a captured launch serves growing sequences.  A CTA that has only some
// pairs of a tile leaves its part in scratch, and the last of the tile's CTAs to arrive joins them in a fixed order.
#include "attention_q4.cuh"
#include "kv_q4.cuh"
#include <algorithm>
#include <atomic>

namespace rlz {

// 3211: a tile's helpers or main warps never answered (bounded wait ran out); 3311: a position beyond the page-table row (the sequence is skipped);
// 3312: a page id outside the cache (read as page 0, not written)
__device__ int g_attn_q4_error = 0;
static std::atomic<bool> attn_q4_ran{false};         // until a launch there is no status to fetch, which takes a synchronous copy

constexpr int QD_STAGES = 3, QD_MAX_SMS = 148, QD_HELPERS = 128;
constexpr int QD_PAIR = 2 * Q4_PAGE;          // tokens of a pair of pages
constexpr int QD_TILE_COST = 40;              // a second tile costs a CTA about as much time as this many pairs
constexpr int QD_FLUSH = 8;                   // pairs whose values a warp adds up in the tensor core's accumulators, a power of two
// p x scale' as fp16: p is at most 2^QD_LAG, by which a score may pass the running maximum before that moves, and scale' carries a power of
// two that keeps it below QD_TOP, so that the product stays below 2^15 and what its fp16 head leaves, times QD_REST, below 2^14
constexpr int QD_LAG = 4;
constexpr float QD_TOP = 63.f / 64.f * (float)(1 << (15 - QD_LAG)), QD_REST = 2048.f;
constexpr int QD_POSITIONS = 512;
constexpr int QD_MAX_PARTS = 64;              // CTAs that share a tile: bounds the time of the last one, which joins their parts
// query heads of a CTA (HN tiles of 4) and its main warps: with the four others 16 warps of 128 registers, or 12 of 168
constexpr int qd_heads(int hn) { return 4 * hn; }
constexpr int qd_warps(int hn) { return hn == 1 ? 12 : 8; }

template <int D, int HN> struct QdSmem {
  static constexpr int NF = D / 32 + (D % 32 ? 1 : 0), ROWS = 4 * HN;
  uint4 frag[2][HN][NF][32];                  // digits 0 and 1 (x, y), 2 and none (z, w) of the heads, as the main warps' lanes hold them
  float part[2][qd_warps(HN)][ROWS][D + 4];   // per warp and head: sum, then maximum and weight
  float q[ROWS][D];                           // helpers: normalised, rotated and scaled queries
  float qc[2][ROWS], qx[2][ROWS];             // 1 / f of a head whose fragments hold the integer q f, and the sum of q
  uint8_t codes[2][2][D];                     // the new token's rows (key, value)
  uint32_t meta[2][2];
  struct { int n, tok, lo, pos, own; } tile[2];   // pairs, first token, first and last visible position, place of the new token's pair or -1
  int last;
  int pos[QD_POSITIONS];                      // positions of the first sequences, which are asked for again and again
  unsigned long long frag_full[2], part_full[2], part_empty[2], own_full[2];
};

__device__ __forceinline__ int q4_page_id(int raw, int num_pages) {
  if (num_pages > 0 && (unsigned)raw >= (unsigned)num_pages) { atomicExch(&g_attn_q4_error, 3312); return 0; }
  return raw;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// nibbles 0..3 of both halves of a word as fp16, less 8
__device__ __forceinline__ void codes_less_8(uint32_t w, uint32_t (&c)[4]) {
  const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k16th = __half2half2(__ushort_as_half(0x2C00)), k72 = __half2half2(__ushort_as_half(0xD480));
  const uint32_t h = w >> 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = ((i ? h : w) & 0x000F000Fu) | 0x64006400u, y = ((i ? h : w) & 0x00F000F0u) | 0x64006400u;
    const __half2 u = __hsub2(*(const __half2*)&x, k1032), v = __hfma2(*(const __half2*)&y, k16th, k72);
    c[2 * i] = *(const uint32_t*)&u; c[2 * i + 1] = *(const uint32_t*)&v;
  }
}
__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_half(int* c, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(b0));
}
// four codes of 16 bits as bytes
__device__ __forceinline__ uint32_t nib_bytes(uint32_t h) { const uint32_t x = (h | h << 8) & 0x00FF00FFu; return (x | x << 4) & 0x0F0F0F0Fu; }
// an integer below 2^23 x 127 / 128 as three signed bytes, the first in the low bits
__device__ __forceinline__ uint32_t digits(int q) {
  const int d2 = (int)(int8_t)(q & 255), q1 = (q - d2) >> 8, d1 = (int)(int8_t)(q1 & 255), d0 = (q1 - d1) >> 8;
  return (uint32_t)(d0 & 255) | (uint32_t)(d1 & 255) << 8 | (uint32_t)(d2 & 255) << 16;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// fp16 heads of two values (low halves) and QD_REST times what the heads leave (high halves)
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t (&w)[2]) {
  const float2 h = __half22float2(__floats2half2_rn(x0, x1));
  const __half2 a = __floats2half2_rn(x0, (x0 - h.x) * QD_REST), b = __floats2half2_rn(x1, (x1 - h.y) * QD_REST);
  w[0] = *(const uint32_t*)&a; w[1] = *(const uint32_t*)&b;
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
__device__ __forceinline__ float inverse_pow2(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }      // x a power of two from pow2_for
template <int N> __device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&w)[N]) {
  if constexpr (N == 4) { const uint4 v = *(const uint4*)src; w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
  else if constexpr (N == 2) { const uint2 v = *(const uint2*)src; w[0] = v.x; w[1] = v.y; }
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = ((const uint32_t*)src)[i];
  }
}

struct QdSeq { int pos, lo, first_page, n; };                 // n pairs of pages from first_page on; 0: nothing to do
__device__ __forceinline__ QdSeq qd_seq(const AttnDecodeParams& p, const int* cached, int b) {
  QdSeq s = {b < QD_POSITIONS ? cached[b] : p.positions[b], 0, 0, 0};
  if (s.pos < 0) return s;
  if (s.pos / Q4_PAGE >= p.max_pages) { atomicExch(&g_attn_q4_error, 3311); return s; }
  s.lo = p.window > 0 ? max(0, s.pos + 1 - p.window) : 0;
  s.first_page = s.lo / Q4_PAGE;
  s.n = (s.pos / Q4_PAGE - s.first_page) / 2 + 1;
  return s;
}
// the pairs of one tile that a CTA has: `n` of them from the tile's pair `skip` on
struct QdTile { QdSeq s; int b, tile, skip, n; };
// the tile that pair `at` of sequence b's tiles (or the next sequence with any) lies in; the CTA has `left` more pairs
__device__ __forceinline__ QdTile qd_tile(const AttnDecodeParams& p, const int* cached, int b, int at, int left) {
  QdTile t;
  for (;; ++b, at = 0) { t.s = qd_seq(p, cached, b); if (t.s.n) break; }
  t.b = b; t.tile = at / t.s.n; t.skip = at - t.tile * t.s.n; t.n = min(t.s.n - t.skip, left);
  return t;
}
__device__ __forceinline__ QdTile qd_next(const AttnDecodeParams& p, const int* cached, const QdTile& t, int tiles, int left) {
  if (t.tile + 1 == tiles) return qd_tile(p, cached, t.b + 1, 0, left);
  return {t.s, t.b, t.tile + 1, 0, min(t.s.n, left)};
}
// pairs divided evenly: the first one of CTA c (the first `more` have one more than `each`), and the CTA that has pair x
struct QdShare { int each, more; };
__device__ __forceinline__ int qd_first(const QdShare& s, int c) { return c * s.each + min(c, s.more); }
__device__ __forceinline__ int qd_owner(const QdShare& s, int x) {
  const int edge = s.more * (s.each + 1);
  return x < edge ? x / (s.each + 1) : s.more + (x - edge) / s.each;
}
// bounded: false (and the status word) when the barrier's phase does not end
__device__ __forceinline__ bool qd_wait(unsigned long long* bar, uint32_t parity, bool patient) {
  const uint32_t limit = patient ? ATT_WAIT_LIMIT : 1024u;
  for (uint32_t spin = 0; spin < limit; ++spin) if (att_try_wait(bar, parity)) return true;
  atomicExch(&g_attn_q4_error, 3211);
  return false;
}
__device__ __forceinline__ void qd_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(att_smem_u32(bar)) : "memory");
}

template <int D, int HN>
__global__ void __launch_bounds__(32 * qd_warps(HN) + QD_HELPERS, 1) attn_decode_q4_kernel(const __grid_constant__ AttnDecodeParams p) {
  constexpr int ROWS = 4 * HN, NW = qd_warps(HN);
  constexpr int NG = D / 32, TAIL = D % 32 ? 1 : 0, NF = NG + TAIL, NT = 2 * NG + TAIL, PB = q4_page_bytes(D), NP = HeadPairs<D>::NP;
  extern __shared__ __align__(128) uint8_t qd_smem[];
  QdSmem<D, HN>& sm = *(QdSmem<D, HN>*)qd_smem;
  uint8_t* qd_ring = qd_smem + (sizeof(QdSmem<D, HN>) + 127) / 128 * 128;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  if (tid < 8) {
    unsigned long long* bar = tid < 2 ? &sm.frag_full[tid] : tid < 4 ? &sm.part_full[tid - 2] : tid < 6 ? &sm.part_empty[tid - 4] : &sm.own_full[tid - 6];
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(att_smem_u32(bar)), "r"(tid < 2 ? QD_HELPERS : tid < 4 ? NW : tid < 6 ? 1 : 64));
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  for (int b = tid; b < min(p.batch, QD_POSITIONS); b += 32 * NW + QD_HELPERS) sm.pos[b] = __ldg(p.positions + b);
  __syncthreads();

  // ---- my share: pairs [x0, x1) of the sequence of all tiles' pairs.  Every warp works it out, its lanes over the sequences.  (Integer
  // quotients by variables take 100 clocks each, one after another: as few as there can be) ------------------------------------------
  const int G = p.n_heads / p.n_kv_heads, hgroups = (G + ROWS - 1) / ROWS, tiles = p.n_kv_heads * hgroups, c = blockIdx.x;
  int mine = 0, live = 0, longest = 0, b_lo = 0;
  if (p.batch == 1) { mine = longest = qd_seq(p, sm.pos, 0).n; live = mine > 0; }
  else {
    const int per = (p.batch + 31) / 32, b_hi = min((lane + 1) * per, p.batch);
    b_lo = min(lane * per, p.batch);
    for (int b = b_lo; b < b_hi; ++b) { const int n = qd_seq(p, sm.pos, b).n; mine += n; live += n > 0; longest = max(longest, n); }
  }
  int incl = mine, live_incl = live, total = mine, all_tiles = live;
  if (p.batch > 1) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o), w = __shfl_up_sync(0xFFFFFFFFu, live_incl, o);
      if (lane >= o) { incl += v; live_incl += w; }
    }
    total = __shfl_sync(0xFFFFFFFFu, incl, 31); all_tiles = __shfl_sync(0xFFFFFFFFu, live_incl, 31);
    longest = __reduce_max_sync(0xFFFFFFFFu, longest);
  }
  total *= tiles; all_tiles *= tiles;
  if (total == 0) return;
  const int split = min((int)gridDim.x / all_tiles, longest);     // CTAs to a tile, 0: there are more tiles
  const bool by_tile = split > 0 && __fdividef((float)longest, (float)split) < __fdividef((float)total, (float)gridDim.x) + QD_TILE_COST;
  const int ctas = by_tile ? all_tiles * split : min((int)gridDim.x, total);
  if (c >= ctas) return;
  const int my_tile = by_tile ? c / split : 0;
  QdShare share = {0, 0};
  if (!by_tile) { share.each = total / ctas; share.more = total - share.each * ctas; }
  int x0 = qd_first(share, c), x1 = x0 + share.each + (c < share.more ? 1 : 0);
  // the lane whose sequences hold place x0, or (by tile) live tile c / split
  const int want = by_tile ? my_tile : x0;
  int b0 = b_lo, at0 = want;
  if (p.batch == 1) { if (by_tile) at0 *= mine; }
  else {
    const int first = by_tile ? (live_incl - live) * tiles : (incl - mine) * tiles;
    const bool holds = first <= want && want < (by_tile ? live_incl : incl) * tiles;
    at0 -= first;
    if (holds)
      for (;; ++b0) {
        const int n = qd_seq(p, sm.pos, b0).n, m = (by_tile ? n > 0 : n) * tiles;
        if (at0 < m) { if (by_tile) at0 *= n; break; }
        at0 -= m;
      }
    const int holder = __ffs(__ballot_sync(0xFFFFFFFFu, holds)) - 1;
    b0 = __shfl_sync(0xFFFFFFFFu, b0, holder);
    at0 = __shfl_sync(0xFFFFFFFFu, at0, holder);
  }
  if (by_tile) {                                                   // places count from the tile's first pair
    const int n = qd_seq(p, sm.pos, b0).n, parts = min(split, n), part = c - my_tile * split;
    if (part >= parts) return;
    const QdShare in_tile = {n / parts, n % parts};
    x0 = qd_first(in_tile, part); x1 = x0 + in_tile.each + (part < in_tile.more ? 1 : 0); at0 += x0;
  }
  // Pair k of main warp w is pair w + NW k of the CTA's share: the tiles' ends fall on all warps alike.
  auto first_k = [](int w, int x) { return x > w ? (x - w + NW - 1) / NW : 0; };        // first pair of warp w at or behind place x of the share
  bool ok = true;

  if (warp < NW) {
    // ================================ main warps ================================================================================
    uint8_t* my_ring = qd_ring + (size_t)warp * QD_STAGES * 4 * PB;
    // -- the copies, pair after pair of the stream.  Lane i keeps the (page, kv head) row of page i % 2 of the i / 2-th of 16 pairs; the
    // ids of the 16 behind them are on their way
    QdTile f = qd_tile(p, sm.pos, b0, at0, x1 - x0);
    int f_at = 0, row_now, id_next, kvh_next;
    auto fetch = [&](int k) {                                        // ids of pairs k .. k + 15
      while (f_at + f.n < x1 - x0 && warp + NW * k >= f_at + f.n) { f_at += f.n; f = qd_next(p, sm.pos, f, tiles, x1 - x0 - f_at); }
      const int x = warp + NW * (k + (lane >> 1));
      kvh_next = -1;
      if (x < x1 - x0) {
        QdTile t = f;
        int t_at = f_at;
        while (x >= t_at + t.n) { t_at += t.n; t = qd_next(p, sm.pos, t, tiles, x1 - x0 - t_at); }
        const int page = t.s.first_page + 2 * (t.skip + x - t_at) + (lane & 1);
        if (page <= t.s.pos / Q4_PAGE) { id_next = __ldg(p.page_table + (int64_t)t.b * p.pt_stride + page); kvh_next = t.tile / hgroups; }
      }
    };
    auto turn = [&]() { row_now = kvh_next < 0 ? -1 : q4_page_id(id_next, p.num_pages) * p.n_kv_heads + kvh_next; };
    const uint8_t* const my_k = (const uint8_t*)p.k_cache + 16 * lane;
    const int64_t k_to_v = (const uint8_t*)p.v_cache - (const uint8_t*)p.k_cache;
    auto copy_pair = [&](int k, uint32_t to) {
      if ((k & 15) == 0) { turn(); fetch(k + 16); }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = __shfl_sync(0xFFFFFFFFu, row_now, 2 * (k & 15) + j);
        if (row >= 0) {
          const uint8_t* src = my_k + (int64_t)row * PB;
          const uint32_t dst = att_smem_u32(my_ring) + to * (4 * PB) + j * (2 * PB) + 16 * lane;
#pragma unroll
          for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < (PB + 511) / 512; ++i)
              if (512 * (i + 1) <= PB || 512 * i + 16 * lane < PB)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + v * PB + 512 * i), "l"(src + (v ? k_to_v : 0) + 512 * i) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0);
    for (int k = 0; k < QD_STAGES - 1; ++k) copy_pair(k, k);
    uint32_t slot = 0;
    for (int it = 0, at = 0; at < x1 - x0; ++it) {
      const int buf = it & 1;
      const uint32_t phase = (uint32_t)(it >> 1) & 1u;
      ok = qd_wait(&sm.frag_full[buf], phase, ok) && ok;
      if (!ok) break;                                                // the tile's description never came
      const auto s = sm.tile[buf];
      const int end = at + s.n, k0 = first_k(warp, at), k1 = first_k(warp, end);
      if (k0 < k1) {
        const int own = s.own >= 0 && s.own % NW == warp ? s.own / NW : -1;              // my pair that holds the new token
        uint4 qb[HN][NF];
        float qc[HN], qx[HN];
#pragma unroll
        for (int h = 0; h < HN; ++h) {
#pragma unroll
          for (int f = 0; f < NF; ++f) qb[h][f] = sm.frag[buf][h][f][lane];
          qc[h] = sm.qc[buf][4 * h + tq]; qx[h] = sm.qx[buf][4 * h + tq];
        }
        float o[HN][NT][4], m[HN], l[HN], om[HN];                  // om: sum of p (min' + 8 scale')
#pragma unroll
        for (int h = 0; h < HN; ++h) {
#pragma unroll
          for (int n = 0; n < NT; ++n) o[h][n][0] = o[h][n][1] = o[h][n][2] = o[h][n][3] = 0.f;
          m[h] = -INFINITY; l[h] = om[h] = 0.f;
        }
        float vf = 0x1p100f;                                        // power of two that p x scale' carries
        // Every QD_FLUSH pairs the sums go to the warp's part in shared memory: the tensor core cuts off what its 32-bit accumulators do
        // not hold, always towards zero, so that the error of one long sum grows with its length (131072 tokens: 1.2e-6 of the result)
        auto part_at = [&](int h) { return sm.part[buf][warp][4 * h + tq] + 4 * gq; };
        auto for_part = [&](auto f) {                                // f(h, n, k, place in shared memory) for the lane's values
#pragma unroll
          for (int h = 0; h < HN; ++h) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              float4* at4 = (float4*)(part_at(h) + 32 * g);
              float4 v = *at4;
              v.x = f(h, 2 * g, 0, v.x); v.y = f(h, 2 * g, 1, v.y); v.z = f(h, 2 * g + 1, 0, v.z); v.w = f(h, 2 * g + 1, 1, v.w);
              *at4 = v;
            }
            if constexpr (TAIL) {
              float2* at2 = (float2*)(sm.part[buf][warp][4 * h + tq] + 32 * NG + 2 * gq);
              float2 v = *at2;
              v.x = f(h, 2 * NG, 0, v.x); v.y = f(h, 2 * NG, 1, v.y);
              *at2 = v;
            }
          }
        };
        int tok = s.tok + (warp + NW * k0 - at) * QD_PAIR;           // first token of pair k

        int kb = k0;                                                // first pair of the sums in the accumulators
        for (;;) {
          const int ke = min(kb + QD_FLUSH, k1);
          for (int k = kb; k < ke; ++k, tok += NW * QD_PAIR) {          // (of an odd number of pages the last comes with a masked one)
            copy_pair(k + QD_STAGES - 1, slot == 0 ? QD_STAGES - 1 : slot - 1);       // into the slot that the pair before this one left
            asm volatile("cp.async.wait_group %0;" ::"n"(QD_STAGES - 1) : "memory");
            __syncwarp();
            uint8_t* const kp[2] = {my_ring + slot * (4 * PB), my_ring + slot * (4 * PB) + 2 * PB};
            if (own == k) {                                            // the copy may have passed the write of the new row
              ok = qd_wait(&sm.own_full[buf], phase, ok) && ok;
              __syncwarp();
              uint8_t* page = s.pos - tok < Q4_PAGE ? kp[0] : kp[1];
              q4_store_k<D>(page, s.pos % Q4_PAGE, sm.codes[buf][0], sm.meta[buf][0], lane);
              q4_store_v<D>(page + PB, s.pos % Q4_PAGE, sm.codes[buf][1], sm.meta[buf][1], lane);
              __syncwarp();
            }
            // ---- scores: lane has tokens gq and gq + 8 of head tq of a tile ----
            float sc[HN][2][2], sv[2][2], mv[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              int hi[HN][4] = {}, lo[HN][4] = {};                        // digits 0 and 1 of tokens gq and gq + 8, digit 2
              uint32_t wa[NG], wb[NG];
              load_words<NG>(kp[j] + gq * (D / 2) + tq * NG * 4, wa);
              load_words<NG>(kp[j] + (gq + 8) * (D / 2) + tq * NG * 4, wb);
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                const uint32_t a0 = wa[g] & 0x0F0F0F0Fu, a1 = wb[g] & 0x0F0F0F0Fu, a2 = wa[g] >> 4 & 0x0F0F0F0Fu, a3 = wb[g] >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                for (int h = 0; h < HN; ++h) {
                  mma_s8(hi[h], a0, a1, a2, a3, qb[h][g].x, qb[h][g].y);
                  mma_s8(lo[h], a0, a1, a2, a3, qb[h][g].z, qb[h][g].w);
                }
              }
              if constexpr (TAIL) {
                const uint8_t* kt = kp[j] + 16 * NG + 2 * tq;
                const uint32_t a0 = nib_bytes(*(const uint16_t*)(kt + gq * (D / 2))), a1 = nib_bytes(*(const uint16_t*)(kt + (gq + 8) * (D / 2)));
#pragma unroll
                for (int h = 0; h < HN; ++h) { mma_s8_half(hi[h], a0, a1, qb[h][NG].x); mma_s8_half(lo[h], a0, a1, qb[h][NG].z); }
              }
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const uint32_t km = *(const uint32_t*)(kp[j] + 8 * D + (gq + 8 * n) * 4), vm = *(const uint32_t*)(kp[j] + PB + 8 * D + (gq + 8 * n) * 4);
                sv[j][n] = q4_scale(vm); mv[j][n] = fmaf(8.f, sv[j][n], q4_min(vm));
#pragma unroll
                for (int h = 0; h < HN; ++h) {
                  const float dot = fmaf((float)hi[h][2 * n], 65536.f, fmaf((float)hi[h][2 * n + 1], 256.f, (float)lo[h][2 * n]));
                  sc[h][j][n] = fmaf(dot * qc[h], q4_scale(km), q4_min(km) * qx[h]);
                }
              }
            }
            if (tok < s.lo || tok + QD_PAIR - 1 > s.pos) {     // rows outside the window or behind the last token hold anything
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                  const int t = tok + j * Q4_PAGE + gq + 8 * n;
                  if (t < s.lo || t > s.pos) {
                    sv[j][n] = mv[j][n] = 0.f;
#pragma unroll
                    for (int h = 0; h < HN; ++h) sc[h][j][n] = -INFINITY;
                  }
                }
            }
            // ---- running maximum and scale: moved only where they fall behind (QD_LAG, QD_TOP) ----
            float mx[HN], top = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
            bool behind = top * vf > QD_TOP;
#pragma unroll
            for (int h = 0; h < HN; ++h) {
              mx[h] = fmaxf(fmaxf(sc[h][0][0], sc[h][0][1]), fmaxf(sc[h][1][0], sc[h][1][1]));
              behind |= mx[h] > m[h] + (float)QD_LAG;
            }
            if (__any_sync(0xFFFFFFFFu, behind)) {
#pragma unroll
              for (int k = 4; k < 32; k <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
#pragma unroll
                for (int h = 0; h < HN; ++h) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xFFFFFFFFu, mx[h], k));
              }
              const float vn = top * vf > QD_TOP ? pow2_for(top, 13 - QD_LAG) : vf, vr = vn / vf;
              vf = vn;
#pragma unroll
              for (int h = 0; h < HN; ++h) {
                const float mn = fmaxf(m[h], mx[h]), corr = m[h] == -INFINITY ? 0.f : ex2(m[h] - mn), co = corr * vr;
#pragma unroll
                for (int n = 0; n < NT; ++n) { o[h][n][0] *= co; o[h][n][1] *= co; o[h][n][2] *= co; o[h][n][3] *= co; }
                l[h] *= corr; om[h] *= corr; m[h] = mn;
                mx[h] = corr;
              }
              if (kb > k0) for_part([&](int h, int, int, float v) { return v * mx[h]; });
            }
            // ---- O += P V: rows gq and gq + 8 of tile 2 g + k are dims 32 g + 4 gq + 2 k and + 1 ----
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t pb[HN][2];
              const float f[2] = {sv[j][0] * vf, sv[j][1] * vf};
#pragma unroll
              for (int h = 0; h < HN; ++h) {
                const float e[2] = {ex2(sc[h][j][0] - m[h]), ex2(sc[h][j][1] - m[h])};
#pragma unroll
                for (int n = 0; n < 2; ++n) { l[h] += e[n]; om[h] = fmaf(e[n], mv[j][n], om[h]); }
                split_f16(e[0] * f[0], e[1] * f[1], pb[h]);
                pb[h][0] = transpose_8x8(pb[h][0]); pb[h][1] = transpose_8x8(pb[h][1]);
              }
              const uint8_t* vp = kp[j] + PB;
              uint32_t w0[NG], w1[NG];
              load_words<NG>(vp + lane * NG * 4, w0);
              load_words<NG>(vp + 128 * NG + lane * NG * 4, w1);
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                uint32_t a[4], c[4];
                codes_less_8(w0[g], a);
                codes_less_8(w1[g], c);
#pragma unroll
                for (int h = 0; h < HN; ++h) {
                  mma_f16(o[h][2 * g], a[0], a[1], c[0], c[1], pb[h][0], pb[h][1]);
                  mma_f16(o[h][2 * g + 1], a[2], a[3], c[2], c[3], pb[h][0], pb[h][1]);
                }
              }
              if constexpr (TAIL) {
                const uint32_t w = *(const uint32_t*)(vp + 256 * NG + lane * 4);
                uint32_t a[4], c[4];
                codes_less_8(__byte_perm(w, 0u, 0x4140), a);
                codes_less_8(__byte_perm(w, 0u, 0x4342), c);
#pragma unroll
                for (int h = 0; h < HN; ++h) mma_f16(o[h][2 * NG], a[0], a[1], c[0], c[1], pb[h][0], pb[h][1]);
              }
            }
            __syncwarp();                                              // every lane has read the pair: its slot may be filled again
            if (++slot == QD_STAGES) slot = 0;
          }
          if (ke == k1) break;
          if (kb == k0 && it >= 2) ok = qd_wait(&sm.part_empty[buf], phase ^ 1u, ok) && ok;
          const float e0 = inverse_pow2(vf);
          for_part([&](int h, int n, int i, float v) {
            const float add = fmaf(o[h][n][2 * i + 1], 1.f / QD_REST, o[h][n][2 * i]) * e0;
            o[h][n][2 * i] = o[h][n][2 * i + 1] = 0.f;
            return kb == k0 ? add : v + add;
          });
          kb = ke;
        }

        // ---- this warp's part of the tile ----
        const bool begun = kb > k0;
        if (!begun && it >= 2) ok = qd_wait(&sm.part_empty[buf], phase ^ 1u, ok) && ok;
        const float e0 = inverse_pow2(vf);
#pragma unroll
        for (int h = 0; h < HN; ++h)
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) { l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], k); om[h] += __shfl_xor_sync(0xFFFFFFFFu, om[h], k); }
        for_part([&](int h, int n, int i, float v) {
          const float add = fmaf(fmaf(o[h][n][2 * i + 1], 1.f / QD_REST, o[h][n][2 * i]), e0, om[h]);
          return begun ? v + add : add;
        });
#pragma unroll
        for (int h = 0; h < HN; ++h) if (gq == 0) *(float2*)(sm.part[buf][warp][4 * h + tq] + D) = make_float2(m[h], l[h]);
      } else {                                                       // no page of this tile is mine
        if (it >= 2) ok = qd_wait(&sm.part_empty[buf], phase ^ 1u, ok) && ok;
        if (lane < ROWS) *(float2*)(sm.part[buf][warp][lane] + D) = make_float2(-INFINITY, 0.f);
      }
      __syncwarp();
      if (lane == 0) qd_arrive(&sm.part_full[buf]);
      at = end;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  QdTile now = qd_tile(p, sm.pos, b0, at0, x1 - x0);
  // ================================== helper warps ================================================================================
  const int hid = tid - 32 * NW, hw = hid >> 5;
  const RopeArgs rope = {p.rope_table, p.rope_table_len, p.rope_dim, p.rope_type, p.rope_theta};
  const int half = p.rope_dim >> 1;
  const float qscale = p.scale * 1.4426950408889634f;
  auto helpers_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(QD_HELPERS) : "memory"); };
  // queries of a tile's heads (norm, rotation, split into fragments), and the new token's rows where its page is in my share
  auto prepare = [&](const QdTile& t, int buf, int at) {
    if (hid == 0)
      sm.tile[buf] = {t.n, (t.s.first_page + 2 * t.skip) * Q4_PAGE, t.s.lo, t.s.pos, p.no_append || t.skip + t.n < t.s.n ? -1 : at + t.n - 1};
    const int kvh = t.tile / hgroups, g0 = (t.tile - kvh * hgroups) * ROWS, gn = min(ROWS, G - g0);
    const float* row = p.qkv + (int64_t)t.b * p.ld_qkv;
    float2 cs[NP];
    load_rope<D>(rope, t.s.pos, lane, cs);
    float xa[NP], xb[NP];
    auto load = [&](const float* src, int hf, int type, float (&a)[NP], float (&b)[NP]) {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int i = lane + 32 * k;
        a[k] = b[k] = 0.f;
        if (i < D / 2) { const int2 at = pair_dims(i, hf, type); a[k] = src[at.x]; b[k] = src[at.y]; }
      }
    };
    const bool own = !p.no_append && t.skip + t.n == t.s.n && hw >= 2, own_v = hw == 3;
    float ra[NP], rb[NP];
    if (own) load(row + (own_v ? p.v_off : p.k_off) + kvh * D, own_v ? 0 : half, own_v ? 0 : p.rope_type, ra, rb);
    for (int g = hw; g < ROWS; g += QD_HELPERS / 32) {
      float f = 1.f, sum = 0.f;
      int isum = 0;
      if (g < gn) {
        load(row + p.q_off + (int64_t)(kvh * G + g0 + g) * D, half, p.rope_type, xa, xb);
        norm_rope_f<D>(xa, xb, p.q_norm_w, (float)p.eps, rope, cs, lane);
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          xa[k] *= qscale; xb[k] *= qscale;
          top = fmaxf(top, fmaxf(fabsf(xa[k]), fabsf(xb[k]))); sum += xa[k] + xb[k];
        }
        top = warp_max(top); sum = warp_sum(sum);
        f = top > 0.f ? pow2_for(top, 22) * (127.f / 128.f) : 1.f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          const int i = lane + 32 * k;
          if (i < D / 2) {
            const int2 at = pair_dims(i, half, p.rope_type);
            const int ia = __float2int_rn(xa[k] * f), ib = __float2int_rn(xb[k] * f);
            sm.q[g][at.x] = (float)ia; sm.q[g][at.y] = (float)ib;
            isum += ia + ib;
          }
        }
        isum = __reduce_add_sync(0xFFFFFFFFu, isum);
      }
      // the sum of the integers, so that their roundings meet centred keys (NaN and infinite queries stay what they are by the other sum)
      if (lane == 0) { const float qc = g < gn ? 1.f / f : 0.f; sm.qc[buf][g] = qc; sm.qx[buf][g] = fmaf((float)isum, qc, sum * 0.f); }
    }
    helpers_sync();
    // column gq is head gq / 2 of a tile, its digits 0 (even) or 1 (odd), and in the second pair of registers digit 2 (even).  Word tq of
    // a group of 32 dims holds dims 8 tq .. + 7: the low nibbles of its bytes are the even ones, the high nibbles the odd ones
    for (int i = hw; i < HN * NF; i += QD_HELPERS / 32) {
      const int h = i / NF, f = i - h * NF, head = 4 * h + (gq >> 1);
      const float* qr = sm.q[head < gn ? head : 0] + 32 * f;
      uint4 r = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t de = head < gn ? digits(__float2int_rn(f < NG ? qr[8 * tq + 2 * e] : qr[4 * tq + e])) : 0u;
        const uint32_t od = head < gn && f < NG ? digits(__float2int_rn(qr[8 * tq + 2 * e + 1])) : 0u;
        r.x |= (gq & 1 ? de >> 8 & 255u : de & 255u) << 8 * e;
        r.y |= (gq & 1 ? od >> 8 & 255u : od & 255u) << 8 * e;
        if (!(gq & 1)) { r.z |= (de >> 16) << 8 * e; r.w |= (od >> 16) << 8 * e; }
      }
      sm.frag[buf][h][f][lane] = r;
    }
    qd_arrive(&sm.frag_full[buf]);
    // the new token's rows, behind the fragments: only the warp that has its pair waits for them
    if (own) {
      const bool v = own_v;
      if (!v) norm_rope_d<D>(ra, rb, p.q_norm_w ? p.k_norm_w : nullptr, p.eps, rope, cs, lane);
      const uint32_t meta = q4_quantise<D>(ra, rb, v ? 0 : half, v ? 0 : p.rope_type, lane, sm.codes[buf][v]);
      __syncwarp();
      if (lane == 0) sm.meta[buf][v] = meta;
      if (g0 == 0) {                                               // one head group writes the row
        const int raw = p.page_table[(int64_t)t.b * p.pt_stride + t.s.pos / Q4_PAGE];
        if (p.num_pages <= 0 || (unsigned)raw < (unsigned)p.num_pages) {
          uint8_t* dst = (uint8_t*)(v ? p.v_cache : p.k_cache) + ((int64_t)raw * p.n_kv_heads + kvh) * PB;
          if (v) q4_store_v<D>(dst, t.s.pos % Q4_PAGE, sm.codes[buf][1], meta, lane);
          else q4_store_k<D>(dst, t.s.pos % Q4_PAGE, sm.codes[buf][0], meta, lane);
        }
      }
    }
    if (hw >= 2) qd_arrive(&sm.own_full[buf]);
  };

  prepare(now, 0, 0);
  QdTile next;
  for (int it = 0, at = 0; at < x1 - x0; ++it) {
    const int end = at + now.n, buf = it & 1;
    const bool more = end < x1 - x0;
    if (more) {
      next = qd_next(p, sm.pos, now, tiles, x1 - x0 - end);
      helpers_sync();                                              // the fragments before are made: the staging rows are free
      prepare(next, buf ^ 1, end);
    }
    ok = qd_wait(&sm.part_full[buf], (uint32_t)(it >> 1) & 1u, ok) && ok;
    const int tile = now.tile, kvh = tile / hgroups, g0 = (tile - kvh * hgroups) * ROWS, gn = min(ROWS, G - g0);
    const bool whole = now.n == now.s.n;
    float* out = p.out + (int64_t)now.b * p.ld_out + (int64_t)(kvh * G + g0) * D;
    // slots of a CTA in scratch: 0 the tile its pairs begin in, 1 the one they end in
    float* parts = p.partial + (int64_t)(2 * c + (it == 0 ? 0 : 1)) * ROWS * (D + 4);
    for (int i = hid; i < gn * (D / 4); i += QD_HELPERS) {
      const int g = i / (D / 4), j = 4 * (i - g * (D / 4));
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sm.part[buf][w][g][D]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 st = *(const float2*)&sm.part[buf][w][g][D];
        if (st.x == -INFINITY) continue;
        const float e = ex2(st.x - mm);
        const float4 v = *(const float4*)&sm.part[buf][w][g][j];
        ll = fmaf(e, st.y, ll);
        a.x = fmaf(e, v.x, a.x); a.y = fmaf(e, v.y, a.y); a.z = fmaf(e, v.z, a.z); a.w = fmaf(e, v.w, a.w);
      }
      if (whole) {
        float* dst = out + g * D + j;
        dst[0] = a.x / ll; dst[1] = a.y / ll; dst[2] = a.z / ll; dst[3] = a.w / ll;
      } else {
        float* dst = parts + g * (D + 4);
        *(float4*)(dst + j) = a;
        if (j == 0) *(float2*)(dst + D) = make_float2(mm, ll);
      }
    }
    helpers_sync();                                                // the parts are read, and what goes to scratch is written
    if (hid == 0) qd_arrive(&sm.part_empty[buf]);
    if (!whole) {
      // by tile, the CTAs are neighbours; else those that have its first and last pair
      const int t0 = x0 + at - now.skip;
      const int c_lo = by_tile ? c - c % split : qd_owner(share, t0);
      const int c_hi = by_tile ? c_lo + min(split, now.s.n) - 1 : qd_owner(share, t0 + now.s.n - 1);
      if (hid == 0) {
        int32_t* ctr = p.counters + (int64_t)now.b * tiles + tile;
        __threadfence();
        sm.last = atomicAdd(ctr, 1) == c_hi - c_lo;
        if (sm.last) { *ctr = 0; __threadfence(); }                // zero again for the next launch
      }
      helpers_sync();
      if (sm.last) {
        constexpr int BATCH = 8;                                    // parts on their way at once (16 took longer)
        const int lead = by_tile || qd_first(share, c_lo) == t0 ? 0 : 1;
        for (int i = hid; i < gn * (D / 4); i += QD_HELPERS) {
          const int g = i / (D / 4), j = 4 * (i - g * (D / 4));
          float mm = -INFINITY, ll = 0.f;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int q0 = c_lo; q0 <= c_hi; q0 += BATCH) {
            float2 st[BATCH];
            float4 v[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
              const int kc = min(q0 + k, c_hi);
              const float* src = p.partial + ((int64_t)(2 * kc + (kc == c_lo ? lead : 0)) * ROWS + g) * (D + 4);
              st[k] = __ldcg((const float2*)(src + D));
              v[k] = __ldcg((const float4*)(src + j));
            }
            float mn = mm;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) mn = fmaxf(mn, st[k].x);
            const float c0 = mm == -INFINITY ? 0.f : ex2(mm - mn);
            a.x *= c0; a.y *= c0; a.z *= c0; a.w *= c0; ll *= c0; mm = mn;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
              const float e = q0 + k > c_hi || st[k].x == -INFINITY ? 0.f : ex2(st[k].x - mm);
              ll = fmaf(e, st[k].y, ll);
              a.x = fmaf(e, v[k].x, a.x); a.y = fmaf(e, v[k].y, a.y); a.z = fmaf(e, v[k].z, a.z); a.w = fmaf(e, v[k].w, a.w);
            }
          }
          float* dst = out + g * D + j;
          dst[0] = a.x / ll; dst[1] = a.y / ll; dst[2] = a.z / ll; dst[3] = a.w / ll;
        }
      }
    }
    at = end;
    if (more) now = next;
  }
}

template <int D, int HN>
static int launch_decode_q4(const AttnDecodeParams& p, cudaStream_t st) {
  int dev = 0, sms = QD_MAX_SMS;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int hgroups = (p.n_heads / p.n_kv_heads + qd_heads(HN) - 1) / qd_heads(HN);
  const long long tiles = (long long)p.batch * p.n_kv_heads * hgroups;
  const int ctas = (int)std::min<long long>(std::min(sms, QD_MAX_SMS), tiles * QD_MAX_PARTS);
  const size_t smem = (sizeof(QdSmem<D, HN>) + 127) / 128 * 128 + (size_t)qd_warps(HN) * QD_STAGES * 4 * q4_page_bytes(D);
  static SmemOptIn opt;
  if (cudaError_t e = opt.ensure(attn_decode_q4_kernel<D, HN>, smem, 0); e != cudaSuccess) return (int)e;
  return (int)launch(attn_decode_q4_kernel<D, HN>, dim3(ctas), dim3(32 * qd_warps(HN) + QD_HELPERS), smem, st, p);
}

int attn_decode_q4_dispatch(const AttnDecodeParams& p, cudaStream_t st) {
  if (!q4_head_dim_ok(p.head_dim)) return -1;
  if (p.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % p.n_kv_heads || p.batch < 1 || p.max_pages < 1) return -2;
  if (p.rope_dim < 0 || p.rope_dim > p.head_dim || (p.rope_dim & 1)) return -3;
  if (((uintptr_t)p.k_cache & 15) || ((uintptr_t)p.v_cache & 15) || ((uintptr_t)p.partial & 15)) return -4;
  if (p.window < 0) return -5;
  attn_q4_ran.store(true, std::memory_order_relaxed);
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
  return 2LL * QD_MAX_SMS * qd_heads(2) * (head_dim + 4);
}

// 0 / 3211 / 3311 / 3312
int rlz_attn_q4_error(int clear) {
  int v = 0;
  if (!rlz::attn_q4_ran.load(std::memory_order_relaxed)) return 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_attn_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_attn_q4_error, &z, sizeof(int)); }
  return v;
}

}  // extern "C"
