// Causal attention of the rows of a prompt chunk over the 4-bit paged cache (kv_q4.cuh), on the tcgen05 tensor cores.
//
// A CTA has two groups of 128 rows of one kv head, row = (token, query head of the group): the group's heads share the keys and values
// that the CTA turns into fp16, 128 keys at a time.  Per group and half a tile (64 keys):
//   S = Q K^T      128 x 64 x D, accumulated in TMEM
//   P = 2^(S - m + 11)  one thread to a row; P goes back to TMEM as fp16, over the columns of S, and is the A operand of
//   O += P V       128 x D x 64, accumulated in TMEM.  The running maximum m moves only when a score passes it by 4 (a factor of 2^4),
//                  so that O is rarely read, scaled and written back.
// Warps 0..7 do the softmax of the groups, 8..11 decode keys and 12..15 values (code x scale + minimum in fp16, rounded once) into two
// buffers each of swizzled operand tiles, warps 16 and 17 issue the products of a group each.  The scores of one half are computed while
// the softmax is at the other (whole tiles, whose scores have to wait for the product that reads P in their place: 4% more
// than the 271 us of 2048 rows behind 6144 keys, 32 query and 8 kv heads of 128).  Registers are moved from the decoding and issuing warps to
// the softmax.
//
// Bound, for 256 rows and 128 keys of 128 dims, by the chain of product, softmax and product, about 4000 clocks: of them the tensor
// cores work 2560 (products of 64 keys read the queries from shared memory twice as often: 384 instead of 256 clocks), the exponentials
// take 2048 (16 a clock) and the decoding 9% of the issue slots' time.
//
// Range: fp16 holds P from 2^15 down to 2^-14 with all of its bits and to 2^-25 with fewer: weights count in full to 2^-25 of the row's
// largest and at all to 2^-36, which matters where the largest belongs to a value near zero (32768 keys, one with 99.9% of the weight
// and a zero value: the sum of the others is off by 6e-3, which is the rounding of the query to fp16; with P = 2^(S - m) by 0.28).  K and V tiles are scaled by powers of two so that fp16 holds them whatever the cache's scales are (K per tile, undone in the
// softmax scale; V by one that changes only when a tile needs it, with O), q by one to a row.
//
// Split, in tiles of 128 keys.  Few row tiles (256 rows of a kv head): to each a cluster of nsplit CTAs, which take the keys in parts
// and join them out of one another's shared memory, every CTA some of the rows (by way of global memory, written by all and read by the
// last to arrive, 512 rows behind 1536 keys took 38 us).  Many, or a number that would leave SMs idle: one CTA to an SM, and the key
// tiles of all row tiles are divided evenly (nsplit = 0).  There a CTA that has only some keys of a row tile leaves its part in scratch,
// and the last of the tile's CTAs to arrive joins them in a fixed order.  Between two row tiles a CTA starts over: all roles meet and
// the barriers are set up again.  Without scratch and for too many row tiles for clusters, a CTA takes a row tile.
#include "attention_q4.cuh"
#include "kv_q4.cuh"
#include "tcgen05_common.cuh"
#include <algorithm>
#include <atomic>
#include <type_traits>

namespace rlz {

// 3113: a page id outside the cache (read as page 0); 3114: rows beyond the page table (not computed); 3115: a bounded wait ran out
__device__ int g_prefill_q4_error = 0;
static std::atomic<bool> prefill_q4_ran{false};      // until a launch there is no status to fetch, which takes a synchronous copy

constexpr int QP_THREADS = 640, QP_GROUP = 128, QP_ROWS = 2 * QP_GROUP, QP_KEYS = 128, QP_MAX_CTAS = 148;
constexpr int QP_MAX_SPLIT = 8;                // CTAs to a cluster
constexpr int QP_MIN_TILES = 2, QP_SEG_COST = 5;      // least share of a CTA; what another row tile costs it, in key tiles
constexpr int QP_REGS_SOFTMAX = 128, QP_REGS_DECODE = 96, QP_REGS_ISSUE = 32;      // 256, 256 and 128 threads: the launch's 640 x 96
// Weights as fp16: 2^(S - m + QP_SHIFT), at most 2^15, where the maximum m of a row moves only when a score passes it by QP_LAG.  What it may
// not lag is range for small weights; 2048 rows behind 6144 keys of 128 dims: 271 us with 8 and with 4, 278 with 2, 293 with 1
constexpr int QP_LAG = 4, QP_SHIFT = 15 - QP_LAG;
constexpr int QP_SLAB = 128 * 128;            // [128 rows x 64 fp16], 128-byte swizzle
constexpr int QP_COUNTERS = 640;               // floats in front of the parts: arrival counters, one to each of a CTA's two slots and group

// key tiles j0 .. j0 + n - 1 of the `all` of row tile mt of a kv head; the tiles' first key and the first key behind them
struct QpSeg { int kvh, mt, j0, n, all, klo, kend; };
struct QpShape { int G, rows, mtiles, pos0; };
// how the key tiles are divided: `left` is the share of this CTA; of an even division, tiles to a CTA and how many have one more; else
// (each = 0) parts of a row tile
struct QpSched { int left, each, more, parts; QpShape z; };

struct QpSmem {
  unsigned long long q_full[2], s_full[2][2], p_full[2][2], o_full[2][2];        // of the groups, and of the tile's halves (64 keys each)
  unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2];      // of the buffers (empty: an arrival from each group's products)
  float kf[4], vf[2];                         // powers of two that the tiles carry (of K the inverse, read after the buffer is free again)
  float mag[2][2][4];                         // largest magnitudes of K and V seen by the decoding warps, for even and odd tiles
  float qf[2][QP_GROUP];                      // powers of two of the query rows
  float2 ml[2][QP_GROUP];                     // maxima and weights of a part's rows
  uint32_t tmem;
  int last[2];
  QpSched sched;
  QpSeg seg;                                  // row tile that is worked on (n = 0: none is left)
  int done, fail;                             // key tiles of my share in front of it; a wait has run out
};

__device__ __forceinline__ float qp_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t qp_half2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const uint32_t*)&h; }
// 2^(e - exponent of x), x >= 0; 2^100 at most
__device__ __forceinline__ float qp_pow2(float x, int e) {
  const int k = e + 254 - (int)(__float_as_uint(x) >> 23);
  return __uint_as_float((uint32_t)max(1, min(k, 227)) << 23);
}
// Products and their commits, called by a whole warp with the same arguments: one elected lane issues.  (With the warp together the
// descriptors stay in uniform registers; issued from a branch of one lane, a product cost 80 clocks of moves.)
// Operand tiles are given by the low words of their descriptors; the high word is that of all K-major tiles with 128-byte swizzle
constexpr uint32_t QP_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t qp_desc_lo(uint32_t tile) { return (tile >> 4 & 0x3FFFu) | 1u << 16; }
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint32_t lo_a, uint32_t lo_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %6};\n\t"
               "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, {%5, %5, %5, %5}, p;\n\t}\n"
               ::"r"(tmem_d), "r"(lo_a), "r"(lo_b), "r"(idesc), "r"(accumulate), "r"(0u), "n"(QP_DESC_HI) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t lo_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %6};\n\t"
               "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, {%5, %5, %5, %5}, p;\n\t}\n"
               ::"r"(tmem_d), "r"(tmem_a), "r"(lo_b), "r"(idesc), "r"(accumulate), "r"(0u), "n"(QP_DESC_HI) : "memory");
}
__device__ __forceinline__ void umma_commit_warp(unsigned long long* bar) {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
               ::"r"(gm_smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// (the tiles are reached by their 32-bit shared addresses: a generic store takes 64-bit sums for each address)
__device__ __forceinline__ void st_shared(uint32_t at, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ bool qp_wait(unsigned long long* bar, uint32_t parity) {
  if (gm_wait((uint64_t*)bar, parity)) return true;
  atomicExch(&g_prefill_q4_error, 3115);
  return false;
}

// true when it is for all 128 threads of a role (also their barrier)
template <int BAR> __device__ __forceinline__ bool qp_agree(bool mine) {
  uint32_t r;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.and.pred q, %2, 128, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(r) : "r"((uint32_t)mine), "n"(BAR) : "memory");
  return r != 0;
}

// eight codes of a word as fp16: pairs (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void codes_f16(uint32_t w, __half2 (&c)[4]) {
  const __half2 magic = __half2half2(__ushort_as_half(0x6400)), sixteenth = __half2half2(__ushort_as_half(0x2C00)), back = __half2half2(__ushort_as_half(0xD400));
  const uint32_t h = w >> 8;                  // 0x6400 | code is 1024 + code, 0x6400 | 16 code is 1024 + 16 code: both come off exactly
  const uint32_t r[4] = {(w & 0x000F000Fu) | 0x64006400u, (w & 0x00F000F0u) | 0x64006400u, (h & 0x000F000Fu) | 0x64006400u, (h & 0x00F000F0u) | 0x64006400u};
  c[0] = __hsub2(*(const __half2*)&r[0], magic); c[1] = __hfma2(*(const __half2*)&r[1], sixteenth, back);
  c[2] = __hsub2(*(const __half2*)&r[2], magic); c[3] = __hfma2(*(const __half2*)&r[3], sixteenth, back);
}

// shared memory of another CTA of the cluster; the cluster's barrier
__device__ __forceinline__ uint32_t qp_peer(uint32_t at, int rank) { uint32_t r; asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank)); return r; }
__device__ __forceinline__ float qp_ld_peer(uint32_t at) { float v; asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory"); return v; }
__device__ __forceinline__ void qp_cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }

template <int R> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
// the registers go through the wait, so that nothing that uses them can move in front of it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*(uint64_t*)&d) : "l"(*(const uint64_t*)&a), "l"(*(const uint64_t*)&b), "l"(*(const uint64_t*)&c));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(uint64_t*)&d) : "l"(*(const uint64_t*)&a), "l"(*(const uint64_t*)&b));
  return d;
}

// a row tile's keys (all = 0: its rows lie beyond the page table)
__device__ __forceinline__ QpSeg qp_rows(const AttnPrefillParams& p, const QpShape& z, int kvh, int mt) {
  QpSeg s = {kvh, mt, 0, 0, 0, 0, 0};
  const int tok0 = mt * QP_ROWS / z.G, tok1 = min(p.n_tokens, (mt * QP_ROWS + QP_ROWS - 1) / z.G + 1);
  if (z.pos0 < 0 || z.pos0 + (int64_t)tok1 > (int64_t)p.pt_len * Q4_PAGE) { atomicExch(&g_prefill_q4_error, 3114); return s; }
  s.kend = z.pos0 + tok1;
  s.klo = p.window > 0 ? max(0, z.pos0 + tok0 + 1 - p.window) / Q4_PAGE * Q4_PAGE : 0;
  s.all = (s.kend - s.klo + QP_KEYS - 1) / QP_KEYS;
  return s;
}
// the next row tile with keys, of which the CTA has at most `left` tiles (left > 0: there is one)
__device__ __forceinline__ QpSeg qp_next(const AttnPrefillParams& p, const QpShape& z, int kvh, int mt, int left) {
  for (;;) {
    if (++mt == z.mtiles) { mt = 0; ++kvh; }
    QpSeg s = qp_rows(p, z, kvh, mt);
    if (s.all) { s.n = min(s.all, left); return s; }
  }
}

// first key tile of CTA c when all are divided evenly, and the CTA that has a tile: the first `more` of them have one tile more
__device__ __forceinline__ int qp_first(const QpSched& s, int c) { return c * s.each + min(c, s.more); }
__device__ __forceinline__ int qp_owner(const QpSched& s, int t) {
  const int edge = s.more * (s.each + 1);
  return t < edge ? t / (s.each + 1) : s.more + (t - edge) / s.each;
}
// The share of this CTA when all key tiles are divided evenly: worked out by a warp, its lanes over the row tiles; true in the one lane
// that has it
__device__ __forceinline__ bool qp_share(const AttnPrefillParams& p, const QpShape& z, QpSched& out, QpSeg& s) {
  const int lane = threadIdx.x & 31, c = blockIdx.x;
  const int per = (z.mtiles + 31) / 32, mt_lo = min(lane * per, z.mtiles), mt_hi = min(mt_lo + per, z.mtiles);
  int mine = 0;
  for (int mt = mt_lo; mt < mt_hi; ++mt) { s = qp_rows(p, z, 0, mt); mine += s.all; }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  const int per_head = __shfl_sync(0xFFFFFFFFu, incl, 31), total = per_head * p.n_kv_heads;
  const int ctas = min((int)gridDim.x, max(1, total / QP_MIN_TILES));
  out.z = z; out.parts = 0; out.each = total / ctas; out.more = total - out.each * ctas;
  out.left = c < ctas ? out.each + (c < out.more ? 1 : 0) : 0;
  if (out.left == 0) { s.n = 0; return lane == 0; }
  const int x0 = qp_first(out, c), kvh = x0 / per_head, want = x0 - kvh * per_head, before = incl - mine;
  if (want < before || want >= incl) return false;
  int at = want - before;
  for (int mt = mt_lo;; ++mt) {
    if (per > 1) s = qp_rows(p, z, 0, mt);
    if (at < s.all) break;
    at -= s.all;
  }
  s.kvh = kvh; s.j0 = at; s.n = min(s.all - at, out.left);
  return true;
}

template <int D>
__global__ void __launch_bounds__(QP_THREADS, 1) attn_prefill_q4_kernel(const __grid_constant__ AttnPrefillParams p, const int nsplit) {
  constexpr int NG = D / 32, TAIL = D % 32 ? 1 : 0, NSLAB = (D + 63) / 64, PB = q4_page_bytes(D);
  constexpr int Q_BYTES = NSLAB * QP_SLAB, K_BYTES = NSLAB * QP_SLAB, V_BYTES = 2 * D * 128;
  constexpr uint32_t TMEM_COLS = 512;         // S and P of the groups: columns 0.. and 128.., O: 256.. and 384..
  extern __shared__ __align__(1024) uint8_t qp_smem[];
  __shared__ QpSmem sm;
  const uint32_t Qs = (gm_smem_u32(qp_smem) + 1023u) & ~1023u, Ks = Qs + 2 * Q_BYTES, Vs = Ks + 2 * K_BYTES;             // a tile is two slabs of [D rows x 64 keys]
  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;      // (the same in all lanes, for the compiler too)
  const int G = p.n_heads / p.n_kv_heads, rows = p.n_tokens * G;
  auto groups_of = [&](int mt) { return rows - mt * QP_ROWS > QP_GROUP ? 2 : 1; };
  auto init_barriers = [&](int groups) {                          // by a warp
    if (lane < 22) {
      const int count = lane < 2 || (lane >= 6 && lane < 10) || lane == 14 || lane == 15 || lane == 18 || lane == 19 ? 128 : lane >= 16 ? groups : 1;
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(gm_smem_u32(&sm.q_full[0] + lane)), "r"(count));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  };
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gm_smem_u32(&sm.tmem)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    QpShape z = {G, rows, (rows + QP_ROWS - 1) / QP_ROWS, p.pos0_ptr ? *p.pos0_ptr : p.pos0};
    QpSched d;
    QpSeg s = {0, 0, 0, 0, 0, 0, 0};
    bool have = lane == 0;
    if (nsplit > 0) {
      const int tile = blockIdx.x / nsplit, part = blockIdx.x - tile * nsplit, kvh = tile / z.mtiles;
      s = qp_rows(p, z, kvh, z.mtiles - 1 - (tile - kvh * z.mtiles));                 // the longest rows first
      d.z = z; d.each = d.more = 0; d.parts = max(1, min(nsplit, s.all / QP_MIN_TILES));
      if (part < d.parts) { s.j0 = part * s.all / d.parts; s.n = (part + 1) * s.all / d.parts - s.j0; }
      d.left = s.n;
    } else have = qp_share(p, z, d, s);
    if (have) { sm.sched = d; sm.seg = s; sm.done = 0; sm.fail = 0; }
    __syncwarp();
    init_barriers(groups_of(sm.seg.mt));
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = sm.tmem;
  // the CTA's next row tile, false: none is left; all threads come here, role 0 with warp 0
  auto next_rows = [&](bool ok, auto role) {
    if (!ok) sm.fail = 1;
    tc_before();                                                   // O has been read
    asm volatile("bar.sync 0, %0;" ::"n"(QP_THREADS) : "memory");
    if (decltype(role)::value == 0 && warp == 0) {
      if (lane == 0) {
        const int done = sm.done + sm.seg.n;
        sm.done = done;
        if (done < sm.sched.left && !sm.fail) sm.seg = qp_next(p, sm.sched.z, sm.seg.kvh, sm.seg.mt, sm.sched.left - done); else sm.seg.n = 0;
      }
      __syncwarp();
      if (sm.seg.n) {                                              // (every arrival of the tile before has been waited for)
        if (lane < 22) asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(gm_smem_u32(&sm.q_full[0] + lane)) : "memory");
        init_barriers(groups_of(sm.seg.mt));
      }
    }
    asm volatile("bar.sync 0, %0;" ::"n"(QP_THREADS) : "memory");
    tc_after();
    return sm.seg.n > 0;
  };
  const bool any = sm.seg.n > 0;

  if (warp < 8) {
    // ================================ softmax: one thread to a row ================================================================
    regs_up<QP_REGS_SOFTMAX>();
    const int grp = warp >> 2, t = tid & 127;
    auto store_at = [&](int token, int head, int c, const float* v) {      // 16 finished values
      const int64_t at = (int64_t)token * p.ld_out + (int64_t)head * D + c;
      if (p.out_bf16) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        uint4* dst = (uint4*)((__nv_bfloat16*)p.out + at);
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]); dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(float4*)(p.out + at + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    };
    float part_f = 0.f;                                              // of a part of my row that waits in TMEM: 1 / vf
    bool more = any;
    while (more) {
      const int m0 = sm.seg.mt * QP_ROWS, groups = groups_of(sm.seg.mt), kvh = sm.seg.kvh, n_tiles = sm.seg.n, kbeg = sm.seg.klo + sm.seg.j0 * QP_KEYS, pos0 = sm.sched.z.pos0;
      bool ok = true;
      if (grp < groups) {
        const uint32_t lane_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(128 * grp), lane_o = lane_s + 256u;
        const int row = m0 + grp * QP_GROUP + t, token = row / G, head = kvh * G + row - token * G;
        const bool live = row < rows;
        const int pos = pos0 + token;
        // ---- queries: 8 dims to a lane, stored as fp16 in the order in which the keys' codes come out of a word: (0, 4), (1, 5), (2, 6),
        // (3, 7) of every 8 dims.  Not unrolled further: 16 rows at
        // once took 11 us instead of 6 (the instructions run once to a CTA and have to be fetched)
        const uint32_t q_tile = Qs + (uint32_t)(grp * Q_BYTES);
        const bool vec = (((uintptr_t)p.qkv | (uintptr_t)(4 * p.ld_qkv) | (uintptr_t)(4 * p.q_off)) & 15) == 0;
        {
          constexpr int LANES = D == 64 ? 8 : 16, STEP = 32 / LANES, BATCH = 8;     // lanes to a row, rows at once and their loads in flight
          const int x = lane % LANES, r0 = (warp & 3) * 32 + lane / LANES;
          int gr = m0 + grp * QP_GROUP + r0, tk = gr / G, hd = gr - tk * G;
#pragma unroll 1
          for (int r1 = r0; r1 < (warp & 3) * 32 + 32; r1 += BATCH * STEP) {
            float4 v[BATCH][2];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (gr < rows && x < D / 8) {
                const float* src = p.qkv + (int64_t)tk * p.ld_qkv + p.q_off + (int64_t)(kvh * G + hd) * D + 8 * x;
                if (vec) { v[i][0] = __ldg((const float4*)src); v[i][1] = __ldg((const float4*)src + 1); }
                else { v[i][0] = make_float4(__ldg(src), __ldg(src + 1), __ldg(src + 2), __ldg(src + 3)); v[i][1] = make_float4(__ldg(src + 4), __ldg(src + 5), __ldg(src + 6), __ldg(src + 7)); }
              }
              gr += STEP;
              for (hd += STEP; hd >= G; hd -= G) ++tk;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int r = r1 + i * STEP;
              const float4 a = v[i][0], b = v[i][1];
              float top = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))), fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
#pragma unroll
              for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
              const float f = top > 0.f ? qp_pow2(top, 4) : 1.f;
              if (x == 0) sm.qf[grp][r] = f;
              if (x < NSLAB * 8) {
                const uint32_t w[4] = {qp_half2(a.x * f, b.x * f), qp_half2(a.y * f, b.y * f), qp_half2(a.z * f, b.z * f), qp_half2(a.w * f, b.w * f)};
                st_shared(q_tile + (uint32_t)((x >> 3) * QP_SLAB + (r >> 3) * 1024 + (r & 7) * 128 + (((x & 7) ^ (r & 7)) << 4)), w);
              }
            }
          }
        }
        __syncwarp();
        const float qs = p.scale * 1.4426950408889634f / sm.qf[grp][t];    // softmax scale of my row
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        gm_arrive((uint64_t*)&sm.q_full[grp]);

        float m = -INFINITY, vf = 1.f;
        float2 l2 = make_float2(0.f, 0.f);
        const int row_first = m0 + grp * QP_GROUP, row_last = min(rows, row_first + QP_GROUP) - 1;
        const int pos_first = pos0 + row_first / G, lo_last = p.window > 0 ? pos0 + row_last / G + 1 - p.window : 0;     // masks are needed beyond these
        for (int i = 0; ok && i < 2 * n_tiles; ++i) {
          const int j = i >> 1, half = i & 1, k0 = kbeg + 64 * i, buf = j & 1;
          const uint32_t s_at = lane_s + (uint32_t)(64 * half);
          // the scores, and with them the tile's power of two of K; that of V
          ok = qp_wait(&sm.s_full[grp][half], (uint32_t)j & 1u) && (half || qp_wait(&sm.v_full[buf], (uint32_t)(j >> 1) & 1u));
          if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
          tc_after();
          const float sc = qs * sm.kf[j & 3], vn = sm.vf[buf];
          const bool edge = k0 + 63 > pos_first || k0 < lo_last;
          const int vis_hi = live ? pos + 1 - k0 : 0, vis_lo = p.window > 0 ? pos + 1 - p.window - k0 : 0;
          // EDGE: some entries are masked
          auto part = [&](auto edge_c) {
            constexpr bool EDGE = decltype(edge_c)::value;
            uint32_t r[2][32];
            tmem_ld32_async(s_at, r[0]);
            tmem_ld32_async(s_at + 32u, r[1]);
            tmem_wait_ld(r[0]);
            tmem_wait_ld(r[1]);
            auto seen = [&](int key) { return !EDGE || (key < vis_hi && key >= vis_lo); };
            float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
            for (int k = 0; k < 64; k += 4) {
              auto score = [&](int key) { return seen(key) ? __uint_as_float(r[key >> 5][key & 31]) : -INFINITY; };
              top = max3(top, score(k), score(k + 1));
              top1 = max3(top1, score(k + 2), score(k + 3));
            }
            top = fmaxf(top, top1) * sc;
            if (__any_sync(0xFFFFFFFFu, top > m + (float)QP_LAG || vn != vf)) {
              const float mn = fmaxf(m, top), corr = m == -INFINITY ? 0.f : qp_ex2(m - mn), co = corr * (vn / vf);
              if (i > 0) {
                ok = __all_sync(0xFFFFFFFFu, qp_wait(&sm.o_full[grp][half ^ 1], (uint32_t)((i - 1) >> 1) & 1u));      // the product before has ended
                tc_after();
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 16) {
                  uint32_t o[16];
                  tmem_ld16(lane_o + (uint32_t)c0, o);
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * co);
                  tmem_st16(lane_o + (uint32_t)c0, o);
                }
              }
              l2.x *= corr; l2.y *= corr; m = mn; vf = vn;
            }
            const float base = m == -INFINITY ? 0.f : (float)QP_SHIFT - m;              // a row that has seen no key yet: all of its entries are masked
            const float2 sc2 = make_float2(sc, sc), b2 = make_float2(base, base);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t w[16];
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                const float2 y = fma2(make_float2(__uint_as_float(r[c][k]), __uint_as_float(r[c][k + 1])), sc2, b2);
                const float2 e = make_float2(seen(32 * c + k) ? qp_ex2(y.x) : 0.f, seen(32 * c + k + 1) ? qp_ex2(y.y) : 0.f);
                l2 = add2(l2, e);
                w[k >> 1] = qp_half2(e.x, e.y);
              }
              tmem_st16(s_at + (uint32_t)(16 * c), w);                   // over the scores
            }
            tmem_wait_st();
            tc_before();
            gm_arrive((uint64_t*)&sm.p_full[grp][half]);
          };
          if (edge) part(std::true_type{}); else part(std::false_type{});
        }
        if (ok) ok = qp_wait(&sm.o_full[grp][0], (uint32_t)(n_tiles - 1) & 1u) && qp_wait(&sm.o_full[grp][1], (uint32_t)(n_tiles - 1) & 1u);       // the last products
        if (grp == 0 ? qp_agree<1>(ok) : qp_agree<2>(ok)) {
          tc_after();
          const float inv_vf = 1.f / vf, l = l2.x + l2.y;
          auto store = [&](int c, const float* v) { store_at(token, head, c, v); };
          const bool whole = n_tiles == sm.seg.all;
          constexpr int COLS = D % 32 ? 16 : 32;
          // slots of a CTA in scratch: 0 the row tile that its share begins in, 1 the one that it ends in
          constexpr int64_t step = (int64_t)QP_ROWS * (D + 4);
          float* const slots = p.scratch + QP_COUNTERS + (int64_t)grp * QP_GROUP * (D + 4) + t;     // a column to 128 floats: a warp's rows lie together
          float* const slot = slots + (int64_t)(2 * blockIdx.x + (sm.done == 0 ? 0 : 1)) * step;
          if (whole) {
            const float f = inv_vf / l;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t r[16];
              tmem_ld16(lane_o + (uint32_t)c, r);
              float v[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) * f;
              if (live) store(c, v);
            }
          } else if (nsplit > 0) {
            sm.ml[grp][t] = make_float2(m, l);
            part_f = inv_vf;
          } else {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t r[16];
              tmem_ld16(lane_o + (uint32_t)c, r);
#pragma unroll
              for (int i = 0; i < 16; ++i) __stcg(slot + (c + i) * QP_GROUP, __uint_as_float(r[i]) * inv_vf);
            }
            slot[D * QP_GROUP] = m; slot[(D + 1) * QP_GROUP] = l;
            // the row tile's CTAs: those that have its first and last key tile
            const int t0 = qp_first(sm.sched, blockIdx.x) + sm.done - sm.seg.j0;
            const int c_lo = qp_owner(sm.sched, t0), c_hi = qp_owner(sm.sched, t0 + sm.seg.all - 1), lead = qp_first(sm.sched, c_lo) == t0 ? 0 : 1;
            if (grp == 0) asm volatile("bar.sync 1, 128;" ::: "memory"); else asm volatile("bar.sync 2, 128;" ::: "memory");
            if (t == 0) {
              int32_t* ctr = (int32_t*)p.scratch + 2 * (2 * c_lo + lead) + grp;
              __threadfence();
              sm.last[grp] = atomicAdd(ctr, 1) == c_hi - c_lo;
              if (sm.last[grp]) { *ctr = 0; __threadfence(); }          // zero again for the next launch
            }
            if (grp == 0) asm volatile("bar.sync 1, 128;" ::: "memory"); else asm volatile("bar.sync 2, 128;" ::: "memory");
            if (sm.last[grp] && live) {
              auto part_of = [&](int k) { return slots + (int64_t)(2 * k + (k == c_lo ? lead : 0)) * step; };
              float mm = -INFINITY, ll = 0.f;
#pragma unroll 4
              for (int k = c_lo; k <= c_hi; ++k) {
                const float mi = __ldcg(part_of(k) + D * QP_GROUP), li = __ldcg(part_of(k) + (D + 1) * QP_GROUP), mn = fmaxf(mm, mi);
                if (mn != -INFINITY) ll = fmaf(ll, qp_ex2(mm - mn), li * qp_ex2(mi - mn));
                mm = mn;
              }
              const float inv = 1.f / ll;
#pragma unroll 1
              for (int c = 0; c < D; c += COLS) {
                float v[COLS] = {};
#pragma unroll 2
                for (int k = c_lo; k <= c_hi; ++k) {
                  const float* part_i = part_of(k);
                  const float e = qp_ex2(__ldcg(part_i + D * QP_GROUP) - mm) * inv;
#pragma unroll
                  for (int q = 0; q < COLS; ++q) v[q] = fmaf(e, __ldcg(part_i + (c + q) * QP_GROUP), v[q]);
                }
#pragma unroll
                for (int q = 0; q < COLS; q += 16) store(c + q, v + q);
              }
            }
          }
        }
      }
      more = next_rows(ok, std::integral_constant<int, 0>{});
    }
    if (nsplit > 1) {
      // ---- the cluster's parts; the last meeting of the roles has freed the operand tiles: sums by columns of 128 rows
      const int parts = sm.sched.parts, rank = (int)blockIdx.x % nsplit, m0 = sm.seg.mt * QP_ROWS, kvh = sm.seg.kvh;
      if (parts > 1 && rank < parts && grp < groups_of(sm.seg.mt)) {
        const uint32_t lane_o = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(128 * grp) + 256u;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t r[16];
          tmem_ld16(lane_o + (uint32_t)c, r);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(Qs + (uint32_t)(((grp * D + c + i) * QP_GROUP + t) * 4)), "f"(__uint_as_float(r[i]) * part_f) : "memory");
        }
      }
      qp_cluster_sync();
      if (parts > 1) {
        const int n = min(QP_ROWS, rows - m0), r0 = rank * n / nsplit, mine = (rank + 1) * n / nsplit - r0;        // my rows
        for (int i = tid; i < mine * (D / 16); i += 256) {
          const int c = i / mine, row = r0 + i - c * mine, g = row >> 7, tr = row & 127;
          float m[QP_MAX_SPLIT], l[QP_MAX_SPLIT], mm = -INFINITY, ll = 0.f, v[16] = {};
#pragma unroll
          for (int k = 0; k < QP_MAX_SPLIT; ++k) {
            const uint32_t at = qp_peer(gm_smem_u32(&sm.ml[g][tr]), min(k, parts - 1));
            m[k] = k < parts ? qp_ld_peer(at) : -INFINITY; l[k] = k < parts ? qp_ld_peer(at + 4u) : 0.f;
            mm = fmaxf(mm, m[k]);
          }
#pragma unroll
          for (int k = 0; k < QP_MAX_SPLIT; ++k) { m[k] = m[k] == -INFINITY ? 0.f : qp_ex2(m[k] - mm); ll = fmaf(m[k], l[k], ll); }
          const float inv = 1.f / ll;
#pragma unroll
          for (int k = 0; k < QP_MAX_SPLIT; ++k) {
            if (k >= parts) break;
            const uint32_t at = qp_peer(Qs + (uint32_t)(((g * D + 16 * c) * QP_GROUP + tr) * 4), k);
            const float e = m[k] * inv;
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = fmaf(e, qp_ld_peer(at + (uint32_t)(q * QP_GROUP * 4)), v[q]);
          }
          const int token = (m0 + row) / G;
          store_at(token, kvh * G + m0 + row - token * G, 16 * c, v);
        }
      }
      qp_cluster_sync();                                             // the others have read my part
    }
  } else if (warp < 16) {
    // ================================ decoding ======================================================================================
    regs_down<QP_REGS_DECODE>();
    const int t = tid & 127;
    bool more = any;
    while (more) {
      const int n_tiles = sm.seg.n, kbeg = sm.seg.klo + sm.seg.j0 * QP_KEYS, kend = sm.seg.kend, kvh = sm.seg.kvh;
      bool ok = true;
      const int last_page = (kend - 1) / Q4_PAGE * Q4_PAGE;
      auto id_of = [&](int key) { return __ldg(p.page_table + min(key, last_page) / Q4_PAGE); };
      auto row_of = [&](int id) {
        if ((unsigned)id >= (unsigned)p.num_pages) { atomicExch(&g_prefill_q4_error, 3113); id = 0; }
        return ((int64_t)id * p.n_kv_heads + kvh) * PB;
      };
      // largest magnitude that a row's codes can stand for; over all threads of the role
      auto largest = [](uint32_t meta) { return fmaxf(fabsf(q4_min(meta)), fabsf(fmaf(15.f, q4_scale(meta), q4_min(meta)))); };
      if (warp < 12) {
        // -- keys: a token row to a thread
        uint32_t kw[D / 8], km = 0u;
        int id = id_of(kbeg + t);
        auto load = [&](int k0) {
          const int key = k0 + t;
          const uint8_t* src = (const uint8_t*)p.k_cache + row_of(id);
#pragma unroll
          for (int i = 0; i < D / 8; i += 2) {
            const uint2 v = __ldg((const uint2*)(src + (key % Q4_PAGE) * (D / 2) + 4 * i));
            kw[i] = v.x; kw[i + 1] = v.y;
          }
          km = key < kend ? __ldg((const uint32_t*)(src + 8 * D + 4 * (key % Q4_PAGE))) : 0u;         // rows behind the last key count as 0
          id = id_of(key + QP_KEYS);
        };
        load(kbeg);
        for (int j = 0; j < n_tiles; ++j) {
          const int buf = j & 1;
          float top = redux_max(largest(km));
          if (lane == 0) sm.mag[buf][0][warp & 3] = top;
          if (!qp_agree<3>(ok)) break;
          top = fmaxf(fmaxf(sm.mag[buf][0][0], sm.mag[buf][0][1]), fmaxf(sm.mag[buf][0][2], sm.mag[buf][0][3]));
          const float kf = qp_pow2(top, 4);                              // the tile's largest value to [2^4, 2^5)
          if (j >= 2) ok = qp_wait(&sm.k_empty[buf], (uint32_t)((j >> 1) - 1) & 1u);
          if (t == 0) sm.kf[j & 3] = 1.f / kf;
          const __half2 s2 = __float2half2_rn(q4_scale(km) * kf), m2 = __float2half2_rn(q4_min(km) * kf);
          const uint32_t base = Ks + (uint32_t)(buf * K_BYTES + (t >> 3) * 1024 + (t & 7) * (128 + 16));       // 16-byte piece x of a row lies at x ^ (row % 8)
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {                              // word i of the row: 8 dims from 8 x on
            const int x = i < 4 * NG ? 4 * (i % NG) + i / NG : i;
            __half2 c[4];
            codes_f16(kw[i], c);
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) { const __half2 v = __hfma2(c[q], s2, m2); o[q] = *(const uint32_t*)&v; }
            st_shared((base ^ (uint32_t)((x & 7) << 4)) + (uint32_t)((x >> 3) * QP_SLAB), o);
          }
          if (j + 1 < n_tiles) load(kbeg + (j + 1) * QP_KEYS);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          gm_arrive((uint64_t*)&sm.k_full[buf]);
        }
      } else {
        // -- values: half a page to a thread: page t / 16 of the tile, tokens 8 vh .. + 7, units vg of every 32 dims
        uint32_t vw[D / 8], vm[8];
        const int vh = (t >> 3) & 1, vg = t & 7;
        int id = id_of(kbeg + (t >> 4) * Q4_PAGE);
        auto load = [&](int k0) {
          const int key = k0 + (t >> 4) * Q4_PAGE;
          const uint8_t* src = (const uint8_t*)p.v_cache + row_of(id);
          const uint32_t* w = (const uint32_t*)(src + (size_t)vh * 128 * NG + vg * 16 * NG);           // words [tq][g]
#pragma unroll
          for (int i = 0; i < 4 * NG; i += 4) { const uint4 v = __ldg((const uint4*)(w + i)); vw[i] = v.x; vw[i + 1] = v.y; vw[i + 2] = v.z; vw[i + 3] = v.w; }
          if constexpr (TAIL) {                                          // bytes of both halves: mine of each word, as 16 bits
            const uint4 v = __ldg((const uint4*)(src + 256 * NG + vg * 16));
            vw[4 * NG] = __byte_perm(v.x, v.y, vh ? 0x7632 : 0x5410); vw[4 * NG + 1] = __byte_perm(v.z, v.w, vh ? 0x7632 : 0x5410);
          }
          const uint4 a = __ldg((const uint4*)(src + 8 * D + 32 * vh)), b = __ldg((const uint4*)(src + 8 * D + 32 * vh + 16));
          const uint32_t r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) vm[i] = key + 8 * vh + i < kend ? r[i] : 0u;
          id = id_of(key + QP_KEYS);
        };
        load(kbeg);
        float vf = 0x1p100f;
        for (int j = 0; j < n_tiles; ++j) {
          const int buf = j & 1;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, largest(vm[i]));
          top = redux_max(top);
          if (lane == 0) sm.mag[buf][1][warp & 3] = top;
          if (!qp_agree<4>(ok)) break;
          top = fmaxf(fmaxf(sm.mag[buf][1][0], sm.mag[buf][1][1]), fmaxf(sm.mag[buf][1][2], sm.mag[buf][1][3]));
          if (top * vf >= 4096.f) vf = qp_pow2(top, 4);                  // it stays as long as it keeps the values below 2^12
          __half2 s2[4], m2[4];                                          // of the token pairs
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s2[i] = __floats2half2_rn(q4_scale(vm[2 * i]) * vf, q4_scale(vm[2 * i + 1]) * vf);
            m2[i] = __floats2half2_rn(q4_min(vm[2 * i]) * vf, q4_min(vm[2 * i + 1]) * vf);
          }
          if (j >= 2) ok = qp_wait(&sm.v_empty[buf], (uint32_t)((j >> 1) - 1) & 1u);
          if (t == 0) sm.vf[buf] = vf;
          const int chunk = (t >> 3) & 7;                                // eight keys of the 64 of a slab
          // dim 32 g + 4 vg + e is row 4 (vg % 2) + e of the eight of row group 4 g + vg / 2; its keys lie at chunk ^ row
          const uint32_t slab = Vs + (uint32_t)(buf * V_BYTES + (t >> 6) * (D * 128));
          const uint32_t base = slab + (uint32_t)((vg >> 1) * 1024 + (vg & 1) * 512 + ((chunk ^ (vg & 1) << 2) << 4));
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            uint32_t o[4][4];                                            // [dim][token pair]
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              __half2 c[4];
              codes_f16(vw[q * NG + g], c);
#pragma unroll
              for (int e = 0; e < 4; ++e) { const __half2 v = __hfma2(c[e], s2[q], m2[q]); o[e][q] = *(const uint32_t*)&v; }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) st_shared((base ^ (uint32_t)(e << 4)) + (uint32_t)(g * 4096 + e * 128), o[e]);
          }
          if constexpr (TAIL) {
            uint32_t o[2][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t two = vw[4 * NG + (q >> 1)] >> (16 * (q & 1));           // a byte to each token of the pair
              __half2 c[4];
              codes_f16((two & 0xFFu) | (two & 0xFF00u) << 8, c);
#pragma unroll
              for (int e = 0; e < 2; ++e) { const __half2 v = __hfma2(c[e], s2[q], m2[q]); o[e][q] = *(const uint32_t*)&v; }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int dim = 2 * vg + e;
              st_shared(slab + (uint32_t)(NG * 4096 + (dim >> 3) * 1024 + (dim & 7) * 128 + ((chunk ^ (dim & 7)) << 4)), o[e]);
            }
          }
          if (j + 1 < n_tiles) load(kbeg + (j + 1) * QP_KEYS);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          gm_arrive((uint64_t*)&sm.v_full[buf]);
        }
      }
      more = next_rows(ok, std::integral_constant<int, 1>{});
    }
    if (nsplit > 1) { qp_cluster_sync(); qp_cluster_sync(); }
  } else {
    regs_down<QP_REGS_ISSUE>();
    bool more = any;
    while (more) {
      const int n_tiles = sm.seg.n;
      bool ok = true;
      if (warp < 16 + groups_of(sm.seg.mt)) {
        // ================================ the products: a warp to a group, so that no group's waits hold up the other =====================
        const int g = warp - 16;
        const uint32_t id_s = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(QP_GROUP >> 4) << 24);      // fp16 operands, fp32 sums
        const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(QP_GROUP >> 4) << 24);
        const uint32_t q_lo = qp_desc_lo(Qs + g * Q_BYTES), k_lo = qp_desc_lo(Ks), v_lo = qp_desc_lo(Vs), s_col = tmem + 128u * g, o_col = s_col + 256u;
        auto both = [&](unsigned long long* bar, uint32_t parity) { if (ok) { ok = __all_sync(0xFFFFFFFFu, qp_wait(bar, parity)); tc_after(); } };
        // half i of the key tiles: S = Q K^T
        auto scores = [&](int i) {
          const int j = i >> 1, half = i & 1;
          if (half == 0) both(&sm.k_full[j & 1], (uint32_t)(j >> 1) & 1u);
          if (!ok) return;
          const uint32_t b = k_lo + (uint32_t)((j & 1) * (K_BYTES >> 4) + half * (64 * 128 >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (uint32_t)((kk >> 2) * (QP_SLAB >> 4) + 2 * (kk & 3));
            umma_f16_ss(s_col + 64u * half, q_lo + off, b + off, id_s, kk > 0 ? 1u : 0u);
          }
          umma_commit_warp(&sm.s_full[g][half]);
          if (half && j + 2 < n_tiles) umma_commit_warp(&sm.k_empty[j & 1]);
        };
        both(&sm.q_full[g], 0u);
        scores(0);
        scores(1);
        for (int i = 0; ok && i < 2 * n_tiles; ++i) {
          const int j = i >> 1, half = i & 1;
          // O += P V, as P arrives (it comes after the softmax has seen that the values are there)
          both(&sm.p_full[g][half], (uint32_t)j & 1u);
          if (!ok) break;
          const uint32_t pa = s_col + (uint32_t)(64 * half), b = v_lo + (uint32_t)((j & 1) * (V_BYTES >> 4) + half * (D * 128 >> 4));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16_ts(o_col, pa + (uint32_t)(8 * kk), b + (uint32_t)(2 * kk), id_o, i > 0 || kk > 0 ? 1u : 0u);
          umma_commit_warp(&sm.o_full[g][half]);
          if (half && j + 2 < n_tiles) umma_commit_warp(&sm.v_empty[j & 1]);
          // the scores that go where P lay, once the product has ended: while the softmax works on the other half
          if (i + 2 < 2 * n_tiles) { both(&sm.o_full[g][half], (uint32_t)j & 1u); scores(i + 2); }
        }
      }
      more = next_rows(ok, std::integral_constant<int, 1>{});
    }
    if (nsplit > 1) { qp_cluster_sync(); qp_cluster_sync(); }
  }
  tc_before();
  __syncthreads();
  if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

template <int D>
static int launch_prefill_q4(const AttnPrefillParams& p, cudaStream_t st) {
  constexpr int NSLAB = (D + 63) / 64;
  const size_t smem = (size_t)4 * NSLAB * QP_SLAB + 4 * D * 128 + 1024;
  static SmemOptIn opt;
  if (cudaError_t e = opt.ensure(attn_prefill_q4_kernel<D>, smem, 0); e != cudaSuccess) return (int)e;
  // the roles' registers have to fit into what the launch brings, or the softmax would wait for them for good
  static const bool regs_fit = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, attn_prefill_q4_kernel<D>) == cudaSuccess &&
           a.numRegs * QP_THREADS >= 256 * (QP_REGS_SOFTMAX + QP_REGS_DECODE) + 128 * QP_REGS_ISSUE;
  }();
  if (!regs_fit) return -7;
  // row tiles, and key tiles to a row tile at most
  const int tiles = (int)(((int64_t)p.n_tokens * (p.n_heads / p.n_kv_heads) + QP_ROWS - 1) / QP_ROWS) * p.n_kv_heads;
  const int64_t reach = p.pos0_ptr ? (int64_t)p.pt_len * Q4_PAGE : (int64_t)p.pos0 + p.n_tokens;
  const int keys = (int)((p.window > 0 ? std::min<int64_t>(reach, p.window + QP_ROWS) : reach) / QP_KEYS) + 1;
  // as many CTAs to a row tile as fit, in clusters, onto the SMs at once
  static int fits[64][QP_MAX_SPLIT + 1] = {};                        // clusters of a size that a device holds, and one
  int dev = 0, nsplit = 1;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return (int)e;
  for (int n = std::min(QP_MAX_SPLIT, QP_MAX_CTAS / tiles); n > 1 && nsplit == 1; --n) {
    int& f = fits[dev & 63][n];
    if (f == 0) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      cfg.gridDim = dim3(n); cfg.blockDim = dim3(QP_THREADS); cfg.dynamicSmemBytes = smem;
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = n; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = 1;
      int active = 0;
      if (cudaError_t e = cudaOccupancyMaxActiveClusters(&active, attn_prefill_q4_kernel<D>, &cfg); e != cudaSuccess) return (int)e;
      f = active + 1;
    }
    if (tiles < f) nsplit = n;
  }
  int grid = tiles * nsplit;
  if (p.scratch && p.scratch_floats >= 2LL * QP_MAX_CTAS * QP_ROWS * (D + 4) + QP_COUNTERS) {
    // time in key tiles: of the longest CTA, or, of an even share, with the second row tile that it reaches into
    const int waves = (grid + QP_MAX_CTAS - 1) / QP_MAX_CTAS, by_tile = waves * ((keys + nsplit - 1) / nsplit) + (waves - 1) * QP_SEG_COST;
    const int even = (int)((int64_t)keys * tiles / QP_MAX_CTAS) + waves * QP_SEG_COST;
    if (even < by_tile) { nsplit = 0; grid = QP_MAX_CTAS; }
  }
  return (int)launch_cluster(attn_prefill_q4_kernel<D>, dim3(grid), dim3(QP_THREADS), dim3(std::max(nsplit, 1)), smem, st, p, nsplit);
}

int attn_prefill_q4_dispatch(const AttnPrefillParams& given, cudaStream_t st) {
  AttnPrefillParams p = given;
  if (p.num_pages < 1 || p.pt_len < 1 || ((uintptr_t)p.scratch & 15)) return -6;
  if (p.window >= (int64_t)p.pt_len * Q4_PAGE) p.window = 0;        // hides nothing, and differences of positions and a larger one could pass 32 bits
  // row tiles x key tiles are counted in 32 bits
  const int64_t mtiles = ((int64_t)p.n_tokens * (p.n_heads / p.n_kv_heads) + QP_ROWS - 1) / QP_ROWS;
  if (mtiles * p.n_kv_heads * ((int64_t)p.pt_len * Q4_PAGE / QP_KEYS + 2) > INT32_MAX) return -6;
  prefill_q4_ran.store(true, std::memory_order_relaxed);
  switch (p.head_dim) {
    case 64: return launch_prefill_q4<64>(p, st);
    case 80: return launch_prefill_q4<80>(p, st);
    case 96: return launch_prefill_q4<96>(p, st);
    case 128: return launch_prefill_q4<128>(p, st);
    default: return -1;
  }
}

}  // namespace rlz

extern "C" {

// floats of scratch with which the keys can be split, whatever the number of rows is
long long rlz_attn_prefill_q4_scratch_floats(int head_dim) {
  return 2LL * rlz::QP_MAX_CTAS * rlz::QP_ROWS * (head_dim + 4) + rlz::QP_COUNTERS;
}

// 0 / 3113 / 3114 / 3115
int rlz_attn_prefill_q4_error(int clear) {
  int v = 0;
  if (!rlz::prefill_q4_ran.load(std::memory_order_relaxed)) return 0;
  if (cudaMemcpyFromSymbol(&v, rlz::g_prefill_q4_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) { int z = 0; cudaMemcpyToSymbol(rlz::g_prefill_q4_error, &z, sizeof(int)); }
  return v;
}

}  // extern "C"
