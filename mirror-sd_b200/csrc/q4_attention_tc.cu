// Grouped-query attention over the paged 4-bit cache for blocks of query rows
// (more than 16 rows times heads a kv head): tcgen05, both products transposed.
//
//   S^T[128 cached rows, N] = K[128, 128] Q^T      K as f16 straight from TMEM
//   O^T[128 channels, N]   += V^T[128, 128] P^T    V^T and P^T from shared memory
//
// N <= 80 query rows of a (request, kv head) are the instruction's columns, so
// a block of 64 costs 64 columns instead of being padded to 128 rows, and a
// cached row is one TMEM lane: the thread that decodes its 64 bytes stores it
// as the A operand without passing through shared memory.
//
// The pass of a group's query rows over the rows that it shares (kAttnPrefix) has
// the wide form where there are more than 64 of them a kv head: 128 query rows are
// the instruction's rows, so a thread has a query row's scores and forms its maximum
// and its sum alone, P goes back to TMEM, and one decoded tile serves 128 rows:
//
//   S[128 query rows, 128] = Q K^T      both from shared memory
//   O[128 query rows, 128] += P V       P from TMEM, V^T from shared memory
//
// (There one O serves both sides, 16 warps share the softmax, and K goes to shared
// memory; see wide_softmax.)  1,360 query rows a kv head on 2 groups of 16,384 rows
// take 178 us, in the transposed form 270, 10 of them the start (lengths, query rows,
// first tiles) and 5 the end; 1,024 on 4,096 rows 35.  A tile takes 1,900 cycles, of
// which the MMAs need 1,024 and shared memory moves bytes for 1,570 (64 KB for QK^T,
// 32 for PV, 64 of decoded K and V written, 36 of codes in and out).  What would pay
// next: Q as the operand in TMEM with scores of 64 cached rows at a time (bytes for
// 1,310), or pairs of CTAs that decode half of a tile each.
//
// Work: the tiles of 128 cached rows of all items, end to end, in equal runs
// of one CTA per SM (q4_attn.cuh).  The CTAs that share an item write partial
// results, which a second small kernel merges.  No CTA waits for another:
// nothing guarantees that they are all resident (a kernel of another stream, or
// a partition of the GPU, may hold SMs).  (Merged by the last CTA to arrive: 64
// query rows on 1 request of 2,048 rows 29 us, of 32,768 48; this way 21 and 36.)
//
// Roles, each running ahead as far as its buffers allow:
//   2 x 4 warps  softmax of the even and the odd tiles; a thread owns a cached
//       row.  Each side has its own S, P, O and references (the values that a
//       column's scores are measured against), joined when the item ends: two
//       tiles are under way at any time, so one's waits (every hand-over
//       between roles is 100 to 300 cycles) are the other's work.  A column's
//       reference moves only when a score passes it by 2^8, so a tile is one
//       pass (scores to P, a column's partial sums kept per thread) and a vote;
//       column maxima across lanes are only formed when the vote asks for them
//       (always for a side's first tile of an item).
//   4 warps  K codes to f16, into TMEM
//   4 warps  V codes to f16, transposed, into shared memory
//   2 warps  issue the MMAs, one those of S, one those of PV
//   1 warp   page look-up and bulk copies of the packed tiles
//   1 warp   the next item's query rows
// Every wait is bounded; after one expires the roles run to their end without
// waiting and the status word says so.  The code is kept small (rolled loops,
// one kind of tile): the roles share the instruction cache.
//
// What it measures (8 kv heads): 256 requests x 16 rows x 32 heads over a sink of
// 64 and a window of 1,040 rows 250 us, 16 requests of up to 32,768 rows with up to
// 32 rows x 40 heads 218 us, one such request 57 us; HBM would allow 59, 31 and 6,
// the products alone 44, 37 and 13.  What bounds it: a tile takes each role 1,500
// to 2,000 cycles (at 64 columns; 512 of them are MMAs), half the issue slots and
// most of shared memory's bandwidth (V^T and P^T are written and read again), so
// that leaving out all of the decoding and the exponentials saves 15 %; and the
// start and the end of an item are 6 to 8 us together with little beside them:
// short items (the 1,040-row window) pay that every 10 tiles.
//
#include "q4_attn.cuh"

namespace dfl {

constexpr int QB_TILE = kQ4TcTile;
constexpr int QB_BLK = kQ4Block + 32;      // a row block's stride in shared memory: 8 blocks on different banks
constexpr int QB_STAGE = QB_TILE / kQ4Rows * QB_BLK;
constexpr int QB_SEEN = 256;               // flag of a tile that every query of the item sees whole
constexpr int QB_PREFIX = 1 << 16;         // beside an item's number of CTAs: there are sums over its group's rows
constexpr int QB_ITEM = 6;                 // what an item's start and end cost beside its tiles, in tiles (9 to 11 us, 5 at 32 columns)
constexpr int QB_SLACK = 6;
constexpr float QB_RAISE = 8.f;

template <int N_>
struct QbCfg {
  static constexpr int N = N_;
  // Wide: query rows as the instruction's rows, cached rows as its columns (below)
  static constexpr bool WIDE = N > 80;
  static constexpr int CH = N / 16;
  // Query buffers and packed stages.  With 80 columns shared memory holds two and
  // two or one and three (8 requests of 16,384 rows, 160 query rows: 167 and 166 us).
  static constexpr int QB = N <= 64 ? 2 : 1;
  static constexpr int SB = WIDE ? 3 : N <= 64 ? 4 : 2;    // S buffers (TMEM: 128 for K, N for each O and S; wide: 4 N)
  static constexpr int NS = N <= 64 ? 4 : 3;
  static constexpr bool AHEAD = N <= 64;        // registers for the next 16 scores
  static constexpr int SEGS = WIDE ? 4 : 8;     // ring of item records (items run ahead by an S buffer each, and one)
  static constexpr int P_BYTES = (N + 63) / 64 * 16384;       // 64-column chunks of [128 rows][128 B] (wide: of K)
  static constexpr int V_OFF = 0, V_BYTES = 32768;
  static constexpr int P_OFF = V_OFF + 2 * V_BYTES;
  static constexpr int Q_OFF = P_OFF + 2 * P_BYTES, Q_BYTES = N * 256;
  static constexpr int RING_OFF = Q_OFF + QB * Q_BYTES;
  static constexpr int MISC_OFF = RING_OFF + NS * QB_STAGE;
  // 2 x 64 for K, N for each O and S (wide: N for each S, which P takes the place of, and one O)
  static constexpr uint32_t K_COL = 0, O_COL = WIDE ? SB * N : 128, S_COL = WIDE ? 0 : 128 + 2 * N;
  static constexpr int SLOT = N * 130;          // floats of a partial: O [N][128], m [N], l [N]
  // warps: softmax, side by side (even tiles 0-3, odd tiles 4-7), then the others, all
  // in whole warpgroups, whose registers are dealt out anew after the common start
  // (wide: two warps to a side's 32 rows, half the columns each)
  static constexpr int KDEC = WIDE ? 16 : 8, VDEC = KDEC + 4, MMA = VDEC + 4, LOAD = MMA + 1, QUERY = MMA + 2, MMA2 = MMA + 3;
  static constexpr int THREADS = 32 * (MMA + 4);
  // registers a thread at the start: 96, 640 * 96 = 256 * 144 + 384 * 64 (wide: 72, and
  // all keep them; 80 and 56: 266 us where 72 and 72 take 260)
  static constexpr int SOFT_REGS = WIDE ? 72 : 144, REST_REGS = WIDE ? 72 : 64;
};
struct QbSeg {          // a run of tiles of one item
  Item it;
  int sub, q0, head0;   // first query row (row * G + head) and head of the item
  int j0, nt;           // tiles [j0, j0 + nt) of the item
  int item0;            // the item's first tile in the flat order
  int uniform;          // every column has the same score factor
};

template <class C>
struct QbMisc {
  uint64_t full[4], empty[4], kready[2], kfree[2], vready[2], pvdone[2], s_ready[4], s_free[4], p_ready[2];
  uint64_t q_ready[2], q_free[2], o_free, rec_ready[4], begun[4], decided[2][4];
  uint32_t tmem;
  int abort;
  int where[2];                   // request of the CTA's first tile, and that request's first tile
  int run[2], share;              // whole CTAs to an item: this one's tiles, and their number
  int wtot[C::THREADS / 32];
  int2 tile[16];                  // row blocks copied and QB_SEEN, rows below the request's end
  QbSeg seg[C::SEGS];
  alignas(16) float qf[C::WIDE ? 2 : C::SEGS][C::N];   // score factors
  alignas(16) float negm[2][C::N];            // minus the columns' references, of either side
  alignas(16) float fac[2][C::WIDE ? 2 * C::N : C::N];             // rescale factors; at the end what O is multiplied by
  alignas(16) float pre[C::N];                // and what the sums over the group's rows are (kAttnOwn)
  int cmax[2][C::N];                          // column maxima as ordered integers
  alignas(16) int cend[C::N];                 // where each column's keys end
  alignas(16) int coff[C::N];                 // output row of each column, or -1
  float lsum[C::WIDE ? 4 : 8][C::N];
  int4 shared;                    // the item that starts here and reaches past the last tile (q4_tc_shared)
};

// One lane of a converged warp, chosen in a way that the compiler recognises:
// an MMA behind it takes its descriptors from uniform registers.  Behind a
// plain `lane == 0` every MMA costs about 150 cycles to issue, whatever its
// size; behind this one M128 N160 K16 runs at its 80 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// the warpgroup's registers per thread from here on
template <int R, bool MORE>
__device__ __forceinline__ void set_registers() {
  if (MORE)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// columns (MN) contiguous in 128-byte chunks lbo_bytes apart, 8-row K groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_sw128_mn(uint32_t smem_addr, uint32_t lbo_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(lbo_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// A warp's wait for a phase, bounded: when it expires (or once another wait has)
// the flag is set and every later wait returns at once.  All lanes poll: one
// polling lane leaves the warp split, and what follows is issued twice (the
// kernel as a whole took a third longer).  The warp is together afterwards, as
// TMEM accesses need it.
__device__ __forceinline__ void qb_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  uint32_t i = 0;
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*dead) break;
    if (++i == kSpinLimit) *dead = 1;
  }
  __syncwarp();
}

// A warp's arrival: what its lanes did before is ordered before it.  (One
// arrival a warp and not one a thread, some 900 a tile on the shared-memory pipe;
// no difference was measured at the time.)
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
// vote of the THREADS threads of a named barrier
template <int THREADS>
__device__ __forceinline__ bool named_bar_or(int id, bool v) {
  int o;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.s32 q, %2, 0;\n barrier.red.or.pred p, %1, %3, q;\n"
      " selp.s32 %0, 1, 0, p;\n}\n"
      : "=r"(o)
      : "r"(id), "r"((int)v), "n"(THREADS)
      : "memory");
  return o != 0;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t x, y, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t x, y, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t x, y, z, r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// order-preserving map of floats to ints (-inf lowest)
__device__ __forceinline__ int float_key(float f) {
  const int i = __float_as_int(f);
  return i ^ (i >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float key_float(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }
// products of columns 16 c .. of this thread's cached row less the references
__device__ __forceinline__ void scores16(const uint32_t (&s)[16], const float* negm, int c, float2 (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 m = *reinterpret_cast<const float4*>(negm + 16 * c + i);
    y[i / 2] = add2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(m.x, m.y));
    y[i / 2 + 1] = add2(make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), make_float2(m.z, m.w));
  }
}

// What CTA b of the grid leaves behind its partials (two of n queries each): the
// item that starts in its run and ends in a later CTA's, as the item's first
// query row, its query rows, its group and kv head (sub), and the number of CTAs
// that hold it (0: no such item).  Written at every launch.
__host__ __device__ __forceinline__ int4* q4_tc_shared(float* part, int n, int grid) {
  return reinterpret_cast<int4*>(part + (size_t)grid * 2 * n * 130);
}

// 16 bytes of bf16 as floats; returns the largest magnitude.
__device__ __forceinline__ float query_floats(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  float a = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[2 * k] = __uint_as_float(u[k] << 16);
    x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    a = fmaxf(a, fmaxf(fabsf(x[2 * k]), fabsf(x[2 * k + 1])));
  }
  return a;
}
// 16 bytes of a bf16 query row, the row's others in 15 neighbouring lanes, as f16.
// A row whose largest magnitude lies in [2^-3, 2^15] is rounded to f16 as it is (what
// is below 2^-14 loses bits, 2^-22 of that largest at most); any other row is scaled
// by a power of two first, whose exponent is returned (0: none).  All lanes take part;
// rows without `mine` stay as they are.
__device__ __forceinline__ int query_f16(uint4* at, bool mine, int lane) {
  float x[8];
  const float a = __uint_as_float(   // (not negative: ordered as integers)
      __reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, __float_as_uint(query_floats(*at, x))));
  const bool scaled = mine && a != 0.f && !(a >= 0.125f && a <= 32768.f);
  const int e = scaled ? min(max((int)(__float_as_uint(a) >> 23), 1), 253) : 0;
  const float down = scaled ? __uint_as_float((uint32_t)(254 - e) << 23) : 1.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] *= down;
  if (mine) *at = make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
  return e;
}
__device__ __forceinline__ float scaled_factor(float f, int e) { return fminf(f * __uint_as_float((uint32_t)e << 23), 3e38f); }

// ---- softmax of the wide form: of the tiles t with t & 1 == x; thread = query row,
// half of the tile's columns.  Both sides add to one O, so a row has one reference,
// which each tile may raise after the tile before has: the sides hand it on in the
// order of the tiles (`decided`), early in a tile's work, and a raise waits for the
// products that O still takes.  P, as f16, takes the place of the scores that are
// read; with a third buffer S of the next tile is there when a side comes to it.
// (Sides with an O each leave room for two buffers, so that a tile's S waits for PV
// of the tile two before: 2,200 cycles a tile, of which the hand-overs alone are 950.)
template <class C, class Sharers>
__device__ __forceinline__ void wide_softmax(const Q4AttnParams& p, QbMisc<C>& ms, uint8_t* q_smem, uint32_t tmem, int c0, int c1,
                                             volatile int* dead, Sharers sharers) {
  constexpr int N = C::N, SOFT = 32 * C::KDEC;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, x = warp >> 3, half = warp >> 2 & 1;
  const int row = 32 * (warp & 3) + lane, pair = 4 + 4 * x + (warp & 3), G = p.by_g.d;   // barrier of the two warps
  const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
  const uint32_t o_all = tmem + C::O_COL + lanes, o_t = o_all + 64 * half;
  // Query rows: 8 a warp, two at a time (lanes 0-15, 16-31), on their way while the
  // item before is finished.  (One warp for all 128: 8 us an item, 15 in bf16.)
  const float base_f = 16.f * p.scale_log2;
  const int piece = lane & 15, q_row0 = 8 * warp + (lane >> 4);
  uint8_t* const q_dst = q_smem + (piece >> 3) * (N * 128) + q_row0 * 128;
  auto query_at = [&](int i) { return q_dst + 2 * i * 128 + (((piece & 7) ^ (q_row0 + 2 * i & 7)) << 4); };
  auto load_queries = [&](int seg) {
    qb_wait(&ms.rec_ready[seg & 3], (seg >> 2) & 1, dead);
    if (__any_sync(0xffffffffu, *dead)) return;   // (there may be no record)
    const QbSeg& sg = ms.seg[seg % C::SEGS];
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + (size_t)sg.it.row0 * p.q_row + 8 * piece;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = sg.q0 + q_row0 + 2 * i, j = p.by_g.of(r);
      const bool real = j < sg.it.rows;
      cp_async16_zfill(smem_u32(query_at(i)), real ? q + (size_t)j * p.q_row + (size_t)(sg.head0 + r - j * G) * p.q_head : p.q, real);
    }
    cp_async_commit();
  };
  if (c0 < c1) load_queries(0);
  int u = c0, t0 = 0;   // the item's first tile, counted in the CTA
#pragma unroll 1
  for (int seg = 0; u < c1; ++seg) {
    cp_async_wait<0>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = p.bf16 ? query_f16(reinterpret_cast<uint4*>(query_at(i)), true, lane) : 0;
      if (piece == 0) ms.qf[seg & 1][q_row0 + 2 * i] = e ? scaled_factor(base_f, e) : base_f;
    }
    fence_proxy_async_smem();
    warp_arrive(&ms.q_ready[0], lane);
    if ((t0 & 1) == x) qb_wait(&ms.s_ready[t0 % C::SB], (t0 / C::SB) & 1, dead);
    const QbSeg& sg = ms.seg[seg % C::SEGS];
    // after an expired wait there may be no record: run to the end, writing nothing
    const bool bad = named_bar_or<SOFT>(3, *dead);
    const int nt = bad ? c1 - u : sg.nt;
    const float f = score_factor(ms.qf[seg & 1][row]);
    if (threadIdx.x == 0) mbar_arrive(&ms.begun[seg & 3]);
    float negm = kUnset;   // minus the reference
    float2 l = make_float2(0.f, 0.f);

#pragma unroll 1
    for (int k = (t0 & 1) == x ? 0 : 1; k < nt; k += 2) {
      const int t = t0 + k;
      const uint32_t s_t = tmem + C::S_COL + (t % C::SB) * N + 64 * half + lanes;
      if (k > 0) qb_wait(&ms.s_ready[t % C::SB], (t / C::SB) & 1, dead);
      tc_fence_after();
      const int2 info = ms.tile[t & 15];
      if (!(info.x & QB_SEEN)) {   // some key is hidden: its scores to -inf, where they lie
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int left = (info.x >> (4 * half + c) & 1) ? info.y - 64 * half - 16 * c : 0;
          if (left >= 16) continue;
          uint32_t s[16];
          tmem_ld16(s_t + 16 * c, s);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = i < left ? s[i] : 0xff800000u;
          tmem_st16(s_t + 16 * c, s);
        }
        tmem_st_wait();
      }
      uint32_t s[2][16];
      tmem_ld16(s_t, s[0]);
      float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait();
        tmem_ld16(s_t + 16 * ((c + 1) & 3), s[(c + 1) & 1]);   // (at last the first ones again)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          top = max3(top, __uint_as_float(s[c & 1][i]), __uint_as_float(s[c & 1][i + 1]));
          top2 = max3(top2, __uint_as_float(s[c & 1][i + 2]), __uint_as_float(s[c & 1][i + 3]));
        }
      }
      top = fmaxf(top, top2);
      if (k > 0) {
        qb_wait(&ms.decided[x ^ 1][warp & 3], ((t - 1) >> 1) & 1, dead);
        const float now = ms.negm[0][row];
        if (__any_sync(0xffffffffu, now != negm)) {
          const float by = now == negm ? 1.f : exp2_fast((now - negm) * f);   // (0 for a row without a reference before)
          l.x *= by;
          l.y *= by;
          negm = now;
        }
      }
      if (named_bar_or<64>(pair, (top + negm) * f > QB_RAISE)) {   // (a row without a reference: any visible key)
        ms.fac[x][row + half * N] = top;
        named_bar_sync(pair, 64);
        top = fmaxf(top, ms.fac[x][row + (half ^ 1) * N]);
        const float rise = (top + negm) * f;
        float by = 1.f;
        if (rise > QB_RAISE) {
          by = exp2_fast(-rise);
          negm = -top;
        }
        l.x *= by;
        l.y *= by;
        if (k > 0) {   // O, once it holds all tiles before t: half of its channels
          qb_wait(&ms.pvdone[(t - 1) & 1], ((t - 1) >> 1) & 1, dead);
          tc_fence_after();
          tmem_ld_wait();
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            tmem_ld16(o_t + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
            tmem_st16(o_t + 16 * c, o);
          }
          tmem_st_wait();
        }
        if (half == 0) ms.negm[0][row] = negm;
      } else if (k == 0 && half == 0) {
        ms.negm[0][row] = negm;
      }
      warp_arrive(&ms.decided[x][warp & 3], lane);
      const float2 nm = make_float2(negm, negm), ff = make_float2(f, f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait();
        if (c < 3) tmem_ld16(s_t + 16 * (c + 1), s[(c + 1) & 1]);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float2 y = mul2(add2(make_float2(__uint_as_float(s[c & 1][2 * i]), __uint_as_float(s[c & 1][2 * i + 1])), nm), ff);
          y.x = exp2_fast(y.x);
          y.y = exp2_fast(y.y);
          l = add2(l, y);
          w[i] = pack_f16x2(y.x, y.y);
        }
        tmem_st8(s_t + 8 * c, w);   // (over scores that this warp has read)
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&ms.p_ready[x], lane);
    }
    u += nt;
    if (u < c1) {
      qb_wait(&ms.q_free[0], seg & 1, dead);
      load_queries(seg + 1);
    }

    // ---- the item's run is over: both sides' sums and O, a quarter of the channels each
    const int last = t0 + nt - 1;
    // (the row's reference is that of the side with the last tile; the other's sums may have an older one)
    if ((last & 1) != x) {
      qb_wait(&ms.decided[x ^ 1][warp & 3], (last >> 1) & 1, dead);
      const float now = ms.negm[0][row], by = now == negm ? 1.f : exp2_fast((now - negm) * f);
      l.x *= by;
      l.y *= by;
      negm = now;
    }
    ms.lsum[2 * x + half][row] = l.x + l.y;
    qb_wait(&ms.pvdone[last & 1], (last >> 1) & 1, dead);
    named_bar_sync(3, SOFT);
    tc_fence_after();
    Item it{};
    if (!bad) it = sg.it;
    const bool whole = bad || (sg.j0 == 0 && nt == it.ntile);
    const int border = sg.item0 < c0 ? 0 : 1, r = sg.q0 + row, j = p.by_g.of(r);
    const long long at = j < it.rows ? (long long)(it.row0 + j) * p.nq + sg.head0 + r - j * G : -1;   // row of the sums
    float* part = p.part + ((size_t)blockIdx.x * 2 + border) * C::SLOT;
    float* to = whole ? p.pre_o + at * 128 : part + row * 128;
    const bool write = !whole || at >= 0;
    if (x == 0 && half == 0) {
      const float sum = (ms.lsum[0][row] + ms.lsum[1][row]) + (ms.lsum[2][row] + ms.lsum[3][row]);
      const float top = partial_max(negm, f);
      if (!whole) {
        part[N * 128 + row] = top;
        part[N * 129 + row] = sum;
      } else if (at >= 0) {
        p.pre_ml[at] = make_float2(top, sum);
      }
    }
#pragma unroll 1
    for (int c = 2 * (warp >> 2); c < 2 * (warp >> 2) + 2; ++c) {
      uint32_t o[16];
      __syncwarp();
      tmem_ld16(o_all + 16 * c, o);
      tmem_ld_wait();
      if (write) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(to + 16 * c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
    }
    // (merged by the item's first CTA's entry; the others' partials follow its own)
    if (!whole && threadIdx.x == 0 && border == 1)
      ms.shared = make_int4(it.row0, it.rows, sg.sub, sharers(sg.item0, it.ntile));
    tc_fence_before();
    warp_arrive(&ms.o_free, lane);
    t0 += nt;
  }
  if (threadIdx.x == 0) q4_tc_shared(p.part, N, gridDim.x)[blockIdx.x] = ms.shared;
}

template <int N, int PASS>
__global__ void __launch_bounds__(QbCfg<N>::THREADS, 1) q4_attn_tc_kernel(const Q4AttnParams p) {
  using C = QbCfg<N>;
  constexpr int NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  // (an offset, not a rounded pointer: the compiler must still see shared memory)
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  QbMisc<C>& ms = *reinterpret_cast<QbMisc<C>*>(smem + C::MISC_OFF);
  volatile int* dead = &ms.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.by_g.d;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(&ms.full[i], 1); mbar_init(&ms.empty[i], 8); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ms.kready[i], 4); mbar_init(&ms.kfree[i], 1);
      mbar_init(&ms.vready[i], 4); mbar_init(&ms.pvdone[i], 1);
      mbar_init(&ms.p_ready[i], C::WIDE ? 8 : 4);
      mbar_init(&ms.q_ready[i], C::WIDE ? C::KDEC : 1); mbar_init(&ms.q_free[i], 1);
    }
    mbar_init(&ms.o_free, C::KDEC);
    if (C::WIDE) {
      for (int i = 0; i < 4; ++i) { mbar_init(&ms.rec_ready[i], 1); mbar_init(&ms.begun[i], 1); }
      for (int i = 0; i < 8; ++i) mbar_init(&ms.decided[i >> 2][i & 3], 2);
    }
    for (int i = 0; i < C::SB; ++i) { mbar_init(&ms.s_ready[i], 1); mbar_init(&ms.s_free[i], C::WIDE ? 1 : 4); }
    ms.abort = 0;
    ms.shared = make_int4(0, 0, 0, 0);
    ms.run[0] = ms.run[1] = 0;
    fence_mbar_init();
  }
  griddep_wait();
  griddep_launch_dependents();
  if (warp == C::MMA) {
    tmem_alloc(&ms.tmem, 512);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i < 2 * N; i += C::THREADS) ms.cmax[0][i] = float_key(-INFINITY);

  // The CTA's run of tiles [c0, c1), from the lengths.
  auto scan = [&](int v, int* sum) {   // what the threads before hold, and the sum of all
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = tiles_sum(x, y);
    }
    __syncthreads();
    if (lane == 31) ms.wtot[warp] = x;
    __syncthreads();
    int w = lane < C::THREADS / 32 ? ms.wtot[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = tiles_sum(w, y);
    }
    *sum = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return tiles_sum(warp > 0 ? before : 0, x - v);
  };
  const int grid = gridDim.x;
  // Passes over shared and own rows weigh an item's start and end as well, QB_ITEM
  // tiles, where there are items for every CTA: an item is then that many units
  // followed by its tiles, and runs are cut by units.  (Own rows of 64 requests, 16
  // to 1,024 of them: 190 us by tiles, 88 by units; one group of 8 x 2,048 rows: 14
  // by tiles, 20 by units.)
  constexpr int W = PASS == kAttnAll ? 0 : QB_ITEM;
  int units = 0, c1_unit = 0;   // of all items; where the CTA's run ends
  int total = 0, c0 = 0, c1 = 0, items = 0, ntile = 0, first = 0;   // (the last three of request threadIdx.x)
#pragma unroll 1
  for (int i0 = 0; i0 < p.n; i0 += C::THREADS) {
    const int i = i0 + threadIdx.x;
    items = ntile = 0;
    if (i < p.n) {
      const Item it = load_item<QB_TILE, N>(p, i);
      ntile = it.ntile;
      items = it.groups * p.nkv;
      if (blockIdx.x == 0 && p.status && !rows_fit(p, i)) atomicOr(p.status, kPagedRows);
    }
    int sum;
    first = scan(items * ntile, &sum);
    total = tiles_sum(total, sum);
    if (W > 0) {
      scan(items * (ntile + W), &sum);
      units = tiles_sum(units, sum);
    }
  }
  if (total == kTilesFull || units == kTilesFull) total = units = 0;
  const bool weigh = W > 0 && units - total >= W * grid;
  // With few items, whole CTAs to each: a run that crosses from one item into the
  // next pays the start and the end of an item (6 to 8 us together) twice.  An
  // item takes a CTA for every `quota` of its tiles, the least number with which
  // the grid holds them all, if that is at most QB_SLACK tiles more than equal
  // runs would have.  (8 items of 64 tiles 26.8 us in equal runs, 23.9 in whole
  // CTAs; 16 of 257 tiles, 160 query rows, 59.9 and 56.6.)
  int quota = 0;
  if (p.n <= C::THREADS && total > grid) {
    int lo = (total + grid - 1) / grid, hi = lo + QB_SLACK + 1, sum;
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      scan(items * ((ntile + mid - 1) / mid), &sum);
      if (sum <= grid) { hi = mid; quota = mid; } else lo = mid + 1;
    }
  }
  if (quota > 0) {
    const int parts = (ntile + quota - 1) / quota;
    int sum;
    const int rel = (int)blockIdx.x - scan(items * parts, &sum);
    if (rel >= 0 && rel < items * parts) {
      const int sub = rel / parts, part = rel - sub * parts, item0 = first + sub * ntile;
      const Runs runs(ntile, parts);
      ms.where[0] = threadIdx.x;
      ms.where[1] = first;
      ms.run[0] = item0 + runs.start(part);
      ms.run[1] = item0 + runs.start(part + 1);
      ms.share = parts;
    }
  } else if (weigh) {
    const Runs runs(units, min(grid, total));
    const int u0 = runs.start(min((int)blockIdx.x, min(grid, total))), u1 = runs.start(min((int)blockIdx.x + 1, min(grid, total)));
    c1_unit = u1;
    int tiles_before = 0, units_before = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < p.n; i0 += C::THREADS) {
      const int i = i0 + threadIdx.x;
      int m = 0, nt = 0, sum;
      if (i < p.n) {
        const Item it = load_item<QB_TILE, N>(p, i);
        nt = it.ntile;
        m = it.groups * p.nkv;
      }
      const int t = tiles_before + scan(m * nt, &sum);
      tiles_before += sum;
      const int u = units_before + scan(m * (nt + W), &sum);
      units_before += sum;
      auto tile_of = [&](int unit) {   // the first tile at or behind a unit of this request
        const int k = (unit - u) / (nt + W);
        return t + k * nt + max(unit - u - k * (nt + W) - W, 0);
      };
      if (u <= u0 && u0 < u + m * (nt + W)) {
        ms.where[0] = i;
        ms.where[1] = t;
        ms.run[0] = tile_of(u0);
      }
      if (u <= u1 && u1 < u + m * (nt + W)) ms.run[1] = tile_of(u1);
      if (u1 == units && threadIdx.x == 0) ms.run[1] = total;
      if (u0 == units && threadIdx.x == 0) ms.run[0] = total;
    }
  } else {
    const int ctas = min(grid, total);
    const Runs runs(total, ctas);
    if ((int)blockIdx.x < ctas) {
      c0 = runs.start(blockIdx.x);
      c1 = runs.start(blockIdx.x + 1);
    }
    int before = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < p.n; i0 += C::THREADS) {
      const int i = i0 + threadIdx.x;
      int v = 0, sum;
      if (i < p.n) {
        const Item it = load_item<QB_TILE, N>(p, i);
        v = it.ntile * it.groups * p.nkv;
      }
      const int at = tiles_sum(before, scan(v, &sum));
      before = tiles_sum(before, sum);
      if (at <= c0 && c0 < at + v) {
        ms.where[0] = i;
        ms.where[1] = at;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem;
  if (quota > 0 || weigh) {
    c0 = ms.run[0];
    c1 = ms.run[1];
  }
  const int T = c1 - c0;
  // number of CTAs that hold an item of ntile tiles, the first of them tile item0 and in this CTA
  auto sharers = [&](int item0, int ntile) {
    if (quota > 0) return ms.share;
    if (weigh)   // (the run ends inside the item's tiles)
      return Runs(units, min(grid, total)).of(c1_unit + item0 + ntile - c1 - 1) - (int)blockIdx.x + 1;
    const Runs runs(total, min(grid, total));
    return runs.of(item0 + ntile - 1) - runs.of(item0) + 1;
  };

  // ring cursors start at the same place in the producer and the query warp
  auto first_cursor = [&](Cursor& c) {
    c.it = load_item<QB_TILE, N>(p, ms.where[0]);
    const int rel = c0 - ms.where[1];
    c.sub = rel / c.it.ntile;
    c.j = rel - c.sub * c.it.ntile;
  };

  // (registers go from the roles that move data to the two that compute)
  if (warp < C::KDEC) {
    set_registers<C::SOFT_REGS, true>();
    if constexpr (C::WIDE) {
      wide_softmax<C>(p, ms, smem + C::Q_OFF, tmem, c0, c1, dead, sharers);
    } else {
    // ---- softmax of the tiles t with t & 1 == x; thread = cached row, and channel at the end
    const int x = warp >> 2, gt = threadIdx.x & 127;
    const int row = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t o_t = tmem + C::O_COL + x * N + lanes;
    uint8_t* pr = smem + C::P_OFF + x * C::P_BYTES + row * 128;
    const int window = p.window > 0 ? p.window : 1 << 30;   // no cache is longer
    float* negm = ms.negm[x];
    float* facs = ms.fac[x];
    int u = c0, t0 = 0;   // the item's first tile, counted in the CTA
#pragma unroll 1
    for (int seg = 0; u < c1; ++seg) {
      // S of the item's first tile is only issued once its record is there
      if ((t0 & 1) == x) qb_wait(&ms.s_ready[t0 % C::SB], (t0 / C::SB) & 1, dead);
      const QbSeg& sg = ms.seg[seg % C::SEGS];
      // after an expired wait there may be no record: run to the end, writing nothing
      const bool bad = named_bar_or<256>(3, *dead);
      Item it{};
      if (!bad) it = sg.it;
      const int nt = bad ? c1 - u : sg.nt, j0 = bad ? 0 : sg.j0;
      const float* qf = ms.qf[seg % C::SEGS];
      const bool uniform = sg.uniform;
      const float f = p.factor;
      if (gt < N) {
        const int r = sg.q0 + gt, j = p.by_g.of(r);
        const bool real = j < it.rows;
        negm[gt] = real ? kUnset : 0.f;
        if (x == 0) {
          ms.cend[gt] = real ? (p.causal ? it.L - it.rows + j + 1 : it.L) : 0;
          ms.coff[gt] = real ? (it.row0 + j) * p.nq + sg.head0 + r - j * G : -1;
        }
      }
      named_bar_sync(3, 256);
      float2 l[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) l[i] = make_float2(0.f, 0.f);

#pragma unroll 1
      for (int k = (t0 & 1) == x ? 0 : 1; k < nt; k += 2) {
        const int t = t0 + k;
        const uint32_t s_t = tmem + C::S_COL + (t % C::SB) * N + lanes;
        // P is read, and this side's O holds the tiles before t
        auto wait_pv = [&]() {
          if (t >= 2) qb_wait(&ms.pvdone[x], ((t >> 1) - 1) & 1, dead);
        };
        if (k > 0) qb_wait(&ms.s_ready[t % C::SB], (t / C::SB) & 1, dead);
        tc_fence_after();
        const int blocks = ms.tile[t & 15].x;
        if (!(blocks & QB_SEEN) || !uniform) {
          const int key = (blocks >> (row >> 4) & 1) ? item_tile(it, j0 + k) * QB_TILE + row : INT32_MAX;
          // Some key is hidden, or the columns have factors of their own: bring
          // the tile's scores to the common factor, hidden ones to -inf, where
          // they lie; the steps below then know one kind of tile.
          if (!p.causal && uniform) {   // every query sees the same keys
            const bool row_seen = (key < it.L) & ((key < p.sink) | (key >= it.L - window));
#pragma unroll 1
            for (int c = 0; c < C::CH; ++c) {
              uint32_t s[16];
              tmem_ld16(s_t + 16 * c, s);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) s[i] = row_seen ? s[i] : 0xff800000u;
              tmem_st16(s_t + 16 * c, s);
            }
          } else {
            const float inv = 1.f / f;
#pragma unroll 1
            for (int c = 0; c < N; c += 4) {
              uint32_t s[4];
              tmem_ld4(s_t + c, s);
              tmem_ld_wait();
              const int4 e = *reinterpret_cast<const int4*>(&ms.cend[c]);
              const float4 w = *reinterpret_cast<const float4*>(&qf[c]);
              auto one = [&](uint32_t v, int end, float by) {
                const bool seen = (key < end) & ((key < p.sink) | (key >= end - window));   // (no branch)
                return seen ? __float_as_uint(__uint_as_float(v) * (by * inv)) : 0xff800000u;
              };
              s[0] = one(s[0], e.x, w.x);
              s[1] = one(s[1], e.y, w.y);
              s[2] = one(s[2], e.z, w.z);
              s[3] = one(s[3], e.w, w.w);
              tmem_st4(s_t + c, s);
            }
          }
          tmem_st_wait();
        }
        // P = 2^y: f16 to shared memory, and from chunk `add` on added to the
        // thread's sums.  With check it stops (the whole warp) at the first chunk
        // with a y above 8; returns the chunks done.
        auto weigh = [&](bool check, int add) {
          uint32_t sa[16], sb[16];
          if (C::AHEAD) tmem_ld16(s_t, sa);
#pragma unroll
          for (int c = 0; c < C::CH; ++c) {
            uint32_t(&s)[16] = (C::AHEAD && (c & 1)) ? sb : sa;
            if (!C::AHEAD) tmem_ld16(s_t + 16 * c, s);
            tmem_ld_wait();
            if (C::AHEAD && c + 1 < C::CH) tmem_ld16(s_t + 16 * (c + 1), (c & 1) ? sa : sb);   // in flight meanwhile
            uint32_t w[8];
            float2 y[8];
            const float on = c >= add ? 1.f : 0.f;
            scores16(s, negm, c, y);
            float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              top = max3(top, y[i].x, y[i].y);
              top2 = max3(top2, y[i + 1].x, y[i + 1].y);
            }
            if (__any_sync(0xffffffffu, check && fmaxf(top, top2) * f > QB_RAISE)) {
              tmem_ld_wait();
              return c;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y[i] = mul2(y[i], make_float2(f, f));
              y[i].x = exp2_fast(y[i].x);
              y[i].y = exp2_fast(y[i].y);
              l[8 * c + i] = fma2(y[i], make_float2(on, on), l[8 * c + i]);
              w[i] = pack_f16x2(y[i].x, y[i].y);
            }
            if (c == 0) wait_pv();
            uint8_t* d = pr + (c >> 2) * 16384;
            *reinterpret_cast<uint4*>(d + (((2 * (c & 3)) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(d + (((2 * (c & 3) + 1) ^ (row & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
          }
          return C::CH;
        };
        // One round; a second one with new references if the first finds a score
        // that passes its column's by more than 2^8.
        bool raise = k < 2;   // this side's first tile of the item
        int done = 0;
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
          if (raise) {
            // Column maxima of the tile over the lanes, 16 columns at a time through
            // this side's P (its last reader is done), then over the warps.
            wait_pv();
            float* stage = reinterpret_cast<float*>(smem + C::P_OFF + x * C::P_BYTES) + (warp & 3) * (16 * 36);
#pragma unroll 1
            for (int c = 0; c < C::CH; ++c) {
              uint32_t s[16];
              tmem_ld16(s_t + 16 * c, s);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) stage[i * 36 + lane] = __uint_as_float(s[i]);
              __syncwarp();
              float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(stage + (lane >> 1) * 36 + (lane & 1) * 16 + 4 * i);
                top = max3(top, v.x, v.y);
                top2 = max3(top2, v.z, v.w);
              }
              top = fmaxf(top, top2);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
              if (!(lane & 1)) atomicMax(&ms.cmax[x][16 * c + (lane >> 1)], float_key(top));
              __syncwarp();
            }
            named_bar_sync(1 + x, 128);
            if (gt < N) {
              const float nm = negm[gt], top = key_float(ms.cmax[x][gt]);
              const float rise = (top + nm) * p.factor;
              float fac = 1.f;
              if (rise > QB_RAISE) {   // an unset column's: any visible key
                fac = exp2_fast(-rise);
                negm[gt] = -top;
              }
              facs[gt] = fac;
              ms.cmax[x][gt] = float_key(-INFINITY);
            }
            named_bar_sync(1 + x, 128);
            if (k >= 2) {
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < C::CH; ++c) {
                uint32_t o[16];
                tmem_ld16(o_t + 16 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * facs[16 * c + i]);
                tmem_st16(o_t + 16 * c, o);
              }
              tmem_st_wait();
#pragma unroll
              for (int i = 0; i < N / 2; ++i) {
                const float2 fac = *reinterpret_cast<const float2*>(&facs[2 * i]);
                l[i].x *= fac.x;
                l[i].y *= fac.y;
              }
            }
            __syncwarp();
          }
          // (what a round that stopped has added stays: the new references' factors
          // apply to the sums as they stand)
          done = weigh(!raise, done);
          if (raise || !named_bar_or<128>(1 + x, done < C::CH)) break;
          raise = true;
          __syncwarp();
        }
        tc_fence_before();
        warp_arrive(&ms.s_free[t % C::SB], lane);
        fence_proxy_async_smem();
        warp_arrive(&ms.p_ready[x], lane);
      }
      u += nt;

      // ---- the item's run is over: sums over the lanes, then both sides' O
      const bool whole = bad || (j0 == 0 && nt == it.ntile);
      const bool prefix = !bad && has_prefix<PASS>(p, it.seq);
      const int border = sg.item0 < c0 ? 0 : 1;
      const int last = t0 + nt - 1;   // the other side's last tile is last - 1
      qb_wait(&ms.pvdone[last & 1], (last >> 1) & 1, dead);
      if (nt > 1) qb_wait(&ms.pvdone[(last - 1) & 1], ((last - 1) >> 1) & 1, dead);
      {
        // 16 columns at a time through this side's P (its last reader is done):
        // lane i of the warp then adds half of column i / 2
        float* stage = reinterpret_cast<float*>(smem + C::P_OFF + x * C::P_BYTES) + (warp & 3) * (16 * 36);
#pragma unroll
        for (int c = 0; c < C::CH; ++c) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            stage[2 * i * 36 + lane] = l[8 * c + i].x;
            stage[(2 * i + 1) * 36 + lane] = l[8 * c + i].y;
          }
          __syncwarp();
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(stage + (lane >> 1) * 36 + (lane & 1) * 16 + 4 * i);
            sum += (v.x + v.y) + (v.z + v.w);
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          if (!(lane & 1)) ms.lsum[warp][16 * c + (lane >> 1)] = sum;
          __syncwarp();
        }
      }
      named_bar_sync(3, 256);
      float* part = p.part + ((size_t)blockIdx.x * 2 + border) * C::SLOT;
      if (x == 0 && gt < N) {
        // a side without a tile (one-tile run) or a column without a key has sum 0 and counts nothing
        const float ma = -ms.negm[0][gt], mb = -ms.negm[1][gt], m = fmaxf(ma, mb);
        const float wa = ma == -kUnset ? 0.f : exp2_fast((ma - m) * p.factor), wb = mb == -kUnset ? 0.f : exp2_fast((mb - m) * p.factor);
        const float sum = wa * ((ms.lsum[0][gt] + ms.lsum[1][gt]) + (ms.lsum[2][gt] + ms.lsum[3][gt])) +
                          wb * ((ms.lsum[4][gt] + ms.lsum[5][gt]) + (ms.lsum[6][gt] + ms.lsum[7][gt]));
        Finish fin{1.f, 0.f};
        const float top = PASS == kAttnAll && whole ? 0.f : partial_max(-m, p.factor);
        if (whole && ms.coff[gt] >= 0) {
          fin = finish<PASS>(p, prefix, ms.coff[gt], top, sum);
          if (PASS == kAttnPrefix) p.pre_ml[ms.coff[gt]] = make_float2(top, sum);
        }
        ms.fac[0][gt] = wa * fin.own;
        ms.fac[1][gt] = wb * fin.own;
        if (PASS == kAttnOwn) ms.pre[gt] = fin.pre;
        if (!whole) {
          part[N * 128 + gt] = top;
          part[N * 129 + gt] = sum;
        }
      }
      named_bar_sync(3, 256);
      tc_fence_after();
      // thread = channel: 32 lanes write 64 (128) contiguous bytes of a row;
      // the two groups of warps take every other 16 columns
      uint8_t* out = static_cast<uint8_t*>(p.out) + 2 * row;
      // (a side without a tile has factor 0; its O may hold anything, so the
      // other side's is read in its place)
      const uint32_t o_all = tmem + C::O_COL + lanes;
      const uint32_t o_a = nt > 1 || (t0 & 1) == 0 ? o_all : o_all + N, o_b = nt > 1 || (t0 & 1) == 1 ? o_all + N : o_all;
#pragma unroll 1
      for (int c = x; c < C::CH; c += 2) {
        uint32_t oa[16], ob[16];
        __syncwarp();
        tmem_ld16(o_a + 16 * c, oa);
        tmem_ld16(o_b + 16 * c, ob);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 fa = *reinterpret_cast<const float4*>(&ms.fac[0][16 * c + i]);
          const float4 fb = *reinterpret_cast<const float4*>(&ms.fac[1][16 * c + i]);
          const float wa[4] = {fa.x, fa.y, fa.z, fa.w}, wb[4] = {fb.x, fb.y, fb.z, fb.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            oa[i + k] = __float_as_uint(fmaf(__uint_as_float(oa[i + k]), wa[k], __uint_as_float(ob[i + k]) * wb[k]));
        }
        if (!whole) {
          float* dst = part + 16 * c * 128 + row;
#pragma unroll
          for (int i = 0; i < 16; ++i) dst[i * 128] = __uint_as_float(oa[i]);
        } else if (PASS == kAttnPrefix) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int to = ms.coff[16 * c + i];
            if (to >= 0) p.pre_o[(size_t)to * 128 + row] = __uint_as_float(oa[i]);
          }
        } else {
          if (PASS == kAttnOwn && prefix) {
            // (16 loads together: one after another they took 10 us an item)
            float a[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) a[i] = __ldcg(p.pre_o + (size_t)max(ms.coff[16 * c + i], 0) * 128 + row);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (ms.pre[16 * c + i] != 0.f) oa[i] = __float_as_uint(fmaf(a[i], ms.pre[16 * c + i], __uint_as_float(oa[i])));
          }
          if (p.bf16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) oa[i] = pack_bf16x2(__uint_as_float(oa[i]), 0.f);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) oa[i] = pack_f16x2(__uint_as_float(oa[i]), 0.f);
          }
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int4 to = *reinterpret_cast<const int4*>(&ms.coff[16 * c + i]);
            const int at[4] = {to.x, to.y, to.z, to.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (at[k] >= 0) *reinterpret_cast<uint16_t*>(out + (size_t)at[k] * 256) = (uint16_t)oa[i + k];
          }
        }
      }
      tc_fence_before();
      warp_arrive(&ms.o_free, lane);
      if (!whole) {
        // (merged by the item's first CTA's entry; the others' partials follow its own)
        if (threadIdx.x == 0 && border == 1)
          ms.shared = make_int4(it.row0, it.rows, sg.sub,
                                sharers(sg.item0, it.ntile) + (prefix ? QB_PREFIX : 0));
      }
      t0 += nt;
    }

    if (threadIdx.x == 0) q4_tc_shared(p.part, N, grid)[blockIdx.x] = ms.shared;
    }
  } else if (warp < C::VDEC) {
    set_registers<C::REST_REGS, false>();
    // ---- K codes to f16: thread = cached row
    const int dt = threadIdx.x - 32 * C::KDEC;
    const uint32_t kt = tmem + C::K_COL + ((uint32_t)(32 * (warp & 3)) << 16);
    uint8_t* const ks = smem + C::P_OFF + dt * 128;   // (wide: 64 channels of a row in 128 bytes)
#pragma unroll 1
    for (int t = 0; t < T; ++t) {
      const int s = t % NS;
      const uint8_t* st = smem + C::RING_OFF + s * QB_STAGE;
      qb_wait(&ms.full[s], (t / NS) & 1, dead);
      if (t >= 2) qb_wait(&ms.kfree[t & 1], ((t >> 1) - 1) & 1, dead);
      tc_fence_after();
      {
        const int rr = dt & 15;
        const uint8_t* blk = st + (dt >> 4) * QB_BLK;
        const uint2 sc = *reinterpret_cast<const uint2*>(blk + kQ4KS + rr * 8);
#pragma unroll C::WIDE ? 4 : 1
        for (int c = 0; c < 4; ++c) {   // 32 channels: groups 2c and 2c + 1
          const uint4 w4 = *reinterpret_cast<const uint4*>(blk + q4_k_piece(rr, c));
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
          const uint32_t two = scale_pair((c < 2 ? sc.x : sc.y) >> (16 * (c & 1)));
          uint32_t out[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t sp = __byte_perm(two, 0, i < 2 ? 0x1010 : 0x3232), ns = scale_shift(sp);
            out[4 * i] = dequant<0>(w[i], sp, ns);
            out[4 * i + 1] = dequant<1>(w[i], sp, ns);
            out[4 * i + 2] = dequant<2>(w[i], sp, ns);
            out[4 * i + 3] = dequant<3>(w[i], sp, ns);
          }
          if constexpr (C::WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(ks + (t & 1) * C::P_BYTES + (c >> 1) * 16384 + ((((4 * c + i) & 7) ^ (dt & 7)) << 4)) =
                  make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
          } else {
            tmem_st16(kt + (t & 1) * 64 + 16 * c, out);
          }
        }
        if constexpr (C::WIDE) {
          fence_proxy_async_smem();
        } else {
          tmem_st_wait();
          tc_fence_before();
        }
        warp_arrive(&ms.kready[t & 1], lane);
        if (lane == 0) mbar_arrive(&ms.empty[s]);
      }
    }
  } else if (warp < C::MMA) {
    set_registers<C::REST_REGS, false>();
    // ---- V codes to f16, channels as rows: thread = 8 cached rows x 16 channels
    const int dt = threadIdx.x - 32 * C::VDEC;
    const int oct = dt & 7, g = (dt >> 3) & 7, chunk = dt >> 6;
#pragma unroll 1
    for (int t = 0; t < T; ++t) {
      const int s = t % NS;
      const uint8_t* st = smem + C::RING_OFF + s * QB_STAGE;
      qb_wait(&ms.full[s], (t / NS) & 1, dead);
      const int2 info = ms.tile[t & 15];
      if (t >= 2) qb_wait(&ms.pvdone[t & 1], ((t >> 1) - 1) & 1, dead);
      {
        const int b = chunk * 4 + (oct >> 1), par = oct & 1;
        const uint8_t* blk = st + b * QB_BLK;
        uint2 sc = *reinterpret_cast<const uint2*>(blk + kQ4VS + g * 16 + par * 8);
        if ((info.x & 255) != 255 || info.y < QB_TILE) {
          // rows that were not copied, or lie past the end and may never have
          // been written: any bits, so their scale becomes 0
          const int left = (info.x >> b & 1) ? info.y - (16 * b + 8 * par) : 0;
          uint64_t keep = left >= 8 ? ~0ull : left <= 0 ? 0ull : (1ull << (8 * left)) - 1;
          sc.x &= (uint32_t)keep;
          sc.y &= (uint32_t)(keep >> 32);
        }
        uint32_t sp[4], ns[4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          sp[jj] = scale_pair((jj < 2 ? sc.x : sc.y) >> (16 * (jj & 1)));
          ns[jj] = scale_shift(sp[jj]);
        }
        uint8_t* vt = smem + C::V_OFF + (t & 1) * C::V_BYTES + chunk * 16384 + g * 2048;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {   // 8 channels: words 2h and 2h + 1 of each piece
          uint2 w[4];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
            w[jj] = *reinterpret_cast<const uint2*>(blk + kQ4V + q4_v_piece(par * 4 + jj, g) + 8 * h);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            auto value = [&](int jj) {
              const uint32_t word = i < 4 ? w[jj].x : w[jj].y;
              return (i & 3) == 0   ? dequant<0>(word, sp[jj], ns[jj])
                     : (i & 3) == 1 ? dequant<1>(word, sp[jj], ns[jj])
                     : (i & 3) == 2 ? dequant<2>(word, sp[jj], ns[jj])
                                    : dequant<3>(word, sp[jj], ns[jj]);
            };
            // channel 16 g + 8 h + i (its low 3 bits are i)
            *reinterpret_cast<uint4*>(vt + h * 1024 + i * 128 + ((oct ^ i) << 4)) =
                make_uint4(value(0), value(1), value(2), value(3));
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&ms.vready[t & 1], lane);
        if (lane == 0) mbar_arrive(&ms.empty[s]);
      }
    }
  } else {
    set_registers<C::REST_REGS, false>();
    if (warp == C::LOAD && T > 0) {
    // ---- packed tiles, four at a time: lane 8 i + b looks after row block b of
    // tile i.  (One tile at a time, page number and addresses took this warp
    // about 1,700 cycles a tile, as long as a tile takes the other roles.)
    Cursor cur;
    first_cursor(cur);
    const int bits = p.page_shift - 4;
    int page, row0, left, head;   // of the lane's block: page, the tile's first row, rows below the request's end
    bool seen;                    // every query sees every key of the tile
    auto look_up = [&](int t0) {   // tiles t0 .. t0 + 3 of the CTA
      int seq = 0, sub = 0, L = 0, rows = 0;
      row0 = 0;
#pragma unroll 1
      for (int i = 0; i < 4 && t0 + i < T; ++i) {
        if (lane >> 3 == i) {
          row0 = item_tile(cur.it, cur.j) * QB_TILE;
          seq = cur.it.seq;
          sub = cur.sub;
          L = cur.it.L;
          rows = cur.it.rows;
        }
        if (t0 + i + 1 < T) cursor_next<QB_TILE, N>(p, cur);
      }
      left = min(L - row0, QB_TILE);
      seen = row0 + QB_TILE <= (p.causal ? L - rows + 1 : L) &&
             (p.window == 0 || row0 + QB_TILE <= p.sink || row0 >= L - p.window);
      head = sub - p.by_nkv.of(sub) * p.nkv;
      const int pos = row0 + (lane & 7) * kQ4Rows;
      page = -1;
      if (pos < L) page = table_entry<PASS>(p, seq, pos >> p.page_shift);
    };
    look_up(0);
    int t = 0;   // tiles requested
#pragma unroll 1
    while (t < T && !*dead) {
      const bool there = page >= 0 && page < p.num_pages;   // (else hidden, like a masked block)
      const uint8_t* src = p.pool + ((((size_t)(there ? page : 0) * p.nkv + head) << bits) +
                                     (row0 / kQ4Rows + (lane & 7) & ((1 << bits) - 1))) * kQ4Block;
      const uint32_t mask = __ballot_sync(0xffffffffu, there);
      const int rows = left, end = min(t + 4, T), all = seen ? QB_SEEN : 0;
      look_up(t + 4);   // (the next four page numbers travel while these tiles wait for their stages)
#pragma unroll 1
      for (; t < end; ++t) {
        const int s = t % NS, i = t & 3;
        if (t >= NS) qb_wait(&ms.empty[s], ((t / NS) - 1) & 1, dead);
        if (__any_sync(0xffffffffu, *dead)) break;
        if (lane == 8 * i) {
          const uint32_t blocks = mask >> 8 * i & 255;
          ms.tile[t & 15] = make_int2(blocks == 255 ? 255 | all : (int)blocks, rows);
          mbar_arrive_expect_tx(&ms.full[s], __popc(blocks) * kQ4Block);
        }
        __syncwarp();
        if (lane >> 3 == i && there)
          bulk_load(smem + C::RING_OFF + s * QB_STAGE + (lane & 7) * QB_BLK, src, kQ4Block, &ms.full[s]);
      }
    }
    // after an expired wait: what was requested and not yet waited for
    if (t < T)
      for (int i = max(t - NS, 0); i < t; ++i) mbar_wait(&ms.full[i % NS], (i / NS) & 1, nullptr, nullptr);
    zero_rows<PASS>(p, lane, 32);
    } else if (warp == C::LOAD) {
      zero_rows<PASS>(p, lane, 32);
    } else if (warp == C::QUERY && T > 0) {
    // ---- query rows, as f16 with the factor that their scores take
    Cursor cur;
    first_cursor(cur);
    const float base_f = 16.f * p.scale_log2;
    int u = c0;
#pragma unroll 1
    for (int seg = 0; u < c1; ++seg) {
      const int qb = seg % C::QB;
      const int nt = min(cur.it.ntile - cur.j, c1 - u);
      if constexpr (C::WIDE) {   // the softmax warps bring the rows; records run ahead of them, while there is room
        // (that of item seg - 4 is no longer read once item seg - 3 has begun)
        if (seg >= 3) qb_wait(&ms.begun[(seg - 3) & 3], ((seg - 3) >> 2) & 1, dead);
      } else if (seg >= C::QB) {
        qb_wait(&ms.q_free[qb], ((seg / C::QB) - 1) & 1, dead);
      }
      uint8_t* qs = smem + C::Q_OFF + qb * C::Q_BYTES;
      float* qf = ms.qf[C::WIDE ? 0 : seg % C::SEGS];
      const int grp = p.by_nkv.of(cur.sub), q0 = grp * N, head0 = (cur.sub - grp * p.nkv) * G;
      bool uniform = true;
      if constexpr (!C::WIDE) {
        // Every 16-byte piece of the rows at once, 2 rows an instruction.  (One warp does
        // it all: what a row costs is its chain of instructions, so addresses are added
        // up, four rows' under way together.)
        const int piece = lane & 15, side = lane >> 4;
        uint8_t* const dst = qs + (piece >> 3) * (N * 128) + side * 128;
        int j = p.by_g.of(q0 + side), h = q0 + side - j * G;
        const uint16_t* at = static_cast<const uint16_t*>(p.q) + (size_t)(cur.it.row0 + j) * p.q_row + (size_t)(head0 + h) * p.q_head + 8 * piece;
        const long long wrap = p.q_row - G * p.q_head;
#pragma unroll 1
        for (int i = 0; i < N; i += 8) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const bool real = j < cur.it.rows;
            cp_async16_zfill(smem_u32(dst + (i + e) * 128 + (((piece & 7) ^ (e + side)) << 4)), real ? at : p.q, real);
            h += 2;
            at += 2 * p.q_head;
            if (h >= G) { h -= G; ++j; at += wrap; }
            if (h >= G) { h -= G; ++j; at += wrap; }   // (one head a kv head)
          }
        }
        cp_async_commit();
        for (int i = lane; i < N; i += 32) qf[i] = base_f;
        cp_async_wait<0>();
        __syncwarp();
        if (p.bf16) {
          // To f16 in place.  Votes are cheaper than maxima (256 requests of 16 x 4 rows
          // 210 us, all rows by maxima 245), but rows that have to be scaled need these: behind
          // 8 rows of which some were scaled the next 8 go there at once (all scaled: 317 us,
          // with votes first 348).
          const uint32_t half = side == 0 ? 0xffffu : 0xffff0000u;   // the lanes of this lane's row
          bool scaling = false;
#pragma unroll 1
          for (int i = 0; i < N; i += 8) {
            uint32_t left = scaling ? 15u : 0u;
            if (!scaling) {
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                uint4* const to = reinterpret_cast<uint4*>(dst + (i + e) * 128 + (((piece & 7) ^ (e + side)) << 4));
                float x[8];
                const float a = query_floats(*to, x);
                const uint32_t big = __ballot_sync(0xffffffffu, a >= 0.125f), nonzero = __ballot_sync(0xffffffffu, a > 0.f),
                               over = __ballot_sync(0xffffffffu, a > 32768.f);
                if (!(over & half) && (!(nonzero & half) || (big & half)))
                  *to = make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
                else
                  left |= 1u << (e / 2);
              }
            }
            if (__any_sync(0xffffffffu, left != 0)) {
              bool any = false;
#pragma unroll
              for (int k = 0; k < 8; k += 2) {
                const bool mine = left >> (k / 2) & 1;
                const int e = query_f16(reinterpret_cast<uint4*>(dst + (i + k) * 128 + (((piece & 7) ^ (k + side)) << 4)), mine, lane);
                if (e && piece == 0) qf[i + k + side] = scaled_factor(base_f, e);
                any = any || e != 0;
              }
              scaling = __any_sync(0xffffffffu, any);
              uniform = uniform && !scaling;
            }
          }
        }
        uniform = __all_sync(0xffffffffu, uniform);
      }
      if (lane == 0) {
        QbSeg& sg = ms.seg[seg % C::SEGS];
        sg.it = cur.it;
        sg.sub = cur.sub; sg.q0 = q0; sg.head0 = head0;
        sg.j0 = cur.j; sg.nt = nt; sg.item0 = u - cur.j; sg.uniform = uniform;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(C::WIDE ? &ms.rec_ready[seg & 3] : &ms.q_ready[qb]);
      u += nt;
      cur.j += nt - 1;
      if (u < c1) cursor_next<QB_TILE, N>(p, cur);
    }
    } else if (warp == C::MMA && T > 0) {
      // ---- S(t) = K(t) Q^T, as soon as K is there and the softmax has read the buffer's last S
      // (wide: Q K(t)^T, and the P that took its place is read)
      const uint32_t idesc = umma_idesc_f16(128, N, 0);
      const uint64_t qd = umma_desc_sw128(smem_u32(smem + C::Q_OFF)), kd = umma_desc_sw128(smem_u32(smem + C::P_OFF));
      int seg = 0, k = 0, nt = 0;
#pragma unroll 1
      for (int t = 0; t < T; ++t) {
        const int qb = seg % C::QB;
        if (k == 0) {
          qb_wait(&ms.q_ready[qb], (seg / C::QB) & 1, dead);
          nt = ms.seg[seg % C::SEGS].nt;
        }
        if (t >= C::SB) qb_wait(&ms.s_free[t % C::SB], (t / C::SB - 1) & 1, dead);
        qb_wait(&ms.kready[t & 1], (t >> 1) & 1, dead);
        const bool last = ++k == nt;
        if (elect_one()) {
          tc_fence_after();
          const uint32_t d = tmem + C::S_COL + (t % C::SB) * N, ka = tmem + C::K_COL + (t & 1) * 64;
          const uint64_t q = qd + qb * (C::Q_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            if constexpr (C::WIDE)
              umma_f16(d, q + (ks >> 2) * 1024 + 2 * (ks & 3), kd + (t & 1) * (C::P_BYTES >> 4) + (ks >> 2) * 1024 + 2 * (ks & 3),
                       idesc, ks > 0);
            else
              umma_ts(d, ka + ks * 8, q + ((ks >> 2) * (N * 128) >> 4) + 2 * (ks & 3), idesc, ks > 0);
          umma_commit(&ms.s_ready[t % C::SB]);
          umma_commit(&ms.kfree[t & 1]);
          if (last) umma_commit(&ms.q_free[qb]);
        }
        __syncwarp();
        if (last) {
          k = 0;
          ++seg;
        }
      }
    } else if (warp == C::MMA2 && T > 0) {
      // ---- O(side of t) += V^T(t) P^T(t) (wide: O += P(t) V(t), P from TMEM)
      const uint32_t idesc = umma_idesc_f16(128, N, 0) | (C::WIDE ? 0 : 1u << 16);   // B (P^T) with the columns contiguous
      const uint64_t vd = umma_desc_sw128(smem_u32(smem + C::V_OFF)), pd = desc_sw128_mn(smem_u32(smem + C::P_OFF), 16384);
      int seg = 0, k = 0, nt = 0;
#pragma unroll 1
      for (int t = 0; t < T; ++t) {
        qb_wait(&ms.vready[t & 1], (t >> 1) & 1, dead);
        qb_wait(&ms.p_ready[t & 1], (t >> 1) & 1, dead);
        if (k == 0) {
          nt = ms.seg[seg % C::SEGS].nt;
          if (seg > 0) qb_wait(&ms.o_free, (seg - 1) & 1, dead);
        }
        if (elect_one()) {
          tc_fence_after();
          const uint64_t v = vd + (t & 1) * (C::V_BYTES >> 4), pp = pd + (t & 1) * (C::P_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)   // (a side's first tile of the item starts its O)
            if constexpr (C::WIDE)
              umma_ts(tmem + C::O_COL, tmem + C::S_COL + (t % C::SB) * N + (ks >> 2) * 64 + (ks & 3) * 8,
                      v + (ks >> 2) * 1024 + 2 * (ks & 3), idesc, k > 0 || ks > 0);
            else
              umma_f16(tmem + C::O_COL + (t & 1) * N, v + (ks >> 2) * 1024 + 2 * (ks & 3), pp + ks * 128, idesc, k > 1 || ks > 0);
          umma_commit(&ms.pvdone[t & 1]);
          if (C::WIDE) umma_commit(&ms.s_free[t % C::SB]);
        }
        __syncwarp();
        if (++k == nt) {
          k = 0;
          ++seg;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && ms.abort && p.status) atomicOr(p.status, kPagedTimeout);
  if (warp == C::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merges the items that several CTAs of the kernel above hold: CTA (b, y) the
// queries 16 y .. + 15 of the item that starts in CTA b, two a warp.  The item's
// first partial is CTA b's second one, the others are the first ones of the CTAs
// after it.
template <int PASS>
__global__ void __launch_bounds__(256) q4_attn_tc_merge_kernel(const Q4AttnParams p, int n) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  const int4 item = __ldcg(q4_tc_shared(p.part, n, gridDim.x) + b);   // row0, rows, sub, count
  auto slot = [&](int i) { return p.part + ((size_t)(b + i) * 2 + (i == 0 ? 1 : 0)) * n * 130; };
  const int grp = p.by_nkv.of(item.z), G = p.by_g.d;
#pragma unroll 1
  for (int q = 16 * blockIdx.y + warp; q < 16 * blockIdx.y + 16; q += 8) {
    const int r = grp * n + q, j = p.by_g.of(r);
    if (item.w == 0 || j >= item.y) return;
    float v[4], m, l;
    merge_query(PASS == kAttnOwn ? item.w & (QB_PREFIX - 1) : item.w, slot, n, q, lane, v, &m, &l);
    const int head = (item.z - grp * p.nkv) * G + r - j * G;
    const Finish f = finish<PASS>(p, PASS == kAttnOwn && item.w >= QB_PREFIX, (size_t)(item.x + j) * p.nq + head, m, l);
    finish4<PASS>(p, item.x + j, head, 4 * lane, v, f, m, l);
  }
}

// Columns of the instruction for R = max_rows * G query rows of a kv head: the
// fewest groups of at most 80 (a thread keeps a sum for every column), evenly
// filled, in steps of 16 and 32 at least (with fewer a tile costs no less: 32, 48,
// 64 and 80 columns take 115, 120, 134 and 164 us for 16 requests of 16,384 rows).
// 160 rows as two groups of 80 take 303 us there, three of 64 three times 134.
int q4_attn_tc_columns(int max_rows, int nq, int nkv) {
  const long long R = (long long)max_rows * (nq / nkv);
  const long long groups = (R + 79) / 80;
  const int n = (int)(((R + groups - 1) / groups + 15) / 16 * 16);
  return n < 32 ? 32 : n;
}

size_t q4_attn_tc_part_floats(int max_rows, int nq, int nkv, int num_sms) {
  // (for every number of rows up to max_rows: past 80 columns they start again at 48)
  const int columns = (long long)max_rows * (nq / nkv) >= 80 ? 80 : q4_attn_tc_columns(max_rows, nq, nkv);
  return (size_t)num_sms * (2 * columns * 130 + sizeof(int4) / sizeof(float));
}

template <int N, int PASS>
static cudaError_t launch_tc(const Q4AttnParams& p, int num_sms, cudaStream_t st) {
  using C = QbCfg<N>;
  constexpr size_t smem = C::MISC_OFF + sizeof(QbMisc<C>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  DFL_TRY(cudaFuncSetAttribute(q4_attn_tc_kernel<N, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  DFL_TRY(launch_pdl(q4_attn_tc_kernel<N, PASS>, dim3(num_sms), dim3(C::THREADS), smem, st, p));
  return launch_pdl(q4_attn_tc_merge_kernel<PASS>, dim3(num_sms, N / 16), dim3(256), 0, st, p, N);
}

// Query rows of a group's pass past 64 of a kv head: the wide form (us, wide / not:
// 64 rows on 8 groups of 8,192 rows 71 / 66 in f16 and 72 / 71 in bf16, 80 rows 73 / 78
// and 74 / 86; 32 groups of 4,096 rows 139 / 126 and 141 / 146).
static bool wide_pass(int max_rows, int nq, int nkv) { return (long long)max_rows * (nq / nkv) > 64; }

size_t q4_attn_tc_group_floats(int max_rows, int nq, int nkv, int num_sms) {
  const size_t n = wide_pass(max_rows, nq, nkv) ? 128 : 80;
  return (size_t)num_sms * (2 * n * 130 + sizeof(int4) / sizeof(float));
}

template <int PASS>
static cudaError_t launch_pass(const Q4AttnParams& p, int num_sms, cudaStream_t st) {
  if (PASS == kAttnPrefix && wide_pass(p.max_rows, p.nq, p.nkv)) return launch_tc<128, kAttnPrefix>(p, num_sms, st);
  switch (q4_attn_tc_columns(p.max_rows, p.nq, p.nkv)) {
    case 32: return launch_tc<32, PASS>(p, num_sms, st);
    case 48: return launch_tc<48, PASS>(p, num_sms, st);
    case 64: return launch_tc<64, PASS>(p, num_sms, st);
    case 80: return launch_tc<80, PASS>(p, num_sms, st);
  }
  return cudaErrorInvalidValue;
}

cudaError_t q4_attn_tc_launch(const Q4AttnParams& p, int pass, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  return pass == kAttnAll      ? launch_pass<kAttnAll>(p, num_sms, st)
         : pass == kAttnPrefix ? launch_pass<kAttnPrefix>(p, num_sms, st)
                               : launch_pass<kAttnOwn>(p, num_sms, st);
}

}  // namespace dfl
