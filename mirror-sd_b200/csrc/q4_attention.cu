// Grouped-query attention over the paged 4-bit cache (layout: q4.cuh).
//
//   out[j, h] = sum_k softmax_k(scale * q[j, h] . K[k]) V[k],  K, V = (u - 8) s
//
// over the cached rows k that query row j of a request sees (tile_span in
// q4_attn.cuh).  R = rows * G query rows of a request share a kv head (G = NQ / NKV,
// row r = j * G + g), cut into groups of QT = 8 * NT.
//
// Work is split over the cached rows by one rule for every batch: the tiles
// of 64 cached rows of all (request, query group, kv head) items lie end to
// end, every warp of the grid takes an equal run of them, and what a run
// leaves unfinished of an item is merged afterwards (warps of a CTA first,
// then the CTAs that share an item, by the last of them to arrive, always in
// the order of the runs).  The lengths are only known on the GPU, so each CTA
// adds them up itself instead of the host planning a grid.
//
// A warp works alone: its lanes 0-3 keep a ring of tiles filled with bulk
// copies (one 2304-byte row block each), and the block layout makes every
// 16-byte shared-memory read a matrix fragment.  Per 16 cached rows,
//   S^T[16 rows, QT] = K[16, 128] Q^T      8 k-steps of m16n8k16
//   O^T[128, QT]    += V^T[128, 16] P^T    8 channel tiles
// with the rows (then the channels) as the tile's 16 rows, so QT = 8 query
// rows waste no half of the instruction as query-major tiles of 16 would.
// Codes become f16 by bit placement: (w >> k) & 0x00F0 | 0x3C00 is 1 + u/64,
// and one f16 FMA gives x / 16 = (1 + u/64) 4s - 4.5s exactly (every term has
// at most 7 significant bits).  The factors 16 go into the softmax scale and
// the final division.  S^T leaves the products with a lane holding two query
// columns of a row; packing those two and transposing 8x8 blocks (movmatrix)
// makes the P^T fragment.  P is rounded to f16 (2^-12 relative, the operand
// type), sums and statistics stay fp32.
//
// A column's reference (what its scores are measured against) only moves when a
// score passes it by 2^8, then O and the sum are rescaled: P below 256 stays
// in f16's range, and a weight below 2^-14 of the reference's loses 2^-25 of that
// at most.
//
// 256 requests of up to 8,192 rows, 32 heads over 8 kv heads, are 1.34 GB, 205 us
// of HBM; they take 306 to 326 us (4.1 to 4.4 TB/s).  What bounds it is instruction issue and
// latency: 1,300 instructions a tile and warp, 3 warps a scheduler (shared memory
// holds two tiles for each of 12), 60 % of the issue slots taken.  Tiles of 32
// rows, whose upkeep is paid twice as often, took 314 us for 256 requests of
// 4,096 against 269, 16 warps of such tiles 285, 10 warps 326.  One token on
// 2,049 rows takes 11.4 us, a chain of latencies: lengths, page numbers, tiles,
// one tile's work, and two merges.
#include "q4_attn.cuh"

namespace dfl {

constexpr int QA_TILE = kQ4Tile;                     // cached rows of a tile
constexpr int QA_STAGE = QA_TILE / kQ4Rows * kQ4Block;
// Tiles of a CTA at least: a warp for each scheduler.  Fewer tiles spread an item
// over more CTAs, whose partials the last one merges (2,049 rows: 13.3 us with 1,
// 11.7 with 2, 11.4 with 4, 12.3 with 8).
constexpr int QA_LEAST = 4;
constexpr int QA_ITEM = 3;                           // what an item's start and end cost beside its tiles, in tiles
constexpr float QA_RAISE = 8.f;
constexpr size_t QA_SMEM = 225 * 1024;               // dynamic shared memory at most, beside the kernel's static 1.3 KB

// ---- fragments
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float col_max(float v) {   // over the 8 lanes that share lane % 4
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <int NT>
struct QaCfg {
  static constexpr int QT = 8 * NT;
  // as many warps as the registers allow, the rest of shared memory for tiles
  static constexpr int WARPS = NT == 1 ? 12 : 8, STAGES = NT == 1 ? 2 : 3, THREADS = 32 * WARPS;
  static constexpr int SLOT = QT * 130;   // floats of a partial: O [QT][128], m [QT], l [QT]
  static constexpr int RING = WARPS * STAGES * QA_STAGE;
};

// A warp merges the partials of one item that the slots of `mask` hold (slot k
// at at[k]), all queries at once: 8 (16) loads of a partial's O are on their way
// together.  Writes the item's output rows (finish) or one partial at dst.
template <int NT, int PASS>
__device__ __forceinline__ void merge_slots(const Q4AttnParams& p, uint32_t mask, const float* const* at, float* dst,
                                            const Item& it, int sub, bool whole, int lane) {
  constexpr int QT = QaCfg<NT>::QT;
  const int q = lane & (QT - 1);
  float M = -INFINITY, l = 0.f;
#pragma unroll 1
  for (uint32_t m = mask; m; m &= m - 1) M = fmaxf(M, at[__ffs(m) - 1][QT * 128 + q]);
  float4 o[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (uint32_t m = mask; m; m &= m - 1) {
    const float* s = at[__ffs(m) - 1];
    const float mk = s[QT * 128 + q], lk = s[QT * 129 + q];
    float4 v[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) v[i] = *reinterpret_cast<const float4*>(s + i * 128 + 4 * lane);
    const float w = mk == -INFINITY ? 0.f : exp2_fast(mk - M);
    l = fmaf(w, lk, l);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      o[i].x = fmaf(wi, v[i].x, o[i].x);
      o[i].y = fmaf(wi, v[i].y, o[i].y);
      o[i].z = fmaf(wi, v[i].z, o[i].z);
      o[i].w = fmaf(wi, v[i].w, o[i].w);
    }
  }
  if (!whole && lane < QT) {
    dst[QT * 128 + q] = M;
    dst[QT * 129 + q] = l;
  }
  constexpr int END = PASS == kAttnPrefix ? kAttnPrefix : kAttnAll;   // (own rows went on from the group's)
  const int grp = p.by_nkv.of(sub), head0 = (sub - grp * p.nkv) * p.by_g.d;
  const Finish fin = finish<END>(p, false, 0, M, l);
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    if (whole) {
      const Finish f{__shfl_sync(0xffffffffu, fin.own, i), 0.f};
      const float mi = PASS == kAttnPrefix ? __shfl_sync(0xffffffffu, M, i) : 0.f;
      const float li = PASS == kAttnPrefix ? __shfl_sync(0xffffffffu, l, i) : 0.f;
      const int r = grp * QT + i, j = p.by_g.of(r);
      const float v[4] = {o[i].x, o[i].y, o[i].z, o[i].w};
      if (j < it.rows) finish4<END>(p, it.row0 + j, head0 + r - j * p.by_g.d, 4 * lane, v, f, mi, li);
    } else {
      *reinterpret_cast<float4*>(dst + i * 128 + 4 * lane) = o[i];
    }
  }
}

template <int NT, int PASS>
__global__ void __launch_bounds__(QaCfg<NT>::THREADS, 1) q4_attn_kernel(const Q4AttnParams p) {
  using C = QaCfg<NT>;
  constexpr int QT = C::QT;
  constexpr int END = PASS == kAttnPrefix ? kAttnPrefix : kAttnAll;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::RING);          // [warp][stage]
  int* base = reinterpret_cast<int*>(bars + C::WARPS * C::STAGES);       // [n + 1] first tile of each request
  // Passes over shared and own rows weigh an item's start and end as well, QA_ITEM
  // tiles, where there are items for every warp: an item is then that many units
  // followed by its tiles, and runs are cut by units.
  int W = PASS == kAttnAll || !p.weigh ? 0 : QA_ITEM;
  int* ubase = base + p.n + 1;                                           // [n] first unit of each request, if weighed
  __shared__ int wtot[C::WARPS];
  __shared__ int slot_item[2 * C::WARPS];   // unit at which the partial's item starts, or -1
  __shared__ Item slot_info[2 * C::WARPS];
  __shared__ int slot_sub[2 * C::WARPS];
  __shared__ const float* slot_at[2 * C::WARPS];   // the partial: in the warp's ring if its run ended with it, else in p.part
  __shared__ int last_run[2];               // runs (of the CTA's two borders) this CTA must finish
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = p.by_g.d;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::WARPS * C::STAGES; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
    last_run[0] = last_run[1] = -1;
  }
  if (threadIdx.x < 2 * C::WARPS) slot_item[threadIdx.x] = -1;
  griddep_wait();
  griddep_launch_dependents();
  // tiles of every request, added up (kPagedMaxSeqs / C::THREADS passes at most)
  int total = 0, units = 0;
  auto add_up = [&](int i, int v, int* first, int& total) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = tiles_sum(x, y);
    }
    __syncthreads();
    if (lane == 31) wtot[warp] = x;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      if (w < warp) before = tiles_sum(before, wtot[w]);
      total = tiles_sum(total, wtot[w]);
    }
    if (i < p.n) first[i] = tiles_sum(before, x - v);
  };
  for (int i0 = 0; i0 < p.n; i0 += C::THREADS) {
    const int i = i0 + threadIdx.x;
    int v = 0, w = 0;
    if (i < p.n) {
      const Item it = load_item<QA_TILE, QT>(p, i);
      v = it.ntile * it.groups * p.nkv;
      w = (it.ntile + W) * it.groups * p.nkv;
      if (blockIdx.x == 0 && p.status && !rows_fit(p, i)) atomicOr(p.status, kPagedRows);
    }
    add_up(i, v, base, total);
    if (W > 0) add_up(i, w, ubase, units);
  }
  if (total == kTilesFull || units == kTilesFull) total = units = 0;
  if (PASS != kAttnAll && units - total < QA_ITEM * (int)gridDim.x * C::WARPS) W = 0;
  if (threadIdx.x == 0) base[p.n] = total;
  __syncthreads();

  const int ctas = min((int)gridDim.x, (total + QA_LEAST - 1) / QA_LEAST);   // CTAs with work
  const int cta = blockIdx.x;
  if (cta >= ctas) {
    zero_rows<PASS>(p, threadIdx.x, C::THREADS);
    return;
  }
  const Runs runs(W > 0 ? units : total, ctas);
  // the first tile at or behind a unit
  auto tile_at = [&](int unit) {
    if (W == 0) return unit;
    if (unit >= units) return total;
    int lo = 0, hi = p.n - 1;
    while (lo < hi) {   // last request whose first unit is at most that
      const int mid = (lo + hi + 1) >> 1;
      if (ubase[mid] <= unit) lo = mid; else hi = mid - 1;
    }
    const int nt = load_item<QA_TILE, QT>(p, lo).ntile, k = (unit - ubase[lo]) / (nt + W);
    return base[lo] + k * nt + max(unit - ubase[lo] - k * (nt + W) - W, 0);
  };
  // the unit of an item's first tile
  auto unit_of = [&](const Item& it, int item0) {
    return W == 0 ? item0 : ubase[it.seq] + (item0 - base[it.seq]) / it.ntile * (it.ntile + W) + W;
  };
  const int cta_unit = runs.start(cta), c0 = tile_at(cta_unit), c1 = tile_at(runs.start(cta + 1));
  const Runs mine(runs.start(cta + 1) - cta_unit, C::WARPS);
  const int u0 = tile_at(cta_unit + mine.start(warp)), u1 = tile_at(cta_unit + mine.start(warp + 1));

  if (u0 < u1) {
    uint8_t* ring = smem + warp * C::STAGES * QA_STAGE;
    uint64_t* bar = bars + warp * C::STAGES;
    Cursor cur, ahead;
    cursor_at<QA_TILE, QT>(p, base, u0, cur);
    ahead = cur;
    // lane b < 4 looks after row block b of a tile: its page, then its copy
    auto page_of = [&](const Cursor& k) {
      const int pos = item_tile(k.it, k.j) * QA_TILE + (lane & 3) * kQ4Rows;
      return lane < 4 && pos < k.it.L ? table_entry<PASS>(p, k.it.seq, pos >> p.page_shift) : -1;
    };
    int next_page = page_of(ahead);
    uint32_t loaded = 0;   // 4 bits a stage: row blocks that were copied
    int fill = u0, fill_end = u1;   // tiles requested so far; fewer than the run after an expired wait
    auto issue = [&](int s) {
      // (looked at only here, a tile after it was requested)
      const bool there = next_page >= 0 && next_page < p.num_pages;   // else hidden, like a masked block
      const uint32_t mask = __ballot_sync(0xffffffffu, there);
      if (lane == 0) mbar_arrive_expect_tx(&bar[s], __popc(mask) * kQ4Block);
      __syncwarp();
      if (there) {
        const int pos = item_tile(ahead.it, ahead.j) * QA_TILE + lane * kQ4Rows;
        const int head = ahead.sub - p.by_nkv.of(ahead.sub) * p.nkv, bits = p.page_shift - 4;   // 16-row blocks a page: 2^bits
        bulk_load(ring + s * QA_STAGE + lane * kQ4Block,
                  p.pool + ((((size_t)next_page * p.nkv + head) << bits) + (pos / kQ4Rows & ((1 << bits) - 1))) * kQ4Block, kQ4Block,
                  &bar[s]);
      }
      loaded = (loaded & ~(15u << (4 * s))) | mask << (4 * s);
      ++fill;
      if (fill < fill_end) {
        cursor_next<QA_TILE, QT>(p, ahead);
        next_page = page_of(ahead);
      }
    };
#pragma unroll 1
    for (int s = 0; s < C::STAGES && fill < fill_end; ++s) issue(s);

    uint32_t qf[NT][16];
    float qscale[NT][2], negm[NT][2], l[NT][2], o[8][NT][4];
    int key_end[NT][2];
    int u = u0, stage = 0;
    uint32_t phase = 0;
    bool fresh = true, alive = true;
    int seg_first = u0;   // first unit of the running segment
#pragma unroll 1
    while (u < u1) {
      const int item0 = u - cur.j;   // the item's first unit
      if (fresh) {
        fresh = false;
        seg_first = u;
        const int grp = p.by_nkv.of(cur.sub), r0 = grp * QT, head0 = (cur.sub - grp * p.nkv) * G;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = r0 + nt * 8 + g, j = p.by_g.of(r);
          uint4 w[4] = {};
          if (j < cur.it.rows) {
            const uint4* src = reinterpret_cast<const uint4*>(
                static_cast<const uint16_t*>(p.q) + (size_t)(cur.it.row0 + j) * p.q_row +
                (size_t)(head0 + r - j * G) * p.q_head + 32 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __ldg(src + i);
          }
          float f = 1.f;
          uint32_t* qr = qf[nt];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qr[4 * i] = w[i].x; qr[4 * i + 1] = w[i].y; qr[4 * i + 2] = w[i].z; qr[4 * i + 3] = w[i].w;
          }
          if (p.bf16) {
            // bf16 query rows as f16: scaled by a power of two so that the
            // row's largest magnitude lies in [1, 2); only values 2^-14 below
            // it lose bits, 2^-25 of it at most
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              a = fmaxf(a, fmaxf(fabsf(__uint_as_float(qr[i] << 16)), fabsf(__uint_as_float(qr[i] & 0xffff0000u))));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
            const int e = min(max((int)(__float_as_uint(a) >> 23), 1), 253);   // biased exponent
            const float down = __uint_as_float((uint32_t)(254 - e) << 23);
            f = __uint_as_float((uint32_t)e << 23);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              qr[i] = pack_f16x2(__uint_as_float(qr[i] << 16) * down, __uint_as_float(qr[i] & 0xffff0000u) * down);
          }
          f = score_factor(f * 16.f * p.scale_log2);
          // the lane's score columns are queries 2c and 2c + 1 of this group of 8
          qscale[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
          qscale[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int jj = p.by_g.of(r0 + nt * 8 + 2 * c + x);
            key_end[nt][x] = jj < cur.it.rows ? (p.causal ? cur.it.L - cur.it.rows + jj + 1 : cur.it.L) : 0;
            negm[nt][x] = kUnset;
            l[nt][x] = 0.f;
          }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[t][nt][x] = 0.f;
        if (PASS == kAttnOwn && cur.j == 0 && has_prefix<PASS>(p, cur.it.seq)) {
          // the item's first tile goes on from what the pass over its group's rows left
          // (joined at the item's end instead, 256 requests of 512 rows took 74 us, not 62)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int r = r0 + nt * 8 + 2 * c + x, j = p.by_g.of(r);
              if (j >= cur.it.rows) continue;
              const size_t at = (size_t)(cur.it.row0 + j) * p.nq + head0 + r - j * G;
              const float2 ml = __ldcg(p.pre_ml + at);
              const float* src = p.pre_o + at * 128 + 16 * g;
#pragma unroll
              for (int t = 0; t < 8; t += 2) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(src + 2 * t));
                o[t][nt][x] = v.x;
                o[t][nt][2 + x] = v.y;
                o[t + 1][nt][x] = v.z;
                o[t + 1][nt][2 + x] = v.w;
              }
              if (ml.x != -INFINITY) {
                negm[nt][x] = -ml.x / qscale[nt][x];
                l[nt][x] = g == 0 ? ml.y : 0.f;
              }
            }
        }
      }

      const uint32_t have = (loaded >> (4 * stage)) & 15u;
      // after an expired wait nothing more is requested, and what is in flight is still waited for
      if (u < fill && !__all_sync(0xffffffffu, mbar_wait(&bar[stage], (phase >> stage) & 1, nullptr, nullptr))) {
        if (lane == 0 && p.status) atomicOr(p.status, kPagedTimeout);
        alive = false;
        fill_end = fill;
      }
      phase ^= 1u << stage;
      if (have && alive) {
        const uint8_t* tile = ring + stage * QA_STAGE;
        const int row0 = item_tile(cur.it, cur.j) * QA_TILE;
        const bool all_seen = have == 15u && row0 + QA_TILE <= (p.causal ? cur.it.L - cur.it.rows + 1 : cur.it.L) &&
                              (p.window == 0 || row0 + QA_TILE <= p.sink || row0 >= cur.it.L - p.window);
        // Two row blocks at a time: one leaves the pipes idle between dependent
        // steps, and the whole tile unrolled outgrows the instruction cache.
#pragma unroll 1
        for (int b0 = 0; b0 < 4; b0 += 2) {
          if (!(have >> b0 & 3)) continue;
          float sc[2][NT][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint8_t* blk = tile + (b0 + i) * kQ4Block;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x) sc[i][nt][x] = 0.f;
            const uint4 wa = *reinterpret_cast<const uint4*>(blk + q4_k_piece(g, c));
            const uint4 wb = *reinterpret_cast<const uint4*>(blk + 512 + q4_k_piece(g, c));
            const uint32_t s2a = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4KS + g * 8 + 2 * c));
            const uint32_t s2b = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4KS + 64 + g * 8 + 2 * c));
            const uint32_t ka[4] = {wa.x, wa.y, wa.z, wa.w}, kb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {   // channels 32c + 8w .. + 7: group 2c + w / 2
              const uint32_t sa = __byte_perm(s2a, 0, w < 2 ? 0x1010 : 0x3232);
              const uint32_t sb = __byte_perm(s2b, 0, w < 2 ? 0x1010 : 0x3232);
              const uint32_t na = scale_shift(sa), nb = scale_shift(sb);
              const uint32_t a0 = dequant<0>(ka[w], sa, na), a2 = dequant<1>(ka[w], sa, na);
              const uint32_t a1 = dequant<0>(kb[w], sb, nb), a3 = dequant<1>(kb[w], sb, nb);
              const uint32_t e0 = dequant<2>(ka[w], sa, na), e2 = dequant<3>(ka[w], sa, na);
              const uint32_t e1 = dequant<2>(kb[w], sb, nb), e3 = dequant<3>(kb[w], sb, nb);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16_16816(sc[i][nt], a0, a1, a2, a3, qf[nt][4 * w], qf[nt][4 * w + 1]);
                mma_f16_16816(sc[i][nt], e0, e1, e2, e3, qf[nt][4 * w + 2], qf[nt][4 * w + 3]);
              }
            }
          }
          // Scores less the columns' references (negm: minus the largest product that
          // set it), base 2; hidden keys get -inf.  Where one passes 2^8 the references
          // move first.
          float y[2][NT][4];
          auto scores = [&]() {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int x = 0; x < 4; ++x) y[i][nt][x] = (sc[i][nt][x] + negm[nt][x & 1]) * qscale[nt][x & 1];
                if (!all_seen) {
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const int key = row0 + 16 * (b0 + i) + g + 8 * (x >> 1), end = key_end[nt][x & 1];
                    const bool seen = (have >> (b0 + i) & 1) & (key < end) &
                                      ((p.window == 0) | (key < p.sink) | (key >= end - p.window));
                    y[i][nt][x] = seen ? y[i][nt][x] : -INFINITY;
                  }
                }
                top = fmaxf(fmaxf(fmaxf(y[i][nt][0], y[i][nt][1]), fmaxf(y[i][nt][2], y[i][nt][3])), top);
              }
            return top;
          };
          if (__any_sync(0xffffffffu, scores() > QA_RAISE)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                // the column's largest product
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                  for (int h = 0; h < 4; h += 2)
                    if (y[i][nt][h + x] != -INFINITY) top = fmaxf(top, sc[i][nt][h + x]);
                top = col_max(top);
                const float rise = (top + negm[nt][x]) * qscale[nt][x];
                const bool up = rise > QA_RAISE;
                const float f = up ? exp2_fast(-rise) : 1.f;
                negm[nt][x] = up ? -top : negm[nt][x];
                l[nt][x] *= f;
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                  o[t][nt][x] *= f;
                  o[t][nt][2 + x] *= f;
                }
              }
            scores();
          }
          uint32_t pb[2][NT][2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float p0 = exp2_fast(y[i][nt][0]), p1 = exp2_fast(y[i][nt][1]);
              const float p2 = exp2_fast(y[i][nt][2]), p3 = exp2_fast(y[i][nt][3]);
              l[nt][0] += p0 + p2;
              l[nt][1] += p1 + p3;
              pb[i][nt][0] = transpose8x8(pack_f16x2(p0, p1));
              pb[i][nt][1] = transpose8x8(pack_f16x2(p2, p3));
            }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint8_t* blk = tile + (b0 + i) * kQ4Block;
            const uint4 wa = *reinterpret_cast<const uint4*>(blk + kQ4V + q4_v_piece(c, g));
            const uint4 wb = *reinterpret_cast<const uint4*>(blk + kQ4V + q4_v_piece(c + 4, g));
            uint32_t sa = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4VS + g * 16 + 2 * c));
            uint32_t sb = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4VS + g * 16 + 8 + 2 * c));
            if (!all_seen) {
              // rows that were not copied, or lie past the end and may never have
              // been written: any bits, so their scale becomes 0
              const int left = (have >> (b0 + i) & 1) ? cur.it.L - (row0 + 16 * (b0 + i)) : 0;
              sa &= (2 * c < left ? 0xffffu : 0u) | (2 * c + 1 < left ? 0xffff0000u : 0u);
              sb &= (2 * c + 8 < left ? 0xffffu : 0u) | (2 * c + 9 < left ? 0xffff0000u : 0u);
            }
            const uint32_t na = scale_shift(sa), nb = scale_shift(sb);
            const uint32_t va[4] = {wa.x, wa.y, wa.z, wa.w}, vb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {   // channels 16g + 4w .. + 3: tiles 2w and 2w + 1
              const uint32_t a0 = dequant<0>(va[w], sa, na), a1 = dequant<1>(va[w], sa, na);
              const uint32_t a2 = dequant<0>(vb[w], sb, nb), a3 = dequant<1>(vb[w], sb, nb);
              const uint32_t e0 = dequant<2>(va[w], sa, na), e1 = dequant<3>(va[w], sa, na);
              const uint32_t e2 = dequant<2>(vb[w], sb, nb), e3 = dequant<3>(vb[w], sb, nb);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16_16816(o[2 * w][nt], a0, a1, a2, a3, pb[i][nt][0], pb[i][nt][1]);
                mma_f16_16816(o[2 * w + 1][nt], e0, e1, e2, e3, pb[i][nt][0], pb[i][nt][1]);
              }
            }
          }
        }
      }
      __syncwarp();   // every lane has read the stage
      if (fill < fill_end) issue(stage);
      stage = stage + 1 == C::STAGES ? 0 : stage + 1;
      ++u;

      const bool item_end = cur.j + 1 == cur.it.ntile;
      if (item_end || u == u1) {
        const bool whole = item_end && seg_first == item0;
        const int grp = p.by_nkv.of(cur.sub), r0 = grp * QT, G0 = (cur.sub - grp * p.nkv) * G;
        // the first slot of a warp: a segment that began before the run or fills it
        const int slot = 2 * warp + (seg_first == u0 ? 0 : 1);
        float* part = u == u1 ? reinterpret_cast<float*>(ring) : p.part + ((size_t)cta * C::WARPS + warp) * C::SLOT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float sum = col_sum(l[nt][x]);
            const int q = nt * 8 + 2 * c + x, r = r0 + q, j = p.by_g.of(r);
            const float m = PASS != kAttnPrefix ? 0.f : partial_max(negm[nt][x], qscale[nt][x]);
            Finish f{1.f, 0.f};
            if (whole) f = finish<END>(p, false, 0, m, sum);
#pragma unroll
            for (int t = 0; t < 8; t += 2) {
              const float v[4] = {o[t][nt][x], o[t][nt][2 + x], o[t + 1][nt][x], o[t + 1][nt][2 + x]};
              if (!whole)
                *reinterpret_cast<float4*>(part + q * 128 + 16 * g + 2 * t) = make_float4(v[0], v[1], v[2], v[3]);
              else if (j < cur.it.rows)
                finish4<END>(p, cur.it.row0 + j, G0 + r - j * G, 16 * g + 2 * t, v, f, m, sum);
            }
            if (!whole && g == 0) {
              part[QT * 128 + q] = partial_max(negm[nt][x], qscale[nt][x]);
              part[QT * 129 + q] = sum;
            }
          }
        if (!whole && lane == 0) {
          slot_item[slot] = item0;
          slot_info[slot] = cur.it;
          slot_sub[slot] = cur.sub;
          slot_at[slot] = part;
        }
        fresh = true;
      }
      if (u < u1) cursor_next<QA_TILE, QT>(p, cur);
    }
  }
  __syncthreads();   // partials of the CTA's warps are written (and visible to its threads)

  // Slots that belong to one item lie side by side; the items go to the warps in
  // turn.  An item inside the CTA's range ends here; one that reaches past a
  // border leaves one partial of the CTA and the last CTA to arrive finishes it.
  float* cta_part = p.part + (size_t)gridDim.x * C::WARPS * C::SLOT;
  {
    const int held = lane < 2 * C::WARPS ? slot_item[lane] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, held);
    uint32_t heads = __ballot_sync(0xffffffffu, held >= 0 && lane == __ffs(same) - 1);
#pragma unroll 1
    for (int run = 0; heads; heads &= heads - 1, ++run) {
      const int first = __ffs(heads) - 1;
      const uint32_t mask = __shfl_sync(0xffffffffu, same, first);
      if (run % C::WARPS != warp) continue;
      const int item0 = slot_item[first];
      const Item it = slot_info[first];
      const bool inside = item0 >= c0 && item0 + it.ntile <= c1;
      const int border = item0 < c0 ? 0 : 1;
      merge_slots<NT, PASS>(p, mask, slot_at, cta_part + ((size_t)cta * 2 + border) * C::SLOT, it, slot_sub[first], inside, lane);
      if (!inside) {
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          // CTAs that hold part of the item: counted at the one holding its first tile
          const int from = runs.of(unit_of(it, item0));
          const int to = runs.of(unit_of(it, item0) + it.ntile - 1);
          if (atomicAdd(&p.counters[from], 1) == to - from) {
            p.counters[from] = 0;   // for the next call
            __threadfence();
            last_run[border] = first;
          }
        }
      }
    }
  }
  __syncthreads();
  for (int border = 0; border < 2; ++border) {
    const int first = last_run[border];
    if (first < 0) continue;
    __threadfence();
    const int item0 = slot_item[first], sub = slot_sub[first];
    const Item it = slot_info[first];
    const int from = runs.of(unit_of(it, item0)), to = runs.of(unit_of(it, item0) + it.ntile - 1);
    // the first CTA holds the item's start, at its right border; the others have it at their left one
#pragma unroll 1
    for (int q = warp; q < QT; q += C::WARPS) {
      const int grp = p.by_nkv.of(sub), r = grp * QT + q, j = p.by_g.of(r);
      if (j >= it.rows) continue;
      float v[4], m, l;
      merge_query(to - from + 1, [&](int k) { return cta_part + ((size_t)(from + k) * 2 + (k == 0 ? 1 : 0)) * C::SLOT; }, QT,
                  q, lane, v, &m, &l);
      const int head = (sub - grp * p.nkv) * G + r - j * G;
      const Finish f = finish<END>(p, false, 0, m, l);
      finish4<END>(p, it.row0 + j, head, 4 * lane, v, f, m, l);
    }
  }
  zero_rows<PASS>(p, threadIdx.x, C::THREADS);
}

// 8 or 16 query columns.  8 query rows, us with 8 columns / 16: 1 request of
// 32,768 rows 22 / 26, 16 of 16,384 81 / 114, 256 of 1,024 83 / 121.
int q4_attn_columns(int max_rows, int nq, int nkv) { return (long long)max_rows * (nq / nkv) <= 8 ? 8 : 16; }

size_t q4_attn_part_floats(int max_rows, int nq, int nkv, int num_sms) {
  return (size_t)num_sms * (q4_attn_columns(max_rows, nq, nkv) == 8 ? (QaCfg<1>::WARPS + 2) * QaCfg<1>::SLOT : (QaCfg<2>::WARPS + 2) * QaCfg<2>::SLOT);
}

template <int NT, int PASS>
static cudaError_t launch(Q4AttnParams p, int num_sms, cudaStream_t st) {
  size_t smem = QaCfg<NT>::RING + QaCfg<NT>::WARPS * QaCfg<NT>::STAGES * 8 + ((size_t)p.n + 1) * sizeof(int);
  // (beside the ring there is room for the units of about a thousand requests, which have items enough for
  // even runs without)
  p.weigh = PASS != kAttnAll && smem + (size_t)p.n * sizeof(int) <= QA_SMEM;
  if (p.weigh) smem += (size_t)p.n * sizeof(int);
  DFL_TRY(cudaFuncSetAttribute(q4_attn_kernel<NT, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return launch_pdl(q4_attn_kernel<NT, PASS>, dim3(num_sms), dim3(QaCfg<NT>::THREADS), smem, st, p);
}

template <int PASS>
static cudaError_t launch_pass(const Q4AttnParams& p, int num_sms, cudaStream_t st) {
  return q4_attn_columns(p.max_rows, p.nq, p.nkv) == 8 ? launch<1, PASS>(p, num_sms, st) : launch<2, PASS>(p, num_sms, st);
}

cudaError_t q4_attn_launch(const Q4AttnParams& p, int pass, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  return pass == kAttnAll      ? launch_pass<kAttnAll>(p, num_sms, st)
         : pass == kAttnPrefix ? launch_pass<kAttnPrefix>(p, num_sms, st)
                               : launch_pass<kAttnOwn>(p, num_sms, st);
}

}  // namespace dfl
