// Grouped-query attention over the paged 4-bit cache (layout: q4.cuh).
//
//   out[j, h] = sum_k softmax_k(scale * q[j, h] . K[k]) V[k],  K, V = (u - 8) s
//
// over the cached rows k that query row j of a request sees (q4_visible
// below).  R = rows * G query rows of a request share a kv head (G = NQ / NKV,
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
// Codes become f16 by bit placement: (w >> k) & 0x03C0 | 0x3C00 is 1 + u/16,
// and one f16 FMA gives x / 16 = (1 + u/16) s - 1.5 s exactly (every term has
// at most 7 significant bits).  The factors 16 go into the softmax scale and
// the final division.  S^T leaves the products with a lane holding two query
// columns of a row; packing those two and transposing 8x8 blocks (movmatrix)
// makes the P^T fragment.  P is rounded to f16 (2^-12 relative, the operand
// type), sums and statistics stay fp32.
//
// The running maximum is only raised when a score passes it by 2^8 (then O
// and the sum are rescaled), as P below 256 loses nothing in f16.
#include "q4_attn.cuh"

namespace dfl {

constexpr int QA_WARPS = 8;
constexpr int QA_THREADS = QA_WARPS * 32;
constexpr int QA_TILE = 64;                      // cached rows of a tile
constexpr int QA_STAGE = QA_TILE / kQ4Rows * kQ4Block;
constexpr int QA_STAGES = 3;
constexpr float QA_RAISE = 8.f;

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
  static constexpr int SLOT = QT * 130;   // floats of a partial: O [QT][128], m [QT], l [QT]
  static constexpr int RING = QA_WARPS * QA_STAGES * QA_STAGE;
};

// write 4 consecutive output values of one query row
__device__ __forceinline__ void store_out4(const Q4AttnParams& p, int row, int head, int d, const float (&v)[4]) {
  const size_t off = ((size_t)row * p.nq + head) * 128 + d;
  const uint2 w = p.bf16 ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                         : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + off) = w;
}

// Merge `count` partials (slot k at slots(k)) of one item and write either the
// item's output rows (out_item != nullptr) or another partial at dst.  `t` of
// `nt` threads; every thread takes whole groups of 4 channels of a query row.
template <int NT, class SlotAt>
__device__ __forceinline__ void merge_partials(const Q4AttnParams& p, int count, SlotAt slots, float* dst,
                                               const Item* out_item, int sub, int t, int nt) {
  constexpr int QT = QaCfg<NT>::QT;
  const int G = p.by_g.d;
  for (int e = t; e < QT * 32; e += nt) {
    const int q = e >> 5, d = (e & 31) * 4;
    float M = -INFINITY;
    for (int k = 0; k < count; ++k) M = fmaxf(M, __ldcg(slots(k) + QT * 128 + q));
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < count; ++k) {
      const float* s = slots(k);
      const float m = __ldcg(s + QT * 128 + q);
      const float w = m == -INFINITY ? 0.f : exp2_fast(m - M);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(s + q * 128 + d));
      l = fmaf(w, __ldcg(s + QT * 129 + q), l);
      o[0] = fmaf(w, v.x, o[0]);
      o[1] = fmaf(w, v.y, o[1]);
      o[2] = fmaf(w, v.z, o[2]);
      o[3] = fmaf(w, v.w, o[3]);
    }
    if (out_item) {
      const int grp = p.by_nkv.of(sub), r = grp * QT + q, j = p.by_g.of(r);
      if (j < out_item->rows) {
        const float f = l == 0.f ? 0.f : 16.f / l;
        for (int x = 0; x < 4; ++x) o[x] *= f;
        store_out4(p, out_item->row0 + j, (sub - grp * p.nkv) * G + r - j * G, d, o);
      }
    } else {
      *reinterpret_cast<float4*>(dst + q * 128 + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) {
        dst[QT * 128 + q] = M;
        dst[QT * 129 + q] = l;
      }
    }
  }
}

template <int NT>
__global__ void __launch_bounds__(QA_THREADS, 1) q4_attn_kernel(const Q4AttnParams p) {
  using C = QaCfg<NT>;
  constexpr int QT = C::QT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::RING);          // [warp][stage]
  int* base = reinterpret_cast<int*>(bars + QA_WARPS * QA_STAGES);       // [n + 1] first tile of each request
  __shared__ int wtot[QA_WARPS];
  __shared__ int slot_item[2 * QA_WARPS];   // unit at which the partial's item starts, or -1
  __shared__ int slot_info[2 * QA_WARPS][2];   // request, sub
  __shared__ int last_run[2];               // runs (of the CTA's two borders) this CTA must finish
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = p.by_g.d;

  if (threadIdx.x == 0) {
    for (int i = 0; i < QA_WARPS * QA_STAGES; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
    last_run[0] = last_run[1] = -1;
  }
  if (threadIdx.x < 2 * QA_WARPS) slot_item[threadIdx.x] = -1;
  // tiles of every request, added up (kPagedMaxSeqs / QA_THREADS passes at most)
  int total = 0;
  for (int i0 = 0; i0 < p.n; i0 += QA_THREADS) {
    const int i = i0 + threadIdx.x;
    int v = 0;
    if (i < p.n) {
      const Item it = load_item<QA_TILE, QT>(p, i);
      v = it.ntile * it.groups * p.nkv;
    }
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) wtot[warp] = x;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < QA_WARPS; ++w) {
      if (w < warp) before += wtot[w];
      total += wtot[w];
    }
    if (i < p.n) base[i] = before + x - v;
  }
  if (threadIdx.x == 0) base[p.n] = total;
  __syncthreads();

  const int ctas = min((int)gridDim.x, total);   // CTAs with work
  const int cta = blockIdx.x;
  if (cta >= ctas) return;
  const Runs runs(total, ctas);
  const int c0 = runs.start(cta), c1 = runs.start(cta + 1);
  const Runs mine(c1 - c0, QA_WARPS);
  const int u0 = c0 + mine.start(warp), u1 = c0 + mine.start(warp + 1);

  if (u0 < u1) {
    uint8_t* ring = smem + warp * QA_STAGES * QA_STAGE;
    uint64_t* bar = bars + warp * QA_STAGES;
    Cursor cur, ahead;
    cursor_at<QA_TILE, QT>(p, base, u0, cur);
    ahead = cur;
    // lane b < 4 looks after row block b of a tile: its page, then its copy
    auto page_of = [&](const Cursor& k) {
      const int pos = item_tile(k.it, k.j) * QA_TILE + (lane & 3) * kQ4Rows;
      int pg = -1;
      if (lane < 4 && pos < k.it.L) {
        pg = __ldg(p.table + (size_t)k.it.seq * p.table_ld + (pos >> p.page_shift));
        if (pg < 0 || pg >= p.num_pages) pg = -1;   // hidden, like a masked block
      }
      return pg;
    };
    int next_page = page_of(ahead);
    uint32_t loaded = 0;   // 4 bits a stage: row blocks that were copied
    int fill = u0, fill_end = u1;   // tiles requested so far; fewer than the run after an expired wait
    auto issue = [&](int s) {
      const uint32_t mask = __ballot_sync(0xffffffffu, next_page >= 0);
      if (lane == 0) mbar_arrive_expect_tx(&bar[s], __popc(mask) * kQ4Block);
      __syncwarp();
      if (next_page >= 0) {
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
    for (int s = 0; s < QA_STAGES && fill < fill_end; ++s) issue(s);

    uint32_t qf[NT][16];
    float qscale[NT][2], m[NT][2], l[NT][2], o[8][NT][4];
    int key_end[NT][2];
    int u = u0, stage = 0;
    uint32_t phase = 0;
    bool fresh = true, alive = true;
    int seg_first = u0;   // first unit of the running segment
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
          f *= 16.f * p.scale_log2;
          // the lane's score columns are queries 2c and 2c + 1 of this group of 8
          qscale[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
          qscale[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int jj = p.by_g.of(r0 + nt * 8 + 2 * c + x);
            key_end[nt][x] = jj < cur.it.rows ? (p.causal ? cur.it.L - cur.it.rows + jj + 1 : cur.it.L) : 0;
            m[nt][x] = -INFINITY;
            l[nt][x] = 0.f;
          }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[t][nt][x] = 0.f;
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
        float sc[4][NT][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[b][nt][x] = 0.f;
          if (!(have >> b & 1)) continue;
          const uint8_t* blk = tile + b * kQ4Block;
          const uint4 wa = *reinterpret_cast<const uint4*>(blk + q4_k_piece(g, c));
          const uint4 wb = *reinterpret_cast<const uint4*>(blk + 512 + q4_k_piece(g, c));
          const uint32_t s2a = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4KS + g * 8 + 2 * c));
          const uint32_t s2b = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4KS + 64 + g * 8 + 2 * c));
          const uint32_t ka[4] = {wa.x, wa.y, wa.z, wa.w}, kb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {   // channels 32c + 8w .. + 7: group 2c + w / 2
            const uint32_t sa = __byte_perm(s2a, 0, w < 2 ? 0x1010 : 0x3232);
            const uint32_t sb = __byte_perm(s2b, 0, w < 2 ? 0x1010 : 0x3232);
            const uint32_t na = hmul2_u(sa, 0xBE00BE00u), nb = hmul2_u(sb, 0xBE00BE00u);   // -1.5 s
            const uint32_t a0 = dequant<0>(ka[w], sa, na), a2 = dequant<1>(ka[w], sa, na);
            const uint32_t a1 = dequant<0>(kb[w], sb, nb), a3 = dequant<1>(kb[w], sb, nb);
            const uint32_t e0 = dequant<2>(ka[w], sa, na), e2 = dequant<3>(ka[w], sa, na);
            const uint32_t e1 = dequant<2>(kb[w], sb, nb), e3 = dequant<3>(kb[w], sb, nb);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16_16816(sc[b][nt], a0, a1, a2, a3, qf[nt][4 * w], qf[nt][4 * w + 1]);
              mma_f16_16816(sc[b][nt], e0, e1, e2, e3, qf[nt][4 * w + 2], qf[nt][4 * w + 3]);
            }
          }
        }
        // base-2 scores; hidden keys get -inf
        const bool all_seen = have == 15u && row0 + QA_TILE <= (p.causal ? cur.it.L - cur.it.rows + 1 : cur.it.L) &&
                              (p.window == 0 || row0 + QA_TILE <= p.sink || row0 >= cur.it.L - p.window);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float y = sc[b][nt][x] * qscale[nt][x & 1];
              if (!all_seen) {
                const int key = row0 + 16 * b + g + 8 * (x >> 1), end = key_end[nt][x & 1];
                const bool seen = (have >> b & 1) && key < end &&
                                  (p.window == 0 || key < p.sink || key >= end - p.window);
                if (!seen) y = -INFINITY;
              }
              sc[b][nt][x] = y;
              top[x & 1] = fmaxf(top[x & 1], y);
            }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            top[x] = col_max(top[x]);
            if (top[x] > m[nt][x] + QA_RAISE) {   // also the first visible key (m = -inf)
              const float f = exp2_fast(m[nt][x] - top[x]);
              m[nt][x] = top[x];
              l[nt][x] *= f;
#pragma unroll
              for (int t = 0; t < 8; ++t) {
                o[t][nt][x] *= f;
                o[t][nt][2 + x] *= f;
              }
            }
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (!(have >> b & 1)) continue;
          uint32_t pb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            // a column without a visible key so far: every score is -inf, P = 0
            const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
            const float p0 = exp2_fast(sc[b][nt][0] - m0), p1 = exp2_fast(sc[b][nt][1] - m1);
            const float p2 = exp2_fast(sc[b][nt][2] - m0), p3 = exp2_fast(sc[b][nt][3] - m1);
            l[nt][0] += p0 + p2;
            l[nt][1] += p1 + p3;
            pb[nt][0] = transpose8x8(pack_f16x2(p0, p1));
            pb[nt][1] = transpose8x8(pack_f16x2(p2, p3));
          }
          const uint8_t* blk = tile + b * kQ4Block;
          const uint4 wa = *reinterpret_cast<const uint4*>(blk + kQ4V + q4_v_piece(c, g));
          const uint4 wb = *reinterpret_cast<const uint4*>(blk + kQ4V + q4_v_piece(c + 4, g));
          uint32_t sa = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4VS + g * 16 + 2 * c));
          uint32_t sb = scale_pair(*reinterpret_cast<const uint16_t*>(blk + kQ4VS + g * 16 + 8 + 2 * c));
          if (row0 + 16 * b + 16 > cur.it.L) {
            // rows past the end may never have been written: their scale could be any bits
            const int left = cur.it.L - (row0 + 16 * b);
            sa &= (2 * c < left ? 0xffffu : 0u) | (2 * c + 1 < left ? 0xffff0000u : 0u);
            sb &= (2 * c + 8 < left ? 0xffffu : 0u) | (2 * c + 9 < left ? 0xffff0000u : 0u);
          }
          const uint32_t na = hmul2_u(sa, 0xBE00BE00u), nb = hmul2_u(sb, 0xBE00BE00u);
          const uint32_t va[4] = {wa.x, wa.y, wa.z, wa.w}, vb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {   // channels 16g + 4w .. + 3: tiles 2w and 2w + 1
            const uint32_t a0 = dequant<0>(va[w], sa, na), a1 = dequant<1>(va[w], sa, na);
            const uint32_t a2 = dequant<0>(vb[w], sb, nb), a3 = dequant<1>(vb[w], sb, nb);
            const uint32_t e0 = dequant<2>(va[w], sa, na), e1 = dequant<3>(va[w], sa, na);
            const uint32_t e2 = dequant<2>(vb[w], sb, nb), e3 = dequant<3>(vb[w], sb, nb);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16_16816(o[2 * w][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
              mma_f16_16816(o[2 * w + 1][nt], e0, e1, e2, e3, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
      __syncwarp();   // every lane has read the stage
      if (fill < fill_end) issue(stage);
      stage = stage + 1 == QA_STAGES ? 0 : stage + 1;
      ++u;

      const bool item_end = cur.j + 1 == cur.it.ntile;
      if (item_end || u == u1) {
        const bool whole = item_end && seg_first == item0;
        const int grp = p.by_nkv.of(cur.sub), r0 = grp * QT, G0 = (cur.sub - grp * p.nkv) * G;
        // the first slot of a warp: a segment that began before the run or fills it
        const int slot = 2 * warp + (seg_first == u0 ? 0 : 1);
        float* part = p.part + ((size_t)cta * 2 * QA_WARPS + slot) * C::SLOT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float sum = col_sum(l[nt][x]);
            const int q = nt * 8 + 2 * c + x, r = r0 + q, j = p.by_g.of(r);
            const float f = whole ? (sum == 0.f ? 0.f : 16.f / sum) : 1.f;
#pragma unroll
            for (int t = 0; t < 8; t += 2) {
              const float v[4] = {o[t][nt][x] * f, o[t][nt][2 + x] * f, o[t + 1][nt][x] * f, o[t + 1][nt][2 + x] * f};
              if (!whole)
                *reinterpret_cast<float4*>(part + q * 128 + 16 * g + 2 * t) = make_float4(v[0], v[1], v[2], v[3]);
              else if (j < cur.it.rows)
                store_out4(p, cur.it.row0 + j, G0 + r - j * G, 16 * g + 2 * t, v);
            }
            if (!whole && g == 0) {
              part[QT * 128 + q] = m[nt][x];
              part[QT * 129 + q] = sum;
            }
          }
        if (!whole && lane == 0) {
          slot_item[slot] = item0;
          slot_info[slot][0] = cur.it.seq;
          slot_info[slot][1] = cur.sub;
        }
        fresh = true;
      }
      if (u < u1) cursor_next<QA_TILE, QT>(p, cur);
    }
  }
  __syncthreads();   // partials of the CTA's warps are written (and visible to its threads)

  // Runs of slots that belong to one item, in order; run k goes to warp k % 8.
  // An item inside the CTA's range ends here; one that reaches past a border
  // leaves one partial of the CTA and the last CTA to arrive finishes it.
  float* cta_part = p.part + (size_t)gridDim.x * 2 * QA_WARPS * C::SLOT;
  {
    int run = 0, k = 0;
    while (k < 2 * QA_WARPS) {
      if (slot_item[k] < 0) { ++k; continue; }
      const int item0 = slot_item[k], first = k;
      int last = k;
      for (++k; k < 2 * QA_WARPS; ++k) {
        if (slot_item[k] < 0) continue;
        if (slot_item[k] != item0) break;
        last = k;
      }
      if (run++ % QA_WARPS != warp) continue;
      const Item it = load_item<QA_TILE, QT>(p, slot_info[first][0]);
      const int sub = slot_info[first][1];
      int list[2 * QA_WARPS], count = 0;
      for (int x = first; x <= last; ++x)
        if (slot_item[x] >= 0) list[count++] = x;
      const float* parts = p.part + (size_t)cta * 2 * QA_WARPS * C::SLOT;
      const bool inside = item0 >= c0 && item0 + it.ntile <= c1;
      const int border = item0 < c0 ? 0 : 1;
      float* dst = cta_part + ((size_t)cta * 2 + border) * C::SLOT;
      merge_partials<NT>(p, count, [&](int x) { return parts + (size_t)list[x] * C::SLOT; }, dst,
                         inside ? &it : nullptr, sub, lane, 32);
      if (!inside) {
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          // CTAs that hold part of the item: counted at the one holding its first tile
          const int from = runs.of(item0);
          const int to = runs.of(item0 + it.ntile - 1);
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
    const int item0 = slot_item[first], sub = slot_info[first][1];
    const Item it = load_item<QA_TILE, QT>(p, slot_info[first][0]);
    const int from = runs.of(item0);
    const int to = runs.of(item0 + it.ntile - 1);
    // the first CTA holds the item's start, so its part is at its right border
    // unless the item also began before that CTA's range, which it did not
    merge_partials<NT>(p, to - from + 1,
                       [&](int x) { return cta_part + ((size_t)(from + x) * 2 + (x == 0 ? 1 : 0)) * C::SLOT; },
                       nullptr, &it, sub, threadIdx.x, QA_THREADS);
  }
}

static int q4_attn_nt(int max_rows, int nq, int nkv) { return (long long)max_rows * (nq / nkv) <= 8 ? 1 : 2; }

size_t q4_attn_part_floats(int max_rows, int nq, int nkv, int num_sms) {
  const int nt = q4_attn_nt(max_rows, nq, nkv);
  return (size_t)num_sms * (2 * QA_WARPS + 2) * (nt == 1 ? QaCfg<1>::SLOT : QaCfg<2>::SLOT);
}

template <int NT>
static cudaError_t launch(const Q4AttnParams& p, int num_sms, cudaStream_t st) {
  const size_t smem = QaCfg<NT>::RING + QA_WARPS * QA_STAGES * 8 + ((size_t)p.n + 1) * 4;
  DFL_TRY(cudaFuncSetAttribute(q4_attn_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  q4_attn_kernel<NT><<<num_sms, QA_THREADS, smem, st>>>(p);
  return cudaGetLastError();
}

cudaError_t q4_attn_launch(const Q4AttnParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  return q4_attn_nt(p.max_rows, p.nq, p.nkv) == 1 ? launch<1>(p, num_sms, st) : launch<2>(p, num_sms, st);
}

}  // namespace dfl
