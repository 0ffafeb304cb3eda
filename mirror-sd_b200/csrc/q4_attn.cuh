// Device code shared by the two attention kernels over the 4-bit cache
// (q4_attention.cu, q4_attention_tc.cu): which cached rows a request's queries
// see, the flat order of the work, and codes to f16.
#pragma once
#include "q4.cuh"

namespace dfl {

// ---- which cached rows a request's queries see ------------------------------
// Query row j of `rows` of a request with L cached rows ends at key
// e = causal ? L - rows + j + 1 : L and sees k < e with k < sink or
// k >= e - window (window 0: all of them).  The request as a whole touches
// tiles [0, a) (sink) and [b, c).
struct TileSpan {
  int a, b, c;   // count = a + c - b
};
template <int TILE>
__device__ __forceinline__ TileSpan tile_span(const Q4AttnParams& p, int L, int rows) {
  TileSpan t{0, 0, (L + TILE - 1) / TILE};
  if (p.window > 0) {
    const int lo = max((p.causal ? L - rows + 1 : L) - p.window, 0);
    t.a = (min(p.sink, L) + TILE - 1) / TILE;
    t.b = max(min(lo, L) / TILE, t.a);
  }
  return t;
}

struct Item {          // one (request, query group, kv head)
  int seq, L, rows, row0;   // cached rows, query rows, first packed query row
  TileSpan span;
  int ntile;           // tiles that hold keys its queries see
  int groups;          // query groups of the request; 0 where it has no rows or sees no key
};

__device__ __forceinline__ int seq_rows(const Q4AttnParams& p, int i, int* row0) {
  int a = i * p.max_rows, b = a + p.max_rows;
  if (p.starts) {
    a = __ldg(p.starts + i);
    b = __ldg(p.starts + i + 1);
  }
  // device data the host has not seen: stay inside the query array
  a = min(max(a, 0), p.T);
  b = min(max(b, a), p.T);
  *row0 = a;
  return min(b - a, p.max_rows);
}
// Whether they are the rows that the caller meant; the host has not seen starts,
// so what does not fit is cut off above and reported.
__device__ __forceinline__ bool rows_fit(const Q4AttnParams& p, int i) {
  if (!p.starts) return true;
  const int a = __ldg(p.starts + i), b = __ldg(p.starts + i + 1);
  return a >= 0 && a <= b && b <= p.T && b - a <= p.max_rows;
}
template <int TILE, int QT>
__device__ __forceinline__ Item load_item(const Q4AttnParams& p, int i) {
  Item it;
  it.seq = i;
  it.rows = seq_rows(p, i, &it.row0);
  it.L = min(max(__ldg(p.lens + i), 0), p.max_pages << p.page_shift);
  it.span = tile_span<TILE>(p, it.L, it.rows);
  it.ntile = it.span.a + it.span.c - it.span.b;
  it.groups = it.ntile > 0 ? (it.rows * p.by_g.d + QT - 1) / QT : 0;
  return it;
}
// The rows of requests without a cached row belong to no tile: zeros, from
// thread t of `threads` of every CTA, which share the requests out.
__device__ __forceinline__ void zero_rows(const Q4AttnParams& p, int t, int threads) {
#pragma unroll 1
  for (int i = blockIdx.x; i < p.n; i += gridDim.x) {
    if (__ldg(p.lens + i) > 0) continue;
    int row0;
    const int rows = seq_rows(p, i, &row0);
    uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + (size_t)row0 * p.nq * 128);
#pragma unroll 1
    for (int e = t; e < rows * p.nq * 16; e += threads) out[e] = make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ int item_tile(const Item& it, int j) {
  return j < it.span.a ? j : j - it.span.a + it.span.b;
}

// Sum of two tile counts that stays at kTilesFull once it is there.  The host
// bounds the tiles by the rows of q, which holds for ascending starts only; a
// call whose sum is full does nothing (its starts are reported, rows_fit).
constexpr int kTilesFull = INT32_MAX;
__device__ __forceinline__ int tiles_sum(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kTilesFull); }

// The tiles of all items in one row, cut into `parts` runs whose lengths differ
// by at most one.
struct Runs {
  int each, longer;   // run length, and how many runs have one more
  __device__ __forceinline__ Runs(int total, int parts) : each(total / parts), longer(total - total / parts * parts) {}
  __device__ __forceinline__ int start(int i) const { return i * each + min(i, longer); }
  __device__ __forceinline__ int of(int u) const {   // the run that holds tile u
    const int head = longer * (each + 1);
    return u < head ? u / (each + 1) : longer + (u - head) / each;
  }
};

// a place in the row of tiles
struct Cursor {
  Item it;
  int sub;    // query group * NKV + kv head
  int j;      // tile of the item
};

template <int TILE, int QT>
__device__ __forceinline__ void cursor_at(const Q4AttnParams& p, const int* base, int u, Cursor& c) {
  int lo = 0, hi = p.n - 1;
  while (lo < hi) {   // last request whose first tile is <= u
    const int mid = (lo + hi + 1) >> 1;
    if (base[mid] <= u) lo = mid; else hi = mid - 1;
  }
  c.it = load_item<TILE, QT>(p, lo);
  const int rel = u - base[lo];
  c.sub = rel / c.it.ntile;
  c.j = rel - c.sub * c.it.ntile;
}
template <int TILE, int QT>
__device__ __forceinline__ void cursor_next(const Q4AttnParams& p, Cursor& c) {
  if (++c.j < c.it.ntile) return;
  c.j = 0;
  if (++c.sub < c.it.groups * p.nkv) return;
  c.sub = 0;
  int i = c.it.seq;
#pragma unroll 1
  do {
    if (++i >= p.n) return;   // past the end: the caller's run is over
    c.it = load_item<TILE, QT>(p, i);
  } while (c.it.groups == 0);
}

// ---- fragments --------------------------------------------------------------
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Scales as dequant takes them: 4 s.  From a u16 holding two scale bytes (the f16
// bits of s are byte << 7), and what goes with it, -4.5 s.
__device__ __forceinline__ uint32_t scale_pair(uint32_t two) {
  return hmul2_u(__byte_perm(two, 0, 0x1404) >> 1, 0x44004400u);
}
__device__ __forceinline__ uint32_t scale_shift(uint32_t s4) { return hmul2_u(s4, 0xBC80BC80u); }
// Nibble n of both halves of w -> (x / 16) pair: (w >> k) & 0x00F0 | 0x3C00 is
// 1 + u / 64, and times 4 s less 4.5 s it is exactly (u - 8) s / 16.  (n = 1 needs
// no shift.  The masking is written as one three-input logic operation: with the
// constants visible the compiler makes it two, a seventh of the decode kernel's
// instructions, 383 against 339 us for 256 requests at the time.)
template <int N>
__device__ __forceinline__ uint32_t dequant(uint32_t w, uint32_t s4, uint32_t shift) {
  const uint32_t t = N == 0 ? w << 4 : N == 1 ? w : w >> (4 * N - 4);
  uint32_t h;
  asm("{\n .reg .b32 m, o;\n mov.b32 m, 0x00F000F0;\n mov.b32 o, 0x3C003C00;\n lop3.b32 %0, %1, m, o, 0xEA;\n}\n" : "=r"(h) : "r"(t));
  return hfma2_u(h, s4, shift);
}
// Scores are measured as (s - reference) * f, s as the products leave it and f
// its factor to base 2: exactly 0 for the key that set the reference, however
// large the score (s * f less a rounded reference is off by the rounding, which
// from 2^27 on hides every key).  A column that has seen no key has -kUnset for
// its reference; no s comes near (|s| < 2^36, or scores beyond fp32), and with f
// in this range, which no s tells from its ends, the difference raises it.
constexpr float kUnset = 3e38f;
__host__ __device__ __forceinline__ float score_factor(float f) { return fminf(fmaxf(f, 0x1p-100f), 3e38f); }
// the reference of a partial result in base-2 units, finite
__device__ __forceinline__ float partial_max(float negm, float f) {
  return negm == kUnset ? -INFINITY : fminf(fmaxf(-negm * f, -3e38f), 3e38f);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A warp merges one query's partials of `count` runs: slots(k) holds O at
// q * 128, m at qt * 128 + q and l at qt * 129 + q.  Returns channels 4 lane ..
// of the output row.  8 loads of O are on their way together, the first ones
// with those of m and l: few partials cost one round trip to L2.
template <class SlotAt>
__device__ __forceinline__ void merge_query(int count, SlotAt slots, int qt, int q, int lane, float (&v)[4]) {
  float4 x[8];
  auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < count) x[i] = __ldcg(reinterpret_cast<const float4*>(slots(k + i) + q * 128 + 4 * lane));
  };
  load(0);
  float m = -INFINITY, s = 0.f;
  if (lane < count) {
    m = __ldcg(slots(lane) + qt * 128 + q);
    s = __ldcg(slots(lane) + qt * 129 + q);
  }
  float M = m;
#pragma unroll 1
  for (int k = lane + 32; k < count; k += 32) M = fmaxf(M, __ldcg(slots(k) + qt * 128 + q));
  M = warp_max(M);
  float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < count; k0 += 32) {
    if (k0 > 0) {
      m = -INFINITY;
      if (k0 + lane < count) {
        m = __ldcg(slots(k0 + lane) + qt * 128 + q);
        s = __ldcg(slots(k0 + lane) + qt * 129 + q);
      }
    }
    const float w = m == -INFINITY ? 0.f : exp2_fast(m - M);
    l = fmaf(w, s, l);
    const int n = min(count - k0, 32);
#pragma unroll 1
    for (int k = 0; k < n; k += 8) {
      if (k0 + k > 0) load(k0 + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, k + i);
        if (k + i < n) {
          o[0] = fmaf(wi, x[i].x, o[0]);
          o[1] = fmaf(wi, x[i].y, o[1]);
          o[2] = fmaf(wi, x[i].z, o[2]);
          o[3] = fmaf(wi, x[i].w, o[3]);
        }
      }
    }
  }
  l = warp_sum(l);
  const float f = l == 0.f ? 0.f : 16.f / l;
  for (int i = 0; i < 4; ++i) v[i] = o[i] * f;
}

// write 4 consecutive output values of one query row
__device__ __forceinline__ void store_out4(const Q4AttnParams& p, int row, int head, int d, const float (&v)[4]) {
  const size_t off = ((size_t)row * p.nq + head) * 128 + d;
  const uint2 w = p.bf16 ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                         : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + off) = w;
}

}  // namespace dfl
