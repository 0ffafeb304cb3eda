// Rotary positions:  (a, b) -> f (a cos t - b sin t, b cos t + a sin t),
// t = position * frequency_i, for the pairs (i, i + r / 2) ("half") or
// (2 i, 2 i + 1) ("interleaved") of the first r channels of every head; the
// other channels pass.
//
// The angle is formed in turns and in 64 bits, where a position of 2^22 leaves
// 2^-31 of a turn; its fraction then goes to 32 bits.  (In 32 bits throughout,
// position 2^20 is off by 0.06 rad at the first frequency.)
//
// A stream: every element is read and written once, the rotation is 6
// operations a pair, and the angles, shared by all heads of a row, are made once
// a row into shared memory while the first elements are on their way.  65,521 rows
// of 40 heads in bf16 are 1.34 GB in and out, 204 us at the rate of a copy; they
// take 206.  256 rows take a launch.
#include "decode.cuh"

namespace dfl {

constexpr int RP_THREADS = 128;
constexpr int RP_FLY = 4;          // units whose loads are on their way together

template <int TYPE, int V, bool ALIGNED>
struct RopeUnit {
  using T = typename std::conditional<TYPE == kElemF32, float, uint16_t>::type;
  static constexpr int BYTES = V * sizeof(T);
  T v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (ALIGNED && BYTES == 16) {
      uint4 w;   // (not through the non-coherent path: out may be x)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
      memcpy(v, &w, 16);
    } else if constexpr (ALIGNED && BYTES == 8) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      memcpy(v, &w, 8);
    } else if constexpr (ALIGNED && BYTES == 4) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
      memcpy(v, &w, 4);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (ALIGNED && BYTES == 16) {
      uint4 w;
      memcpy(&w, v, 16);
      *reinterpret_cast<uint4*>(p) = w;
    } else if constexpr (ALIGNED && BYTES == 8) {
      uint2 w;
      memcpy(&w, v, 8);
      *reinterpret_cast<uint2*>(p) = w;
    } else if constexpr (ALIGNED && BYTES == 4) {
      uint32_t w;
      memcpy(&w, v, 4);
      *reinterpret_cast<uint32_t*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = v[i];
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (TYPE == kElemF32) return v[i];
    else if constexpr (TYPE == kElemBf16) return __uint_as_float((uint32_t)v[i] << 16);
    else return __half2float(__ushort_as_half(v[i]));
  }
  __device__ __forceinline__ void set(int i, float f) {
    if constexpr (TYPE == kElemF32) v[i] = f;
    else if constexpr (TYPE == kElemBf16) v[i] = __bfloat16_as_ushort(__float2bfloat16_rn(f));
    else v[i] = __half_as_ushort(__float2half_rn(f));
  }
};

// x / d for x below 2^31 (m = ceil(2^(31 + s) / d), s = ceil(log2 d))
struct Div31 {
  uint32_t m;
  int s, d;
  Div31() = default;
  explicit Div31(int by) : s(0), d(by) {
    while ((1ll << s) < by) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + by - 1) / by);
  }
  __device__ __forceinline__ int of(int x) const { return (int)(((unsigned long long)(uint32_t)x * m) >> (31 + s)); }
};

struct RopeShape {
  int rows_cta, units, turned;   // rows of a CTA; units of a (row, head), the first `turned` of them rotated
  Div31 by_units, by_heads;
};

template <int TYPE, int V, bool ALIGNED, bool HALF>
__global__ void __launch_bounds__(RP_THREADS) rope_kernel(const RopeParams p, const RopeShape s) {
  using U = RopeUnit<TYPE, V, ALIGNED>;
  using T = typename U::T;
  // (cosine, sine) of the rows' pairs, [rows_cta][rot / 2]; those of a unit's pairs lie
  // `turned` apart two by two (one by one where it has one), so that neighbouring
  // lanes read neighbouring addresses
  constexpr int PAIRS = HALF ? V : V / 2, TWO = PAIRS > 1 ? 2 : 1;
  extern __shared__ __align__(16) float2 cs[];
  const int row0 = blockIdx.x * s.rows_cta, rows = min(s.rows_cta, p.rows - row0);
  const int half = p.rot / 2, total = rows * p.heads * s.units;
  const T* x = static_cast<const T*>(p.x);
  T* out = static_cast<T*>(p.out);
  griddep_wait();
  griddep_launch_dependents();

  U a[RP_FLY], b[RP_FLY];
  int row[RP_FLY], head[RP_FLY], unit[RP_FLY];
  auto fetch = [&](int k, int t) {
    const int rh = s.by_units.of(t);
    unit[k] = t - rh * s.units;
    row[k] = s.by_heads.of(rh);
    head[k] = rh - row[k] * p.heads;
    const T* src = x + (row0 + row[k]) * p.x_row + head[k] * p.x_head;
    if (unit[k] < s.turned) {
      a[k].load(src + unit[k] * V);
      if (HALF) b[k].load(src + half + unit[k] * V);
    } else {
      a[k].load(src + p.rot + (unit[k] - s.turned) * V);
    }
  };
#pragma unroll
  for (int k = 0; k < RP_FLY; ++k) {
    const int t = threadIdx.x + k * RP_THREADS;
    if (t < total) fetch(k, t);
  }
  // the rows' angles
  __shared__ int owned_end;
  if (threadIdx.x == 0) owned_end = p.positions ? p.rows : min(max(__ldg(p.starts + p.n), 0), p.rows);
  for (int i = threadIdx.x; i < rows * half; i += RP_THREADS) {
    const int r = i / half, c = i - r * half;
    double pos;
    if (p.positions) {
      pos = p.wide ? (double)__ldg(static_cast<const long long*>(p.positions) + row0 + r)
                   : (double)__ldg(static_cast<const int32_t*>(p.positions) + row0 + r);
    } else {   // row r of request i: its length less the rows behind r
      int lo = 0, hi = p.n - 1;
      while (lo < hi) {   // the first request that ends behind the row
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.starts + mid + 1) > row0 + r) hi = mid; else lo = mid + 1;
      }
      pos = (double)__ldg(p.lens + lo) - __ldg(p.starts + lo + 1) + (row0 + r);
    }
    const double t = pos * __ldg(p.turns + c);
    float sn, cn;
    sincospif(2.f * (float)(t - rint(t)), &sn, &cn);
    const int u = c / PAIRS, e = c - u * PAIRS;
    cs[r * half + (e / TWO * s.turned + u) * TWO + e % TWO] = make_float2(cn * p.factor, (p.inverse ? -sn : sn) * p.factor);
  }
  __syncthreads();
  const int end = owned_end - row0;   // rows of no request are left alone
#pragma unroll 1
  for (int t0 = threadIdx.x; t0 < total; t0 += RP_FLY * RP_THREADS) {
    if (t0 != threadIdx.x)
#pragma unroll
      for (int k = 0; k < RP_FLY; ++k)
        if (t0 + k * RP_THREADS < total) fetch(k, t0 + k * RP_THREADS);
#pragma unroll
    for (int k = 0; k < RP_FLY; ++k) {
      if (t0 + k * RP_THREADS >= total || row[k] >= end) continue;
      T* dst = out + (row0 + row[k]) * p.out_row + head[k] * p.out_head;
      if (unit[k] >= s.turned) {
        a[k].store(dst + p.rot + (unit[k] - s.turned) * V);
        continue;
      }
      float2 w[PAIRS];
#pragma unroll
      for (int i = 0; i < PAIRS; i += TWO) {
        const float2* at = cs + row[k] * half + (i / TWO * s.turned + unit[k]) * TWO;
        if constexpr (TWO == 2) {
          const float4 two = *reinterpret_cast<const float4*>(at);
          w[i] = make_float2(two.x, two.y);
          w[i + 1] = make_float2(two.z, two.w);
        } else {
          w[i] = *at;
        }
      }
      if constexpr (HALF) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 c = w[i];
          const float u = a[k].get(i), v = b[k].get(i);
          a[k].set(i, u * c.x - v * c.y);
          b[k].set(i, v * c.x + u * c.y);
        }
        a[k].store(dst + unit[k] * V);
        b[k].store(dst + half + unit[k] * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float2 c = w[i / 2];
          const float u = a[k].get(i), v = a[k].get(i + 1);
          a[k].set(i, u * c.x - v * c.y);
          a[k].set(i + 1, v * c.x + u * c.y);
        }
        a[k].store(dst + unit[k] * V);
      }
    }
  }
}

template <int TYPE, int V, bool ALIGNED>
static cudaError_t launch(const RopeParams& p, int num_sms, cudaStream_t st) {
  RopeShape s;
  const bool in_place = p.out == p.x && p.out_row == p.x_row && p.out_head == p.x_head;
  s.turned = p.interleaved ? p.rot / V : p.rot / 2 / V;
  s.units = s.turned + (in_place ? 0 : (p.dim - p.rot) / V);
  s.by_units = Div31(s.units);
  s.by_heads = Div31(p.heads);
  // four units a thread where there are rows enough for every SM, so that all of a
  // CTA's loads are on their way while the angles are made (eight: 4,128 rows of 48
  // heads 18.6 us in place of 15.8, 65,521 of 40 heads 215 in place of 202)
  const long long per_row = (long long)p.heads * s.units;
  long long rows = (RP_FLY * RP_THREADS + per_row - 1) / per_row, most = (p.rows + 2 * num_sms - 1) / (2 * num_sms);
  const long long room = 32768 / (p.rot * 4);
  if (rows > most) rows = most;
  if (rows > room) rows = room;
  s.rows_cta = rows < 1 ? 1 : (int)rows;
  const size_t smem = (size_t)s.rows_cta * (p.rot / 2) * sizeof(float2);
  const dim3 grid((p.rows + s.rows_cta - 1) / s.rows_cta);
  auto kernel = rope_kernel<TYPE, V, ALIGNED, true>;
  if constexpr (V > 1)
    if (p.interleaved) kernel = rope_kernel<TYPE, V, ALIGNED, false>;
  return launch_pdl(kernel, grid, dim3(RP_THREADS), smem, st, p, s);
}

template <int TYPE, int V>
static cudaError_t launch_aligned(const RopeParams& p, int num_sms, cudaStream_t st) {
  const long long bytes = V * elem_bytes(TYPE);
  const unsigned long long all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out) |
                                 (unsigned long long)((p.x_row | p.x_head | p.out_row | p.out_head) * elem_bytes(TYPE));
  return all % bytes == 0 ? launch<TYPE, V, true>(p, num_sms, st) : launch<TYPE, V, false>(p, num_sms, st);
}

cudaError_t rope_launch(const RopeParams& p, int num_sms, cudaStream_t st) {
  if (p.rows < 1) return cudaErrorInvalidValue;
  // the widest units that the rotated and the passing channels divide into
  const int turned = p.interleaved ? p.rot : p.rot / 2, rest = p.dim - p.rot;
  int v = p.type == kElemF32 ? 4 : 8;
  while (v > 1 && (turned % v || rest % v)) v /= 2;
  if (p.interleaved && v < 2) return cudaErrorInvalidValue;   // (dim and rot are even)
  switch (p.type) {
    case kElemF32:
      return v == 4 ? launch_aligned<kElemF32, 4>(p, num_sms, st)
             : v == 2 ? launch_aligned<kElemF32, 2>(p, num_sms, st) : launch_aligned<kElemF32, 1>(p, num_sms, st);
    case kElemBf16:
      return v == 8 ? launch_aligned<kElemBf16, 8>(p, num_sms, st) : v == 4 ? launch_aligned<kElemBf16, 4>(p, num_sms, st)
             : v == 2 ? launch_aligned<kElemBf16, 2>(p, num_sms, st) : launch_aligned<kElemBf16, 1>(p, num_sms, st);
    case kElemF16:
      return v == 8 ? launch_aligned<kElemF16, 8>(p, num_sms, st) : v == 4 ? launch_aligned<kElemF16, 4>(p, num_sms, st)
             : v == 2 ? launch_aligned<kElemF16, 2>(p, num_sms, st) : launch_aligned<kElemF16, 1>(p, num_sms, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace dfl
