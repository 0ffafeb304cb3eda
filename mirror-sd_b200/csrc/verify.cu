// Verification of drafted tokens by sampling.  With p_j the softmax of logits
// row j over the temperature, u the request's uniform numbers and q_j what the
// draft was sampled from (1 at the draft itself where it was not sampled):
//
//   draft d_j is accepted while u_j q_j(d_j) < p_j(d_j);
//   the token behind the accepted ones is sampled from r = max(p_a - q_a, 0) at
//   the first refused place a, from r = p_a behind the last draft: the first
//   token in vocabulary order whose running sum of r passes u_last sum(r).
//
// A cluster of CTAs owns a request and cuts the vocabulary into slices; rows
// behind the first refused draft are never read.  One pass over a row gives the
// softmax's maximum and sum: 2^((x - m) c) in 32 bits, c = log2(e) / T, against a
// reference m of each thread that moves when a logit passes it by 2^8 (so the
// exponents that matter are small and exact to 2^-24 of themselves), summed over
// threads in 64 bits.  The row that the token comes from is read once more, in
// 64 bits throughout: u times the sum must fall between the same two of up to
// 150,000 running sums, whatever order they are added up in, and sums in 32 bits are
// off by more than an unlikely token weighs.
//
// Logits: NaN counts as -inf, a weight of 0; what lies beyond +-1e30 counts as
// that.  A row that leaves no token refuses its draft and gives token -1.
#include "decode.cuh"

namespace dfl {

constexpr int VF_THREADS = 512, VF_WARPS = VF_THREADS / 32;
constexpr int VF_ROWS = 16;              // rows between two exchanges at most
constexpr int VF_CLUSTER = 16;           // CTAs of a request at most
constexpr float VF_BIG = 1e30f;
constexpr float VF_RAISE = 8.f;

template <int TYPE>
struct Logits {
  static constexpr int E = TYPE == kElemF32 ? 4 : 8;   // entries of 16 bytes
  const char* base;     // the 16-byte piece that the row starts in
  int skip, vocab;      // entries of that piece before the row
  int pieces;
  __device__ __forceinline__ Logits(const void* row, int V) : vocab(V) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    skip = (int)(at & 15) / (16 / E);
    base = reinterpret_cast<const char*>(at & ~(uintptr_t)15);
    pieces = (V + skip + E - 1) / E;
  }
  __device__ __forceinline__ bool whole(int piece) const { return (piece > 0 || skip == 0) && (piece + 1) * E - skip <= vocab; }
  __device__ __forceinline__ uint4 load(int piece) const { return __ldg(reinterpret_cast<const uint4*>(base) + piece); }
  static __device__ __forceinline__ float bits(uint32_t u, int hi) {   // entry of a 16-bit pair
    if (TYPE == kElemBf16) return __uint_as_float(hi ? u & 0xffff0000u : u << 16);
    return __half2float(__ushort_as_half((unsigned short)(hi ? u >> 16 : u)));
  }
  static __device__ __forceinline__ void split(const uint4& w, float (&x)[E]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kElemF32) {
        x[i] = __uint_as_float(u[i]);
      } else {
        x[2 * i] = bits(u[i], 0);
        x[2 * i + 1] = bits(u[i], 1);
      }
    }
  }
  __device__ __forceinline__ float at(int i) const {   // entry i of the row
    const char* p = base + (long long)(i + skip) * (16 / E);
    if (TYPE == kElemF32) return __ldg(reinterpret_cast<const float*>(p));
    return bits(__ldg(reinterpret_cast<const unsigned short*>(p)), 0);
  }
  // the entries of a piece, those outside the row as -inf
  __device__ __forceinline__ void get(int piece, float (&x)[E]) const {
    if (whole(piece)) {
      split(load(piece), x);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int k = piece * E - skip + i;
        x[i] = k >= 0 && k < vocab ? at(k) : -INFINITY;
      }
    }
  }
};

// a logit as the definition takes it: NaN is -inf, and finite ones (and +inf) lie within +-1e30
__device__ __forceinline__ float clean(float x) {
  if (!(x > -INFINITY)) return -INFINITY;
  return fminf(fmaxf(x, -VF_BIG), VF_BIG);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct RowStat {   // over a part of a row: reference and sum, or the largest entry and its place
  float m;
  int at;
  double sum;
};

// Sum of 2^((x - m) c) over the pieces lo + t, lo + t + threads, ... < hi.
template <int TYPE, bool CAREFUL>
__device__ __forceinline__ void row_sum(const Logits<TYPE>& row, int lo, int hi, float c, float& m, float& s) {
  constexpr int E = Logits<TYPE>::E, FLY = 4;
  m = CAREFUL ? -2 * VF_BIG : -VF_BIG;
  s = 0.f;
  float lim = m;   // (the first logit above raises it)
  auto take = [&](float (&x)[E]) {
    if (CAREFUL) {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = clean(x[i]);
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
    if (top > lim) {
      s *= ex2((m - top) * c);
      m = top;
      lim = top + VF_RAISE / c;
    }
    float y[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      y[i] = ex2((x[i] - m) * c);
      if (CAREFUL && x[i] == -INFINITY) y[i] = 0.f;
    }
#pragma unroll
    for (int k = E / 2; k > 0; k /= 2)
#pragma unroll
      for (int i = 0; i < k; ++i) y[i] += y[i + k];
    s += y[0];
  };
  int i = lo + threadIdx.x;
#pragma unroll 1
  for (; i + (FLY - 1) * VF_THREADS < hi; i += FLY * VF_THREADS) {
    uint4 w[FLY];
    bool whole = true;
#pragma unroll
    for (int k = 0; k < FLY; ++k) whole = whole && row.whole(i + k * VF_THREADS);
    if (whole) {
#pragma unroll
      for (int k = 0; k < FLY; ++k) w[k] = row.load(i + k * VF_THREADS);
#pragma unroll
      for (int k = 0; k < FLY; ++k) {
        float x[E];
        Logits<TYPE>::split(w[k], x);
        take(x);
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < FLY; ++k) {
        float x[E];
        row.get(i + k * VF_THREADS, x);
        take(x);
      }
    }
  }
#pragma unroll 1
  for (; i < hi; i += VF_THREADS) {
    float x[E];
    row.get(i, x);
    take(x);
  }
}

// Largest entry (NaN aside) and its first place.
template <int TYPE>
__device__ __forceinline__ void row_top(const Logits<TYPE>& row, int lo, int hi, float& m, int& at) {
  constexpr int E = Logits<TYPE>::E;
  m = -INFINITY;
  at = INT32_MAX;
#pragma unroll 4
  for (int i = lo + threadIdx.x; i < hi; i += VF_THREADS) {
    float x[E];
    row.get(i, x);
    float top = x[0];
#pragma unroll
    for (int k = 1; k < E; ++k) top = fmaxf(top, x[k]);
    if (top > m) {
      m = top;
#pragma unroll
      for (int k = E - 1; k >= 0; --k)
        if (x[k] == top) at = i * E - row.skip + k;
    }
  }
}

struct Weights {   // of the row that the token comes from
  double c, m;           // 2^((x - m) c)
  const float* q;        // subtract total * q, or NULL
  double total;
  int drop;              // entry without weight, or -1
};
__device__ __forceinline__ double weight(const Weights& w, float x, int i) {
  x = clean(x);
  if (x == -INFINITY || i == w.drop) return 0.0;
  double y = exp2(((double)x - w.m) * w.c);
  if (w.q) {
    const float q = __ldg(w.q + i);
    y = q > 0.f ? fmax(y - (double)q * w.total, 0.0) : y;
  }
  return y;
}

// Sum of the weights of the pieces [lo, hi), by a warp.
template <int TYPE>
__device__ __forceinline__ double warp_run_sum(const Logits<TYPE>& row, const Weights& w, int lo, int hi) {
  constexpr int E = Logits<TYPE>::E;
  const int lane = threadIdx.x & 31;
  double s = 0.0;
#pragma unroll 2
  for (int i = lo + lane; i < hi; i += 32) {
    float x[E];
    row.get(i, x);
#pragma unroll
    for (int k = 0; k < E; ++k) s += weight(w, x[k], i * E - row.skip + k);
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

__device__ __forceinline__ int cut(int lo, int hi, int i, int parts) { return lo + (int)((long long)(hi - lo) * i / parts); }

// A warp's entries y, E consecutive ones a lane, added up in order from `base`:
// the first entry that weighs anything and whose running sum passes x.  Returns
// its index (lane * E + e), -1 if there is none, with `heavy` the last entry that
// weighs anything (or -1); *before: what lies before the one that is found (or
// before heavy), *total: base and all entries.
template <int E>
__device__ __forceinline__ int warp_find(const double (&y)[E], double x, double base, int* heavy, double* before,
                                         double* total) {
  const int lane = threadIdx.x & 31;
  double mine = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += y[e];
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const double v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  double run = __shfl_up_sync(0xffffffffu, upto, 1), first = 0.0, last = 0.0;
  run = base + (lane == 0 ? 0.0 : run);
  int found = -1, some = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (y[e] > 0.0) {
      some = e;
      last = run;
      if (found < 0 && run + y[e] > x) {
        found = e;
        first = run;
      }
    }
    run += y[e];
  }
  const uint32_t pass = __ballot_sync(0xffffffffu, found >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
  *total = base + __shfl_sync(0xffffffffu, upto, 31);
  const int l = any ? 31 - __clz(any) : 0;
  *heavy = any ? l * E + __shfl_sync(0xffffffffu, some, l) : -1;
  if (!pass) {
    *before = __shfl_sync(0xffffffffu, last, l);
    return -1;
  }
  const int f = __ffs(pass) - 1;
  *before = __shfl_sync(0xffffffffu, first, f);
  return f * E + __shfl_sync(0xffffffffu, found, f);
}

__device__ __forceinline__ double ld_cluster_f64(const double* local, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_s32(const int* local, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(local, rank)) : "memory");
  return v;
}

template <int TYPE>
__global__ void __launch_bounds__(VF_THREADS) verify_kernel(const VerifyParams p, int ctas, int window) {
  __shared__ RowStat warp_stat[VF_ROWS][VF_WARPS];
  __shared__ RowStat cta_stat[2][VF_ROWS];
  __shared__ double run_sum[2][VF_WARPS];
  __shared__ int verdict[VF_ROWS];       // 1 accepted, 0 refused, 2 to be read once more with care
  __shared__ RowStat row_stat[VF_ROWS];  // of the whole rows
  __shared__ struct { double total, x; int run; } place;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x / ctas, rank = blockIdx.x - seq * ctas;
  griddep_wait();
  griddep_launch_dependents();
  const int count = p.counts ? min(max(__ldg(p.counts + seq), 0), p.block - 1) : p.block - 1;
  const float temp = p.temps ? __ldg(p.temps + seq) : p.temp;
  const bool greedy = !(temp >= 1e-5f);
  const float c = greedy ? 0.f : (float)(1.4426950408889634 / (double)temp);
  const int32_t* drafts = p.drafts + (size_t)seq * (p.block - 1);
  const float* u = p.uniforms + (size_t)seq * p.block;
  auto row_of = [&](int j) {
    return Logits<TYPE>(static_cast<const char*>(p.logits) + (seq * p.l_seq + j * p.l_row) * (16 / Logits<TYPE>::E), p.vocab);
  };

  // ---- the first refused draft
  int stop = -1, at = 0, buf = 0;
  bool careful = false;
  RowStat st{};
#pragma unroll 1
  while (stop < 0) {
    const int rows = careful ? 1 : min(window, count + 1 - at);
#pragma unroll 1
    for (int w = 0; w < rows; ++w) {
      const Logits<TYPE> row = row_of(at + w);
      const int lo = cut(0, row.pieces, rank, ctas), hi = cut(0, row.pieces, rank + 1, ctas);
      float m, s = 0.f;
      int idx = 0;
      if (greedy) row_top(row, lo, hi, m, idx);
      else if (careful) row_sum<TYPE, true>(row, lo, hi, c, m, s);
      else row_sum<TYPE, false>(row, lo, hi, c, m, s);
      double sum = s;
#pragma unroll
      for (int o = 16; o > 0; o /= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        if (greedy) {
          const int oi = __shfl_xor_sync(0xffffffffu, idx, o);
          if (om > m || (om == m && oi < idx)) idx = oi;
          m = fmaxf(m, om);
        } else {
          const double os = __shfl_xor_sync(0xffffffffu, sum, o);
          const float M = fmaxf(m, om);
          sum = sum * ex2((m - M) * c) + os * ex2((om - M) * c);
          m = M;
        }
      }
      if (lane == 0) warp_stat[w][warp] = {m, idx, sum};
    }
    __syncthreads();
    // one warp a row: the CTA's warps, then the cluster's CTAs
    auto join = [&](RowStat a) {   // lanes 0 .. 15 hold parts
#pragma unroll
      for (int o = 8; o > 0; o /= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, a.m, o);
        const int oi = __shfl_xor_sync(0xffffffffu, a.at, o);
        const double os = __shfl_xor_sync(0xffffffffu, a.sum, o);
        if (greedy) {
          if (om > a.m || (om == a.m && oi < a.at)) a.at = oi;
          a.m = fmaxf(a.m, om);
        } else {
          const float M = fmaxf(a.m, om);
          a.sum = a.sum * ex2((a.m - M) * c) + os * ex2((om - M) * c);
          a.m = M;
        }
      }
      return a;
    };
    const RowStat none{greedy ? -INFINITY : -2 * VF_BIG, INT32_MAX, 0.0};
    if (warp < rows) {
      const RowStat a = join(warp_stat[warp][lane & (VF_WARPS - 1)]);
      if (lane == 0) cta_stat[buf][warp] = a;
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp < rows) {
      RowStat a = none;
      if ((lane & 15) < ctas) {
        const RowStat* s = &cta_stat[buf][warp];
        a.m = ld_cluster_f32(&s->m, lane & 15);
        a.at = ld_cluster_s32(&s->at, lane & 15);
        a.sum = ld_cluster_f64(&s->sum, lane & 15);
      }
      a = join(a);
      if (lane == 0) {
        const int j = at + warp;
        int v = 0;
        if (!greedy && !careful && !(a.sum > 0.0 && a.sum < 1e300 && a.m < VF_BIG)) {
          v = 2;   // a NaN, an infinity, or nothing above -1e30
        } else if (j < count) {
          const int d = __ldg(drafts + j);
          if (d >= 0 && d < p.vocab) {
            double pd;
            if (greedy) {
              pd = d == a.at ? 1.0 : 0.0;
            } else {
              const float x = clean(row_of(j).at(d));
              pd = x == -INFINITY || !(a.sum > 0.0) ? 0.0 : exp2(((double)x - (double)a.m) * (double)c) / a.sum;
            }
            const double q = p.probs ? (double)__ldg(p.probs + seq * p.q_seq + j * p.q_row + d) : 1.0;
            v = (double)__ldg(u + j) * q < pd;
          }
        }
        verdict[warp] = v;
        row_stat[warp] = a;
      }
    }
    __syncthreads();
    int w = 0;
    while (w < rows && verdict[w] == 1) ++w;
    at += w;
    careful = false;
    if (w < rows) {
      careful = verdict[w] == 2;
      if (!careful) stop = at;
      st = row_stat[w];
    }
    buf ^= 1;
    __syncthreads();   // verdict and row_stat are read
  }

  // ---- the token
  int token = -1;
  if (greedy) {
    token = st.at == INT32_MAX ? -1 : st.at;
  } else if (st.sum > 0.0) {
    const Logits<TYPE> row = row_of(stop);
    const int lo = cut(0, row.pieces, rank, ctas), hi = cut(0, row.pieces, rank + 1, ctas);
    Weights w{1.4426950408889634 / (double)temp, (double)st.m, nullptr, 0.0, -1};
    int which = 0;
    // Sums over the cluster's runs, a warp each, added up in the same order by
    // every CTA: `total`, and the run that u_last times it falls into.
    auto add_up = [&]() {
      const double s = warp_run_sum(row, w, cut(lo, hi, warp, VF_WARPS), cut(lo, hi, warp + 1, VF_WARPS));
      which ^= 1;
      if (lane == 0) run_sum[which][warp] = s;
      cluster_arrive_release();
      cluster_wait_acquire();
      if (warp == 0) {
        constexpr int E = VF_CLUSTER * VF_WARPS / 32;
        double y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int k = lane * E + e;
          y[e] = k < ctas * VF_WARPS ? ld_cluster_f64(&run_sum[which][k & (VF_WARPS - 1)], k / VF_WARPS) : 0.0;
        }
        int heavy;
        double before, all;
        warp_find(y, INFINITY, 0.0, &heavy, &before, &all);
        const double x = (double)__ldg(u + p.block - 1) * all;
        int k = warp_find(y, x, 0.0, &heavy, &before, &all);
        if (k < 0) k = heavy;   // (a uniform number of 1)
        if (lane == 0) {
          place.total = all;
          place.x = x - before;
          place.run = k;
        }
      }
      __syncthreads();
    };
    if (stop < count) {
      if (p.probs) {
        add_up();
        w.total = place.total;
        w.q = p.probs + seq * p.q_seq + stop * p.q_row;
      } else {
        w.drop = __ldg(drafts + stop);
      }
    }
    add_up();
    if (!(place.total > 0.0) && (w.q || w.drop >= 0)) {   // nothing is left of p: all of it
      w.q = nullptr;
      w.drop = -1;
      add_up();
    }
    const int owner = place.run;
    // the CTA that holds it goes on alone: its warps share the run, then one warp the rest
    if (owner >= 0 && owner / VF_WARPS == rank) {
      const int a = cut(lo, hi, owner % VF_WARPS, VF_WARPS), b = cut(lo, hi, owner % VF_WARPS + 1, VF_WARPS);
      const double s = warp_run_sum(row, w, cut(a, b, warp, VF_WARPS), cut(a, b, warp + 1, VF_WARPS));
      which ^= 1;
      if (lane == 0) run_sum[which][warp] = s;
      __syncthreads();
      if (warp == 0) {
        constexpr int E = Logits<TYPE>::E;
        double x = place.x, before, all;
        int heavy;
        const double part[1] = {lane < VF_WARPS ? run_sum[which][lane] : 0.0};
        int k = warp_find(part, x, 0.0, &heavy, &before, &all);
        if (k < 0) k = heavy;
        x -= before;
        const int from = cut(a, b, k, VF_WARPS), to = k < 0 ? from : cut(a, b, k + 1, VF_WARPS);
        double sum = 0.0;
#pragma unroll 1
        for (int i0 = from; i0 < to; i0 += 32) {
          const int i = i0 + lane;
          double y[E];
          float l[E];
          if (i < to) row.get(i, l);
#pragma unroll
          for (int e = 0; e < E; ++e) y[e] = i < to ? weight(w, l[e], i * E - row.skip + e) : 0.0;
          const int f = warp_find(y, x, sum, &heavy, &before, &sum);
          if (f >= 0 || heavy >= 0) token = i0 * E - row.skip + (f >= 0 ? f : heavy);
          if (f >= 0) break;
        }
      }
    }
    if (owner >= 0 && owner / VF_WARPS != rank) stop = -1;   // (that CTA writes)
    if (owner < 0 && rank > 0) stop = -1;
  } else if (rank > 0) {
    stop = -1;
  }
  if (greedy && rank > 0) stop = -1;
  if (threadIdx.x == 0 && stop >= 0) {
    p.accepted[seq] = stop;
    p.tokens[seq] = token;
  }
  cluster_arrive_release();   // no CTA leaves while its sums are read
  cluster_wait_acquire();
}

template <int TYPE>
static cudaError_t launch(const VerifyParams& p, int num_sms, cudaStream_t st) {
  // CTAs of a request: enough for two waves of CTAs at most, and a slice of 4 KB at least
  int ctas = VF_CLUSTER;
  const long long bytes = (long long)p.vocab * elem_bytes(p.type);
  while (ctas > 1 && ((long long)p.n * ctas > 4 * num_sms || bytes / ctas < 4096)) ctas /= 2;
  const int window = (long long)p.n * ctas <= num_sms ? 4 : 1;
  DFL_TRY(cudaFuncSetAttribute(verify_kernel<TYPE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  return launch_pdl_cluster(verify_kernel<TYPE>, dim3(p.n * ctas), dim3(VF_THREADS), ctas, st, p, ctas, window);
}

cudaError_t verify_launch(const VerifyParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.block < 1 || p.vocab < 1) return cudaErrorInvalidValue;
  switch (p.type) {
    case kElemF16: return launch<kElemF16>(p, num_sms, st);
    case kElemBf16: return launch<kElemBf16>(p, num_sms, st);
    case kElemF32: return launch<kElemF32>(p, num_sms, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace dfl
