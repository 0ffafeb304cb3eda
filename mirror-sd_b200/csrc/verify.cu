// Verification of drafted tokens by sampling.  With p_j the softmax of logits
// row j over the temperature, u the request's uniform numbers and q_j what the
// draft was sampled from (1 at the draft itself where it was not sampled):
//
//   draft d_j is accepted while u_j q_j(d_j) < p_j(d_j);
//   the token behind the accepted ones is sampled from r = max(p_a - q_a, 0) at
//   the first refused place a, from r = p_a behind the last draft: the first
//   token in vocabulary order whose running sum of r passes u_last sum(r).
//
// A cluster of CTAs owns a request.  Its warps stream the request's rows, one after
// another, each warp a run of its own of every row: one pass of 2^((x - m) c) in 32
// bits, c = log2(e) / T, against a reference m of each thread that moves when a logit
// passes it by 2^8 (so the exponents that matter are small, and exact to 2^-24 of
// themselves).  One more warp joins the runs' parts of a row (in 64 bits) and decides
// its draft, while the others are at work on the next rows already: rows behind the
// first refused draft do not count, but waiting for each decision would take 5 us a
// row (load latency, two exchanges, a decision) of which the bytes of a row are 1 or
// 2.  So up to `ahead` of them are read all the same.
//
// 256 requests of up to 16 rows of 151,936 bf16 logits, 4.9 rows each on average:
// 150 us, where the rows' bytes are 47 us of HBM (all rows of all requests: 200 us).
// What bounds it is the longest chains: a request whose drafts are all accepted
// takes 16 rows one after another, each 4 to 8 us while others share its SMs, and the
// token costs 10 to 25 us.  One request: 17 to 25 us, all of it such a chain.  (Rounds of a
// few rows of all requests, a launch each, when this took 180 us: 188; each such launch
// costs 12 us beside its bytes.  Rings filled by bulk copies in place of 8 loads a lane,
// when it took 155: 180.)
//
// The row that the token comes from is read once more, from L2, with weights to 2^-31
// of themselves and sums in 64 bits: u times the sum must fall between the same two
// of up to 150,000 running sums, whatever order they are added up in, and weights to
// 2^-22 of themselves move running sums by more than an unlikely token weighs.  (Where p
// and q agree to 2^-30 of p everywhere, what is left of p is rounding, and so is its
// token; a draft that q proposes is refused there once in 2^30 times at most.)
//
// Logits: NaN counts as -inf, a weight of 0; what lies beyond +-1e30 counts as
// that, but for greedy requests (T < 1e-5), which compare logits as they are, as an
// argmax does.  A row that leaves no token refuses its draft and gives token -1.
#include <algorithm>

#include "decode.cuh"

namespace dfl {

constexpr int VF_THREADS = 256, VF_WARPS = VF_THREADS / 32, VF_CTAS = 4;   // of a CTA; CTAs an SM
constexpr int VF_FLY = 8;                // 16-byte pieces of a lane on their way together
constexpr int VF_BLOCK = 32 * VF_FLY;
constexpr int VS_FLY = 4, VS_BLOCK = 32 * VS_FLY;   // the same where a token is sampled
constexpr int VF_CLUSTER = 16;           // CTAs of a request at most
constexpr int VF_DEPTH = 8;              // rows whose parts are kept
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

// a logit as a sampled request takes it: NaN is -inf, and finite ones (and +inf) lie within +-1e30
__device__ __forceinline__ float clean(float x) {
  if (!(x > -INFINITY)) return -INFINITY;
  return fminf(fmaxf(x, -VF_BIG), VF_BIG);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- arithmetic on pairs
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
// the largest entry of some pieces, NaN aside
template <int TYPE, int FLY>
__device__ __forceinline__ float top_of(const uint4 (&w)[FLY]) {
  uint32_t u[4 * FLY];
#pragma unroll
  for (int k = 0; k < FLY; ++k) {
    u[4 * k] = w[k].x;
    u[4 * k + 1] = w[k].y;
    u[4 * k + 2] = w[k].z;
    u[4 * k + 3] = w[k].w;
  }
#pragma unroll
  for (int k = 2 * FLY; k > 0; k /= 2)
#pragma unroll
    for (int i = 0; i < k; ++i) {
      if constexpr (TYPE == kElemF32) u[i] = __float_as_uint(fmaxf(__uint_as_float(u[i]), __uint_as_float(u[i + k])));
      else if constexpr (TYPE == kElemBf16) asm("max.bf16x2 %0, %0, %1;" : "+r"(u[i]) : "r"(u[i + k]));
      else asm("max.f16x2 %0, %0, %1;" : "+r"(u[i]) : "r"(u[i + k]));
    }
  if constexpr (TYPE == kElemF32) return __uint_as_float(u[0]);
  else return fmaxf(Logits<TYPE>::bits(u[0], 0), Logits<TYPE>::bits(u[0], 1));
}

// a warp's largest m and the first of its places
__device__ __forceinline__ void warp_first(float& m, int& at) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (om > m || (om == m && oi < at)) {
      m = om;
      at = oi;
    }
  }
}

// Sum of 2^((x - m) c) over what a lane sees of a row.
template <int TYPE>
struct SoftSum {
  static constexpr int E = Logits<TYPE>::E;
  float c, m = -VF_BIG, lim = -VF_BIG;   // (the first logit above raises it)
  float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
  __device__ __forceinline__ explicit SoftSum(float c) : c(c) {}
  __device__ __forceinline__ void raise(float top) {
    const float f = ex2((m - top) * c);
    sum[0] = mul2(sum[0], make_float2(f, f));
    sum[1] = mul2(sum[1], make_float2(f, f));
    m = top;
    lim = top + VF_RAISE / c;
  }
  __device__ __forceinline__ void block(const uint4 (&w)[VF_FLY]) {
    const float top = top_of<TYPE>(w);
    if (top > lim) raise(top);
    const float2 nm = make_float2(-m, -m), cc = make_float2(c, c);
#pragma unroll
    for (int k = 0; k < VF_FLY; ++k) {
      float x[E];
      Logits<TYPE>::split(w[k], x);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        float2 y = mul2(add2(make_float2(x[i], x[i + 1]), nm), cc);
        y.x = ex2(y.x);
        y.y = ex2(y.y);
        sum[i / 2 & 1] = add2(sum[i / 2 & 1], y);
      }
    }
  }
  __device__ __forceinline__ void one(float x) {
    if (x > lim) raise(x);
    sum[0].x += ex2((x - m) * c);
  }
  __device__ __forceinline__ float total() const { return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y); }
};

// The same by the definition's rules for NaN, infinities and what lies beyond +-1e30.
template <int TYPE>
__device__ __noinline__ void row_sum_careful(const Logits<TYPE>& row, float c, float& m, float& s) {
  m = -2 * VF_BIG;
  s = 0.f;
  float lim = m;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < row.vocab; i += 32) {
    const float x = clean(row.at(i));
    if (x > lim) {
      s *= ex2((m - x) * c);
      m = x;
      lim = x + VF_RAISE / c;
    }
    if (x > -INFINITY) s += ex2((x - m) * c);
  }
}

// ---- the weights of the row that the token comes from, 2^((x - m) c) in 64 bits
struct Weights {
  double c, m;
  const float* q;        // subtract total * q, or NULL
  double total;
  int drop;              // entry without weight, or -1
  // 2^(x c - mc) = 2^(k + j / 256) 2^r: x c + grid, grid = 1.5 * 2^44 - mc, has k and j in its lowest 32 bits (mc
  // a multiple of 2^-8), 2^(j / 256) comes from a table, 2^r = 1 + r ln 2 + (r ln 2)^2 / 2 for |r| <= 2^-9 is off by
  // 2^-31 at most.  Logits outside [low, high] (2^-990, 2^960) are taken for
  // those.
  bool fast;
  double grid;
  float low, high;
  const double* table;
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
constexpr double kLn2 = 0.69314718055994530942;
// 2^(k + j / 256) and the factor 2^r
struct FastWeight {
  double c, grid;
  float low, high;
  const double* table;
  __device__ __forceinline__ double operator()(float x, double* factor) const {
    const double X = (double)fminf(fmaxf(x, low), high);   // (NaN and -inf: low)
    const double n = fma(X, c, grid), r = fma(X, c, grid - n);
    *factor = fma(r, fma(r, kLn2 * kLn2 / 2, kLn2), 1.0);
    const int lo = __double2loint(n);
    const double t = table[lo & 255];
    return __hiloint2double(__double2hiint(t) + ((lo >> 8) << 20), __double2loint(t));
  }
};

__device__ __forceinline__ void refer(Weights* w, float m) {
  const double mc = rint((double)m * w->c * 256.0) / 256.0;
  w->fast = w->c > 1e-3 && fabs(mc) < 0x1p20;
  w->m = w->fast ? mc / w->c : m;   // (both forms of a weight to the same scale)
  w->grid = 0x1.8p44 - mc;
  w->low = (float)((double)m - 990.0 / w->c);
  w->high = (float)((double)m + 960.0 / w->c);
}
// Sum of the weights of one 16-byte piece.
template <int TYPE>
__device__ __forceinline__ double piece_sum(const Logits<TYPE>& row, const Weights& w, const FastWeight& fast, int drop, int piece,
                                            const float (&x)[Logits<TYPE>::E]) {
  constexpr int E = Logits<TYPE>::E;
  double s = 0.0;
  if (!w.fast || piece == drop) {
#pragma unroll 1
    for (int k = 0; k < E; ++k) s += weight(w, x[k], piece * E - row.skip + k);
  } else if (w.q) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int i = piece * E - row.skip + k;
      const float q = i >= 0 && i < row.vocab ? __ldg(w.q + i) : 0.f;
      double f;
      const double t = fast(x[k], &f), y = t * f;
      s += q > 0.f ? fmax(y - (double)q * w.total, 0.0) : y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      double f;
      const double t = fast(x[k], &f);
      s = fma(t, f, s);
    }
  }
  return s;
}
__device__ __forceinline__ double warp_sum64(double s) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s > 0x1p-900 ? s : 0.0;   // (masked entries at 2^-990 are none)
}
// Sum of the weights of the pieces [lo, hi), by a warp.
template <int TYPE>
__device__ __forceinline__ double warp_run_sum(const Logits<TYPE>& row, const Weights& w, int lo, int hi) {
  constexpr int E = Logits<TYPE>::E;
  const FastWeight fast{w.c, w.grid, w.low, w.high, w.table};
  const int drop = w.drop >= 0 ? (w.drop + row.skip) / E : -1;
  const int a = max(lo, row.skip ? 1 : 0), b = min(hi, (row.vocab + row.skip) / E);   // whole pieces
  const int lane = threadIdx.x & 31;
  double s = 0.0;
  int i = a + lane;
  if (w.fast && !w.q) {
    double t[2] = {0.0, 0.0};
#pragma unroll 1
    for (; i - lane + VS_BLOCK <= b; i += VS_BLOCK) {
      uint4 v[VS_FLY];
#pragma unroll
      for (int k = 0; k < VS_FLY; ++k) v[k] = row.load(i + 32 * k);
      if (drop >= i - lane && drop < i - lane + VS_BLOCK) {
#pragma unroll 1
        for (int k = 0; k < VS_FLY; ++k) {
          float x[E];
          row.get(i + 32 * k, x);
          s += piece_sum(row, w, fast, drop, i + 32 * k, x);
        }
        continue;
      }
#pragma unroll
      for (int k = 0; k < VS_FLY; ++k) {
        float x[E];
        Logits<TYPE>::split(v[k], x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          double f;
          const double y = fast(x[e], &f);
          t[e & 1] = fma(y, f, t[e & 1]);
        }
      }
    }
    s += t[0] + t[1];
  }
#pragma unroll 1
  for (; i < b; i += 32) {
    float x[E];
    Logits<TYPE>::split(row.load(i), x);
    s += piece_sum(row, w, fast, drop, i, x);
  }
  if (lane == 0 && (lo < a || b < hi))
    for (int e = lo; e < hi; e = e + 1 < a ? e + 1 : max(e + 1, b))
      if (e < a || e >= b) {
        float x[E];
        row.get(e, x);
        s += piece_sum(row, w, fast, drop, e, x);
      }
  return warp_sum64(s);
}

// where part i of [lo, hi) begins, of equal parts but for the last ones (in 32 bits: a division of 64 takes a microsecond)
__device__ __forceinline__ int cut(int lo, int hi, int i, int parts) {
  const int len = (hi - lo + parts - 1) / parts;
  return min(lo + i * len, hi);
}

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
template <int TYPE>
__device__ __forceinline__ Logits<TYPE> logits_row(const VerifyParams& p, int seq, int j) {
  return Logits<TYPE>(static_cast<const char*>(p.logits) + (seq * p.l_seq + j * p.l_row) * (16 / Logits<TYPE>::E), p.vocab);
}
__device__ __forceinline__ int drafts_of(const VerifyParams& p, int seq) {
  return p.counts ? min(max(__ldg(p.counts + seq), 0), p.block - 1) : p.block - 1;
}
__device__ __forceinline__ float temperature_of(const VerifyParams& p, int seq) { return p.temps ? __ldg(p.temps + seq) : p.temp; }
__device__ __forceinline__ bool is_greedy(float temp) { return !(temp >= 1e-5f); }

struct alignas(8) Part {   // of a row, by a warp (stored as 64 bits)
  float m;                 // reference, or the largest entry
  int s;                   // bits of the sum, or the entry's place
};
static_assert(sizeof(Part) == 8 && alignof(Part) == 8, "st_cluster_u64 stores it whole");
// What a cluster's CTAs know of their request: rows whose drafts are accepted so
// far, or -1 - stop once that is known, and the bits of the last decided row's
// reference (its first largest entry, where the request is greedy).
struct Progress {
  int rows, row;
};
__device__ __forceinline__ Progress progress_of(const unsigned long long* at) {
  const unsigned long long v = *reinterpret_cast<const volatile unsigned long long*>(at);
  return {(int)(v >> 32), (int)v};
}
__device__ __forceinline__ void st_cluster_u64(uint32_t remote, unsigned long long v) {
  asm volatile("st.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}
// Bounded wait for parts that other CTAs of the cluster have stored.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

template <int TYPE>
__global__ void __launch_bounds__(VF_THREADS, VF_CTAS) verify_kernel(const VerifyParams p, int ctas, int ahead) {
  constexpr int E = Logits<TYPE>::E;
  constexpr uint32_t NONE = TYPE == kElemF16 ? 0xfc00fc00u : TYPE == kElemBf16 ? 0xff80ff80u : 0xff800000u;
  __shared__ Part parts[VF_DEPTH][VF_CLUSTER * VF_WARPS];   // (the first CTA's are used)
  __shared__ uint64_t full[VF_DEPTH];
  __shared__ unsigned long long progress;
  __shared__ double run_sum[2][VF_WARPS];
  __shared__ float warp_top[VF_WARPS], cta_top;
  __shared__ struct { double total, x; int run; } place;
  __shared__ double table[256];          // 2^(i / 256)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x / ctas, rank = blockIdx.x - seq * ctas;
  const int streams = ctas * VF_WARPS - 1;   // the first CTA's last warp decides
  if (threadIdx.x == 0) {
    for (int i = 0; i < VF_DEPTH; ++i) mbar_init(&full[i], streams);
    fence_mbar_init();
    progress = 0;
  }
  for (int i = threadIdx.x; i < 256; i += VF_THREADS) table[i] = exp2(i / 256.0);
  __syncthreads();
  cluster_arrive_release();
  cluster_wait_acquire();
  griddep_wait();
  griddep_launch_dependents();
  const int count = drafts_of(p, seq);
  const float temp = temperature_of(p, seq);
  const bool greedy = is_greedy(temp);
  const float c = greedy ? 0.f : (float)(1.4426950408889634 / (double)temp);
  // (a sampled token's row needs no pass of its own: only greedy requests take the row behind the last draft)
  const int rows = greedy ? count + 1 : count;

  if (rank > 0 || warp < VF_WARPS - 1) {
    // ---- the rows, a run of each
    const int me = rank == 0 ? warp : rank * VF_WARPS + warp - 1;
    const int len = ((p.vocab + 2 * E - 2) / E + streams - 1) / streams, lo = me * len;   // (whatever a row's alignment)
#pragma unroll 1
    for (int j = 0; j < rows; ++j) {
      const Logits<TYPE> row = logits_row<TYPE>(p, seq, j);
      const int hi = min(lo + len, row.pieces);
      const int a = max(lo, row.skip ? 1 : 0), b = min(hi, (p.vocab + row.skip) / E);   // whole pieces
      int done = 0;
#pragma unroll 1
      for (uint32_t i = 0; i < kSpinLimit; ++i) {
        done = progress_of(&progress).rows;
        if (done < 0 || j <= done + ahead) break;
        __nanosleep(40);
      }
      if (__any_sync(0xffffffffu, done < 0 || j > done + ahead)) break;
      bool over = false;
      // its blocks, one after another: f(pieces, first piece of the lane), missing ones as -inf
      auto blocks_to = [&](auto f) {
        int i = a + lane;
#pragma unroll 1
        for (; i - lane + VF_BLOCK <= b; i += VF_BLOCK) {
          uint4 v[VF_FLY];
#pragma unroll
          for (int k = 0; k < VF_FLY; ++k) v[k] = row.load(i + 32 * k);
          over = __any_sync(0xffffffffu, progress_of(&progress).rows < 0);
          if (over) return;
          f(v, i);
        }
        if (i - lane < b) {
          uint4 v[VF_FLY];
#pragma unroll
          for (int k = 0; k < VF_FLY; ++k) {
            v[k] = make_uint4(NONE, NONE, NONE, NONE);
            if (i + 32 * k < b) v[k] = row.load(i + 32 * k);
          }
          f(v, i);
        }
      };
      // the row's ragged ends in the run, by lane 0
      auto ends_to = [&](auto f) {
        if (lane == 0 && (lo < a || b < hi))
          for (int e = 0; e < 2; ++e) {
            const int piece = e == 0 ? 0 : row.pieces - 1;
            if (piece < lo || piece >= hi || (piece >= a && piece < b) || (e == 1 && row.pieces == 1)) continue;
            float x[E];
            row.get(piece, x);
            f(x, piece);
          }
      };
      float m;
      int part;   // the sum's bits, or the place
      if (greedy) {
        int block = -1, at = INT32_MAX;   // the lane's first piece of the block that its largest entry is in
        m = -INFINITY;
        blocks_to([&](const uint4(&v)[VF_FLY], int piece) {
          const float top = top_of<TYPE>(v);
          block = top > m ? piece : block;
          m = fmaxf(m, top);
        });
        if (over) break;
        if (block >= 0) {
#pragma unroll 1
          for (int k = 0; k < VF_FLY && block + 32 * k < b; ++k) {
            float x[E];
            row.get(block + 32 * k, x);
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (x[e] == m) at = min(at, (block + 32 * k) * E - row.skip + e);
          }
        }
        ends_to([&](const float(&x)[E], int piece) {
          for (int k = 0; k < E; ++k) {
            const int i = piece * E - row.skip + k;
            if (x[k] > m || (x[k] == m && i < at && m > -INFINITY)) {
              m = x[k];
              at = i;
            }
          }
        });
        warp_first(m, at);
        part = at;
      } else {
        SoftSum<TYPE> s(c);
        blocks_to([&](const uint4(&v)[VF_FLY], int) { s.block(v); });
        if (over) break;
        ends_to([&](const float(&x)[E], int) {
          for (int k = 0; k < E; ++k) s.one(x[k]);
        });
        m = warp_max(s.m);
        part = __float_as_int(warp_sum(s.total() * ex2((s.m - m) * c)));
      }
      if (lane == 0) {
        st_cluster_u64(mapa_shared(&parts[j % VF_DEPTH][me], 0),
                       (unsigned long long)(uint32_t)part << 32 | (uint32_t)__float_as_int(m));
        mbar_arrive_cluster(mapa_shared(&full[j % VF_DEPTH], 0));
      }
      __syncwarp();
    }
  } else {
    // ---- the decisions
    int j = 0, last = 0;   // bits of the last row's reference or place
    int my_d = -1;
    float my_x = -INFINITY;
    double my_u = 1.0;
    bool good = true;
#pragma unroll 1
    for (; j < rows; ++j) {
      // what the decisions need beside the rows' sums, of 32 rows at a time, a lane each
      if (j % 32 == 0) {
        const int k = j + lane;
        my_d = -1;
        if (k < count) {
          my_d = __ldg(p.drafts + (size_t)seq * (p.block - 1) + k);
          my_u = __ldg(p.uniforms + (size_t)seq * p.block + k);
          if (my_d >= 0 && my_d < p.vocab) {
            my_x = clean(logits_row<TYPE>(p, seq, k).at(my_d));
            if (p.probs) my_u = (double)my_u * (double)__ldg(p.probs + seq * p.q_seq + k * p.q_row + my_d);
          } else {
            my_d = -1;
          }
        }
      }
      const int d = __shfl_sync(0xffffffffu, my_d, j % 32);
      const float x = __shfl_sync(0xffffffffu, my_x, j % 32);
      const double uq = __shfl_sync(0xffffffffu, my_u, j % 32);
      good = __all_sync(0xffffffffu, wait_cluster(&full[j % VF_DEPTH], (j / VF_DEPTH) & 1));
      if (!good) break;
      constexpr int N = VF_CLUSTER * VF_WARPS / 32;
      Part v[N];
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[k] = lane + 32 * k < streams ? parts[j % VF_DEPTH][lane + 32 * k]
                                       : Part{greedy ? -INFINITY : -VF_BIG, greedy ? INT32_MAX : 0};
      bool accepted;
      if (greedy) {
        float M = v[0].m;
        int at = v[0].s;
#pragma unroll
        for (int k = 1; k < N; ++k)
          if (v[k].m > M || (v[k].m == M && v[k].s < at)) {
            M = v[k].m;
            at = v[k].s;
          }
        warp_first(M, at);
        last = at;
        accepted = d >= 0 && uq < (d == at ? 1.0 : 0.0);
      } else {
        float m = v[0].m;
#pragma unroll
        for (int k = 1; k < N; ++k) m = fmaxf(m, v[k].m);
        m = warp_max(m);
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < N; ++k) sum += (double)(__int_as_float(v[k].s) * ex2((v[k].m - m) * c));
#pragma unroll
        for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!(sum > 0.0 && sum < 1e300 && m < VF_BIG)) {
          // a NaN, an infinity, or nothing above -1e30: this warp takes the row again, with care
          float M, s;
          row_sum_careful(logits_row<TYPE>(p, seq, j), c, M, s);
          m = warp_max(M);
          sum = (double)s * ex2((M - m) * c);
#pragma unroll
          for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        last = __float_as_int(m);
        accepted = d >= 0 && x > -INFINITY && sum > 0.0 && uq * sum < exp2(((double)x - (double)m) * (double)c);
      }
      if (!__all_sync(0xffffffffu, accepted)) break;
      if (j + 1 < rows && lane < ctas)
        st_cluster_u64(mapa_shared(&progress, lane), (unsigned long long)(uint32_t)(j + 1) << 32 | (uint32_t)last);
    }
    if (lane < ctas)   // (INT32_MIN: a wait expired)
      st_cluster_u64(mapa_shared(&progress, lane), (unsigned long long)(uint32_t)(good ? -1 - j : INT32_MIN) << 32 | (uint32_t)last);
  }
  __syncwarp();
  cluster_arrive_release();
  cluster_wait_acquire();

  // ---- the token behind the accepted drafts
  const Progress end = progress_of(&progress);
  const bool failed = end.rows >= 0 || end.rows == INT32_MIN;
  const int stop = failed ? -1 : -1 - end.rows;
  if (rank == 0 && threadIdx.x == 0) {
    p.accepted[seq] = stop;
    if (failed || greedy) p.tokens[seq] = failed || end.row == INT32_MAX ? -1 : end.row;
  }
  if (failed || greedy) return;   // (all CTAs of the cluster)
  const Logits<TYPE> row = logits_row<TYPE>(p, seq, stop);
  const double u = __ldg(p.uniforms + (size_t)seq * p.block + p.block - 1);
  const int lo = cut(0, row.pieces, rank, ctas), hi = cut(0, row.pieces, rank + 1, ctas);
  const bool refused = stop < count;
  Weights w;
  w.c = 1.4426950408889634 / (double)temp;
  w.table = table;
  w.total = 0.0;
  w.drop = refused && !p.probs ? __ldg(p.drafts + (size_t)seq * (p.block - 1) + stop) : -1;
  {
    // a reference near the row's largest logit: its own or, behind the last draft, that of the row before
    const float near = __int_as_float(end.row);
    refer(&w, fabsf(near) < VF_BIG ? near : 0.f);
  }
  int which = 0;
  // Sums over the cluster's runs, a warp each, added up in the same order by every
  // CTA: their total, and the run that u times it falls into.
  auto add_up = [&]() {
    const double s = warp_run_sum(row, w, cut(lo, hi, warp, VF_WARPS), cut(lo, hi, warp + 1, VF_WARPS));
    which ^= 1;
    if (lane == 0) run_sum[which][warp] = s;
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp == 0) {
      constexpr int N = VF_CLUSTER * VF_WARPS / 32;
      double y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int k = lane * N + e;
        y[e] = k < ctas * VF_WARPS ? ld_cluster_f64(&run_sum[which][k % VF_WARPS], k / VF_WARPS) : 0.0;
      }
      int heavy;
      double before, all;
      warp_find(y, INFINITY, 0.0, &heavy, &before, &all);
      const double x = u * all;
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
  // All of p, unless a draft was refused: what the draft distribution leaves of it.
  const bool sampled = refused && p.probs;
  auto residual = [&]() {
    w.q = nullptr;
    add_up();
    if (sampled) {
      w.total = place.total;
      w.q = p.probs + seq * p.q_seq + stop * p.q_row;
      add_up();
    }
  };
  residual();
  if (const double t = w.q ? w.total : place.total; !(t > 0x1p-500 && t < 0x1p900)) {
    // the reference was none for this row (or nothing but the draft weighs anything): the row's largest logit
    float top = -INFINITY;
    for (int i = lo + threadIdx.x; i < hi; i += VF_THREADS) {
      float x[E];
      row.get(i, x);
#pragma unroll
      for (int k = 0; k < E; ++k) top = fmaxf(top, clean(x[k]));
    }
    top = warp_max(top);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < VF_WARPS; ++k) top = fmaxf(top, warp_top[k]);
      cta_top = top;
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    for (int k = 0; k < ctas; ++k) top = fmaxf(top, ld_cluster_f32(&cta_top, k));
    w.m = top == -INFINITY ? 0.f : top;
    w.fast = false;
    residual();
  }
  if (!(place.total > 0.0) && (w.q || w.drop >= 0)) {   // nothing is left of p: all of it
    w.q = nullptr;
    w.drop = -1;
    add_up();
  }
  const int owner = place.run;   // rank * VF_WARPS + warp
  // the CTA that holds it goes on alone: its warps share the run, then one warp the rest
  if (owner >= 0 && owner / VF_WARPS == rank) {
    const int a = cut(lo, hi, owner % VF_WARPS, VF_WARPS), b = cut(lo, hi, owner % VF_WARPS + 1, VF_WARPS);
    const double s = warp_run_sum(row, w, cut(a, b, warp, VF_WARPS), cut(a, b, warp + 1, VF_WARPS));
    which ^= 1;
    if (lane == 0) run_sum[which][warp] = s;
    __syncthreads();
    if (warp == 0) {
      int token = -1;
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
      if (lane == 0) p.tokens[seq] = token;
    }
  } else if (owner < 0 && rank == 0 && threadIdx.x == 0) {
    p.tokens[seq] = -1;
  }
  cluster_arrive_release();   // no CTA leaves while its sums are read
  cluster_wait_acquire();
}

template <int TYPE>
static cudaError_t launch(const VerifyParams& p, int num_sms, cudaStream_t st) {
  // CTAs of a request: 8 KB of a row each at least, and at most twice as many CTAs
  // in all as are resident together.  us with 1 / 2 / 4 / 8 / 16 CTAs, the rule's in brackets:
  //   256 requests, 16 rows of 151,936   247 / 154 / [150] / 180 / 255
  //   256 requests, 16 rows of 32,003     80 /  72 /  [75] / 110 / 215
  //    64 requests, 16 rows of 151,936   200 / 101 /  76 / 71 / [75]
  //    64 requests, 8 rows of 32,003      40 /  31 / [28] / 33 / 55
  //   512 requests, 8 rows of 32,003      84 / [92] / 113 / 187 / 395
  // 1,024 requests, 4 rows of 8,192      [47] / 70 / 124 / 240 / 563
  //     1 request, 16 rows of 151,936     83 /  46 /  34 / 28 / [23]
  const long long bytes = (long long)p.vocab * elem_bytes(p.type);
  int ctas = VF_CLUSTER;
  while (ctas > 1 && (p.n * (long long)ctas > 2 * VF_CTAS * num_sms || bytes / ctas < 8192)) ctas /= 2;
  // Rows to run ahead: one where the requests fill the GPU, as many as there is room
  // for where they do not (none / one / two / seven: 256 requests of 151,936 156 / 150 /
  // 151 / 152 us, of 32,003 78 / 75 / 76 / 76, 16 requests of 151,936 54 / 48 / 48 / 47).
  const int ahead = p.n * (long long)ctas > VF_CTAS * num_sms ? 1 : VF_DEPTH - 1;
  DFL_TRY(cudaFuncSetAttribute(verify_kernel<TYPE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  return launch_pdl_cluster(verify_kernel<TYPE>, dim3(p.n * ctas), dim3(VF_THREADS), ctas, st, p, ctas, ahead);
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
