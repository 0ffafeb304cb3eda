// Prefix sums over the requests of a paged call (paged.cu, paged_share.cu).
#pragma once
#include "q4.cuh"

namespace dfl {

constexpr int PG_THREADS = 512;

// inclusive scan of (a, b) over the block; *ta / *tb receive the totals
__device__ __forceinline__ void block_scan2(long long& a, int& b, long long* ta, int* tb) {
  __shared__ long long wa[PG_THREADS / 32];
  __shared__ int wb[PG_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long xa = __shfl_up_sync(0xffffffffu, a, o);
    const int xb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += xa; b += xb; }
  }
  __syncthreads();  // wa / wb of the previous call are read
  if (lane == 31) { wa[warp] = a; wb[warp] = b; }
  __syncthreads();
  long long sa = 0, all_a = 0;
  int sb = 0, all_b = 0;
#pragma unroll
  for (int w = 0; w < PG_THREADS / 32; ++w) {
    if (w < warp) { sa += wa[w]; sb += wb[w]; }
    all_a += wa[w];
    all_b += wb[w];
  }
  a += sa;
  b += sb;
  *ta = all_a;
  *tb = all_b;
}

// last index i in [0, n) with first[i] <= x (first ascending, first[0] <= x)
__device__ __forceinline__ int last_le(const int* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace dfl
