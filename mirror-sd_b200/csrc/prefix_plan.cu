// Which cached rows the requests of a group share, from the block tables: the
// pages on which the rows of all its members with query rows begin alike, cut to
// those that every query row sees whole.  Once a step, for all layers.
//
// One CTA a group; a warp compares a member's table row with the first member's,
// 32 columns at a time, up to the first difference that any warp has found.  Nothing
// is compared where the lengths alone leave fewer rows to spare than are asked for.
// What the tables spare is known once all groups are compared: one group's CTA sees
// that for itself, several groups' is added up by a second kernel.  Few numbers, so
// what both take is latency.
#include "q4.cuh"

namespace dfl {

constexpr int PP_THREADS = 512;

__global__ void __launch_bounds__(PP_THREADS) prefix_plan_kernel(const PrefixPlanParams p) {
  extern __shared__ int sm[];
  int* bound = sm;                // [g + 1] where the groups begin, never falling
  int* limits = bound + p.g + 1;  // [g] pages at most that members with query rows can share
  int* counts = limits + p.g;     // [g] their number
  __shared__ int first, limit, warp_top[PP_THREADS / 32];
  __shared__ unsigned long long spared;
  const int k = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    first = INT32_MAX;
    spared = 0;
  }
  griddep_wait();
  griddep_launch_dependents();
  // groups[] as boundaries that never fall (device data that the host has not seen): running maxima
  int carry = 0;
  for (int i0 = 0; i0 <= p.g; i0 += PP_THREADS) {
    const int i = i0 + threadIdx.x;
    int v = i <= p.g ? min(max(__ldg(p.groups + i), 0), p.n) : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, x);
    }
    __syncthreads();
    if (lane == 31) warp_top[warp] = v;
    __syncthreads();
    v = max(v, carry);
    for (int w = 0; w < PP_THREADS / 32; ++w) {
      if (w < warp) v = max(v, warp_top[w]);
      carry = max(carry, warp_top[w]);
    }
    if (i <= p.g) bound[i] = v;
    if (i < p.g) {
      limits[i] = p.max_pages;
      counts[i] = 0;
    }
  }
  __syncthreads();
  const int a = bound[k], b = bound[k + 1];
  auto start = [&](int i) { return p.starts ? __ldg(p.starts + i) : i * p.max_rows; };
  auto rows = [&](int i) { return start(i + 1) - start(i); };
  auto length = [&](int i) { return (int)min((long long)max(__ldg(p.lens + i), 0), (long long)p.max_pages * p.page_size); };
  // What sharing could spare at most, by the lengths, of all groups together: every CTA adds it up for itself.
  for (int i = bound[0] + threadIdx.x; i < bound[p.g]; i += PP_THREADS) {
    const int m = rows(i);
    if (m <= 0) continue;
    int lo = 0, hi = p.g - 1;
    while (lo < hi) {   // the last group that begins at or before the request
      const int mid = (lo + hi + 1) >> 1;
      if (bound[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const int seen = max(length(i) - (p.causal ? m - 1 : 0), 0);   // keys that all its query rows see
    atomicMin(&limits[lo], seen / p.page_size);
    atomicAdd(&counts[lo], 1);
    if (lo == k) atomicMin(&first, i);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.g; i += PP_THREADS)
    if (counts[i] > 1) atomicAdd(&spared, (unsigned long long)(counts[i] - 1) * limits[i] * p.page_size);
  __syncthreads();
  if (threadIdx.x == 0) limit = counts[k] < 2 || spared < (unsigned long long)p.least ? 0 : limits[k];
  __syncthreads();
  const int ref = first == INT32_MAX ? a : first;
  const int32_t* one = p.table + (size_t)ref * p.table_ld;
  for (int i = a + warp; i < b; i += PP_THREADS / 32) {
    if (i == ref || rows(i) <= 0) continue;
    const int32_t* other = p.table + (size_t)i * p.table_ld;
    int most = 0;   // (read by one lane: the votes below need the whole warp, and other warps lower it meanwhile)
    if (lane == 0) most = *reinterpret_cast<volatile int*>(&limit);
    most = __shfl_sync(0xffffffffu, most, 0);
#pragma unroll 4
    for (int c0 = 0; c0 < most; c0 += 32) {
      const int c = c0 + lane;
      const uint32_t differ = __ballot_sync(0xffffffffu, c < most && __ldg(one + c) != __ldg(other + c));
      if (differ) {
        most = c0 + __ffs(differ) - 1;
        if (lane == 0) atomicMin(&limit, most);
        break;
      }
    }
  }
  __syncthreads();
  int pages = limit;
  if (p.g == 1 && (counts[0] - 1ll) * pages * p.page_size < p.least) pages = 0;
  auto plan = [&](int i, int skip) {
    p.skip[i] = skip;
    p.own_lens[i] = max(length(i) - skip * p.page_size, 0);
  };
  for (int i = a + threadIdx.x; i < b; i += PP_THREADS) plan(i, rows(i) > 0 ? pages : 0);
  if (threadIdx.x == 0) {
    p.prefix[k] = pages * p.page_size;
    p.row_of[k] = min(ref, p.n - 1);
    p.group_starts[k] = start(a);
    if (k == p.g - 1) p.group_starts[p.g] = start(b);
  }
  // requests of no group
  if (k == 0)
    for (int i = threadIdx.x; i < a; i += PP_THREADS) plan(i, 0);
  if (k == p.g - 1)
    for (int i = b + threadIdx.x; i < p.n; i += PP_THREADS) plan(i, 0);
}

// A plan that spares fewer than `least` rows (each sharing member's shared rows, less
// once a group) shares nothing.
__global__ void __launch_bounds__(PP_THREADS) prefix_least_kernel(const PrefixPlanParams p) {
  __shared__ long long part[PP_THREADS / 32];
  griddep_wait();
  griddep_launch_dependents();
  long long spared = 0;
  for (int i = threadIdx.x; i < p.n; i += PP_THREADS) spared += (long long)p.skip[i] * p.page_size;
  for (int k = threadIdx.x; k < p.g; k += PP_THREADS) spared -= p.prefix[k];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) spared += __shfl_xor_sync(0xffffffffu, spared, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = spared;
  __syncthreads();
  spared = 0;
  for (int w = 0; w < PP_THREADS / 32; ++w) spared += part[w];
  if (spared >= p.least) return;
  for (int i = threadIdx.x; i < p.n; i += PP_THREADS) {
    p.own_lens[i] += p.skip[i] * p.page_size;
    p.skip[i] = 0;
  }
  for (int k = threadIdx.x; k < p.g; k += PP_THREADS) p.prefix[k] = 0;
}

cudaError_t prefix_plan_launch(const PrefixPlanParams& p, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs || p.g < 1 || p.g > kPagedMaxSeqs) return cudaErrorInvalidValue;
  DFL_TRY(launch_pdl(prefix_plan_kernel, dim3(p.g), dim3(PP_THREADS), ((size_t)3 * p.g + 1) * sizeof(int), st, p));
  // (nothing spares 2^42 rows, 2,048 requests of 2^31: the first kernel has then shared nothing)
  if (p.g == 1 || p.least <= 0 || p.least > 1ll << 42) return cudaSuccess;
  return launch_pdl(prefix_least_kernel, dim3(1), dim3(PP_THREADS), 0, st, p);
}

}  // namespace dfl
