// Block tables and slot maps of the paged cache, built on the GPU from the
// requests' lengths (no host round trip between acceptance, which sets the
// lengths on the device, and the next step's cache writes).
//
// Reserve and release are prefix sums over at most 2048 requests followed by an
// even spread of small copies.  They move a few bytes per request and row, so
// what bounds them is latency: one launch, in which every CTA repeats the
// prefix sums for itself (the requests' counts are a few KB out of L2) instead
// of waiting for another CTA, and then writes its own share.  Calls one after
// another take 5.5 us (reserve, 1 or 256 requests), 4.2 us (release, 256) and
// 5.7 to 6.7 us (release, 1,000 requests with 250 finished, 0.6 MB of table read);
// all but the last are bound by the host's 4 to 7 us a call.
#include "paged_scan.cuh"

namespace dfl {

// Requests are served in order.  need = pages beyond those held; a request
// whose inclusive prefix of needs passes the free pages gets none, so neither
// does any later one that needs a page.  Row r of request i (rows packed in
// order) lies at position len + r - starts[i]; its page is the table's where
// the request held it already, else the free list's, so no thread reads a
// table entry that another one writes.
__global__ void __launch_bounds__(PG_THREADS) paged_reserve_kernel(const ReserveParams p) {
  extern __shared__ int sm[];
  const int n = p.n;
  int* first_row = sm;              // [n] packed row at which the request starts (clamped)
  int* first_need = first_row + n;  // [n] pages taken before it
  int* len = first_need + n;        // [n]
  int* held = len + n;              // [n] pages held before; -1 - held when turned away
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const int head = min(max(__ldg(p.head), 0), p.num_pages);
  const int room = p.num_pages - head;
  long long carry_r = 0;
  int carry_p = 0, bits = 0;
  const bool writer = blockIdx.x == 0;
  for (int i0 = 0; i0 < n; i0 += PG_THREADS) {
    const int i = i0 + threadIdx.x;
    const int li = i < n ? max(__ldg(p.lens + i), 0) : 0;
    const int ni = i < n ? max(__ldg(p.new_rows + i), 0) : 0;
    const int hi = i < n ? max(__ldg(p.pages + i), 0) : 0;
    // (li + ni) rows in 64 bits: arguments are device data the host has not seen
    const long long want = ((long long)li + ni + p.page_size - 1) / p.page_size;
    const bool too_long = want > p.max_pages;
    long long rows = ni, tot_r;
    // whether the slots hold this request's rows needs the row prefix first
    int zero = 0, tot_z;
    block_scan2(rows, zero, &tot_r, &tot_z);
    const long long row_end = carry_r + rows;
    const bool over = row_end > p.num_slots;
    const int need = (too_long || over || want <= hi) ? 0 : (int)want - hi;
    int upto = need, tot_p;
    long long zl = 0, tot_zl;
    block_scan2(zl, upto, &tot_zl, &tot_p);
    upto += carry_p;
    const bool dry = need > 0 && upto > room;
    const bool served = !(too_long || over || dry);
    if (i < n) {
      first_row[i] = (int)min(row_end - ni, (long long)INT32_MAX);
      first_need[i] = upto - need;
      len[i] = li;
      held[i] = served ? hi : -1 - hi;
      if (served && need > 0) atomicMax(&taken, upto);
      if (writer) {
        bits |= (dry ? kPagedDry : 0) | (too_long ? kPagedLong : 0) | (over ? kPagedSlots : 0);
        p.starts[i + 1] = (int)min(row_end, (long long)INT32_MAX);
        p.lens_out[i] = served ? li + ni : li;
        p.pages_out[i] = served ? max(hi, (int)want) : hi;
        if (p.refused && ni > 0) p.refused[i] = !served;
      }
    }
    carry_r += tot_r;
    carry_p = (int)min((long long)carry_p + tot_p, (long long)INT32_MAX / 2);
  }
  if (writer && bits && p.status) atomicOr(p.status, bits);
  __syncthreads();
  if (writer && threadIdx.x == 0) {
    p.starts[0] = 0;
    *p.head_out = head + taken;
  }
  const int tid = blockIdx.x * PG_THREADS + threadIdx.x, stride = gridDim.x * PG_THREADS;
  // pages into the table
  for (int t = tid; t < taken; t += stride) {
    const int i = last_le(first_need, n, t);  // the last of equal prefixes is the one that needs the page
    p.table[(size_t)i * p.table_ld + held[i] + (t - first_need[i])] = __ldg(p.free_pages + head + t);
  }
  // slots of the new rows
  const int total = (int)min(carry_r, (long long)p.num_slots);
  for (int r = tid; r < p.num_slots; r += stride) {
    int slot = -1;
    if (r < total) {
      const int i = last_le(first_row, n, r);
      if (held[i] >= 0) {
        const int pos = len[i] + r - first_row[i];
        const int pg = pos / p.page_size;
        const int entry = pg < held[i] ? p.table[(size_t)i * p.table_ld + pg]
                                       : __ldg(p.free_pages + head + first_need[i] + pg - held[i]);
        // (append and attention check pages against their pool; here only the product has to fit)
        if (entry >= 0 && entry < INT32_MAX / p.page_size) slot = entry * p.page_size + pos % p.page_size;
      }
    }
    p.slots[r] = slot;
  }
}

// Request i keeps ceil(keep / page_size) of its pages; the others go back to
// the free list below its head, in order of (request, table column).
__global__ void __launch_bounds__(PG_THREADS) paged_release_kernel(const ReleaseParams p) {
  extern __shared__ int sm[];
  const int n = p.n;
  int* first = sm;         // [n] pages given back before this request
  int* left = first + n;   // [n] pages kept
  griddep_wait();
  griddep_launch_dependents();
  const int head = min(max(__ldg(p.head), 0), p.num_pages);
  int carry = 0;
  for (int i0 = 0; i0 < n; i0 += PG_THREADS) {
    const int i = i0 + threadIdx.x;
    const int ki = i < n ? max(__ldg(p.keep + i), 0) : 0;
    const int hi = i < n ? min(max(__ldg(p.pages + i), 0), p.max_pages) : 0;
    const int li = min(hi, (int)(((long long)ki + p.page_size - 1) / p.page_size));
    int upto = hi - li, tot;
    long long zl = 0, tot_zl;
    block_scan2(zl, upto, &tot_zl, &tot);
    if (i < n) {
      first[i] = carry + upto - (hi - li);
      left[i] = li;
    }
    carry += tot;
  }
  __syncthreads();
  const bool bad = carry > head;
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < n; i += PG_THREADS) p.pages_out[i] = bad ? __ldg(p.pages + i) : left[i];
    if (threadIdx.x == 0) {
      *p.head_out = bad ? head : head - carry;
      if (bad && p.status) atomicOr(p.status, kPagedCorrupt);
    }
  }
  if (bad) return;
  const int stride = gridDim.x * PG_THREADS;
  for (int t = blockIdx.x * PG_THREADS + threadIdx.x; t < carry; t += stride) {
    const int i = last_le(first, n, t);
    p.free_pages[head - carry + t] = __ldg(p.table + (size_t)i * p.table_ld + left[i] + (t - first[i]));
  }
}

__global__ void __launch_bounds__(256) paged_trim_kernel(const int32_t* lens, const int32_t* counts, int count,
                                                         const int32_t* refused, int n, int32_t* lens_out) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (i >= n) return;
  const int drop = refused && refused[i] ? 0 : max(counts ? counts[i] : count, 0);
  lens_out[i] = max(max(lens[i], 0) - drop, 0);
}

cudaError_t paged_reserve_launch(const ReserveParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  const int want = (p.num_slots + 4 * PG_THREADS - 1) / (4 * PG_THREADS);
  const int grid = want < 1 ? 1 : want > num_sms ? num_sms : want;
  return launch_pdl(paged_reserve_kernel, dim3(grid), dim3(PG_THREADS), (size_t)p.n * 16, st, p);
}

cudaError_t paged_release_launch(const ReleaseParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  const long long want = ((long long)p.n * p.max_pages + 16 * PG_THREADS - 1) / (16 * PG_THREADS);
  const int grid = want < 1 ? 1 : want > num_sms ? num_sms : (int)want;
  return launch_pdl(paged_release_kernel, dim3(grid), dim3(PG_THREADS), (size_t)p.n * 8, st, p);
}

cudaError_t paged_trim_launch(const int32_t* lens, const int32_t* counts, int count, const int32_t* refused, int n,
                              int32_t* lens_out, cudaStream_t st) {
  return launch_pdl(paged_trim_kernel, dim3((n + 255) / 256), dim3(256), 0, st, lens, counts, count, refused, n, lens_out);
}

}  // namespace dfl
