// Pages of the paged cache that several requests hold: fork, reserve with copy
// on write, release that counts holders, and the copies themselves.
//
// A page's count is the number of requests beyond the first that hold it, so
// pages fresh off the free list need no entry.  Fork copies table rows and
// counts; it moves no cached row.  Before a request writes into a page that
// others hold (the last page it holds rows on, when that is not full), reserve
// gives it a page of its own: of all requests that write into one page in a call,
// the first ones in order take copies, as many as there are other holders; where
// every holder writes, the last one keeps the page.  (Pages behind a request's
// rows, left there by a trim, must be its own: release gives the others up.)
// Release returns a page when its last holder gives it up, in the order of (request,
// column) of that.
//
// All but the copies is latency, of searches, table entries and counts that wait for
// one another (512 requests: reserve and release 9 us each, 16 with cold tables):
// they run as one cluster of 8 CTAs, whose barrier (0.3 us) separates reading the
// tables and counts from changing them, where a second launch would cost 2 us.  The copies stream: 2304 bytes for
// every 16 rows of a kv head, of all layers in one launch, and only the row
// blocks that hold rows.
#include "paged_scan.cuh"

namespace dfl {

constexpr int SH_CTAS = 8;

__device__ __forceinline__ void cluster_sync() {
  cluster_arrive_release();
  cluster_wait_acquire();
}
__device__ __forceinline__ int ld_cluster_int(const int* local, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(local, rank)) : "memory");
  return v;
}

// ---- fork: a warp per 256 columns of a pair's table row
__global__ void __launch_bounds__(PG_THREADS) paged_fork_kernel(const ForkParams p) {
  extern __shared__ int first[];   // [n] the first pair that names the request as its destination
  griddep_wait();
  griddep_launch_dependents();
  for (int i = threadIdx.x; i < p.n; i += PG_THREADS) first[i] = INT32_MAX;
  __syncthreads();
  for (int j = threadIdx.x; j < p.m; j += PG_THREADS) {
    const int d = __ldg(p.dst + j);
    if (d >= 0 && d < p.n) atomicMin(&first[d], j);
  }
  __syncthreads();
  auto held = [&](int i) { return min(max(__ldg(p.pages + i), 0), p.max_pages); };
  auto good = [&](int j) {   // an empty destination, named once before, and a source
    const int s = __ldg(p.src + j), d = __ldg(p.dst + j);
    return s >= 0 && s < p.n && d >= 0 && d < p.n && first[d] == j && __ldg(p.pages + d) <= 0 && __ldg(p.lens + d) <= 0;
  };
  auto length = [&](int j) {   // rows that the fork takes over; its pages follow from them
    const int s = __ldg(p.src + j);
    int len = max(__ldg(p.lens + s), 0);
    if (p.rows) len = min(len, max(__ldg(p.rows + j), 0));
    return (int)min((long long)len, (long long)held(s) * p.page_size);
  };
  if (blockIdx.x == 0) {
    int bits = 0;
    for (int j = threadIdx.x; j < p.m; j += PG_THREADS) bits |= good(j) ? 0 : kPagedFork;
    if (bits && p.status) atomicOr(p.status, bits);
    for (int i = threadIdx.x; i < p.n; i += PG_THREADS) {
      const int j = first[i];
      const bool forked = j < p.m && good(j);
      const int len = forked ? length(j) : 0;
      p.lens_out[i] = forked ? len : __ldg(p.lens + i);
      p.pages_out[i] = forked ? (len + p.page_size - 1) / p.page_size : __ldg(p.pages + i);
      if (forked && p.refused) p.refused[i] = 0;
    }
  }
  const int chunks = (p.max_pages + 255) / 256, lane = threadIdx.x & 31;
  const int warps = gridDim.x * (PG_THREADS / 32);
  for (long long w = blockIdx.x * (PG_THREADS / 32) + (threadIdx.x >> 5); w < (long long)p.m * chunks; w += warps) {
    const int j = (int)(w / chunks), c0 = (int)(w - (long long)j * chunks) * 256;
    if (!good(j)) continue;
    const int take = (length(j) + p.page_size - 1) / p.page_size;
    const int32_t* from = p.table + (size_t)__ldg(p.src + j) * p.table_ld;
    int32_t* to = p.table + (size_t)__ldg(p.dst + j) * p.table_ld;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = c0 + 32 * k + lane;
      if (c >= take) break;
      const int page = from[c];
      to[c] = page;
      if (page >= 0 && page < p.num_pages) atomicAdd(p.holders + page, 1);
    }
  }
}

// ---- reserve, as paged_reserve_kernel, and copies of pages that are written into.
// A request that writes into a shared page counts as one that needs a page, also
// the one that ends up keeping it: after the first that finds too few, it is
// turned away too, for one before it may still hold the page.
__global__ void __launch_bounds__(PG_THREADS) paged_reserve_forked_kernel(const ReserveParams p, int32_t* holders, int32_t* copies) {
  extern __shared__ __align__(16) int words[];
  const int n = p.n, n4 = (n + 3) & ~3;
  int* tail = words;                // [n4] page written into, -1: it is the request's own (read 16 bytes at a time)
  int* first_row = tail + n4;       // [n]
  int* first_need = first_row + n;  // [n]
  int* len = first_need + n;        // [n]
  int* held = len + n;              // [n] pages held before; -1 - held when turned away
  uint8_t* state = reinterpret_cast<uint8_t*>(held + n);   // [n] bit 0: cannot be served, 1: writes into a shared page, 2: takes a copy
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  griddep_wait();
  griddep_launch_dependents();
  const int head = min(max(__ldg(p.head), 0), p.num_pages);
  const int room = p.num_pages - head;
  const bool writer = blockIdx.x == 0;
  int bits = 0;
  long long carry_r = 0;
  bool shares = false;
  for (int i0 = 0; i0 < n4; i0 += PG_THREADS) {
    const int i = i0 + threadIdx.x;
    const int li = i < n ? max(__ldg(p.lens + i), 0) : 0;
    const int ni = i < n ? max(__ldg(p.new_rows + i), 0) : 0;
    const int hi = i < n ? max(__ldg(p.pages + i), 0) : 0;
    const long long want = ((long long)li + ni + p.page_size - 1) / p.page_size;
    long long rows = ni, tot_r;
    int zero = 0, tot_z;
    block_scan2(rows, zero, &tot_r, &tot_z);
    const long long row_end = carry_r + rows;
    carry_r += tot_r;
    const bool too_long = want > p.max_pages, over = row_end > p.num_slots;
    auto shared = [&](int c) {   // the page of column c, -1: it is the request's own
      const int page = p.table[(size_t)i * p.table_ld + c];
      return page >= 0 && page < p.num_pages && holders[page] > 0 ? page : -1;
    };
    int page = -1;
    bool surplus = false;
    if (i < n && ni > 0 && !too_long && !over) {
      for (int c = (li + p.page_size - 1) / p.page_size; c < min(hi, (int)want); ++c) surplus = surplus || shared(c) >= 0;
      if (!surplus && li % p.page_size && li / p.page_size < hi) page = shared(li / p.page_size);
    }
    if (i < n4) tail[i] = page;
    shares = shares || page >= 0;
    if (i < n) {
      first_row[i] = (int)min(row_end - ni, (long long)INT32_MAX);
      len[i] = li;
      held[i] = hi;
      state[i] = (too_long || over || surplus ? 1 : 0) | (page >= 0 ? 2 : 0);
      if (writer) {
        bits |= (too_long ? kPagedLong : 0) | (over ? kPagedSlots : 0) | (surplus ? kPagedSurplus : 0);
        p.starts[i + 1] = (int)min(row_end, (long long)INT32_MAX);
      }
    }
  }
  if (__syncthreads_or(shares)) {
    // how many requests before it write into the same page
    for (int i = threadIdx.x; i < n; i += PG_THREADS) {
      const int page = tail[i];
      if (page < 0) continue;
      int rank = 0;
      for (int k = 0; k < i; k += 4) {
        const int4 t = *reinterpret_cast<const int4*>(tail + k);
        rank += (t.x == page) + (k + 1 < i && t.y == page) + (k + 2 < i && t.z == page) + (k + 3 < i && t.w == page);
      }
      if (rank < holders[page]) state[i] |= 4;
    }
    __syncthreads();
  }
  int carry_p = 0;
  for (int i0 = 0; i0 < n; i0 += PG_THREADS) {
    const int i = i0 + threadIdx.x;
    int need = 0, li = 0, ni = 0, hi = 0, want = 0, st = 1;
    if (i < n) {
      li = len[i];
      hi = held[i];
      st = state[i];
      ni = max(__ldg(p.new_rows + i), 0);
      if (!(st & 1)) {
        want = (int)(((long long)li + ni + p.page_size - 1) / p.page_size);
        need = max(want - hi, 0) + (st >> 2 & 1);
      }
    }
    int upto = need, tot_p;
    long long zl = 0, tot_zl;
    block_scan2(zl, upto, &tot_zl, &tot_p);
    upto += carry_p;
    const bool dry = (need > 0 || (st & 2)) && upto > room;
    const bool served = !(st & 1) && !dry;
    if (i < n) {
      first_need[i] = upto - need;
      if (!served) held[i] = -1 - hi;
      if (served && need > 0) atomicMax(&taken, upto);
      if (writer) {
        bits |= dry ? kPagedDry : 0;
        p.lens_out[i] = served ? li + ni : li;
        p.pages_out[i] = served ? max(hi, want) : hi;
        if (p.refused && ni > 0) p.refused[i] = !served;
      }
    }
    carry_p = (int)min((long long)carry_p + tot_p, (long long)INT32_MAX / 2);
  }
  if (writer && bits && p.status) atomicOr(p.status, bits);
  cluster_sync();   // tables and counts are read by all, and now change
  if (writer && threadIdx.x == 0) {
    p.starts[0] = 0;
    *p.head_out = head + taken;
  }
  const int tid = blockIdx.x * PG_THREADS + threadIdx.x, stride = gridDim.x * PG_THREADS;
  auto copied = [&](int i) { return held[i] >= 0 ? state[i] >> 2 & 1 : 0; };
  for (int i = tid; i < n; i += stride) {
    int from = -1, to = -1, rows = 0;
    if (copied(i)) {
      from = tail[i];
      to = __ldg(p.free_pages + head + first_need[i]);
      rows = len[i] % p.page_size;
      p.table[(size_t)i * p.table_ld + len[i] / p.page_size] = to;
      atomicAdd(holders + from, -1);
    }
    copies[3 * i] = from;
    copies[3 * i + 1] = to;
    copies[3 * i + 2] = rows;
  }
  for (int t = tid; t < taken; t += stride) {
    const int i = last_le(first_need, n, t), k = t - first_need[i] - copied(i);
    if (k >= 0) p.table[(size_t)i * p.table_ld + held[i] + k] = __ldg(p.free_pages + head + t);
  }
  const int total = (int)min(carry_r, (long long)p.num_slots);
  for (int r = tid; r < p.num_slots; r += stride) {
    int slot = -1;
    if (r < total) {
      const int i = last_le(first_row, n, r);
      if (held[i] >= 0) {
        const int pos = len[i] + r - first_row[i];
        const int pg = pos / p.page_size, mine = copied(i);
        const int entry = pg >= held[i] ? __ldg(p.free_pages + head + first_need[i] + mine + pg - held[i])
                          : mine && pg == len[i] / p.page_size ? __ldg(p.free_pages + head + first_need[i])
                                                               : p.table[(size_t)i * p.table_ld + pg];
        if (entry >= 0 && entry < INT32_MAX / p.page_size) slot = entry * p.page_size + pos % p.page_size;
      }
    }
    p.slots[r] = slot;
  }
}

// ---- release: pages beyond those kept are given up; the last holder's come back
__global__ void __launch_bounds__(PG_THREADS) paged_release_forked_kernel(const ReleaseParams p, int32_t* holders) {
  extern __shared__ int sm[];
  const int n = p.n;
  int* first = sm;         // [n] pages given up before this request
  int* left = first + n;   // [n] pages kept
  __shared__ int warp_back[PG_THREADS / 32], cta_back;
  griddep_wait();
  griddep_launch_dependents();
  const int head = min(max(__ldg(p.head), 0), p.num_pages);
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += PG_THREADS) {
    const int i = i0 + threadIdx.x;
    const int ki = i < n ? max(__ldg(p.keep + i), 0) : 0;
    const int hi = i < n ? min(max(__ldg(p.pages + i), 0), p.max_pages) : 0;
    const int li = min(hi, (int)(((long long)ki + p.page_size - 1) / p.page_size));
    int upto = hi - li, tot;
    long long zl = 0, tot_zl;
    block_scan2(zl, upto, &tot_zl, &tot);
    if (i < n) {
      first[i] = total + upto - (hi - li);
      left[i] = li;
    }
    total += tot;
  }
  __syncthreads();
  int32_t* last = holders + p.num_pages;
  auto page_of = [&](int t) {   // -1 where it is none of the pool's
    const int i = last_le(first, n, t);
    const int page = __ldg(p.table + (size_t)i * p.table_ld + left[i] + (t - first[i]));
    return page >= 0 && page < p.num_pages ? page : -1;
  };
  const int tid = blockIdx.x * PG_THREADS + threadIdx.x, stride = gridDim.x * PG_THREADS;
  int bits = 0;
  for (int t = tid; t < total; t += stride) {
    const int page = page_of(t);
    if (page < 0) {
      bits |= kPagedCorrupt;
      continue;
    }
    atomicAdd(holders + page, -1);
    atomicMax(last + page, t + 1);
  }
  cluster_sync();
  // the pages that come back: a run of the given-up ones for each warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = gridDim.x * (PG_THREADS / 32);
  const int me = blockIdx.x * (PG_THREADS / 32) + warp;
  const int t0 = (int)((long long)total * me / warps), t1 = (int)((long long)total * (me + 1) / warps);
  auto returns = [&](int t, int* page) {
    *page = page_of(t);
    if (*page < 0) return false;
    const int c = __ldcg(holders + *page);
    if (c < -1) bits |= kPagedCorrupt;
    return c < 0 && __ldcg(last + *page) == t + 1;
  };
  int back = 0;
#pragma unroll 4
  for (int t = t0 + lane; t < t1; t += 32) {
    int page;
    back += returns(t, &page);
  }
  back = __reduce_add_sync(0xffffffffu, back);
  if (lane == 0) warp_back[warp] = back;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int w = 0; w < PG_THREADS / 32; ++w) s += warp_back[w];
    cta_back = s;
  }
  cluster_sync();
  int before = 0, all = 0;
  for (int k = 0; k < (int)gridDim.x; ++k) {
    const int v = ld_cluster_int(&cta_back, k);
    if (k < (int)blockIdx.x) before += v;
    all += v;
  }
  for (int w = 0; w < warp; ++w) before += warp_back[w];
  const bool bad = all > head;
  if (bad) bits |= kPagedCorrupt;
  if (!bad) {
    int at = head - all + before;
    for (int b = t0; b < t1; b += 32) {
      const int t = b + lane;
      int page = -1;
      const bool r = t < t1 && returns(t, &page);
      const uint32_t mask = __ballot_sync(0xffffffffu, r);
      if (r) p.free_pages[at + __popc(mask & ((1u << lane) - 1))] = page;
      at += __popc(mask);
    }
  }
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < n; i += PG_THREADS) p.pages_out[i] = bad ? __ldg(p.pages + i) : left[i];
    if (threadIdx.x == 0) *p.head_out = bad ? head : head - all;
  }
  cluster_sync();   // counts are read
  for (int t = tid; t < total; t += stride) {
    const int page = page_of(t);
    if (page < 0) continue;
    if (bad)
      atomicAdd(holders + page, 1);
    else if (__ldcg(holders + page) < 0)
      holders[page] = 0;
    last[page] = 0;
  }
  if (bits && p.status) atomicOr(p.status, bits);
}

// ---- copies: the CTAs share the (copy, layer) pairs out evenly.  A page that many
// requests fork from is read by many copies, from L2 (plain loads), and what is written
// leaves the caches first: 480 copies from 32 pages over 16 layers, 323 MB written, take
// 63 us (5.1 TB/s), with streaming loads 65, with ordinary stores 66, with both 72.
constexpr int CP_THREADS = 256, CP_FLY = 4;
__global__ void __launch_bounds__(CP_THREADS) q4_copy_kernel(const __grid_constant__ CopyParams p) {
  __shared__ int list[kPagedMaxSeqs];   // the copies to make, in order
  __shared__ int warp_count[CP_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch_dependents();
  int count = 0;
  for (int i0 = 0; i0 < p.n; i0 += CP_THREADS) {
    const int i = i0 + threadIdx.x;
    bool there = false;
    if (i < p.n) {
      const int from = __ldg(p.copies + 3 * i), to = __ldg(p.copies + 3 * i + 1);
      there = from >= 0 && from < p.num_pages && to >= 0 && to < p.num_pages && from != to && __ldg(p.copies + 3 * i + 2) > 0;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, there);
    if (lane == 0) warp_count[warp] = __popc(mask);
    __syncthreads();
    int at = count + __popc(mask & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < CP_THREADS / 32; ++w) {
      if (w < warp) at += warp_count[w];
      count += warp_count[w];
    }
    if (there) list[at] = i;
    __syncthreads();
  }
  const int blocks_page = 1 << (p.page_shift - 4);
  const size_t page_bytes = (size_t)p.nkv * blocks_page * kQ4Block;
  for (long long u = blockIdx.x; u < (long long)count * p.layers; u += gridDim.x) {
    const int layer = (int)(u / count), i = list[u - (long long)layer * count];
    const int blocks = min((__ldg(p.copies + 3 * i + 2) + kQ4Rows - 1) / kQ4Rows, blocks_page);
    const uint8_t* from = p.pools[layer] + __ldg(p.copies + 3 * i) * page_bytes;
    uint8_t* to = p.pools[layer] + __ldg(p.copies + 3 * i + 1) * page_bytes;
    const int run = blocks * (kQ4Block / 16), total = run * p.nkv;   // 16-byte pieces of a head, of all
    for (int e0 = threadIdx.x; e0 < total; e0 += CP_FLY * CP_THREADS) {
      uint4 w[CP_FLY];
      int at[CP_FLY];
#pragma unroll
      for (int k = 0; k < CP_FLY; ++k) {
        const int e = e0 + k * CP_THREADS, head = e / run;
        at[k] = head * blocks_page * (kQ4Block / 16) + e - head * run;
        if (e < total) w[k] = __ldcg(reinterpret_cast<const uint4*>(from) + at[k]);
      }
#pragma unroll
      for (int k = 0; k < CP_FLY; ++k)
        if (e0 + k * CP_THREADS < total) __stcs(reinterpret_cast<uint4*>(to) + at[k], w[k]);
    }
  }
}

cudaError_t paged_fork_launch(const ForkParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs || p.m < 1 || p.m > kPagedMaxSeqs) return cudaErrorInvalidValue;
  const long long warps = (long long)p.m * ((p.max_pages + 255) / 256), ctas = (warps + PG_THREADS / 32 - 1) / (PG_THREADS / 32);
  return launch_pdl(paged_fork_kernel, dim3((int)(ctas < num_sms ? ctas : num_sms)), dim3(PG_THREADS), (size_t)p.n * 4, st, p);
}

cudaError_t paged_reserve_forked_launch(const ReserveParams& p, int32_t* holders, int32_t* copies, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  const size_t smem = ((size_t)p.n + 3) / 4 * 16 + (size_t)p.n * 17;
  return launch_pdl_cluster_smem(paged_reserve_forked_kernel, dim3(SH_CTAS), dim3(PG_THREADS), SH_CTAS, smem, st, p, holders, copies);
}

cudaError_t paged_release_forked_launch(const ReleaseParams& p, int32_t* holders, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs) return cudaErrorInvalidValue;
  return launch_pdl_cluster_smem(paged_release_forked_kernel, dim3(SH_CTAS), dim3(PG_THREADS), SH_CTAS, (size_t)p.n * 8, st, p, holders);
}

cudaError_t q4_copy_launch(const CopyParams& p, int num_sms, cudaStream_t st) {
  if (p.n < 1 || p.n > kPagedMaxSeqs || p.layers < 1 || p.layers > kCopyPools) return cudaErrorInvalidValue;
  const long long units = (long long)p.n * p.layers;
  // (16 CTAs an SM in all: 8 take 68 us, 64 65)
  return launch_pdl(q4_copy_kernel, dim3((int)(units < 16 * num_sms ? units : 16 * num_sms)), dim3(CP_THREADS), 0, st, p);
}

}  // namespace dfl
