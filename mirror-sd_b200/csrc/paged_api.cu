// C ABI of the paged 4-bit K/V cache (include/dflash_b200.h): argument checks
// and launches of paged.cu, q4_cache.cu and q4_attention.cu.
#include <algorithm>
#include <cmath>

#include "api_error.cuh"
#include "q4_attn.cuh"

using namespace dfl;

namespace {

bool page_size_ok(int page_size) { return page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int page_size) {
  int b = 0;
  while ((1 << b) < page_size) ++b;
  return b;
}

int num_sms(int* sms) {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  CK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return DFLASH_OK;
}

int check_paging(int n, int page_size, long long table_ld, int max_pages, int num_pages) {
  if (n < 1 || n > DFLASH_PAGED_MAX_SEQS)
    return fail(DFLASH_ERR_INVALID, "n %d outside [1, %d]", n, DFLASH_PAGED_MAX_SEQS);
  if (!page_size_ok(page_size))
    return fail(DFLASH_ERR_INVALID, "page_size must be 16, 32, 64, 128 or 256 (got %d)", page_size);
  if (max_pages < 1 || table_ld < max_pages)
    return fail(DFLASH_ERR_INVALID, "max_pages %d, table_ld %lld", max_pages, table_ld);
  if ((long long)n * max_pages > INT32_MAX || (long long)max_pages * page_size > INT32_MAX)
    return fail(DFLASH_ERR_INVALID, "block table of %d x %d entries is too large", n, max_pages);
  if (num_pages < 0 || (long long)num_pages * page_size > INT32_MAX)
    return fail(DFLASH_ERR_INVALID, "num_pages %d (x page_size must stay below 2^31)", num_pages);
  return DFLASH_OK;
}

int check_pool(int rows, int nkv, const void* pool, int num_pages, int page_size) {
  if (rows < 0 || nkv < 1 || nkv > 65535) return fail(DFLASH_ERR_INVALID, "rows %d, nkv %d", rows, nkv);
  if (!page_size_ok(page_size))
    return fail(DFLASH_ERR_INVALID, "page_size must be 16, 32, 64, 128 or 256 (got %d)", page_size);
  if (num_pages < 1 || (long long)num_pages * page_size > INT32_MAX)
    return fail(DFLASH_ERR_INVALID, "num_pages %d (x page_size must stay below 2^31)", num_pages);
  if (!aligned16(pool)) return fail(DFLASH_ERR_INVALID, "pool must be 16-byte aligned");
  return DFLASH_OK;
}

// whether out [rows, nq, 128] touches a row of q (strides in elements)
bool overlap(const uint16_t* out, const uint16_t* q, long long q_row, long long q_head, long long rows, int nq) {
  const long long heads = (nq - 1) * q_head, all = (rows - 1) * q_row;
  const long long span = (heads < 0 ? -heads : heads) + 128, stride = q_row < 0 ? -q_row : q_row;   // a row's elements
  const long long lowest = (heads < 0 ? heads : 0) + (all < 0 ? all : 0);
  // out in elements from q's lowest one on: [a, b)
  const long long a = ((long long)(uintptr_t)out - (long long)(uintptr_t)q) / 2 - lowest, b = a + rows * nq * 128;
  if (b <= 0) return false;
  if (stride == 0) return a < span;
  const long long first = a < span ? 0 : (a - span) / stride + 1;   // first row that ends behind a
  return first < rows && first * stride < b;
}

constexpr size_t kCounterBytes = 4096;   // two counters per SM, then the partials

// Checks of an attention call and its parameters; n, rows and max_rows of the
// pass.  *few: which kernel (up to 16 query rows a kv head each warp multiplies on
// its own (mma.sync, no hand-over between warps); above, tcgen05 with the rows as
// columns).
int attention_params(const uint16_t* q, int64_t q_row, int64_t q_head, int bf16, const uint8_t* pool, int num_pages, int page_size,
                     const int32_t* table, int64_t table_ld, int max_pages, const int32_t* lens, const int32_t* starts, int n,
                     int rows, int max_rows, int nq, int nkv, int causal, int sink, int window, float scale, uint16_t* out,
                     int32_t* status, int item_units, Q4AttnParams* params, bool* few) {
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  if (int rc = check_pool(rows, nkv, pool, num_pages, page_size)) return rc;
  // (the kernels add a tile, a window or the query rows to a position in 32 bits)
  if ((long long)max_pages * page_size > 1ll << 30)
    return fail(DFLASH_ERR_INVALID, "%d pages of %d rows a request: at most 2^30 rows", max_pages, page_size);
  if (nq < nkv || nq % nkv) return fail(DFLASH_ERR_INVALID, "nq %d must be a multiple of nkv %d", nq, nkv);
  if (max_rows < 1 || max_rows > DFLASH_Q4_MAX_ROWS)
    return fail(DFLASH_ERR_INVALID, "max_rows %d outside [1, %d]", max_rows, DFLASH_Q4_MAX_ROWS);
  if (!starts && (long long)n * max_rows != rows)
    return fail(DFLASH_ERR_INVALID, "without starts every request has max_rows rows (%d x %d, got %d)", n, max_rows, rows);
  if (sink < 0 || window < 0) return fail(DFLASH_ERR_INVALID, "sink %d, window %d", sink, window);
  if (sink > 0 && window == 0) return fail(DFLASH_ERR_INVALID, "sink needs a window (window 0 sees every row)");
  // A window as wide as the table hides nothing; the kernels subtract the others
  // from lengths less query rows, in 32 bits.
  if (window >= max_pages * page_size) sink = window = 0;
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(DFLASH_ERR_INVALID, "scale must be positive and finite");
  if (!aligned16(q) || !aligned16(out) || q_row % 8 || q_head % 8)
    return fail(DFLASH_ERR_INVALID, "q, out and workspace must be 16-byte aligned, q's strides whole 16 bytes");
  const int G = nq / nkv;
  *few = (long long)max_rows * G <= kQ4FewRows;
  const double columns = *few ? q4_attn_columns(max_rows, nq, nkv) : q4_attn_tc_columns(max_rows, nq, nkv);
  if (G > 256 || nkv > 1024 || ((double)max_rows * G / columns + 1) * nkv * nkv > 4e9)
    return fail(DFLASH_ERR_INVALID, "%d query heads a kv head, %d kv heads, %d rows: too many", G, nkv, max_rows);
  // Tiles of all items together are counted in 32 bits: a full table for each
  // group of query rows, of which every request with rows has one in part.
  // (and what the passes over shared and own rows add to an item)
  const double units = (std::ceil((double)max_pages * page_size / (*few ? kQ4Tile : kQ4TcTile)) + item_units) * nkv *
                       ((double)rows * G / columns + (n < rows ? n : rows));
  if ((long long)rows * nq > INT32_MAX) return fail(DFLASH_ERR_INVALID, "rows x nq must stay below 2^31");
  if (units >= INT32_MAX) return fail(DFLASH_ERR_INVALID, "n x table x heads x rows is too large for one call");
  Q4AttnParams& p = *params;
  p = Q4AttnParams{};
  p.q = q; p.q_row = q_row; p.q_head = q_head; p.bf16 = bf16 != 0; p.pool = pool;
  p.table = table; p.lens = lens; p.starts = starts; p.table_ld = table_ld;
  p.n = n; p.T = rows; p.max_rows = p.most_rows = max_rows; p.nq = nq; p.nkv = nkv;
  p.by_g = Divisor(G); p.by_nkv = Divisor(nkv);
  p.page_shift = log2_of(page_size);
  p.max_pages = max_pages; p.num_pages = num_pages; p.causal = causal != 0; p.sink = sink; p.window = window;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.factor = score_factor(16.f * p.scale_log2);
  p.out = out; p.status = status;
  return DFLASH_OK;
}

// The rest of the call, where there are rows: its workspace and the launch.
int attention_launch(Q4AttnParams& p, bool few, int pass, void* workspace, void* stream) {
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  if ((size_t)sms * 2 * sizeof(int) > kCounterBytes) return fail(DFLASH_ERR_INVALID, "%d SMs", sms);
  p.counters = static_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  if (few)
    CK(q4_attn_launch(p, pass, sms, static_cast<cudaStream_t>(stream)));
  else
    CK(q4_attn_tc_launch(p, pass, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

}  // namespace

extern "C" {

int dflash_paged_reserve(const int32_t* lens, const int32_t* new_rows, const int32_t* pages, int n, int page_size,
                         int32_t* table, int64_t table_ld, int max_pages, const int32_t* free_pages, int num_pages,
                         const int32_t* head, int32_t* starts, int32_t* slots, int num_slots, int32_t* lens_out,
                         int32_t* pages_out, int32_t* head_out, int32_t* status, void* stream) {
  return dflash_paged_reserve_tracked(lens, new_rows, pages, n, page_size, table, table_ld, max_pages, free_pages, num_pages,
                                      head, starts, slots, num_slots, lens_out, pages_out, head_out, nullptr, status, stream);
}

int dflash_paged_reserve_tracked(const int32_t* lens, const int32_t* new_rows, const int32_t* pages, int n, int page_size,
                                 int32_t* table, int64_t table_ld, int max_pages, const int32_t* free_pages, int num_pages,
                                 const int32_t* head, int32_t* starts, int32_t* slots, int num_slots, int32_t* lens_out,
                                 int32_t* pages_out, int32_t* head_out, int32_t* refused, int32_t* status, void* stream) {
  if (!lens || !new_rows || !pages || !table || (num_pages > 0 && !free_pages) || !head || !starts || !lens_out || !pages_out ||
      !head_out || (num_slots > 0 && !slots))
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (num_slots < 0) return fail(DFLASH_ERR_INVALID, "num_slots %d", num_slots);
  if (lens_out == lens || pages_out == pages || head_out == head)
    return fail(DFLASH_ERR_INVALID, "lens_out, pages_out and head_out must not be the inputs");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  ReserveParams p{};
  p.lens = lens; p.new_rows = new_rows; p.pages = pages; p.free_pages = free_pages; p.head = head;
  p.table = table; p.n = n; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages;
  p.num_slots = num_slots; p.table_ld = table_ld;
  p.starts = starts; p.slots = slots; p.lens_out = lens_out; p.pages_out = pages_out; p.head_out = head_out;
  p.refused = refused; p.status = status;
  CK(paged_reserve_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_paged_release(const int32_t* keep, const int32_t* pages, int n, int page_size, const int32_t* table,
                         int64_t table_ld, int max_pages, int32_t* free_pages, int num_pages, const int32_t* head,
                         int32_t* pages_out, int32_t* head_out, int32_t* status, void* stream) {
  if (!keep || !pages || !table || (num_pages > 0 && !free_pages) || !head || !pages_out || !head_out)
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (pages_out == pages || head_out == head)
    return fail(DFLASH_ERR_INVALID, "pages_out and head_out must not be the inputs");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  ReleaseParams p{};
  p.keep = keep; p.pages = pages; p.table = table; p.head = head; p.free_pages = free_pages;
  p.n = n; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages; p.table_ld = table_ld;
  p.pages_out = pages_out; p.head_out = head_out; p.status = status;
  CK(paged_release_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_paged_fork(const int32_t* src, const int32_t* dst, const int32_t* rows, int m, const int32_t* lens,
                      const int32_t* pages, int n, int page_size, int32_t* table, int64_t table_ld, int max_pages,
                      int32_t* holders, int num_pages, int32_t* lens_out, int32_t* pages_out, int32_t* refused,
                      int32_t* status, void* stream) {
  if ((m > 0 && (!src || !dst)) || !lens || !pages || !table || !holders || !lens_out || !pages_out)
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (m < 0 || m > DFLASH_PAGED_MAX_SEQS) return fail(DFLASH_ERR_INVALID, "%d forks outside [0, %d]", m, DFLASH_PAGED_MAX_SEQS);
  if (lens_out == lens || pages_out == pages) return fail(DFLASH_ERR_INVALID, "lens_out and pages_out must not be the inputs");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  if (m == 0) {
    CK(cudaMemcpyAsync(lens_out, lens, (size_t)n * 4, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream)));
    CK(cudaMemcpyAsync(pages_out, pages, (size_t)n * 4, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream)));
    return DFLASH_OK;
  }
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  ForkParams p{};
  p.src = src; p.dst = dst; p.rows = rows; p.lens = lens; p.pages = pages; p.table = table; p.holders = holders;
  p.m = m; p.n = n; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages; p.table_ld = table_ld;
  p.lens_out = lens_out; p.pages_out = pages_out; p.refused = refused; p.status = status;
  CK(paged_fork_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_paged_reserve_forked(const int32_t* lens, const int32_t* new_rows, const int32_t* pages, int n, int page_size,
                                int32_t* table, int64_t table_ld, int max_pages, const int32_t* free_pages, int num_pages,
                                const int32_t* head, int32_t* holders, int32_t* starts, int32_t* slots, int num_slots,
                                int32_t* lens_out, int32_t* pages_out, int32_t* head_out, int32_t* copies, int32_t* refused,
                                int32_t* status, void* stream) {
  if (!lens || !new_rows || !pages || !table || (num_pages > 0 && !free_pages) || !head || !holders || !starts || !lens_out ||
      !pages_out || !head_out || !copies || (num_slots > 0 && !slots))
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (num_slots < 0) return fail(DFLASH_ERR_INVALID, "num_slots %d", num_slots);
  if (lens_out == lens || pages_out == pages || head_out == head)
    return fail(DFLASH_ERR_INVALID, "lens_out, pages_out and head_out must not be the inputs");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  ReserveParams p{};
  p.lens = lens; p.new_rows = new_rows; p.pages = pages; p.free_pages = free_pages; p.head = head;
  p.table = table; p.n = n; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages;
  p.num_slots = num_slots; p.table_ld = table_ld;
  p.starts = starts; p.slots = slots; p.lens_out = lens_out; p.pages_out = pages_out; p.head_out = head_out;
  p.refused = refused; p.status = status;
  CK(paged_reserve_forked_launch(p, holders, copies, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_paged_release_forked(const int32_t* keep, const int32_t* pages, int n, int page_size, const int32_t* table,
                                int64_t table_ld, int max_pages, int32_t* free_pages, int num_pages, const int32_t* head,
                                int32_t* holders, int32_t* pages_out, int32_t* head_out, int32_t* status, void* stream) {
  if (!keep || !pages || !table || (num_pages > 0 && !free_pages) || !head || !holders || !pages_out || !head_out)
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (pages_out == pages || head_out == head)
    return fail(DFLASH_ERR_INVALID, "pages_out and head_out must not be the inputs");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, num_pages)) return rc;
  ReleaseParams p{};
  p.keep = keep; p.pages = pages; p.table = table; p.head = head; p.free_pages = free_pages;
  p.n = n; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages; p.table_ld = table_ld;
  p.pages_out = pages_out; p.head_out = head_out; p.status = status;
  CK(paged_release_forked_launch(p, holders, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_q4_copy_pages(uint8_t* const* pools, int layers, int num_pages, int nkv, int page_size, const int32_t* copies, int n,
                         void* stream) {
  if (layers < 0 || n < 0) return fail(DFLASH_ERR_INVALID, "layers %d, n %d", layers, n);
  if ((layers > 0 && !pools) || (n > 0 && !copies)) return fail(DFLASH_ERR_INVALID, "NULL pointer");
  for (int i = 0; i < layers; ++i) {
    if (!pools[i]) return fail(DFLASH_ERR_INVALID, "NULL pointer");
    if (int rc = check_pool(0, nkv, pools[i], num_pages, page_size)) return rc;
  }
  if (layers == 0 || n == 0) return DFLASH_OK;
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  CopyParams p{};
  p.nkv = nkv; p.page_shift = log2_of(page_size); p.num_pages = num_pages;
  for (int l = 0; l < layers; l += kCopyPools) {
    p.layers = layers - l < kCopyPools ? layers - l : kCopyPools;
    for (int i = 0; i < p.layers; ++i) p.pools[i] = pools[l + i];
    for (int i = 0; i < n; i += DFLASH_PAGED_MAX_SEQS) {
      p.copies = copies + 3 * (size_t)i;
      p.n = n - i < DFLASH_PAGED_MAX_SEQS ? n - i : DFLASH_PAGED_MAX_SEQS;
      CK(q4_copy_launch(p, sms, static_cast<cudaStream_t>(stream)));
    }
  }
  return DFLASH_OK;
}

int dflash_paged_trim(const int32_t* lens, const int32_t* counts, int count, const int32_t* refused, int n,
                      int32_t* lens_out, void* stream) {
  if (!lens || !lens_out) return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (n < 1 || n > DFLASH_PAGED_MAX_SEQS)
    return fail(DFLASH_ERR_INVALID, "n %d outside [1, %d]", n, DFLASH_PAGED_MAX_SEQS);
  CK(paged_trim_launch(lens, counts, count, refused, n, lens_out, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

size_t dflash_q4_page_bytes(int nkv, int page_size) {
  if (nkv < 1 || !page_size_ok(page_size)) return 0;
  return (size_t)nkv * (page_size / kQ4Rows) * kQ4Block;
}

int dflash_q4_append(const uint16_t* k, int64_t k_row, int64_t k_head, const uint16_t* v, int64_t v_row,
                     int64_t v_head, int bf16, const int32_t* slots, int rows, int nkv, uint8_t* pool, int num_pages,
                     int page_size, int32_t* status, void* stream) {
  if (!pool || (rows > 0 && (!k || !v || !slots))) return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (int rc = check_pool(rows, nkv, pool, num_pages, page_size)) return rc;
  if (!aligned16(k) || !aligned16(v) || k_row % 8 || k_head % 8 || v_row % 8 || v_head % 8)
    return fail(DFLASH_ERR_INVALID, "k and v must be 16-byte aligned with strides of whole 16 bytes");
  if (rows == 0) return DFLASH_OK;
  Q4AppendParams p{};
  p.k = k; p.v = v; p.k_row = k_row; p.k_head = k_head; p.v_row = v_row; p.v_head = v_head;
  p.bf16 = bf16 != 0; p.slots = slots; p.T = rows; p.nkv = nkv; p.page_shift = log2_of(page_size);
  p.num_slots = num_pages * page_size; p.pool = pool; p.status = status;
  CK(q4_append_launch(p, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_q4_read(const uint8_t* pool, int num_pages, int page_size, const int32_t* slots, int rows, int nkv,
                   int bf16, uint16_t* k, uint16_t* v, void* stream) {
  if (!pool || (rows > 0 && (!k || !v || !slots))) return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (int rc = check_pool(rows, nkv, pool, num_pages, page_size)) return rc;
  if (!aligned16(k) || !aligned16(v)) return fail(DFLASH_ERR_INVALID, "k and v must be 16-byte aligned");
  if (rows == 0) return DFLASH_OK;
  Q4ReadParams p{};
  p.pool = pool; p.slots = slots; p.T = rows; p.nkv = nkv; p.page_shift = log2_of(page_size);
  p.num_slots = num_pages * page_size; p.bf16 = bf16 != 0; p.k = k; p.v = v;
  CK(q4_read_launch(p, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

size_t dflash_q4_attention_workspace_size(int max_rows, int nq, int nkv) {
  if (max_rows < 1 || nkv < 1 || nq < nkv || nq % nkv) return 0;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // either kernel (fewer rows than max_rows may run in a later call)
  const size_t few = q4_attn_part_floats(max_rows, nq, nkv, sms);
  const size_t many = (long long)max_rows * (nq / nkv) <= kQ4FewRows ? 0 : q4_attn_tc_part_floats(max_rows, nq, nkv, sms);
  return kCounterBytes + (few > many ? few : many) * sizeof(float);
}

int dflash_q4_attention(const uint16_t* q, int64_t q_row, int64_t q_head, int bf16, const uint8_t* pool, int num_pages,
                        int page_size, const int32_t* table, int64_t table_ld, int max_pages, const int32_t* lens,
                        const int32_t* starts, int n, int rows, int max_rows, int nq, int nkv, int causal, int sink,
                        int window, float scale, uint16_t* out, int32_t* status, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (!pool || !table || !lens || !workspace || (rows > 0 && (!q || !out)))
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  Q4AttnParams p;
  bool few;
  if (int rc = attention_params(q, q_row, q_head, bf16, pool, num_pages, page_size, table, table_ld, max_pages, lens, starts, n,
                                rows, max_rows, nq, nkv, causal, sink, window, scale, out, status, 0, &p, &few))
    return rc;
  if (!aligned16(workspace))
    return fail(DFLASH_ERR_INVALID, "q, out and workspace must be 16-byte aligned, q's strides whole 16 bytes");
  if (workspace_bytes < dflash_q4_attention_workspace_size(max_rows, nq, nkv))
    return fail(DFLASH_ERR_INVALID, "workspace too small (%zu < %zu)", workspace_bytes,
                dflash_q4_attention_workspace_size(max_rows, nq, nkv));
  if (rows == 0) return DFLASH_OK;
  // (the kernels read q through the non-coherent path, some rows after others are finished)
  if (overlap(out, q, q_row, q_head, rows, nq)) return fail(DFLASH_ERR_INVALID, "out overlaps q");
  return attention_launch(p, few, kAttnAll, workspace, stream);
}

int dflash_paged_prefix_plan(const int32_t* table, int64_t table_ld, int max_pages, const int32_t* lens, const int32_t* starts,
                             int n, int max_rows, int page_size, const int32_t* groups, int num_groups, int causal,
                             int64_t least, int32_t* group_starts, int32_t* prefix, int32_t* row_of, int32_t* skip, int32_t* own_lens,
                             void* stream) {
  if (!table || !lens || !groups || !group_starts || !prefix || !row_of || !skip || !own_lens)
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (int rc = check_paging(n, page_size, table_ld, max_pages, 0)) return rc;
  if (max_rows < 1 || max_rows > DFLASH_Q4_MAX_ROWS)
    return fail(DFLASH_ERR_INVALID, "max_rows %d outside [1, %d]", max_rows, DFLASH_Q4_MAX_ROWS);
  if (num_groups < 1 || num_groups > DFLASH_PAGED_MAX_SEQS)
    return fail(DFLASH_ERR_INVALID, "%d groups outside [1, %d]", num_groups, DFLASH_PAGED_MAX_SEQS);
  if (least < 0) return fail(DFLASH_ERR_INVALID, "least %lld", (long long)least);
  if (own_lens == lens) return fail(DFLASH_ERR_INVALID, "own_lens must not be lens");
  PrefixPlanParams p{};
  p.table = table; p.lens = lens; p.starts = starts; p.groups = groups; p.table_ld = table_ld;
  p.n = n; p.g = num_groups; p.max_rows = max_rows; p.page_size = page_size; p.max_pages = max_pages; p.causal = causal != 0;
  p.least = least;
  p.group_starts = group_starts; p.prefix = prefix; p.row_of = row_of; p.skip = skip; p.own_lens = own_lens;
  CK(prefix_plan_launch(p, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

size_t dflash_q4_prefix_workspace_size(int rows, int max_rows, int max_group, int nq, int nkv) {
  if (rows < 0 || max_rows < 1 || max_group < 1 || (long long)max_rows * max_group > DFLASH_Q4_MAX_ROWS) return 0;
  const size_t own = dflash_q4_attention_workspace_size(max_rows, nq, nkv);
  size_t group = dflash_q4_attention_workspace_size(max_rows * max_group, nq, nkv);
  if (own == 0 || group == 0 || (long long)rows * nq > INT32_MAX) return 0;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const size_t wide = kCounterBytes + q4_attn_tc_group_floats(max_rows * max_group, nq, nkv, sms) * sizeof(float);
  if (group < wide) group = wide;
  return ((own > group ? own : group) + 15) / 16 * 16 + (size_t)rows * nq * 130 * sizeof(float);
}

int dflash_q4_prefix_attention(const uint16_t* q, int64_t q_row, int64_t q_head, int bf16, const uint8_t* pool, int num_pages,
                               int page_size, const int32_t* table, int64_t table_ld, int max_pages, const int32_t* starts,
                               int n, int rows, int max_rows, const int32_t* group_starts, const int32_t* prefix,
                               const int32_t* row_of, int num_groups, int max_group, const int32_t* skip,
                               const int32_t* own_lens, int nq, int nkv, int causal, float scale, uint16_t* out,
                               int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  if (!pool || !table || !group_starts || !prefix || !row_of || !skip || !own_lens || !workspace || (rows > 0 && (!q || !out)))
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (num_groups < 1 || num_groups > DFLASH_PAGED_MAX_SEQS)
    return fail(DFLASH_ERR_INVALID, "%d groups outside [1, %d]", num_groups, DFLASH_PAGED_MAX_SEQS);
  if (max_group < 1 || (long long)max_rows * max_group > DFLASH_Q4_MAX_ROWS)
    return fail(DFLASH_ERR_INVALID, "groups of %d requests of %d rows: at most %d rows", max_group, max_rows, DFLASH_Q4_MAX_ROWS);
  Q4AttnParams group, own;
  bool few_group, few_own;
  if (int rc = attention_params(q, q_row, q_head, bf16, pool, num_pages, page_size, table, table_ld, max_pages, own_lens, starts,
                                n, rows, max_rows, nq, nkv, causal, 0, 0, scale, out, status, kQ4ItemUnits, &own, &few_own))
    return rc;
  if (int rc = attention_params(q, q_row, q_head, bf16, pool, num_pages, page_size, table, table_ld, max_pages, prefix,
                                group_starts, num_groups, rows, max_rows * max_group, nq, nkv, 0, 0, 0, scale, out, status,
                                kQ4ItemUnits, &group, &few_group))
    return rc;
  if (!aligned16(workspace))
    return fail(DFLASH_ERR_INVALID, "q, out and workspace must be 16-byte aligned, q's strides whole 16 bytes");
  const size_t need = dflash_q4_prefix_workspace_size(rows, max_rows, max_group, nq, nkv);
  if (workspace_bytes < need) return fail(DFLASH_ERR_INVALID, "workspace too small (%zu < %zu)", workspace_bytes, need);
  if (rows == 0) return DFLASH_OK;
  if (overlap(out, q, q_row, q_head, rows, nq)) return fail(DFLASH_ERR_INVALID, "out overlaps q");
  // (the sums lie at the end, where they depend on this call's rows alone)
  const size_t sums = need - (size_t)rows * nq * 130 * sizeof(float);
  group.pre_o = own.pre_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + sums);
  group.pre_ml = own.pre_ml = reinterpret_cast<float2*>(group.pre_o + (size_t)rows * nq * 128);
  group.row_of = row_of;
  group.table_rows = n;
  // The own pass joins what the group pass leaves for every row, so a group of more rows than the caller said (on the
  // device, where nobody has looked) is taken whole: max_rows and max_group choose the kernel, any number of rows runs
  // through it.  The bounds are those of the divisions by G and nkv, x * d < 2^32: millions of rows.
  const double G = nq / nkv, columns = few_group ? q4_attn_columns(group.max_rows, nq, nkv) : q4_attn_tc_columns(group.max_rows, nq, nkv);
  const double by_g = (4294967295.0 / G - 128) / G, by_nkv = (4e9 / ((double)nkv * nkv) - 1) * columns / G;
  group.most_rows = std::max(group.most_rows, (int)std::min({by_g, by_nkv, (double)rows}));
  own.skip = skip;
  if (int rc = attention_launch(group, few_group, kAttnPrefix, workspace, stream)) return rc;
  return attention_launch(own, few_own, kAttnOwn, workspace, stream);
}

}  // extern "C"
