// C ABI of the paged 4-bit K/V cache (include/dflash_b200.h): argument checks
// and launches of paged.cu, q4_cache.cu and q4_attention.cu.
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
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || q_row % 8 || q_head % 8)
    return fail(DFLASH_ERR_INVALID, "q, out and workspace must be 16-byte aligned, q's strides whole 16 bytes");
  const int G = nq / nkv;
  // Up to 16 query rows a kv head each warp multiplies on its own (mma.sync, no
  // hand-over between warps); above, tcgen05 with the rows as columns.
  const bool few = (long long)max_rows * G <= kQ4FewRows;
  const double columns = few ? q4_attn_columns(max_rows, nq, nkv) : q4_attn_tc_columns(max_rows, nq, nkv);
  if (G > 256 || nkv > 1024 || ((double)max_rows * G / columns + 1) * nkv * nkv > 4e9)
    return fail(DFLASH_ERR_INVALID, "%d query heads a kv head, %d kv heads, %d rows: too many", G, nkv, max_rows);
  // Tiles of all items together are counted in 32 bits: a full table for each
  // group of query rows, of which every request with rows has one in part.
  const double units = std::ceil((double)max_pages * page_size / (few ? kQ4Tile : kQ4TcTile)) * nkv *
                       ((double)rows * G / columns + (n < rows ? n : rows));
  if ((long long)rows * nq > INT32_MAX) return fail(DFLASH_ERR_INVALID, "rows x nq must stay below 2^31");
  if (units >= INT32_MAX) return fail(DFLASH_ERR_INVALID, "n x table x heads x rows is too large for one call");
  if (workspace_bytes < dflash_q4_attention_workspace_size(max_rows, nq, nkv))
    return fail(DFLASH_ERR_INVALID, "workspace too small (%zu < %zu)", workspace_bytes,
                dflash_q4_attention_workspace_size(max_rows, nq, nkv));
  if (rows == 0) return DFLASH_OK;
  // (the kernels read q through the non-coherent path, some rows after others are finished)
  if (overlap(out, q, q_row, q_head, rows, nq)) return fail(DFLASH_ERR_INVALID, "out overlaps q");
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  if ((size_t)sms * 2 * sizeof(int) > kCounterBytes) return fail(DFLASH_ERR_INVALID, "%d SMs", sms);
  Q4AttnParams p{};
  p.q = q; p.q_row = q_row; p.q_head = q_head; p.bf16 = bf16 != 0; p.pool = pool;
  p.table = table; p.lens = lens; p.starts = starts; p.table_ld = table_ld;
  p.n = n; p.T = rows; p.max_rows = max_rows; p.nq = nq; p.nkv = nkv;
  p.by_g = Divisor(G); p.by_nkv = Divisor(nkv);
  p.page_shift = log2_of(page_size);
  p.max_pages = max_pages; p.num_pages = num_pages; p.causal = causal != 0; p.sink = sink; p.window = window;
  p.scale_log2 = (float)((double)scale * 1.4426950408889634);
  p.factor = score_factor(16.f * p.scale_log2);
  p.out = out; p.status = status;
  p.counters = static_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  if (few)
    CK(q4_attn_launch(p, sms, static_cast<cudaStream_t>(stream)));
  else
    CK(q4_attn_tc_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

}  // extern "C"
