// Layout of the paged 4-bit K/V cache, its number format, and the host
// launchers of its kernels (paged.cu, q4_cache.cu, q4_attention.cu).
//
// A pool holds pages of `page_size` cached rows (16, 32, 64, 128 or 256):
//   [page][kv head][page_size / 16 row blocks][kQ4Block bytes]
// A row block holds 16 rows of one kv head, K then V:
//   K values  [16 rows][64 B]           4 bits a channel
//   K scales  [16 rows][8 groups]       1 byte a group of 16 channels
//   V values  [8 row pairs][8 groups][16 B]
//   V scales  [8 groups][16 rows]
// so a block is one contiguous copy and its 16-byte pieces are the register
// fragments of a 16x16 matrix tile, K with the rows and V with the channels as
// the tile's rows:
//   K, row r, channel d = 32c + 8w + 2n + h: word w of piece (r, c), bits 16h + 4n .. + 3
//   V, row r = 2j + h, channel d = 16g + 4w + n: word w of piece (j, g), bits 16h + 4n .. + 3
// (half h of a word holds one side of a register's f16 pair).  Pieces are
// permuted inside their rows (q4_k_piece, q4_v_piece) so that 8 lanes read 8
// different 16-byte columns of shared memory whether they hold different rows
// of one piece column (a thread per cached row), or 2 rows and every piece
// (the fragments of mma.sync), or the row halves of different blocks.
//
// Numbers: a group of 16 channels of a row is x = (u - 8) * s, u the 4-bit
// code (1..15 as written here), s a scale with 5 exponent and 3 mantissa bits,
// float16's top bits below the sign: its f16 form is the byte << 7.  u - 8 has
// 3 significant bits and s has 4, so every x is exact in f16 and in bf16.
//   s = the smallest such number >= max |x| / 7.5, within [2^-17, 9216]
//   u - 8 = x / s rounded to nearest, halves away from zero, within [-7, 7]
// NaN is stored as 0 and counts as 0 in the maximum; infinities and values
// beyond 7 * 9216 saturate.  The pool therefore only ever reads back finite
// numbers, so rows hidden by a mask cannot reach a result through 0 * inf.
#pragma once
#include "common.cuh"

namespace dfl {

constexpr int kQ4Rows = 16;            // rows of a block
constexpr int kQ4KS = 1024;            // byte offsets inside a block
constexpr int kQ4V = 1152;
constexpr int kQ4VS = 2176;
constexpr int kQ4Block = 2304;
constexpr int kPagedMaxSeqs = 2048;    // requests of one call

// status bits of the paged operators (device word, or-ed)
enum PagedStatus : int {
  kPagedDry = 1,        // a request found too few free pages
  kPagedLong = 2,       // a request's rows do not fit its row of the block table
  kPagedSlots = 4,      // the new rows do not fit the slot array
  kPagedCorrupt = 8,    // more pages come back than the free list lent out
  kPagedNonFinite = 16, // an appended row held a NaN or an infinity
  kPagedTimeout = 32,   // a bounded wait of the attention kernel expired
  kPagedRows = 64,      // a request's query rows pass max_rows or lie outside the query array
  kPagedFork = 128,     // a fork names no request, or one that holds rows already
  kPagedSurplus = 256,  // new rows would go into a page of others behind the request's rows
};

// byte offsets of the pieces inside the block's K and V values
__host__ __device__ __forceinline__ int q4_k_piece(int r, int c) { return 64 * r + 16 * (c ^ (r >> 1 & 3)); }
__host__ __device__ __forceinline__ int q4_v_piece(int j, int g) { return 16 * (8 * j + (g ^ 2 * (j & 3) ^ j >> 2)); }

struct ReserveParams {
  const int32_t *lens, *new_rows, *pages, *free_pages, *head;
  int32_t* table;
  int n, page_size, max_pages, num_pages, num_slots;
  long long table_ld;
  int32_t *starts, *slots, *lens_out, *pages_out, *head_out, *refused, *status;
};
cudaError_t paged_reserve_launch(const ReserveParams& p, int num_sms, cudaStream_t st);

struct ReleaseParams {
  const int32_t *keep, *pages, *table, *head;
  int32_t* free_pages;
  int n, page_size, max_pages, num_pages;
  long long table_ld;
  int32_t *pages_out, *head_out, *status;
};
cudaError_t paged_release_launch(const ReleaseParams& p, int num_sms, cudaStream_t st);
cudaError_t paged_trim_launch(const int32_t* lens, const int32_t* counts, int count, const int32_t* refused, int n,
                              int32_t* lens_out, cudaStream_t st);

// ---- pages that several requests hold (paged_share.cu)
// holders[p], p < num_pages: the requests beyond the first that hold page p;
// holders[num_pages + p] is the kernels' own and 0 between calls.
struct ForkParams {
  const int32_t *src, *dst, *rows;   // [m]; rows NULL: all
  const int32_t *lens, *pages;       // [n]
  int32_t *table, *holders;
  int m, n, page_size, max_pages, num_pages;
  long long table_ld;
  int32_t *lens_out, *pages_out, *refused, *status;
};
cudaError_t paged_fork_launch(const ForkParams& p, int num_sms, cudaStream_t st);
// copies [n][3]: page to copy, its new page, rows; -1, -1, 0 where there is none
cudaError_t paged_reserve_forked_launch(const ReserveParams& p, int32_t* holders, int32_t* copies, cudaStream_t st);
cudaError_t paged_release_forked_launch(const ReleaseParams& p, int32_t* holders, cudaStream_t st);

constexpr int kCopyPools = 64;
struct CopyParams {
  uint8_t* pools[kCopyPools];
  const int32_t* copies;             // [n][3]
  int n, layers, nkv, page_shift, num_pages;
};
cudaError_t q4_copy_launch(const CopyParams& p, int num_sms, cudaStream_t st);

// Which rows the members of each group share, once a step (prefix_plan.cu).
struct PrefixPlanParams {
  const int32_t *table, *lens, *starts, *groups;   // starts NULL: max_rows rows each; groups [g + 1]
  long long table_ld;
  int n, g, max_rows, page_size, max_pages, causal;
  long long least;                                 // cached rows that it must spare, of all groups, to share any
  int32_t *group_starts, *prefix, *row_of;         // [g + 1], [g] rows, [g]
  int32_t *skip, *own_lens;                        // [n] columns, [n]
};
cudaError_t prefix_plan_launch(const PrefixPlanParams& p, cudaStream_t st);

struct Q4AppendParams {
  const void *k, *v;                 // [T, NKV, 128], f16 or bf16
  long long k_row, k_head, v_row, v_head;   // strides in elements
  int bf16;
  const int32_t* slots;              // [T]; outside [0, num_slots): the row is skipped
  int T, nkv, page_shift, num_slots;  // pages of 2^page_shift rows; num_slots: rows of all pages
  uint8_t* pool;
  int32_t* status;
};
cudaError_t q4_append_launch(const Q4AppendParams& p, cudaStream_t st);

struct Q4ReadParams {
  const uint8_t* pool;
  const int32_t* slots;
  int T, nkv, page_shift, num_slots, bf16;
  void *k, *v;                       // [T, NKV, 128] contiguous
};
cudaError_t q4_read_launch(const Q4ReadParams& p, cudaStream_t st);

// x / d for x * d < 2^32
struct Divisor {
  uint32_t m;
  int d;
  Divisor() = default;
  explicit Divisor(int by) : m((uint32_t)(((1ull << 32) + by - 1) / by)), d(by) {}
  __device__ __forceinline__ int of(int x) const { return d == 1 ? x : (int)__umulhi((uint32_t)x, m); }
};

struct Q4AttnParams {
  const void* q;                     // [T, NQ, 128], f16 or bf16
  long long q_row, q_head;           // strides in elements
  int bf16;
  const uint8_t* pool;
  const int32_t *table, *lens, *starts;   // starts NULL: max_rows rows each
  long long table_ld;
  int n, T, max_rows, nq, nkv, page_shift, max_pages, num_pages;   // pages of 2^page_shift rows
  Divisor by_g, by_nkv;              // G = NQ / NKV; NKV
  int causal, sink, window;
  float scale_log2;                  // softmax scale * log2(e)
  float factor;                      // score_factor of 16 times it (q4_attn.cuh)
  void* out;                         // [T, NQ, 128] contiguous, q's type
  int* counters;                     // [2 * num_sms], zero between calls
  float* part;                       // partial results
  int32_t* status;                   // or NULL
  int most_rows;                     // query rows of a request that are taken (kAttnPrefix: of a group); more are cut off
  // passes over rows that several requests share (AttnPass)
  const int32_t* row_of;             // kAttnPrefix: the table row of each group, of table_rows
  int table_rows;
  const int32_t* skip;               // kAttnOwn: columns of each request's table row that its group's pass covers
  float* pre_o;                      // what that pass leaves: [T, NQ, 128] sums, and their (m, l) [T, NQ]
  float2* pre_ml;
  int weigh;                         // whether the few-rows kernel weighs items (q4_attention.cu)
};
// An ordinary call; the query rows of groups of requests over the rows that each
// group shares, which leaves sums and statistics; the requests' own rows, joined
// with those.
enum AttnPass : int { kAttnAll = 0, kAttnPrefix = 1, kAttnOwn = 2 };
// Each kernel cuts a request's rows of a kv head into groups of `columns`, and
// its cached rows into tiles.
constexpr int kQ4Tile = 64, kQ4TcTile = 128;
constexpr int kQ4ItemUnits = 8;        // at least what either kernel adds to an item where it weighs items
int q4_attn_columns(int max_rows, int nq, int nkv);
int q4_attn_tc_columns(int max_rows, int nq, int nkv);
size_t q4_attn_part_floats(int max_rows, int nq, int nkv, int num_sms);
cudaError_t q4_attn_launch(const Q4AttnParams& p, int pass, int num_sms, cudaStream_t st);
// the same for blocks of query rows (q4_attention_tc.cu)
size_t q4_attn_tc_part_floats(int max_rows, int nq, int nkv, int num_sms);
size_t q4_attn_tc_group_floats(int max_rows, int nq, int nkv, int num_sms);   // of a group's pass
cudaError_t q4_attn_tc_launch(const Q4AttnParams& p, int pass, int num_sms, cudaStream_t st);
// Query rows of a kv head (rows of a request times G) up to which the first
// kernel runs; it takes them 16 at a time and decodes the cache for each group.
// us, first kernel / second, on 1 request of 2,048 rows, 16 of 16,384, 256 of
// 1,024 (8 kv heads): 16 query rows 14 / 15, 116 / 114, 123 / 149; 20 query rows
// 15 / 15, 210 / 114, 220 / 150; 64 query rows 16 / 20, 404 / 134, 412 / 206.
constexpr int kQ4FewRows = 16;

}  // namespace dfl
