// C ABI of the operators around a target's decode step (include/dflash_b200.h):
// argument checks and launches of rope.cu and verify.cu.
#include <cmath>

#include "api_error.cuh"
#include "decode.cuh"

using namespace dfl;

namespace {

bool type_ok(int type) { return type == DFLASH_F16 || type == DFLASH_BF16 || type == DFLASH_F32; }

int current_sms(int* sms) {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  CK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return DFLASH_OK;
}

long long magnitude(long long v) { return v < 0 ? -v : v; }

// bytes [lo, hi) around ptr that rows x heads x dim elements with these strides touch
void extent(const void* ptr, long long row, long long head, int rows, int heads, int dim, int bytes, long long* lo, long long* hi) {
  const long long r = (rows - 1) * row, h = (heads - 1) * head;
  *lo = (long long)reinterpret_cast<uintptr_t>(ptr) + ((r < 0 ? r : 0) + (h < 0 ? h : 0)) * bytes;
  *hi = (long long)reinterpret_cast<uintptr_t>(ptr) + ((r > 0 ? r : 0) + (h > 0 ? h : 0) + dim) * bytes;
}

// whether no two of its elements share an address
bool distinct(long long row, long long head, int rows, int heads, int dim) {
  row = magnitude(row);
  head = magnitude(head);
  if (rows == 1) return heads == 1 || head >= dim;
  if (heads == 1) return row >= dim;
  return (head >= dim && row >= (heads - 1) * head + dim) || (row >= dim && head >= (rows - 1) * row + dim);
}

}  // namespace

extern "C" {

int dflash_rope(const void* x, int64_t x_row, int64_t x_head, int type, int rows, int heads, int dim, int rotary_dim,
                int interleaved, int inverse, const double* turns, float factor, const void* positions, int positions64,
                const int32_t* starts, const int32_t* lens, int n, void* out, int64_t out_row, int64_t out_head,
                void* stream) {
  if (!turns || (rows > 0 && (!x || !out))) return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (!type_ok(type)) return fail(DFLASH_ERR_INVALID, "type %d is neither f16, bf16 nor f32", type);
  if (rows < 0 || heads < 1 || heads > 65535) return fail(DFLASH_ERR_INVALID, "rows %d, heads %d", rows, heads);
  if (dim < 2 || dim > 1024 || dim % 2) return fail(DFLASH_ERR_INVALID, "head dim %d is not even or outside [2, 1024]", dim);
  if (rotary_dim < 2 || rotary_dim > dim || rotary_dim % 2)
    return fail(DFLASH_ERR_INVALID, "rotary dim %d is not even or outside [2, %d]", rotary_dim, dim);
  if (!std::isfinite(factor)) return fail(DFLASH_ERR_INVALID, "factor must be finite");
  if (positions ? starts || lens || n : !starts || !lens)
    return fail(DFLASH_ERR_INVALID, "either positions or the starts and lens of a step");
  if (!positions && (n < 1 || n > DFLASH_PAGED_MAX_SEQS))
    return fail(DFLASH_ERR_INVALID, "n %d outside [1, %d]", n, DFLASH_PAGED_MAX_SEQS);
  const int bytes = elem_bytes(type);
  if (reinterpret_cast<uintptr_t>(x) % bytes || reinterpret_cast<uintptr_t>(out) % bytes)
    return fail(DFLASH_ERR_INVALID, "x and out must be aligned to their type");
  if (rows == 0) return DFLASH_OK;
  if (!distinct(out_row, out_head, rows, heads, dim)) return fail(DFLASH_ERR_INVALID, "rows or heads of out overlap");
  if (x != out || x_row != out_row || x_head != out_head) {
    long long a, b, c, d;
    extent(x, x_row, x_head, rows, heads, dim, bytes, &a, &b);
    extent(out, out_row, out_head, rows, heads, dim, bytes, &c, &d);
    if (a < d && c < b) return fail(DFLASH_ERR_INVALID, "out overlaps x (it must be x itself or lie apart)");
  }
  int sms = 0;
  if (int rc = current_sms(&sms)) return rc;
  RopeParams p{};
  p.x = x; p.out = out; p.x_row = x_row; p.x_head = x_head; p.out_row = out_row; p.out_head = out_head;
  p.turns = turns; p.factor = factor; p.type = type; p.rows = rows; p.heads = heads; p.dim = dim; p.rot = rotary_dim;
  p.interleaved = interleaved != 0; p.inverse = inverse != 0; p.positions = positions; p.wide = positions64 != 0;
  p.starts = starts; p.lens = lens; p.n = n;
  CK(rope_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

int dflash_verify_drafts(const void* logits, int64_t seq_stride, int64_t row_stride, int type, int n, int block, int vocab,
                         const int32_t* drafts, const float* uniforms, const float* temperatures, float temperature,
                         const float* probs, int64_t probs_seq_stride, int64_t probs_row_stride, const int32_t* num_drafts,
                         int32_t* accepted, int32_t* tokens, void* stream) {
  // (a row of 2^22 entries read entry by entry, as one whose logits leave no reference is, takes 0.1 s of the 0.4 s
  // that the kernel's bounded waits last)
  if (n < 0 || block < 1 || vocab < 1 || vocab > 1 << 22 || (long long)n * 16 > INT32_MAX)
    return fail(DFLASH_ERR_INVALID, "n %d, block %d, vocab %d", n, block, vocab);
  if (!type_ok(type)) return fail(DFLASH_ERR_INVALID, "type %d is neither f16, bf16 nor f32", type);
  if (n > 0 && (!logits || (block > 1 && !drafts) || !uniforms || !accepted || !tokens))
    return fail(DFLASH_ERR_INVALID, "NULL pointer");
  if (!temperatures && (!(temperature >= 0.f) || !std::isfinite(temperature)))
    return fail(DFLASH_ERR_INVALID, "temperature %g must be finite and not negative", temperature);
  if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(type)) return fail(DFLASH_ERR_INVALID, "logits must be aligned to their type");
  if (n == 0) return DFLASH_OK;
  int sms = 0;
  if (int rc = current_sms(&sms)) return rc;
  VerifyParams p{};
  p.logits = logits; p.l_seq = seq_stride; p.l_row = row_stride; p.type = type; p.n = n; p.block = block; p.vocab = vocab;
  p.drafts = drafts; p.uniforms = uniforms; p.temps = temperatures; p.temp = temperature;
  p.probs = probs; p.q_seq = probs_seq_stride; p.q_row = probs_row_stride; p.counts = num_drafts;
  p.accepted = accepted; p.tokens = tokens;
  CK(verify_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return DFLASH_OK;
}

}  // extern "C"
