// Parameters and host launchers of the kernels around a target's decode step:
// rotary positions (rope.cu) and verification of drafts by sampling (verify.cu).
#pragma once
#include "common.cuh"

namespace dfl {

enum ElemType : int { kElemF16 = 0, kElemBf16 = 1, kElemF32 = 2 };
__host__ __device__ __forceinline__ int elem_bytes(int type) { return type == kElemF32 ? 4 : 2; }

struct RopeParams {
  const void* x;                       // [rows, heads, dim]
  void* out;
  long long x_row, x_head, out_row, out_head;   // strides in elements
  const double* turns;                 // [rot / 2] turns a position
  float factor;                        // of both cosine and sine
  int type, rows, heads, dim, rot, interleaved, inverse;
  const void* positions;               // [rows], int32 or int64; NULL: of the packed rows of a step
  int wide;                            // positions are int64
  const int32_t *starts, *lens;        // step: [n + 1], [n]
  int n;
};
cudaError_t rope_launch(const RopeParams& p, int num_sms, cudaStream_t st);


struct VerifyParams {
  const void* logits;                  // [n, block, vocab], rows contiguous
  long long l_seq, l_row;              // strides in elements
  int type, n, block, vocab;
  const int32_t* drafts;               // [n, block - 1]
  const float* uniforms;               // [n, block]
  const float* temps;                  // [n], or NULL: temp for all
  float temp;
  const float* probs;                  // [n, block - 1, vocab], rows contiguous; NULL: drafts are certain
  long long q_seq, q_row;
  const int32_t* counts;               // [n] drafts of each request, or NULL: block - 1
  int32_t *accepted, *tokens;          // [n]
};
cudaError_t verify_launch(const VerifyParams& p, int num_sms, cudaStream_t st);

}  // namespace dfl
