// Error reporting shared by the C entry points (dflash_api.cu, paged_api.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/dflash_b200.h"

namespace dfl {
// records the calling thread's last error message and returns code
int fail(int code, const char* fmt, ...);
}  // namespace dfl

#define CK(call)                                                                        \
  do {                                                                                  \
    cudaError_t e_ = (call);                                                            \
    if (e_ != cudaSuccess) {                                                            \
      if (e_ == cudaErrorInvalidValue)                                                  \
        return fail(DFLASH_ERR_INVALID, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), \
                    __FILE__, __LINE__);                                                \
      return fail(e_ == cudaErrorMemoryAllocation ? DFLASH_ERR_OOM : DFLASH_ERR_CUDA,   \
                  "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__);  \
    }                                                                                   \
  } while (0)
