// What the host sides of the library's translation units share: the calling
// thread's error message (pcp_last_error) and the error-returning macros.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "pcp_attn.h"

namespace pcp {

constexpr int kErrChars = 1024;
// The calling thread's message buffer (defined in pcp_attn.cu).
__attribute__((visibility("hidden"))) char* error_buffer();

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(error_buffer(), kErrChars, fmt, ap);
  va_end(ap);
  return code;
}

}  // namespace pcp

#define CUDA_TRY(x)                                                                                              \
  do {                                                                                                           \
    cudaError_t e_ = (x);                                                                                        \
    if (e_ != cudaSuccess)                                                                                       \
      return pcp::fail(e_ == cudaErrorMemoryAllocation ? PCP_ERR_OUT_OF_MEMORY : PCP_ERR_CUDA, "%s: %s (%s:%d)", \
                       #x, cudaGetErrorString(e_), __FILE__, __LINE__);                                          \
  } while (0)

#define PCP_TRY(x)          \
  do {                      \
    int s_ = (x);           \
    if (s_ != PCP_OK) return s_; \
  } while (0)
