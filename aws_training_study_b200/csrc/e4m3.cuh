// Rounding to e4m3fn as the cache writers do it (pcp_cache_write,
// pcp_cache_append).
#pragma once

#include <cuda_fp8.h>
#include <cstdint>

namespace pcp {

// Two fp32 -> two e4m3fn bytes (`a` in the low one), nearest even; magnitudes
// above 464 and non-finite values -> NaN, as tensor.to(torch.float8_e4m3fn).
__device__ __forceinline__ uint16_t e4m3x2_from_floats(float a, float b) {
  uint16_t c = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  // Beyond the rounding range of the largest finite value (448), and NaN/Inf:
  // the NaN code with the input's sign.
  if (!(fabsf(a) <= 464.f)) c = static_cast<uint16_t>((c & 0xFF00u) | 0x7Fu | ((__float_as_uint(a) >> 24) & 0x80u));
  if (!(fabsf(b) <= 464.f))
    c = static_cast<uint16_t>((c & 0x00FFu) | ((0x7Fu | ((__float_as_uint(b) >> 24) & 0x80u)) << 8));
  return c;
}

}  // namespace pcp
