// f8_device.h -- e4m3 codes and their exponents, shared by f8_codec.hip and evict_f8.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qkv_device.h"

namespace qkv {

__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }

// 4 codes times f (a power of two up to 1), rounded to nearest even
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float f) {
  const f2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, w, true);
}

}  // namespace qkv
