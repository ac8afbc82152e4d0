// 8-bit floating-point numbers (e4m3) and the scales of blocks of 128 values.
#pragma once

#include <cuda_fp8.h>

#include "ffm_common.cuh"

namespace ffm {

constexpr int E4M3_BLOCK = 128;  // values of a row, or rows and columns of a matrix, that share a scale

// rounded to nearest, saturating; NaN stays NaN
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// The scale that puts a block's largest magnitude on 448, the largest e4m3 number: at least 2^-126, so that its inverse is finite, and 1
// for a block of zeros. An infinity makes the scale infinite, and the block's numbers 0 and NaN.
__device__ __forceinline__ float e4m3_scale(float amax) { return amax > 0.0f ? fmaxf(amax / 448.0f, 1.17549435e-38f) : 1.0f; }

// The same within two roundings, without a division
__device__ __forceinline__ float e4m3_scale_near(float amax) { return amax > 0.0f ? fmaxf(amax * (1.0f / 448.0f), 1.17549435e-38f) : 1.0f; }

// 1 / x within a rounding or so, for what is then rounded to 8 bits; x is 2^-126 at least
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

}  // namespace ffm
