// 8-bit floating-point numbers (e4m3) and the scales of blocks of 128 values.
#pragma once

#include <cuda_fp8.h>

#include <cfloat>

#include "ffm_common.cuh"
#include "ffm_types.cuh"

namespace ffm {

constexpr int E4M3_BLOCK = 128;  // values of a row, or rows and columns of a matrix, that share a scale

// rounded to nearest, saturating; NaN stays NaN
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// A block's values in 8 bits: the scale is its largest magnitude over 448, the largest e4m3 number, rounded once, at least 2^-126, so that quotients by it
// stay finite, and 1 for a block of zeros. The quotients in fp32 are rounded to 8 bits, ties to even. An infinity makes the scale infinite, and the
// block's numbers 0 and NaN.
//
// 16-bit values often lie halfway between two e4m3 numbers, and a product with 1 / s falls on either side there, so quotients are rounded as
// division rounds them. With a division for every value 32768 x 7168 bf16 rows took 195 us, 8192 x 7168 of the norm 102 (the product alone 124 and 80).
// Instead the product's remainder, which is exact, is divided in the same way and added: the correctly rounded quotient, where 1 / s is
// (P. Markstein, IBM J. Res. Dev. 34, 1990), in 125 and 76 us. Blocks whose remainders may fall below 2^-149, or which are not finite, are left to
// division.

__device__ __forceinline__ bool e4m3_by_division(float amax) { return amax > 0.0f && !(amax >= 0x1p-70f && amax <= FLT_MAX); }

__device__ __forceinline__ float e4m3_scale_divided(float amax) { return amax > 0.0f ? fmaxf(amax / 448.0f, 0x1p-126f) : 1.0f; }

// amax / 448 for the other blocks
__device__ __forceinline__ float e4m3_scale(float amax) {
  amax = amax > 0.0f ? amax : 448.0f;
  constexpr float inverse = 1.0f / 448.0f;
  const float q = amax * inverse;
  return fmaf(fmaf(-q, 448.0f, amax), inverse, q);
}

// 1 / s, s in 2^-80..2^120: a Newton step from within a step or so of it
__device__ __forceinline__ float reciprocal(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return fmaf(r, fmaf(-s, r, 1.0f), r);
}

// Four values over s; `negative_inverse`: -1 / s. Everything is negated, and the codes' signs turned in the end, which keeps -0.
__device__ __forceinline__ uint32_t pack_quotients(float2 a, float2 b, float s, float negative_inverse) {
  const float2 d = both(s), y = both(negative_inverse), qa = mul2(a, y), qb = mul2(b, y);
  a = fma2(fma2(qa, d, a), y, qa);
  b = fma2(fma2(qb, d, b), y, qb);
  return pack_e4m3x4(a.x, a.y, b.x, b.y) ^ 0x80808080u;
}

__device__ __forceinline__ uint32_t pack_divided(float2 a, float2 b, float s) { return pack_e4m3x4(a.x / s, a.y / s, b.x / s, b.y / s); }

// CHUNKS x 2 PAIRS values of a thread, chunk c of a block with magnitudes up to top[c]: to store(c, words of four codes, scale)
template <int CHUNKS, int PAIRS, typename F>
__device__ __forceinline__ void quantize_chunks(const float2 (&v)[CHUNKS][PAIRS], const float (&top)[CHUNKS], F&& store) {
  bool divide = false;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) divide |= e4m3_by_division(top[c]);
  uint32_t word[PAIRS / 2];
  if (!divide) {
    float s[CHUNKS], y[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) s[c] = e4m3_scale(top[c]), y[c] = -reciprocal(s[c]);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int i = 0; i < PAIRS / 2; ++i) word[i] = pack_quotients(v[c][2 * i], v[c][2 * i + 1], s[c], y[c]);
      store(c, word, s[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const float s = e4m3_scale_divided(top[c]);
#pragma unroll
      for (int i = 0; i < PAIRS / 2; ++i) word[i] = pack_divided(v[c][2 * i], v[c][2 * i + 1], s);
      store(c, word, s);
    }
  }
}

template <int N>
__device__ __forceinline__ void store_words(uint8_t* to, const uint32_t (&word)[N]) {
  if constexpr (N == 2) {
    *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
  } else {
    *reinterpret_cast<uint32_t*>(to) = word[0];
  }
}

}  // namespace ffm
