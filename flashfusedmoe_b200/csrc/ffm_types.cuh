// Eight values at a time of the element types that the operators beside the layer take (FFM_TYPE_*): layer norm and AdamW.
#pragma once

#include <cuda_fp16.h>

#include "ffm_common.cuh"

namespace ffm {

typedef __half fp16;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(fp16 v) { return __half2float(v); }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ fp16 from_float<fp16>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }

// p on a 16-byte boundary
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
__device__ __forceinline__ void load8(const fp16* p, float (&v)[8]) {
  uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(fp16* p, const float (&v)[8]) {
  uint4 u;
  __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// The same for a type known only at run time (uniform over the grid), i elements into p.
__device__ __forceinline__ float load1_as(const void* p, int type, long long i) {
  if (type == FFM_TYPE_BF16) return to_float(static_cast<const bf16*>(p)[i]);
  if (type == FFM_TYPE_FP16) return to_float(static_cast<const fp16*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store1_as(void* p, int type, long long i, float v) {
  if (type == FFM_TYPE_BF16) {
    static_cast<bf16*>(p)[i] = from_float<bf16>(v);
  } else if (type == FFM_TYPE_FP16) {
    static_cast<fp16*>(p)[i] = from_float<fp16>(v);
  } else {
    static_cast<float*>(p)[i] = v;
  }
}
__device__ __forceinline__ void load8_as(const void* p, int type, long long i, float (&v)[8]) {
  if (type == FFM_TYPE_BF16) {
    load8(static_cast<const bf16*>(p) + i, v);
  } else if (type == FFM_TYPE_FP16) {
    load8(static_cast<const fp16*>(p) + i, v);
  } else {
    load8(static_cast<const float*>(p) + i, v);
  }
}
__device__ __forceinline__ void store8_as(void* p, int type, long long i, const float (&v)[8]) {
  if (type == FFM_TYPE_BF16) {
    store8(static_cast<bf16*>(p) + i, v);
  } else if (type == FFM_TYPE_FP16) {
    store8(static_cast<fp16*>(p) + i, v);
  } else {
    store8(static_cast<float*>(p) + i, v);
  }
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ unsigned long long bits2(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 of_bits2(unsigned long long v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return of_bits2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return of_bits2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return of_bits2(d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

inline bool is_type(int type) { return type == FFM_TYPE_BF16 || type == FFM_TYPE_FP16 || type == FFM_TYPE_FP32; }
inline int type_bytes(int type) { return type == FFM_TYPE_FP32 ? 4 : 2; }

}  // namespace ffm
