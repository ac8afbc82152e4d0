// AdamW step over many tensors in one launch, with the two moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        (t: steps taken, this one included)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Eight bits: blocks of 128 values of a tensor share a power of two; m / 2^k and sqrt(v) / 2^k are e4m3 numbers, k being the
// least for which the block's largest magnitude fits (448 * 2^k). With a power of two the scaling rounds nothing, so that a state
// that is read and written back unchanged stays. The root of v, because its e4m3 numbers then span 2^34 in v. m is rounded to nearest.
// sqrt(v) is rounded up or down at random, in proportion: v moves by 1 - b2 of itself a step at most when gradients fall, its
// root by 2.5 % at b2 = 0.95, and two e4m3 numbers are 6-12 % apart: to nearest it would never leave its number. A positive v
// does not become zero (its least is 2^-18 of the block's scale squared): the quotient would explode. The update itself uses
// the new m and v before they are rounded.
//
// Bytes a value: bf16 parameters, gradients and 8-bit states move 10, with fp32 states 22, with an fp32 master as well 28. With
// 32-bit states memory is the bound (5.4-5.9 TB/s read and written). 8-bit states take 55-64 instructions a value: 60-69 % of the issue
// slots at 59 % of the memory's rate (3.8 TB/s without a master, 5.1 with one), neither of them full, so that waiting for loads, of which 24
// warps an SM have two halves of a chunk in flight, is what is left. Tensors of mixed types (bf16 parameters with fp32 gradients) go value
// by value where their states are: 96 M in 1.88 ms with 32-bit states, 0.81 with 8-bit ones.
// A block walks chunks of 4096 values, twice eight neighbours a thread, over all tensors as one list. Steps are counted on the
// device, so that a captured step can be replayed: every block reads them, and the last block to finish raises them.
#include "ffm_types.cuh"

#include "ffm_gemm_common.cuh"
#include "ffm_internal.h"

namespace ffm {

namespace {

constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_CHUNK = ADAMW_THREADS * 16;
constexpr int ADAMW_BLOCK = 128;  // values that share a scale: 16 threads

struct AdamWTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* master;
  uint8_t* m_scale;
  uint8_t* v_scale;
  int32_t* step;
  long long n;
  long long chunks_end;  // chunks of this tensor and all before it
  int p_type, g_type;
  int wide;  // every pointer allows 16-byte accesses (8-byte ones to 8-bit states)
};

template <int MAX>
struct AdamWJob {
  AdamWTensor tensor[MAX];
  int count;
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, weight_decay;
  double beta1_wide, beta2_wide;
  const float* lr_device;   // instead of lr
  const float* grad_scale;  // device scalar or null
  uint32_t seed;
  unsigned int* ticket;  // zero before and after
};

// b^t by squaring
__device__ __forceinline__ double power(double b, int t) {
  double r = 1.0;
  for (unsigned int e = t > 0 ? t : 0; e != 0; e >>= 1) {
    if (e & 1) r *= b;
    b *= b;
  }
  return r;
}

__device__ __forceinline__ float exponent_of_two(int k) { return __int_as_float((k + 127) << 23); }

// The least k for which top <= 448 * 2^k (448 = 1.75 * 2^8), within what the scale's byte and fp32 can say.
__device__ __forceinline__ int block_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int k = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(k, -126), 120);
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(two)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Two values of at most 448 (or NaN) to e4m3, to nearest.
__device__ __forceinline__ uint32_t e4m3x2_nearest(float2 v) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// x from 2^-6 to 448 to e4m3, up with probability (distance from the lower neighbour) / (distance of the neighbours): 16 random
// bits and a half, as a fraction, are added to the bits that are cut off, and the code is what is left of this from bit 20 on.
// random: 20 bits, the last four of them 8. For a smaller x the code is below 8, or not below 128.
__device__ __forceinline__ uint32_t e4m3_random(float x, uint32_t random) { return __float_as_uint(x) + random - (120u << 23); }

// The code for any v, x being its root, correctly rounded, times 1 / the scale. Below 2^-6 codes are multiples of 2^-9. Never zero for a
// positive v; NaN for one that is not finite.
__device__ __noinline__ uint32_t e4m3_random_any(float v, float scale, uint32_t random) {
  if (!(fabsf(v) <= 3.402823466e38f)) return 0x7fu;
  const float x = __fsqrt_rn(v) * scale, fraction = (static_cast<float>(random >> 4) + 0.5f) * (1.0f / 65536.0f);
  const uint32_t code = x < 0.015625f ? static_cast<uint32_t>(floorf(__fadd_rn(x * 512.0f, fraction))) : e4m3_random(x, random) >> 20;
  return v > 0.0f ? max(code, 1u) : 0u;
}

// Random bits of a pair of neighbouring values (16 each): the finaliser of MurmurHash3 (two rounds of multiply and fold) over a counter.
__device__ __forceinline__ uint32_t random_pair(uint32_t pair, uint32_t key) {
  uint32_t h = pair * 0x9E3779B1u + key;
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// the larger one, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// the larger of either half, over 16 threads
__device__ __forceinline__ uint32_t max16(uint32_t v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = __vmaxu2(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// One instruction each, good to 2 units of the last place; what is below 2^-126 counts as zero.
__device__ __forceinline__ float root_fast(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// eight values as four pairs
__device__ __forceinline__ float (&values(float2 (&v)[4]))[8] { return *reinterpret_cast<float (*)[8]>(&v); }

// What of a call is the same for all values.
struct Step {
  float2 keep, eps;
  float beta1, less1, beta2, less2, eps_one, grad_scale;
  bool scaled, fast;
};

// The update of eight values: m, v and p in place; root is sqrt(v).
template <bool EIGHT>
__device__ __forceinline__ void update8(const Step& h, float rate, float inverse, const float2 (&g)[4], float2 (&p)[4], float2 (&m)[4],
                                        float2 (&v)[4], float2 (&root)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 x = h.scaled ? mul2(g[q], both(h.grad_scale)) : g[q];
    if (EIGHT) {
      // Each product and sum is rounded on its own: the largest of a block decides its scale, and two evaluations that differ in the
      // last place would now and then differ in it. (Pairs of products and sums are put together by the compiler even so.)
      m[q].x = __fadd_rn(__fmul_rn(m[q].x, h.beta1), __fmul_rn(x.x, h.less1));
      m[q].y = __fadd_rn(__fmul_rn(m[q].y, h.beta1), __fmul_rn(x.y, h.less1));
      v[q].x = __fadd_rn(__fmul_rn(v[q].x, h.beta2), __fmul_rn(__fmul_rn(x.x, h.less2), x.x));
      v[q].y = __fadd_rn(__fmul_rn(v[q].y, h.beta2), __fmul_rn(__fmul_rn(x.y, h.less2), x.y));
    } else {
      m[q] = add2(mul2(m[q], both(h.beta1)), mul2(x, both(h.less1)));
      v[q] = add2(mul2(v[q], both(h.beta2)), mul2(mul2(x, both(h.less2)), x));
    }
  }
  if (h.fast) {
    const float2 r = both(-rate), inv = both(inverse);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // (the exact root is the faster one with 32-bit states, 96 M bf16 values with masters: 478 against 503 us; the slower one
      // with 8-bit ones, 128 M: 450 against 412)
      root[q] = EIGHT ? make_float2(root_fast(v[q].x), root_fast(v[q].y)) : make_float2(__fsqrt_rn(v[q].x), __fsqrt_rn(v[q].y));
      const float2 under = fma2(root[q], inv, h.eps);
      p[q] = fma2(r, mul2(m[q], make_float2(reciprocal_fast(under.x), reciprocal_fast(under.y))), mul2(p[q], h.keep));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      values(root)[j] = __fsqrt_rn(values(v)[j]);
      values(p)[j] = fmaf(-rate, __fdiv_rn(values(m)[j], fmaf(values(root)[j], inverse, h.eps_one)), values(p)[j] * h.keep.x);
    }
  }
}

// Eight 8-bit values of either moment with their blocks' scales.
__device__ __forceinline__ void unpack_states(uint2 cm, uint2 cv, uint32_t sm, uint32_t sv, float2 (&m)[4], float2 (&v)[4]) {
  const float2 fm = both(__uint_as_float(sm << 23)), fv = both(__uint_as_float(sv << 23));
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    m[q] = mul2(e4m3x2_to_float2((q < 2 ? cm.x : cm.y) >> (16 * (q & 1)) & 0xffffu), fm);
    v[q] = mul2(e4m3x2_to_float2((q < 2 ? cv.x : cv.y) >> (16 * (q & 1)) & 0xffffu), fv);
    v[q] = mul2(v[q], v[q]);
  }
}

// And back: the 16 threads of a block find its scales. pair0: the first value's place in the tensor, halved.
__device__ __forceinline__ void pack_states(float2 (&m)[4], const float2 (&v)[4], const float2 (&root)[4], uint32_t pair0, uint32_t key,
                                            uint32_t (&cm)[2], uint32_t (&cv)[2], int& km, int& kv) {
  float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    top_m = max_nan(top_m, max_nan(fabsf(m[q].x), fabsf(m[q].y)));
    top_v = max_nan(top_v, max_nan(v[q].x, v[q].y));
  }
  // the exponents grow with the values: both of the block in one maximum, 0x7fff for what is not finite
  const uint32_t mine = static_cast<uint32_t>(finite(top_m) ? block_exponent(top_m) + 127 : 0x7fff) |
                        static_cast<uint32_t>(finite(top_v) ? block_exponent(__fsqrt_rn(top_v)) + 127 : 0x7fff) << 16;
  uint32_t both_k = max16(mine);
  const bool odd = (both_k & 0xffffu) == 0x7fffu || both_k >> 16 == 0x7fffu;
  if (__any_sync(0xffffffffu, odd)) {
    // what is infinite or NaN leaves the scale to the others, and becomes NaN
    float other_m = 0.0f, other_v = 0.0f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (finite(m[q].x)) other_m = fmaxf(other_m, fabsf(m[q].x));
      if (finite(m[q].y)) other_m = fmaxf(other_m, fabsf(m[q].y));
      if (finite(v[q].x)) other_v = fmaxf(other_v, v[q].x);
      if (finite(v[q].y)) other_v = fmaxf(other_v, v[q].y);
      if (!finite(m[q].x)) m[q].x = __int_as_float(0x7fc00000);
      if (!finite(m[q].y)) m[q].y = __int_as_float(0x7fc00000);
    }
    const uint32_t others = max16(static_cast<uint32_t>(block_exponent(other_m) + 127) |
                                  static_cast<uint32_t>(block_exponent(__fsqrt_rn(other_v)) + 127) << 16);
    if (odd) both_k = others;
  }
  km = static_cast<int>(both_k & 0xffffu) - 127;
  kv = static_cast<int>(both_k >> 16) - 127;
  const float2 fm = both(exponent_of_two(-km)), fv = both(exponent_of_two(-kv));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    cm[h] = e4m3x2_nearest(mul2(m[2 * h], fm)) | e4m3x2_nearest(mul2(m[2 * h + 1], fm)) << 16;
    const uint32_t first = random_pair(pair0 + 2 * h, key), second = random_pair(pair0 + 2 * h + 1, key);
    const uint32_t random[4] = {(first << 4 & 0xffff0u) | 8u, (first >> 12 & 0xffff0u) | 8u, (second << 4 & 0xffff0u) | 8u,
                                (second >> 12 & 0xffff0u) | 8u};
    const float2 a = mul2(root[2 * h], fv), b = mul2(root[2 * h + 1], fv);
    const float x[4] = {a.x, a.y, b.x, b.y};
    // The roots are good to a unit or two of their last place, and the code is that of the correctly rounded one: where so little
    // could change it (8 times in 2^20), it is taken again.
    uint32_t c[4];
    bool near = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = e4m3_random(x[j], random[j]);
      near = near || ((c[j] + 4u) & 0xffff8u) == 0;
      c[j] >>= 20;
    }
    cv[h] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    // a code below 8 or above 127 stands for a number below 2^-6, or one that is none: rare as well
    const uint32_t eights = cv[h] & 0x78787878u;
    if (((c[0] | c[1] | c[2] | c[3]) & ~0x7fu) != 0 || ((eights - 0x01010101u) & ~eights & 0x80808080u) != 0 || near || odd) {
      const float y[4] = {v[2 * h].x, v[2 * h].y, v[2 * h + 1].x, v[2 * h + 1].y};
      cv[h] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) cv[h] |= e4m3_random_any(y[j], fv.x, random[j]) << (8 * j);
    }
  }
}

// How a tensor's values lie: a launch is for one of these, so that its kernel knows the loads of a value at compile time. HALF:
// parameter and gradient in the same 16-bit type. ANY: the two in different types.
enum { ANY_LAYOUT = 0, HALF_LAYOUT = 1, HALF_MASTER_LAYOUT = 2, F32_LAYOUT = 3, LAYOUTS = 4 };

// Eight values as they come from memory.
template <int LAYOUT, bool EIGHT>
struct Raw {
  static constexpr int P = LAYOUT == HALF_LAYOUT ? 1 : 2, G = LAYOUT == F32_LAYOUT ? 2 : 1;
  uint4 p[P], g[G], m[EIGHT ? 1 : 2], v[EIGHT ? 1 : 2];  // 8-bit states: the first half
  uint32_t sm, sv;

  template <int N>
  __device__ __forceinline__ static void get(uint4 (&to)[N], const void* from) {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = static_cast<const uint4*>(from)[i];
  }
  template <int N>
  __device__ __forceinline__ static void as_pairs(const uint4 (&from)[N], bool fp16s, float2 (&to)[4]) {
    if constexpr (N == 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        to[2 * i] = make_float2(__uint_as_float(from[i].x), __uint_as_float(from[i].y));
        to[2 * i + 1] = make_float2(__uint_as_float(from[i].z), __uint_as_float(from[i].w));
      }
    } else {
      const uint32_t word[4] = {from[0].x, from[0].y, from[0].z, from[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        to[i] = fp16s ? __half22float2(*reinterpret_cast<const __half2*>(&word[i]))
                      : make_float2(__uint_as_float(word[i] << 16), __uint_as_float(word[i] & 0xffff0000u));
      }
    }
  }

  __device__ __forceinline__ void load(const AdamWTensor& a, long long e) {
    get(g, static_cast<const char*>(a.g) + e * (G == 2 ? 4 : 2));
    get(p, LAYOUT == HALF_MASTER_LAYOUT ? static_cast<const void*>(a.master + e) : static_cast<const char*>(a.p) + e * (P == 2 ? 4 : 2));
    if constexpr (EIGHT) {
      const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + e);
      const uint2 y = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + e);
      m[0] = make_uint4(x.x, x.y, 0, 0);
      v[0] = make_uint4(y.x, y.y, 0, 0);
      sm = a.m_scale[e / ADAMW_BLOCK];
      sv = a.v_scale[e / ADAMW_BLOCK];
    } else {
      get(m, static_cast<const float*>(a.m) + e);
      get(v, static_cast<const float*>(a.v) + e);
    }
  }
  __device__ __forceinline__ void step(const AdamWTensor& a, long long e, const Step& h, float rate, float inverse, uint32_t key) {
    float2 gf[4], pf[4], mf[4], vf[4], root[4];
    const bool fp16s = a.p_type == FFM_TYPE_FP16;
    as_pairs(g, fp16s, gf);
    as_pairs(p, fp16s, pf);
    if constexpr (EIGHT) {
      unpack_states(make_uint2(m[0].x, m[0].y), make_uint2(v[0].x, v[0].y), sm, sv, mf, vf);
    } else {
      as_pairs(m, false, mf);
      as_pairs(v, false, vf);
    }
    update8<EIGHT>(h, rate, inverse, gf, pf, mf, vf, root);
    if constexpr (LAYOUT == HALF_MASTER_LAYOUT) store8(a.master + e, values(pf));
    if constexpr (LAYOUT == F32_LAYOUT) {
      store8(static_cast<float*>(a.p) + e, values(pf));
    } else if (fp16s) {
      store8(static_cast<fp16*>(a.p) + e, values(pf));
    } else {
      store8(static_cast<bf16*>(a.p) + e, values(pf));
    }
    if constexpr (EIGHT) {
      uint32_t cm[2], cv[2];
      int km, kv;
      pack_states(mf, vf, root, static_cast<uint32_t>(e >> 1), key, cm, cv, km, kv);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + e) = make_uint2(cm[0], cm[1]);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + e) = make_uint2(cv[0], cv[1]);
      if ((threadIdx.x & 15) == 0) {
        a.m_scale[e / ADAMW_BLOCK] = static_cast<uint8_t>(km + 127);
        a.v_scale[e / ADAMW_BLOCK] = static_cast<uint8_t>(kv + 127);
      }
    } else {
      store8(static_cast<float*>(a.m) + e, values(mf));
      store8(static_cast<float*>(a.v) + e, values(vf));
    }
  }
};

// Up to eight values of any types at any address, from value e of the tensor on: the ends of tensors, tensors off 16 bytes, and
// the ANY layout.
template <bool EIGHT>
__device__ __forceinline__ void step_any(const AdamWTensor& a, long long e, const Step& h, float rate, float inverse, uint32_t key) {
  const int left = static_cast<int>(min(a.n - e, 8ll));  // none where <= 0
  const bool whole = left == 8 && a.wide != 0;
  float2 g[4], p[4], m[4], v[4], root[4];
  if (whole) {
    load8_as(a.g, a.g_type, e, values(g));
    if (a.master != nullptr) {
      load8(a.master + e, values(p));
    } else {
      load8_as(a.p, a.p_type, e, values(p));
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (whole) break;
    values(g)[j] = j < left ? load1_as(a.g, a.g_type, e + j) : 0.0f;
    values(p)[j] = j < left ? (a.master != nullptr ? a.master[e + j] : load1_as(a.p, a.p_type, e + j)) : 0.0f;
  }
  if (EIGHT) {
    uint2 cm = make_uint2(0, 0), cv = make_uint2(0, 0);
    uint32_t sm = 0, sv = 0;
    if (left > 0) {
      sm = a.m_scale[e / ADAMW_BLOCK];
      sv = a.v_scale[e / ADAMW_BLOCK];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < left) {
        const uint32_t x = static_cast<const uint8_t*>(a.m)[e + j], y = static_cast<const uint8_t*>(a.v)[e + j];
        if (j < 4) {
          cm.x |= x << (8 * j), cv.x |= y << (8 * j);
        } else {
          cm.y |= x << (8 * j - 32), cv.y |= y << (8 * j - 32);
        }
      }
    }
    unpack_states(cm, cv, sm, sv, m, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      values(m)[j] = j < left ? static_cast<const float*>(a.m)[e + j] : 0.0f;
      values(v)[j] = j < left ? static_cast<const float*>(a.v)[e + j] : 0.0f;
    }
  }
  update8<EIGHT>(h, rate, inverse, g, p, m, v, root);
  if (whole) {
    if (a.master != nullptr) store8(a.master + e, values(p));
    store8_as(a.p, a.p_type, e, values(p));
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < left && !whole) {
      if (a.master != nullptr) a.master[e + j] = values(p)[j];
      store1_as(a.p, a.p_type, e + j, values(p)[j]);
    }
  }
  if (EIGHT) {
    uint32_t cm[2], cv[2];
    int km, kv;
    pack_states(m, v, root, static_cast<uint32_t>(e >> 1), key, cm, cv, km, kv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < left) {
        static_cast<uint8_t*>(a.m)[e + j] = static_cast<uint8_t>(cm[j >> 2] >> (8 * (j & 3)));
        static_cast<uint8_t*>(a.v)[e + j] = static_cast<uint8_t>(cv[j >> 2] >> (8 * (j & 3)));
      }
    }
    if (left > 0 && (threadIdx.x & 15) == 0) {
      a.m_scale[e / ADAMW_BLOCK] = static_cast<uint8_t>(km + 127);
      a.v_scale[e / ADAMW_BLOCK] = static_cast<uint8_t>(kv + 127);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < left) {
        static_cast<float*>(a.m)[e + j] = values(m)[j];
        static_cast<float*>(a.v)[e + j] = values(v)[j];
      }
    }
  }
}

template <int MAX, int LAYOUT, bool EIGHT>
__global__ void __launch_bounds__(ADAMW_THREADS, EIGHT ? 3 : 2)
adamw_kernel(const __grid_constant__ AdamWJob<MAX> job) {
  __shared__ float rate[MAX], inverse[MAX];  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  __shared__ uint32_t keys[MAX];
  __shared__ bool last;
  const float lr = job.lr_device != nullptr ? *job.lr_device : job.lr;
  for (int i = threadIdx.x; i < job.count; i += ADAMW_THREADS) {
    const int t = *job.tensor[i].step + 1;
    rate[i] = static_cast<float>(lr / (1.0 - power(job.beta1_wide, t)));
    inverse[i] = static_cast<float>(1.0 / sqrt(1.0 - power(job.beta2_wide, t)));
    keys[i] = static_cast<uint32_t>(t) * 0x85EBCA77u + job.seed * 0xC2B2AE3Du;
  }
  __syncthreads();
  Step h;
  h.keep = both(1.0f - lr * job.weight_decay);
  h.eps = both(job.eps);
  h.eps_one = job.eps;
  h.beta1 = job.beta1, h.less1 = job.one_minus_beta1, h.beta2 = job.beta2, h.less2 = job.one_minus_beta2;
  h.scaled = job.grad_scale != nullptr;
  h.grad_scale = h.scaled ? *job.grad_scale : 1.0f;
  // with eps from here on a root of a v below 2^-126 (10^-19) makes no difference to the update
  h.fast = job.eps >= 1e-12f;
  const long long chunks = job.tensor[job.count - 1].chunks_end;
  int i = 0;
  for (long long chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    while (chunk >= job.tensor[i].chunks_end) ++i;  // the chunk's tensor, for the whole block alike
    const AdamWTensor& a = job.tensor[i];
    const long long c0 = (chunk - (i > 0 ? job.tensor[i - 1].chunks_end : 0)) * ADAMW_CHUNK, e0 = c0 + threadIdx.x * 8;
    if constexpr (LAYOUT != ANY_LAYOUT) {
      if (a.wide && c0 + ADAMW_CHUNK <= a.n) {
        // both halves' loads first: twice as much in flight
        Raw<LAYOUT, EIGHT> first, second;
        first.load(a, e0);
        second.load(a, e0 + ADAMW_CHUNK / 2);
        if (EIGHT) {
          // one copy of the code (128 M bf16 values with masters: 408 us, with two copies 428; without masters 350 and 352)
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            first.step(a, e0 + half * (ADAMW_CHUNK / 2), h, rate[i], inverse[i], keys[i]);
            first = second;
          }
        } else {
          // bound by memory; the stores of one half then lie beside the other's arithmetic (96 M bf16 values with masters: 475 us, with one copy
          // of the code 536; fp32 values 514 and 519)
          first.step(a, e0, h, rate[i], inverse[i], keys[i]);
          second.step(a, e0 + ADAMW_CHUNK / 2, h, rate[i], inverse[i], keys[i]);
        }
        continue;
      }
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) step_any<EIGHT>(a, e0 + half * (ADAMW_CHUNK / 2), h, rate[i], inverse[i], keys[i]);
  }
  // every block has read the steps before it takes a ticket; the last one raises them
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(job.ticket, 1u) == gridDim.x - 1;
    if (last) *job.ticket = 0;
  }
  __syncthreads();
  if (last) {
    for (int k = threadIdx.x; k < job.count; k += ADAMW_THREADS) *job.tensor[k].step += 1;
  }
}

template <int MAX, int LAYOUT, bool EIGHT>
int launch_adamw(const ffm_adamw_tensor* t, int count, const ffm_adamw_args& h, cudaStream_t stream) {
  AdamWJob<MAX> job;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    AdamWTensor& a = job.tensor[i];
    a.p = t[i].param;
    a.g = t[i].grad;
    a.m = t[i].exp_avg;
    a.v = t[i].exp_avg_sq;
    a.master = static_cast<float*>(t[i].master);
    a.m_scale = static_cast<uint8_t*>(t[i].exp_avg_scale);
    a.v_scale = static_cast<uint8_t*>(t[i].exp_avg_sq_scale);
    a.step = t[i].step;
    a.n = t[i].elements;
    a.p_type = static_cast<int>(t[i].param_type);
    a.g_type = static_cast<int>(t[i].grad_type);
    const uintptr_t states = reinterpret_cast<uintptr_t>(a.m) | reinterpret_cast<uintptr_t>(a.v);
    a.wide = !off_16_bytes(a.p, a.g, a.master) && states % (EIGHT ? 8 : 16) == 0;
    chunks += (a.n + ADAMW_CHUNK - 1) / ADAMW_CHUNK;
    a.chunks_end = chunks;
  }
  job.count = count;
  job.lr = static_cast<float>(h.lr);
  job.beta1 = static_cast<float>(h.beta1);
  job.one_minus_beta1 = static_cast<float>(1.0 - h.beta1);
  job.beta2 = static_cast<float>(h.beta2);
  job.one_minus_beta2 = static_cast<float>(1.0 - h.beta2);
  job.eps = static_cast<float>(h.eps);
  job.weight_decay = static_cast<float>(h.weight_decay);
  job.beta1_wide = h.beta1;
  job.beta2_wide = h.beta2;
  job.lr_device = h.lr_device;
  job.grad_scale = h.grad_scale;
  job.seed = static_cast<uint32_t>(h.seed);
  job.ticket = static_cast<unsigned int*>(h.ticket);
  auto kernel = adamw_kernel<MAX, LAYOUT, EIGHT>;
  static PerDevice resident;
  const int most = resident.get([&] {
    int blocks = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, ADAMW_THREADS, 0) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return blocks * num_sms();
  });
  if (most <= 0) return FFM_ERR_LAUNCH;
  kernel<<<static_cast<unsigned>(chunks < most ? (chunks > 0 ? chunks : 1) : most), ADAMW_THREADS, 0, stream>>>(job);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

int adamw_layout(const ffm_adamw_tensor& t) {
  if (t.param_type != t.grad_type) return ANY_LAYOUT;
  if (t.param_type == FFM_TYPE_FP32) return t.master == nullptr ? F32_LAYOUT : ANY_LAYOUT;
  return t.master != nullptr ? HALF_MASTER_LAYOUT : HALF_LAYOUT;
}

template <int MAX>
int launch_adamw_as(int layout, bool eight, const ffm_adamw_tensor* t, int count, const ffm_adamw_args& h, cudaStream_t stream) {
  switch (layout) {
    case HALF_LAYOUT: return eight ? launch_adamw<MAX, HALF_LAYOUT, true>(t, count, h, stream) : launch_adamw<MAX, HALF_LAYOUT, false>(t, count, h, stream);
    case HALF_MASTER_LAYOUT:
      return eight ? launch_adamw<MAX, HALF_MASTER_LAYOUT, true>(t, count, h, stream) : launch_adamw<MAX, HALF_MASTER_LAYOUT, false>(t, count, h, stream);
    case F32_LAYOUT: return eight ? launch_adamw<MAX, F32_LAYOUT, true>(t, count, h, stream) : launch_adamw<MAX, F32_LAYOUT, false>(t, count, h, stream);
    default: return eight ? launch_adamw<MAX, ANY_LAYOUT, true>(t, count, h, stream) : launch_adamw<MAX, ANY_LAYOUT, false>(t, count, h, stream);
  }
}

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" int ffm_adamw_step(const ffm_adamw_tensor* tensors, int count, const ffm_adamw_args* args, ffm_stream_t stream) {
  if (count < 0 || !args || (count > 0 && !tensors)) return FFM_ERR_BAD_ARG;
  if (count == 0) return FFM_OK;
  const ffm_adamw_args& h = *args;
  if (!h.ticket || (h.bits != 8 && h.bits != 32)) return FFM_ERR_BAD_ARG;
  if (!(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0 && h.eps >= 0.0)) return FFM_ERR_BAD_ARG;
  const bool eight = h.bits == 8;
  for (int i = 0; i < count; ++i) {
    const ffm_adamw_tensor& t = tensors[i];
    if (t.elements < 0 || !t.step || !is_type(static_cast<int>(t.param_type)) || !is_type(static_cast<int>(t.grad_type))) return FFM_ERR_BAD_ARG;
    if (t.elements == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return FFM_ERR_BAD_ARG;
    if (eight && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return FFM_ERR_BAD_ARG;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ffm_adamw_tensor some[FFM_ADAMW_MAX];
  for (int layout = 0; layout < LAYOUTS; ++layout) {
    int n = 0;
    for (int i = 0; i < count; ++i) {
      if (adamw_layout(tensors[i]) == layout) some[n++] = tensors[i];
      if (n == FFM_ADAMW_MAX || (i + 1 == count && n > 0)) {
        const int rc = n <= FFM_ADAMW_FEW ? launch_adamw_as<FFM_ADAMW_FEW>(layout, eight, some, n, h, s)
                                          : launch_adamw_as<FFM_ADAMW_MAX>(layout, eight, some, n, h, s);
        if (rc != FFM_OK) return rc;
        n = 0;
        if (h.launched != nullptr) ++*h.launched;
      }
    }
  }
  return FFM_OK;
}
