// Rows of 16-bit or fp32 values as the norms' teams of threads hold them (ffm_norm.cu, ffm_rms.cu): where a thread's values lie, packed
// loads and stores, asynchronous copies to shared memory, sums over a team.
#pragma once

#include <type_traits>

#include "ffm_gemm_common.cuh"
#include "ffm_types.cuh"

namespace ffm {

template <typename T>
constexpr int VALUES = 16 / static_cast<int>(sizeof(T));  // of a chunk

// How a row lies in a team: where value j of chunk c of a thread is, and whether it is in the row. 16-byte accesses want
// neighbours in a thread; single accesses want neighbours in neighbouring threads.
template <typename T, bool VEC>
struct Place {
  int t, team, D, count;  // count: chunks (single accesses: values) that this thread has

  __device__ __forceinline__ Place(int team_, int D_) : t(threadIdx.x % team_), team(team_), D(D_) {
    const int all = VEC ? D / VALUES<T> : D;
    count = all > t ? (all - t + team - 1) / team : 0;
  }
  __device__ __forceinline__ int column(int c, int j) const {
    return VEC ? (c * team + t) * VALUES<T> + j : (c * VALUES<T> + j) * team + t;
  }
  __device__ __forceinline__ bool has(int c, int j) const { return (VEC ? c : c * VALUES<T> + j) < count; }
};

// A thread's part of a row stays packed, as it lies in memory: half the registers of its fp32 values, and what a block holds
// in registers decides how much it has in flight.
template <typename T>
__device__ __forceinline__ T bits_as(uint32_t bits);
template <>
__device__ __forceinline__ bf16 bits_as<bf16>(uint32_t bits) { return __ushort_as_bfloat16(static_cast<unsigned short>(bits)); }
template <>
__device__ __forceinline__ fp16 bits_as<fp16>(uint32_t bits) { return __ushort_as_half(static_cast<unsigned short>(bits)); }

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[VALUES<T>]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  } else {
    const uint32_t word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = to_float(bits_as<T>(word[q] & 0xffffu));
      v[2 * q + 1] = to_float(bits_as<T>(word[q] >> 16));
    }
  }
}

template <typename T, int CH, bool VEC>
__device__ __forceinline__ void load_row(const T* p, const Place<T, VEC>& at, uint4 (&raw)[CH]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if constexpr (VEC) {
      raw[c] = at.has(c, 0) ? *reinterpret_cast<const uint4*>(p + at.column(c, 0)) : make_uint4(0, 0, 0, 0);
    } else {
      uint32_t word[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (sizeof(T) == 4) {
          word[q] = at.has(c, q) ? reinterpret_cast<const uint32_t*>(p)[at.column(c, q)] : 0u;
        } else {
          const unsigned short* bits = reinterpret_cast<const unsigned short*>(p);
          const uint32_t low = at.has(c, 2 * q) ? bits[at.column(c, 2 * q)] : 0u;
          word[q] = low | (at.has(c, 2 * q + 1) ? static_cast<uint32_t>(bits[at.column(c, 2 * q + 1)]) << 16 : 0u);
        }
      }
      raw[c] = make_uint4(word[0], word[1], word[2], word[3]);
    }
  }
}

// Unpacked again afterwards: without this the compiler keeps the fp32 values from the first pass over the row to the last.
template <int CH>
__device__ __forceinline__ void stay_packed(uint4 (&raw)[CH]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) asm volatile("" : "+r"(raw[c].x), "+r"(raw[c].y), "+r"(raw[c].z), "+r"(raw[c].w));
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(T* p, const Place<T, VEC>& at, int c, const float (&v)[VALUES<T>]) {
  if constexpr (VEC) {
    if (at.has(c, 0)) {
      const int col = at.column(c, 0);
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p + col) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        store8(p + col, v);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < VALUES<T>; ++j) {
      if (at.has(c, j)) p[at.column(c, j)] = from_float<T>(v[j]);
    }
  }
}

// weight or bias of a thread's chunk; `fill` where there is none
template <typename T, bool VEC>
__device__ __forceinline__ void load_vector(const void* p, int type, const Place<T, VEC>& at, int c, float fill,
                                            float (&v)[VALUES<T>]) {
#pragma unroll
  for (int j = 0; j < VALUES<T>; ++j) v[j] = fill;
  if (p == nullptr) return;
  if constexpr (VEC && sizeof(T) == 2) {
    if (at.has(c, 0)) load8_as(p, type, at.column(c, 0), v);
  } else {
#pragma unroll
    for (int j = 0; j < VALUES<T>; ++j) {
      if (at.has(c, j)) v[j] = load1_as(p, type, at.column(c, j));
    }
  }
}

// a thread's chunk of the weight in shared memory
template <typename T, bool VEC>
__device__ __forceinline__ void load_scale(const float* scale, const Place<T, VEC>& at, int c, float (&w)[VALUES<T>]) {
  if constexpr (VEC) {
    const int col = min(at.column(c, 0), at.D - VALUES<T>);  // past the row's end: any
#pragma unroll
    for (int j = 0; j < VALUES<T>; j += 4) {
      const float4 f = *reinterpret_cast<const float4*>(scale + col + j);
      w[j] = f.x, w[j + 1] = f.y, w[j + 2] = f.z, w[j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VALUES<T>; ++j) w[j] = scale[min(at.column(c, j), at.D - 1)];
  }
}

// Sums over a team (a power of two of threads up to 32, whole warps beyond), the same in each of its threads. A team of more than a warp meets in shared
// memory: every thread of the block has to come here, and `part` (a slot a warp) must not be the one of the call before.
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N], int team, float (*part)[32]) {
  for (int o = (team < 32 ? team : 32) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  }
  if (team <= 32) return;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) part[n][threadIdx.x >> 5] = v[n];
  }
  __syncthreads();
  const int first = threadIdx.x / team * (team >> 5);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = 0.0f;
    for (int i = 0; i < team >> 5; ++i) v[n] += part[n][first + i];
  }
}

// zeros where there is nothing to copy (`valid` is any address of the tensor then)
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, bool any, const void* valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(any ? src : valid), "r"(any ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void team_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// team_sum() for teams that do not keep step with one another: a barrier for each, from BARRIER on (16 teams of more than a
// warp at most, 14 in the backward kernel, which meets as a block at barrier 0 in the end).
template <int BARRIER, int N>
__device__ __forceinline__ void own_team_sum(float (&v)[N], int team, float (*part)[32]) {
  for (int o = (team < 32 ? team : 32) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  }
  if (team <= 32) return;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) part[n][threadIdx.x >> 5] = v[n];
  }
  const int index = threadIdx.x / team;
  team_barrier(BARRIER + index, team);
  const int first = index * (team >> 5), lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = lane < team >> 5 ? part[n][first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  }
}

__device__ __forceinline__ uint4 read_shared_16(uint32_t at) {
  uint4 v;
  ld_shared_v4(at, v);
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack2(const uint4& u, float2 (&v)[VALUES<T> / 2]) {
  const uint32_t word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int q = 0; q < VALUES<T> / 2; ++q) {
    if constexpr (sizeof(T) == 4) {
      v[q] = make_float2(__uint_as_float(word[2 * q]), __uint_as_float(word[2 * q + 1]));
    } else if constexpr (std::is_same<T, bf16>::value) {
      v[q] = make_float2(__uint_as_float(word[q] << 16), __uint_as_float(word[q] & 0xffff0000u));
    } else {
      v[q] = __half22float2(*reinterpret_cast<const __half2*>(&word[q]));
    }
  }
}

template <typename T>
__device__ __forceinline__ void store2(T* p, const float2 (&v)[VALUES<T> / 2]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
  } else {
    const float values[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    store8(p, values);
  }
}

}  // namespace ffm
