// Layer norm over the last dimension and its backward pass.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w:  dx = r (g - mean(g) - xh mean(g xh))      dw = sum over rows of dy xh      db = sum over rows of dy
//
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx. A row is held in the registers of a team
// of 1 to 1024 threads, up to 64 bytes each, so that the variance is the mean of squared differences (not a difference of
// sums, which loses everything for rows far from zero) and memory is read once. In the backward pass every thread keeps the
// same columns for all of its rows and sums their dw and db in registers; a block leaves one fp32 row of each behind and a
// second kernel adds those in a fixed order, so results do not depend on the order in which blocks run.
#include <type_traits>

#include "ffm_types.cuh"

#include "ffm_device.h"
#include "ffm_gemm_common.cuh"
#include "ffm_internal.h"

namespace ffm {

namespace {

// Chunks of 16 bytes of a row that a thread holds. With two, the backward kernel needs about 80 registers (32 of them sums of
// dw and db) and 768 threads fit on an SM; with four it spills, and is used where a row does not fit otherwise.
constexpr int NORM_CHUNKS = 2;
constexpr int NORM_CHUNKS_LONG = 4;
constexpr int NORM_TEAM = 512;        // threads of a row at most, with two chunks
constexpr int NORM_TEAM_LONG = 1024;  // and with four
constexpr int NORM_THREADS = 256;     // of a block, about, unless one row takes more
constexpr int NORM_SM_THREADS = 768;  // of the backward kernel's blocks on an SM

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

// THREADS: of an SM, so that the compiler knows how many registers a thread may have
template <typename T, int CH, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1)
layer_norm_forward_kernel(const T* __restrict__ x, long long stride, const void* __restrict__ weight, int w_type,
                          const void* __restrict__ bias, int b_type, long long rows, int D, float eps, int team,
                          T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>;
  const Place<T, VEC> at(team, D);
  const int teams = blockDim.x / team;
  const float width = static_cast<float>(D);
  for (long long row0 = static_cast<long long>(blockIdx.x) * teams; row0 < rows;
       row0 += static_cast<long long>(gridDim.x) * teams) {
    const bool active = row0 + threadIdx.x / team < rows;
    const long long row = active ? row0 + threadIdx.x / team : row0;
    uint4 raw[CH];
    load_row<T, CH, VEC>(x + row * stride, at, raw);
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V];
      unpack<T>(raw[c], v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[j];
    }
    team_sum(s, team, part[0]);
    const float mu = s[0] / width;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V];
      unpack<T>(raw[c], v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (at.has(c, j)) s[0] = fmaf(v[j] - mu, v[j] - mu, s[0]);
      }
    }
    team_sum(s, team, part[1]);
    const float r = 1.0f / sqrtf(s[0] / width + eps);
    if (!active) continue;  // whole teams; the block's trips are the same for all
    if (at.t == 0 && mean != nullptr) {
      mean[row] = mu;
      rstd[row] = r;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], w[V], b[V];
      unpack<T>(raw[c], v);
      load_vector<T, VEC>(weight, w_type, at, c, 1.0f, w);
      load_vector<T, VEC>(bias, b_type, at, c, 0.0f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - mu) * r, w[j], b[j]);
      store_chunk<T, VEC>(y + row * D, at, c, v);
    }
  }
}

// dx (skipped where null), and of every block one row of partial sums of dw and db (skipped where null).
template <typename T, int CH, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1)
layer_norm_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, long long stride,
                           const void* __restrict__ weight, int w_type, const float* __restrict__ mean,
                           const float* __restrict__ rstd, long long rows, int D, int team, T* __restrict__ dx,
                           float* __restrict__ part_w, float* __restrict__ part_b) {
  __shared__ float part[2][2][32];
  extern __shared__ __align__(16) float scale[];  // [D] the weight in fp32
  float* sums = scale + D;                        // [2][D] where several warps have the same columns
  constexpr int V = VALUES<T>;
  for (int c = threadIdx.x; c < D; c += blockDim.x) scale[c] = weight != nullptr ? load1_as(weight, w_type, c) : 1.0f;
  __syncthreads();
  const Place<T, VEC> at(team, D);
  const int teams = blockDim.x / team;
  const float width = static_cast<float>(D);
  float aw[CH][V], ab[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) aw[c][j] = ab[c][j] = 0.0f;
  }
  int parity = 0;
  for (long long row0 = static_cast<long long>(blockIdx.x) * teams; row0 < rows;
       row0 += static_cast<long long>(gridDim.x) * teams, parity ^= 1) {
    const bool active = row0 + threadIdx.x / team < rows;
    const long long row = active ? row0 + threadIdx.x / team : row0;
    uint4 raw_x[CH], raw_g[CH];
    load_row<T, CH, VEC>(x + row * stride, at, raw_x);
    load_row<T, CH, VEC>(dy + row * D, at, raw_g);
    const float mu = mean[row], r = rstd[row];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], g[V], w[V];
      unpack<T>(raw_x[c], v);
      unpack<T>(raw_g[c], g);
      load_scale<T, VEC>(scale, at, c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (v[j] - mu) * r;  // past the row's end times g = 0
        if (active) {
          aw[c][j] = fmaf(g[j], xh, aw[c][j]);
          ab[c][j] += g[j];
        }
        s[0] = fmaf(g[j], w[j], s[0]);
        s[1] = fmaf(g[j] * w[j], xh, s[1]);
      }
    }
    if (dx == nullptr) continue;  // for all threads alike
    team_sum(s, team, part[parity]);
    stay_packed(raw_x);
    stay_packed(raw_g);
    const float s1 = s[0] / width, s2 = s[1] / width;
    if (!active) continue;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], g[V], w[V];
      unpack<T>(raw_x[c], v);
      unpack<T>(raw_g[c], g);
      load_scale<T, VEC>(scale, at, c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = r * (fmaf(g[j], w[j], -s1) - (v[j] - mu) * r * s2);
      store_chunk<T, VEC>(dx + row * D, at, c, v);
    }
  }
  if (part_w == nullptr && part_b == nullptr) return;
  // first the teams of a warp, then the warps that hold the same columns, one after the other
  for (int o = team; o < 32; o <<= 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        aw[c][j] += __shfl_xor_sync(0xffffffffu, aw[c][j], o);
        ab[c][j] += __shfl_xor_sync(0xffffffffu, ab[c][j], o);
      }
    }
  }
  const int wide = team < 32 ? 32 : team, turns = blockDim.x / wide;
  const bool mine = (threadIdx.x & 31) < team || team >= 32;
  for (int k = 0; k < turns; ++k) {
    if (static_cast<int>(threadIdx.x) / wide == k && mine) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int col = at.column(c, j);
          if (at.has(c, j)) {
            const float w = aw[c][j] + (k > 0 ? sums[col] : 0.0f), b = ab[c][j] + (k > 0 ? sums[D + col] : 0.0f);
            if (k + 1 < turns) {
              sums[col] = w;
              sums[D + col] = b;
            } else {
              if (part_w != nullptr) part_w[static_cast<long long>(blockIdx.x) * D + col] = w;
              if (part_b != nullptr) part_b[static_cast<long long>(blockIdx.x) * D + col] = b;
            }
          }
        }
      }
    }
    if (k + 1 < turns) __syncthreads();
  }
}

// out[col] = sum over p of parts[p][col], in an order that depends on the number of parts alone: 32 columns a block, eight
// warps that take every eighth part. blockIdx.y: weight or bias.
__global__ void __launch_bounds__(256)
layer_norm_sum_kernel(const float* __restrict__ part_w, const float* __restrict__ part_b, int parts, int D,
                      void* __restrict__ dweight, int w_type, void* __restrict__ dbias, int b_type) {
  __shared__ float s[8][33];
  const float* part = blockIdx.y == 0 ? part_w : part_b;
  void* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (col < D) {
    for (int p = warp; p < parts; p += 32) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (p + 8 * u < parts) a[u] += part[static_cast<long long>(p + 8 * u) * D + col];
      }
    }
  }
  s[warp][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (warp == 0 && col < D) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += s[w][lane];
    store1_as(out, blockIdx.y == 0 ? w_type : b_type, col, total);
  }
}

int max_columns(int type) { return NORM_TEAM_LONG * NORM_CHUNKS_LONG * (16 / type_bytes(type)); }

struct NormShape {
  int team, chunks, threads, teams;
};

// Up to a warp the team is the smallest power of two that holds the row, beyond that the fewest warps: a width just above a
// power of two leaves few threads idle.
NormShape norm_shape(int D, int type) {
  const int values = 16 / type_bytes(type);
  const int pieces = (D + values - 1) / values;
  NormShape s;
  s.chunks = pieces <= NORM_TEAM * NORM_CHUNKS ? NORM_CHUNKS : NORM_CHUNKS_LONG;
  s.team = 1;
  while (s.team < 32 && s.team * s.chunks < pieces) s.team *= 2;
  if (s.team * s.chunks < pieces) s.team = (pieces + 32 * s.chunks - 1) / (32 * s.chunks) * 32;
  s.teams = s.team < NORM_THREADS ? NORM_THREADS / s.team : 1;
  s.threads = s.team * s.teams;
  return s;
}

// Blocks of the backward pass: one row of partial sums each.
int backward_blocks(int64_t rows, int D, int type) {
  const NormShape s = norm_shape(D, type);
  const int64_t want = (rows + s.teams - 1) / s.teams, cap = static_cast<int64_t>(num_sms()) * (s.chunks == NORM_CHUNKS ? NORM_SM_THREADS / s.threads : 1);
  return static_cast<int>(want < cap ? (want > 0 ? want : 1) : cap);
}

template <typename T, int CH, bool VEC, int THREADS>
int forward_as(const void* x, int64_t stride, const void* w, int w_type, const void* b, int b_type, int64_t rows, int D, float eps,
               const NormShape& s, void* y, float* mean, float* rstd, cudaStream_t stream) {
  const int64_t groups = (rows + s.teams - 1) / s.teams;
  const int64_t cap = static_cast<int64_t>(num_sms()) * (2048 / s.threads);
  layer_norm_forward_kernel<T, CH, VEC, THREADS><<<static_cast<unsigned>(groups < cap ? groups : cap), s.threads, 0, stream>>>(
      static_cast<const T*>(x), stride, w, w_type, b, b_type, rows, D, eps, s.team, static_cast<T*>(y), mean, rstd);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

template <typename T, int CH, bool VEC, int THREADS>
int backward_as(const void* dy, const void* x, int64_t stride, const void* w, int w_type, const float* mean, const float* rstd,
                int64_t rows, int D, const NormShape& s, void* dx, float* part_w, float* part_b, int blocks, cudaStream_t stream) {
  // 4 bytes a column for the weight, and 8 for the sums of warps that share columns (D < 4096 then)
  const int smem = D * static_cast<int>(sizeof(float)) * (s.threads > (s.team < 32 ? 32 : s.team) ? 3 : 1);
  static PerDevice room;
  const int allowed = room.get([&] {
    const int most = max_columns(FFM_TYPE_BF16) * static_cast<int>(sizeof(float));
    if (cudaFuncSetAttribute(layer_norm_backward_kernel<T, CH, VEC, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) !=
        cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return most;
  });
  if (smem > allowed) return FFM_ERR_LAUNCH;
  layer_norm_backward_kernel<T, CH, VEC, THREADS><<<blocks, s.threads, smem, stream>>>(
      static_cast<const T*>(dy), static_cast<const T*>(x), stride, w, w_type, mean, rstd, rows, D, s.team, static_cast<T*>(dx),
      part_w, part_b);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

// f(type tag, chunks, vector accesses, threads of an SM) for the run-time values of a call
template <typename F>
int dispatch_norm(int type, const NormShape& s, bool vec, F&& f) {
  auto with_vec = [&](auto tag, auto ch, auto threads) {
    return vec ? f(tag, ch, std::true_type{}, threads) : f(tag, ch, std::false_type{}, threads);
  };
  auto with_chunks = [&](auto tag) {
    return s.chunks == NORM_CHUNKS ? with_vec(tag, std::integral_constant<int, NORM_CHUNKS>{}, std::integral_constant<int, NORM_SM_THREADS>{})
                                   : with_vec(tag, std::integral_constant<int, NORM_CHUNKS_LONG>{},
                                              std::integral_constant<int, NORM_TEAM_LONG>{});
  };
  if (type == FFM_TYPE_BF16) return with_chunks(bf16{});
  if (type == FFM_TYPE_FP16) return with_chunks(fp16{});
  return with_chunks(float{});
}

// 16-byte accesses: every row of every operand starts on a 16-byte boundary and is a whole number of them
template <typename... P>
bool norm_vectors(int type, int64_t stride, int D, const P*... p) {
  return static_cast<int64_t>(D) * type_bytes(type) % 16 == 0 && (stride * type_bytes(type)) % 16 == 0 && !off_16_bytes(p...);
}

bool norm_arguments(int x_type, int64_t rows, int64_t stride, int D, const void* w, int w_type) {
  return is_type(x_type) && rows >= 0 && D > 0 && (stride >= D || rows <= 1) && (w == nullptr || is_type(w_type));
}

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" int ffm_layer_norm_forward(const void* x, int x_type, int64_t rows, int64_t row_stride, int D, const void* weight,
                                      int w_type, const void* bias, int b_type, float eps, void* y, float* mean, float* rstd,
                                      ffm_stream_t stream) {
  if (!norm_arguments(x_type, rows, row_stride, D, weight, w_type) || (bias != nullptr && !is_type(b_type))) return FFM_ERR_BAD_ARG;
  if (!(eps >= 0.0f) || (mean == nullptr) != (rstd == nullptr)) return FFM_ERR_BAD_ARG;
  if (D > max_columns(x_type)) return FFM_ERR_UNSUPPORTED;
  if (rows == 0) return FFM_OK;
  if (!x || !y) return FFM_ERR_BAD_ARG;
  const NormShape s = norm_shape(D, x_type);
  return dispatch_norm(x_type, s, norm_vectors(x_type, row_stride, D, x, y, weight, bias), [&](auto tag, auto ch, auto vec, auto threads) {
    return forward_as<decltype(tag), decltype(ch)::value, decltype(vec)::value, decltype(threads)::value>(
        x, row_stride, weight, w_type, bias, b_type, rows, D, eps, s, y, mean, rstd, static_cast<cudaStream_t>(stream));
  });
}

extern "C" size_t ffm_layer_norm_workspace_bytes(int64_t rows, int D, int x_type) {
  if (rows < 0 || !is_type(x_type) || D <= 0 || D > max_columns(x_type)) return 0;
  return static_cast<size_t>(2) * backward_blocks(rows, D, x_type) * D * sizeof(float);
}

extern "C" int ffm_layer_norm_backward(const void* dy, const void* x, int x_type, int64_t rows, int64_t row_stride, int D,
                                       const void* weight, int w_type, const float* mean, const float* rstd, void* dx,
                                       void* dweight, void* dbias, int b_type, void* workspace, size_t workspace_bytes,
                                       ffm_stream_t stream) {
  if (!norm_arguments(x_type, rows, row_stride, D, weight, w_type)) return FFM_ERR_BAD_ARG;
  if ((dweight != nullptr && !is_type(w_type)) || (dbias != nullptr && !is_type(b_type))) return FFM_ERR_BAD_ARG;
  if (D > max_columns(x_type)) return FFM_ERR_UNSUPPORTED;
  if (rows > 0 && (!dy || !x || !mean || !rstd)) return FFM_ERR_BAD_ARG;
  const bool parts = dweight != nullptr || dbias != nullptr;
  if (parts && (workspace == nullptr || workspace_bytes < ffm_layer_norm_workspace_bytes(rows, D, x_type))) return FFM_ERR_WORKSPACE;
  if (!parts && (dx == nullptr || rows == 0)) return FFM_OK;
  const NormShape s = norm_shape(D, x_type);
  const int blocks = backward_blocks(rows, D, x_type);
  float* part_w = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  float* part_b = dbias != nullptr ? static_cast<float*>(workspace) + static_cast<size_t>(blocks) * D : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vectors = norm_vectors(x_type, row_stride, D, dy, x, dx);
  const int rc = dispatch_norm(x_type, s, vectors, [&](auto tag, auto ch, auto vec, auto threads) {
    return backward_as<decltype(tag), decltype(ch)::value, decltype(vec)::value, decltype(threads)::value>(
        dy, x, row_stride, weight, w_type, mean, rstd, rows, D, s, dx, part_w, part_b, blocks, st);
  });
  if (rc != FFM_OK || !parts) return rc;
  layer_norm_sum_kernel<<<dim3((D + 31) / 32, 2), 256, 0, st>>>(part_w, part_b, blocks, D, dweight, w_type, dbias, b_type);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}
