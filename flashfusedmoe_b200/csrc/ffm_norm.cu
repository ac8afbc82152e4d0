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
#include "ffm_device.h"
#include "ffm_internal.h"
#include "ffm_norm_common.cuh"

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
// The streaming kernels (many rows of 16-byte boundaries): one block an SM, four chunks a thread, a ring of rows a team.
constexpr int STREAM_CHUNKS = 4, STREAM_STAGES = 2;
constexpr int STREAM_BACK_STAGES = 3;     // where they fit (up to 8192 16-bit columns), else 2
constexpr int STREAM_THREADS = 1024;      // forward: 64 registers
constexpr int STREAM_BACK_THREADS = 512;  // backward: 128, 64 of them sums of dw and db
static_assert(STREAM_THREADS / 64 <= 16 && STREAM_BACK_THREADS / 64 <= 15, "a barrier for every team of more than a warp");
constexpr int STREAM_SMEM = 226 << 10;
// The same for rows off 16-byte boundaries. A stage is being filled while a row is worked on; the backward kernel needs 168
// registers (at 512 threads there are 128: it spilled, and took 98 us for 16384 x 1025 bf16, where it takes 55).
constexpr int SHIFTED_THREADS = 768, SHIFTED_BACK_THREADS = 384, SHIFTED_STAGES = 3;

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

// The block's row of partial sums: first the teams of a warp, then the warps that hold the same columns, one after the other
// (sums: 2 D values of shared memory).
template <typename T, int CH, bool VEC>
__device__ __forceinline__ void add_teams(const Place<T, VEC>& at, int team, float* sums, int D, float (&aw)[CH][VALUES<T>],
                                          float (&ab)[CH][VALUES<T>], float* part_w, float* part_b) {
  constexpr int V = VALUES<T>;
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
  add_teams<T, CH, VEC>(at, team, sums, D, aw, ab, part_w, part_b);
}

// ---- many rows of 16-byte boundaries ------------------------------------------------------------------------------------
//
// What a block holds in registers is too little to be in flight all the time: reading a row, two exchanges and writing it
// follow one another (32768 x 7168 bf16: 354 us forward, 563 backward; here 167 and 225, 5.6 and 6.3 TB/s). Here every thread copies its chunks of the next rows
// to shared memory (cp.async; it reads back what it copied itself, so nothing but its own wait stands between), and teams of
// one block go their own way with a barrier each. Weight and bias lie in shared memory in fp32.

// A vector of D values in shared memory in fp32, four neighbours of every thread side by side: threads then read 16 bytes each
// without a bank in common. Filled by the whole block.
template <typename T>
__device__ __forceinline__ void fill_vector(float* to, const void* p, int type, float fill, int D, int team) {
  constexpr int V = VALUES<T>, PARTS = V / 4;
  for (int i = threadIdx.x; i < team * STREAM_CHUNKS * V; i += blockDim.x) {
    const int j = i & 3, quad = i >> 2, t = quad % team, part = quad / team;
    const int col = (part / PARTS * team + t) * V + part % PARTS * 4 + j;
    to[i] = p != nullptr && col < D ? load1_as(p, type, col) : fill;
  }
}

template <typename T>
__device__ __forceinline__ void read_vector(uint32_t thread_base, int c, int team, float2 (&v)[VALUES<T> / 2]) {
  constexpr int PARTS = VALUES<T> / 4;
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    const uint4 u = read_shared_16(thread_base + (c * PARTS + h) * team * 16);
    v[2 * h] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[2 * h + 1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
}

// Rows of a team: its own, and how often its loop runs (teams of a warp or less go in step with their warp's first).
struct Trips {
  int mine, all;
  __device__ __forceinline__ Trips(long long rows, long long first, long long step, int team) {
    auto count = [&](long long from) { return from < rows ? static_cast<int>((rows - from + step - 1) / step) : 0; };
    mine = count(first);
    all = team < 32 ? count(first - (threadIdx.x & 31) / team) : mine;
  }
};

// s / n, rounded as a division would for whole results, with inv = 1 / n: one step of correction by the residual, Markstein's method
__device__ __forceinline__ float quotient(float s, float n, float inv) {
  const float q = s * inv;
  return fmaf(fmaf(-q, n, s), inv, q);
}

template <typename T>
__global__ void __launch_bounds__(STREAM_THREADS, 1)
layer_norm_forward_stream_kernel(const T* __restrict__ x, long long stride, const void* __restrict__ weight, int w_type,
                                 const void* __restrict__ bias, int b_type, long long rows, int D, float eps, int team,
                                 T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  extern __shared__ __align__(16) float scale[];  // weight, bias, ring
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>, CH = STREAM_CHUNKS, S = STREAM_STAGES;
  const Place<T, true> at(team, D);
  float* shift = scale + team * CH * V;
  const uint32_t my_scale = smem_u32(scale) + at.t * 16, my_shift = smem_u32(shift) + at.t * 16;
  const uint32_t ring = smem_u32(shift + team * CH * V) + threadIdx.x * 16, slot = blockDim.x * 16;
  const int teams = blockDim.x / team;
  const float width = static_cast<float>(D), inv = 1.0f / width;
  const long long first = static_cast<long long>(blockIdx.x) * teams + threadIdx.x / team, step = static_cast<long long>(gridDim.x) * teams;
  const Trips trips(rows, first, step, team);
  const T* source = x + first * stride + at.t * V;  // of the next row to fetch
  auto fetch = [&](int k, uint32_t to) {
    const int chunks = k < trips.mine ? at.count : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) copy_async_16(to + c * slot, source + c * team * V, c < chunks, x);
    copy_async_commit();
    source += step * stride;
  };
  const uint32_t row_bytes = CH * slot;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, ring + s * row_bytes);
  fill_vector<T>(scale, weight, w_type, 1.0f, D, team);
  fill_vector<T>(shift, bias, b_type, 0.0f, D, team);
  __syncthreads();
  uint32_t here = ring;  // the row's stage
  T* out = y + first * D + at.t * V;
  for (int k = 0; k < trips.all; ++k, out += step * D) {
    copy_async_wait<S - 1>();
    float2 s2 = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) s2 = add2(s2, v[j]);
    }
    float s[1] = {s2.x + s2.y};
    own_team_sum<0>(s, team, part[0]);
    const float mu = quotient(s[0], width, inv);
    s2 = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float2 less = both(c < at.count ? -mu : 0.0f);
      float2 v[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        v[j] = add2(v[j], less);
        s2 = fma2(v[j], v[j], s2);
      }
    }
    s[0] = s2.x + s2.y;
    own_team_sum<0>(s, team, part[1]);
    const float r = rsqrtf(fmaf(s[0], inv, eps));
    const int chunks = k < trips.mine ? at.count : 0;  // to write
    if (at.t == 0 && chunks > 0 && mean != nullptr) {
      mean[first + k * step] = mu;
      rstd[first + k * step] = r;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], w[V / 2], b[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
      read_vector<T>(my_scale, c, team, w);
      read_vector<T>(my_shift, c, team, b);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) w[j] = fma2(mul2(add2(v[j], both(-mu)), both(r)), w[j], b[j]);
      if (c < chunks) store2<T>(out + c * team * V, w);
    }
    fetch(k + S, here);  // this thread's chunks have been read
    here = here == ring + (S - 1) * row_bytes ? ring : here + row_bytes;
  }
  copy_async_wait<0>();
}

template <typename T, int S>
__global__ void __launch_bounds__(STREAM_BACK_THREADS, 1)
layer_norm_backward_stream_kernel(const T* __restrict__ dy, const T* __restrict__ x, long long stride,
                                  const void* __restrict__ weight, int w_type, const float* __restrict__ mean,
                                  const float* __restrict__ rstd, long long rows, int D, int team, T* __restrict__ dx,
                                  float* __restrict__ part_w, float* __restrict__ part_b) {
  extern __shared__ __align__(16) float scale[];  // weight, ring; the ring's place then holds sums [2][D]
  __shared__ float part[2][2][32];
  constexpr int V = VALUES<T>, CH = STREAM_CHUNKS;
  const Place<T, true> at(team, D);
  const uint32_t my_scale = smem_u32(scale) + at.t * 16;
  const uint32_t ring = smem_u32(scale + team * CH * V) + threadIdx.x * 16, slot = blockDim.x * 16;
  const int teams = blockDim.x / team;
  const float inv = 1.0f / static_cast<float>(D);
  const long long first = static_cast<long long>(blockIdx.x) * teams + threadIdx.x / team, step = static_cast<long long>(gridDim.x) * teams;
  const Trips trips(rows, first, step, team);
  const T *source = x + first * stride + at.t * V, *source_dy = dy + first * D + at.t * V;  // of the next row to fetch
  auto fetch = [&](int k, uint32_t to) {
    const int chunks = k < trips.mine ? at.count : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      copy_async_16(to + c * slot, source + c * team * V, c < chunks, x);
      copy_async_16(to + (CH + c) * slot, source_dy + c * team * V, c < chunks, x);
    }
    copy_async_commit();
    source += step * stride;
    source_dy += step * D;
  };
  const uint32_t row_bytes = 2 * CH * slot;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, ring + s * row_bytes);
  fill_vector<T>(scale, weight, w_type, 1.0f, D, team);
  __syncthreads();
  float2 aw[CH][V / 2], ab[CH][V / 2];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) aw[c][j] = ab[c][j] = both(0.0f);
  }
  int parity = 0;
  uint32_t here = ring;  // the row's stage
  const float *mean_next = mean + first, *rstd_next = rstd + first;
  float mu_next = 0.0f, r_next = 0.0f;
  if (trips.mine > 0) mu_next = *mean_next, r_next = *rstd_next;
  T* out = dx + first * D + at.t * V;
  for (int k = 0; k < trips.all; ++k, parity ^= 1, out += step * D) {
    // a row past the end has r = 0 and dy = 0: nothing in any sum
    const float r = r_next, base = -mu_next * r_next;
    mu_next = r_next = 0.0f;
    mean_next += step;
    rstd_next += step;
    if (k + 1 < trips.mine) mu_next = *mean_next, r_next = *rstd_next;
    copy_async_wait<S - 1>();
    float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], g[V / 2], w[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
      unpack2<T>(read_shared_16(here + (CH + c) * slot), g);
      read_vector<T>(my_scale, c, team, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 xh = fma2(v[j], both(r), both(base));
        aw[c][j] = fma2(g[j], xh, aw[c][j]);
        ab[c][j] = add2(ab[c][j], g[j]);
        g[j] = mul2(g[j], w[j]);
        s0 = add2(s0, g[j]);
        s1 = fma2(g[j], xh, s1);
      }
    }
    float s[2] = {s0.x + s0.y, s1.x + s1.y};
    own_team_sum<1>(s, team, part[parity]);
    const int chunks = dx != nullptr && k < trips.mine ? at.count : 0;  // to write
    const float2 c1 = both(-r * (s[0] * inv)), c2 = both(-r * (s[1] * inv));
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], g[V / 2], w[V / 2];
      // read again: held from the first pass on, they would take 32 of 128 registers, and others would be spilled
      unpack2<T>(read_shared_16(here + c * slot), v);
      unpack2<T>(read_shared_16(here + (CH + c) * slot), g);
      read_vector<T>(my_scale, c, team, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        v[j] = fma2(fma2(v[j], both(r), both(base)), c2, fma2(mul2(g[j], w[j]), both(r), c1));
      }
      if (c < chunks) store2<T>(out + c * team * V, v);
    }
    fetch(k + S, here);  // this thread's chunks have been read
    here = here == ring + (S - 1) * row_bytes ? ring : here + row_bytes;
  }
  copy_async_wait<0>();
  if (part_w == nullptr && part_b == nullptr) return;
  __syncthreads();
  // every thread leaves its sums in the ring's place, [team][weight, bias][chunk and quarter][thread], and the block adds up the teams
  constexpr int PARTS = V / 4;
  float4* sums = reinterpret_cast<float4*>(scale + team * CH * V);
  const int quads = CH * PARTS * team;
  float4* my_sums = sums + threadIdx.x / team * 2 * quads + at.t;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      my_sums[(c * PARTS + h) * team] = make_float4(aw[c][2 * h].x, aw[c][2 * h].y, aw[c][2 * h + 1].x, aw[c][2 * h + 1].y);
      my_sums[quads + (c * PARTS + h) * team] = make_float4(ab[c][2 * h].x, ab[c][2 * h].y, ab[c][2 * h + 1].x, ab[c][2 * h + 1].y);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * quads; i += blockDim.x) {
    const int q = i < quads ? i : i - quads;
    float* out_row = i < quads ? part_w : part_b;
    const int col = (q / team / PARTS * team + q % team) * V + q / team % PARTS * 4;
    if (out_row == nullptr || col >= D) continue;
    float4 total = sums[i];
    for (int n = 1; n < teams; ++n) {
      const float4 f = sums[n * 2 * quads + i];
      total.x += f.x, total.y += f.y, total.z += f.z, total.w += f.w;
    }
    float* to = out_row + static_cast<long long>(blockIdx.x) * D + col;
    to[0] = total.x, to[1] = total.y, to[2] = total.z, to[3] = total.w;
  }
}

// ---- many rows off 16-byte boundaries -----------------------------------------------------------------------------------
//
// Rows of odd width start anywhere. Read value by value they took ten times as long as their bytes (4093 x 2051 fp16: 48 us
// forward, 80 backward; here 20 and 27, bound by instructions: two to four times the time of rows on 16 bytes). Here the 16-byte pieces that cover a row are copied to shared memory as they lie, and values are taken from there: a
// thread has pairs of neighbours (fp32: single values), side by side with its neighbours' pairs, out of two words and a shift where
// the row starts in the middle of one. What a piece has beside the row, up to 14 bytes in front of and behind a
// tensor's memory, belongs to rows or allocations beside it, may be written by others meanwhile, and is not looked at. This is intended, and cannot
// fault: a 16-byte piece never lies in two pages. A thread reads what others copied, so a team also meets before a
// row; that it then is past the row before frees that row's place for the next fetch.

// What a thread has of a row: PAIRS pairs of values, and how they lie. WORDS (16-bit types): a pair is a word of memory, for all of a
// team's rows alike; where they start in the middle of one, pairs begin a value before the row (`before` = 1).
template <typename T, bool WORDS>
struct Shifted {
  static constexpr int PAIRS = STREAM_CHUNKS * VALUES<T> / 2;
  int t, team, D, before;
  int firsts, seconds;  // pairs whose first, and whose second value is in the row (the first pair's first: has_first)

  __device__ __forceinline__ Shifted(int t_, int team_, int D_, int before_) : t(t_), team(team_), D(D_), before(WORDS ? before_ : 0) {
    const int d = 2 * team;  // from a thread's pair to its next
    const int a = first(0), b = second(0);
    firsts = a < D ? (D - a + d - 1) / d : 0;
    seconds = b < D ? (D - b + d - 1) / d : 0;
  }
  __device__ __forceinline__ int first(int k) const { return sizeof(T) == 2 ? 2 * (k * team + t) - before : 2 * k * team + t; }
  __device__ __forceinline__ int second(int k) const { return sizeof(T) == 2 ? first(k) + 1 : first(k) + team; }
  __device__ __forceinline__ bool has_first(int k) const { return k < firsts && !(WORDS && k == 0 && t < before); }

  __device__ __forceinline__ static float2 of_word(uint32_t word) {
    if constexpr (std::is_same<T, bf16>::value) {
      return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
    } else {
      return __half22float2(*reinterpret_cast<const __half2*>(&word));
    }
  }
  // row: shared address of the row's first value
  __device__ __forceinline__ float2 read(uint32_t row, int k) const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(read_word_as_float(row + first(k) * 4), read_word_as_float(row + second(k) * 4));
    } else if constexpr (WORDS) {
      return of_word(read_word(row + first(k) * 2));
    } else {
      const uint32_t at = row + first(k) * 2, word = at & ~3u;
      return of_word(__funnelshift_r(read_word(word), read_word(word + 4), (at & 2u) * 8));
    }
  }
  // of a vector in fp32, which is there `before` places further on for WORDS
  __device__ __forceinline__ float2 read_vector(uint32_t vector, int k) const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(read_word_as_float(vector + first(k) * 4), read_word_as_float(vector + second(k) * 4));
    } else {
      float2 v;
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(vector + 8 * (k * team + t)) : "memory");
      return v;
    }
  }
  // words: the row starts at a word (WORDS: pairs do)
  __device__ __forceinline__ void write(T* row, int k, float2 v, bool words) const {
    if constexpr (sizeof(T) == 2) {
      if ((WORDS || words) && k < seconds && has_first(k)) {
        const T pair[2] = {from_float<T>(v.x), from_float<T>(v.y)};
        *reinterpret_cast<uint32_t*>(row + first(k)) = *reinterpret_cast<const uint32_t*>(pair);
        return;
      }
    }
    if (has_first(k)) row[first(k)] = from_float<T>(v.x);
    if (k < seconds) row[second(k)] = from_float<T>(v.y);
  }
  // zero beside the row. (Leaving the loops where no thread of a team has a pair any more breaks them into pieces: 8192 x 4097 bf16
  // took 84 us forward for 56, 121 backward for 90.)
  __device__ __forceinline__ float2 inside(int k, float2 v) const {
    return make_float2(has_first(k) ? v.x : 0.0f, k < seconds ? v.y : 0.0f);
  }

  __device__ __forceinline__ static uint32_t read_word(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
  }
  __device__ __forceinline__ static float read_word_as_float(uint32_t at) { return __uint_as_float(read_word(at)); }

  // copies the pieces that cover `row` to shared memory from `to` on; the row's first value then lies (address of row) % 16
  // further
  __device__ __forceinline__ void fetch(uint32_t to, const T* row, bool any) const {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(row), end = begin + D * sizeof(T), from = begin & ~static_cast<uintptr_t>(15);
#pragma unroll
    for (int c = 0; c < STREAM_CHUNKS; ++c) {
      const uintptr_t piece = from + (c * team + t) * 16;
      copy_async_16(to + (c * team + t) * 16, reinterpret_cast<const void*>(piece), any && piece < end, reinterpret_cast<const void*>(from));
    }
  }
};

template <typename T>
__device__ __forceinline__ uint32_t phase(const T* row) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15);
}

// every thread of a team, for what the others wrote to shared memory
__device__ __forceinline__ void team_meet(int barrier, int team) {
  if (team > 32) {
    team_barrier(barrier + threadIdx.x / team, team);
  } else {
    __syncwarp();
  }
}

// A vector of D values in shared memory in fp32, `fill` past its end; with WORDS twice, the second time a place further on, for teams whose
// pairs begin before the row. Filled by the whole block.
template <bool WORDS>
__device__ __forceinline__ void fill_shifted(float* to, const void* p, int type, float fill, int D, int room) {
  for (int c = threadIdx.x; c < room; c += blockDim.x) {
    to[c] = p != nullptr && c < D ? load1_as(p, type, c) : fill;
    if (WORDS) to[room + c] = p != nullptr && c > 0 && c <= D ? load1_as(p, type, c - 1) : fill;
  }
}

template <typename T, bool WORDS>
__global__ void __launch_bounds__(SHIFTED_THREADS, 1)
layer_norm_forward_shifted_kernel(const T* __restrict__ x, long long stride, const void* __restrict__ weight, int w_type,
                                  const void* __restrict__ bias, int b_type, long long rows, int D, float eps, int team,
                                  T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  extern __shared__ __align__(16) float scale[];  // weight, bias, ring
  __shared__ float part[2][1][32];
  constexpr int S = SHIFTED_STAGES, PAIRS = Shifted<T, WORDS>::PAIRS, COPIES = WORDS ? 2 : 1;
  const int room = team * STREAM_CHUNKS * VALUES<T>;
  fill_shifted<WORDS>(scale, weight, w_type, 1.0f, D, room);
  fill_shifted<WORDS>(scale + COPIES * room, bias, b_type, 0.0f, D, room);
  const int teams = blockDim.x / team;
  const uint32_t row_bytes = team * STREAM_CHUNKS * 16, ring = smem_u32(scale + 2 * COPIES * room) + threadIdx.x / team * S * row_bytes;
  const float width = static_cast<float>(D), inv = 1.0f / width;
  const long long first = static_cast<long long>(blockIdx.x) * teams + threadIdx.x / team, step = static_cast<long long>(gridDim.x) * teams;
  const Trips trips(rows, first, step, team);
  const T *source = x + first * stride, *here_source = source;
  const Shifted<T, WORDS> at(static_cast<int>(threadIdx.x) % team, team, D, static_cast<int>(phase(source) >> 1 & 1));
  const uint32_t my_scale = smem_u32(scale + at.before * room), my_shift = smem_u32(scale + (COPIES + at.before) * room);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    at.fetch(ring + s * row_bytes, s < trips.mine ? source : x, s < trips.mine);
    copy_async_commit();
    source += step * stride;
  }
  __syncthreads();
  uint32_t here = ring, free = ring + (S - 1) * row_bytes;
  T* out = y + first * D;
  for (int k = 0; k < trips.all; ++k, out += step * D, here_source += step * stride) {
    copy_async_wait<S - 2>();
    team_meet(0, team);
    at.fetch(free, k + S - 1 < trips.mine ? source : x, k + S - 1 < trips.mine);
    copy_async_commit();
    source += step * stride;
    const uint32_t row = here + phase(here_source);
    free = here;
    here = here == ring + (S - 1) * row_bytes ? ring : here + row_bytes;
    float2 v[PAIRS], s2 = both(0.0f);
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      v[j] = at.inside(j, at.read(row, j));
      s2 = add2(s2, v[j]);
    }
    float s[1] = {s2.x + s2.y};
    own_team_sum<0>(s, team, part[0]);
    const float mu = quotient(s[0], width, inv);
    s2 = both(0.0f);
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      v[j] = at.inside(j, add2(v[j], both(-mu)));
      s2 = fma2(v[j], v[j], s2);
    }
    s[0] = s2.x + s2.y;
    own_team_sum<0>(s, team, part[1]);
    const float r = rsqrtf(fmaf(s[0], inv, eps));
    if (k >= trips.mine) continue;
    if (at.t == 0 && mean != nullptr) {
      mean[first + k * step] = mu;
      rstd[first + k * step] = r;
    }
    const bool words = phase(out) % 4 == 0;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      at.write(out, j, fma2(mul2(v[j], both(r)), at.read_vector(my_scale, j), at.read_vector(my_shift, j)), words);
    }
  }
  copy_async_wait<0>();
}

template <typename T, bool WORDS>
__global__ void __launch_bounds__(SHIFTED_BACK_THREADS, 1)
layer_norm_backward_shifted_kernel(const T* __restrict__ dy, const T* __restrict__ x, long long stride,
                                   const void* __restrict__ weight, int w_type, const float* __restrict__ mean,
                                   const float* __restrict__ rstd, long long rows, int D, int team, T* __restrict__ dx,
                                   float* __restrict__ part_w, float* __restrict__ part_b) {
  extern __shared__ __align__(16) float scale[];  // weight, ring; the ring's place then holds the teams' sums
  __shared__ float part[2][2][32];
  constexpr int S = SHIFTED_STAGES, PAIRS = Shifted<T, WORDS>::PAIRS, COPIES = WORDS ? 2 : 1;
  const int room = team * STREAM_CHUNKS * VALUES<T>;
  fill_shifted<WORDS>(scale, weight, w_type, 1.0f, D, room);
  const int teams = blockDim.x / team;
  const uint32_t row_bytes = team * STREAM_CHUNKS * 16, ring = smem_u32(scale + COPIES * room) + threadIdx.x / team * S * 2 * row_bytes;
  const float inv = 1.0f / static_cast<float>(D);
  const long long first = static_cast<long long>(blockIdx.x) * teams + threadIdx.x / team, step = static_cast<long long>(gridDim.x) * teams;
  const Trips trips(rows, first, step, team);
  const T *source = x + first * stride, *source_dy = dy + first * D, *here_source = source, *here_dy = source_dy;
  const Shifted<T, WORDS> at(static_cast<int>(threadIdx.x) % team, team, D, static_cast<int>(phase(source) >> 1 & 1));
  const uint32_t my_scale = smem_u32(scale + at.before * room);
  auto fetch = [&](int k, uint32_t to) {
    at.fetch(to, k < trips.mine ? source : x, k < trips.mine);
    at.fetch(to + row_bytes, k < trips.mine ? source_dy : x, k < trips.mine);
    copy_async_commit();
    source += step * stride;
    source_dy += step * D;
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, ring + s * 2 * row_bytes);
  __syncthreads();
  float2 aw[PAIRS], ab[PAIRS];
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) aw[j] = ab[j] = both(0.0f);
  uint32_t here = ring, free = ring + (S - 1) * 2 * row_bytes;
  int parity = 0;
  const float *mean_next = mean + first, *rstd_next = rstd + first;
  float mu_next = 0.0f, r_next = 0.0f;
  if (trips.mine > 0) mu_next = *mean_next, r_next = *rstd_next;
  T* out = dx + first * D;
  for (int k = 0; k < trips.all; ++k, parity ^= 1, out += step * D, here_source += step * stride, here_dy += step * D) {
    // a row past the end has r = 0 and dy = 0: nothing in any sum
    const float r = r_next, base = -mu_next * r_next;
    mu_next = r_next = 0.0f;
    mean_next += step;
    rstd_next += step;
    if (k + 1 < trips.mine) mu_next = *mean_next, r_next = *rstd_next;
    copy_async_wait<S - 2>();
    team_meet(1, team);
    fetch(k + S - 1, free);
    const bool mine = k < trips.mine;
    const uint32_t row = here + phase(here_source), row_dy = here + row_bytes + phase(here_dy);
    free = here;
    here = here == ring + (S - 1) * 2 * row_bytes ? ring : here + 2 * row_bytes;
    float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const float2 xh = fma2(at.inside(j, at.read(row, j)), both(r), both(base));
      float2 g = at.inside(j, at.read(row_dy, j));
      aw[j] = fma2(g, xh, aw[j]);
      ab[j] = add2(ab[j], g);
      g = mul2(g, at.read_vector(my_scale, j));
      s0 = add2(s0, g);
      s1 = fma2(g, xh, s1);
    }
    float s[2] = {s0.x + s0.y, s1.x + s1.y};
    own_team_sum<1>(s, team, part[parity]);
    if (dx == nullptr || !mine) continue;
    const float2 c1 = both(-r * (s[0] * inv)), c2 = both(-r * (s[1] * inv));
    const bool words = phase(out) % 4 == 0;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const float2 xh = fma2(at.read(row, j), both(r), both(base)), g = mul2(at.read(row_dy, j), at.read_vector(my_scale, j));
      at.write(out, j, fma2(xh, c2, fma2(g, both(r), c1)), words);
    }
  }
  copy_async_wait<0>();
  if (part_w == nullptr && part_b == nullptr) return;
  __syncthreads();
  // [team][weight, bias], and there a value at its column
  float* sums = scale + COPIES * room;
  float* my_sums = sums + threadIdx.x / team * 2 * D;
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    if (at.has_first(j)) my_sums[at.first(j)] = aw[j].x, my_sums[D + at.first(j)] = ab[j].x;
    if (j < at.seconds) my_sums[at.second(j)] = aw[j].y, my_sums[D + at.second(j)] = ab[j].y;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) {
    float* out_row = c < D ? part_w : part_b;
    if (out_row == nullptr) continue;
    float total = sums[c];
    for (int n = 1; n < teams; ++n) total += sums[n * 2 * D + c];
    out_row[static_cast<long long>(blockIdx.x) * D + (c < D ? c : c - D)] = total;
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

// Blocks of the backward pass at most (a streaming kernel has one an SM): one row of partial sums each.
int backward_blocks(int64_t rows, int D, int type) {
  const NormShape s = norm_shape(D, type);
  const int64_t want = (rows + s.teams - 1) / s.teams, cap = static_cast<int64_t>(num_sms()) * (s.chunks == NORM_CHUNKS ? NORM_SM_THREADS / s.threads : 1);
  return static_cast<int>(want < cap ? (want > 0 ? want : 1) : cap);
}

// The streaming kernels' team and block: as many whole teams as fit. Rows off 16-byte boundaries lie in one piece more.
NormShape stream_shape(int D, int type, int most, bool vec) {
  const int values = 16 / type_bytes(type);
  const int pieces = (D + values - 1 + (vec ? 0 : values - 1)) / values;
  NormShape s;
  s.chunks = STREAM_CHUNKS;
  s.team = 1;
  while (s.team < 32 && s.team * s.chunks < pieces) s.team *= 2;
  if (s.team * s.chunks < pieces) s.team = (pieces + 32 * s.chunks - 1) / (32 * s.chunks) * 32;
  s.teams = most / s.team;
  s.threads = s.team * s.teams;
  return s;
}

// Shared memory: `vectors` fp32 vectors of the row's width, and the ring of `stages` times `inputs` rows a team, or at least
// the sums that lie in its place in the end; and 16 bytes, for the word past a value in the ring's last row.
int stream_smem(const NormShape& s, int type, int vectors, int inputs, int stages, int least) {
  const int ring = stages * inputs * STREAM_CHUNKS * s.threads * 16;
  return vectors * s.team * STREAM_CHUNKS * (16 / type_bytes(type)) * static_cast<int>(sizeof(float)) + (ring > least ? ring : least) + 16;
}

// A ring pays where a team has several rows to go through.
bool streams(int64_t rows, const NormShape& s, int smem) {
  return s.teams > 0 && smem <= STREAM_SMEM && rows > 2ll * num_sms() * s.teams && rows < 1ll << 31;
}

// `kernel` with STREAM_SMEM allowed, once for a device
template <typename K>
bool allow_stream_smem(K kernel, PerDevice& room) {
  return room.get([&] {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return 1;
  }) > 0;
}

// How the streaming kernels read a row: as 16-byte pieces, as words (16-bit values, two a word, where every operand's rows start alike in a word),
// as single values.
enum { STREAM_PIECES = 0, STREAM_WORDS = 1, STREAM_VALUES = 2 };

template <typename T>
int forward_stream(int how, const void* x, int64_t stride, const void* w, int w_type, const void* b, int b_type, int64_t rows, int D,
                   float eps, const NormShape& s, int smem, void* y, float* mean, float* rstd, cudaStream_t stream) {
  static PerDevice room[3];
  auto kernel = how == STREAM_PIECES  ? layer_norm_forward_stream_kernel<T>
                : how == STREAM_WORDS ? layer_norm_forward_shifted_kernel<T, sizeof(T) == 2>
                                      : layer_norm_forward_shifted_kernel<T, false>;
  if (!allow_stream_smem(kernel, room[how])) return FFM_ERR_LAUNCH;
  kernel<<<num_sms(), s.threads, smem, stream>>>(static_cast<const T*>(x), stride, w, w_type, b, b_type, rows, D, eps, s.team,
                                                 static_cast<T*>(y), mean, rstd);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

// stages: of STREAM_PIECES
template <typename T>
int backward_stream(int how, int stages, const void* dy, const void* x, int64_t stride, const void* w, int w_type, const float* mean, const float* rstd,
                    int64_t rows, int D, const NormShape& s, int smem, void* dx, float* part_w, float* part_b, cudaStream_t stream) {
  static PerDevice room[4];
  auto kernel = how == STREAM_WORDS              ? layer_norm_backward_shifted_kernel<T, sizeof(T) == 2>
                : how == STREAM_VALUES           ? layer_norm_backward_shifted_kernel<T, false>
                : stages == STREAM_BACK_STAGES ? layer_norm_backward_stream_kernel<T, STREAM_BACK_STAGES>
                                               : layer_norm_backward_stream_kernel<T, STREAM_STAGES>;
  if (!allow_stream_smem(kernel, room[how == STREAM_PIECES && stages == STREAM_BACK_STAGES ? 3 : how])) return FFM_ERR_LAUNCH;
  kernel<<<num_sms(), s.threads, smem, stream>>>(static_cast<const T*>(dy), static_cast<const T*>(x), stride, w, w_type, mean, rstd, rows, D,
                                                 s.team, static_cast<T*>(dx), part_w, part_b);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
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

template <typename F>
int with_type(int type, F&& f) {
  if (type == FFM_TYPE_BF16) return f(bf16{});
  if (type == FFM_TYPE_FP16) return f(fp16{});
  return f(float{});
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
  return with_type(type, with_chunks);
}

// 16-byte accesses: every row of every operand starts on a 16-byte boundary and is a whole number of them
template <typename... P>
bool norm_vectors(int type, int64_t stride, int D, const P*... p) {
  return static_cast<int64_t>(D) * type_bytes(type) % 16 == 0 && (stride * type_bytes(type)) % 16 == 0 && !off_16_bytes(p...);
}

// 16-bit rows of all operands start alike in a word, and so do all rows of a team (an even number of rows apart).
template <typename... P>
bool norm_words(int type, int64_t stride, int D, const NormShape& s, const void* x, const P*... p) {
  const uintptr_t base = reinterpret_cast<uintptr_t>(x);
  return type != FFM_TYPE_FP32 && (stride - D) % 2 == 0 && (D % 2 == 0 || num_sms() * s.teams % 2 == 0) &&
         ((p == nullptr || (reinterpret_cast<uintptr_t>(p) - base) % 4 == 0) && ...);
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
  if (!(eps >= 0.0f)) return FFM_ERR_BAD_ARG;
  if (D > max_columns(x_type)) return FFM_ERR_UNSUPPORTED;
  if (rows == 0) return FFM_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return FFM_ERR_BAD_ARG;
  const NormShape s = norm_shape(D, x_type);
  const bool vec = norm_vectors(x_type, row_stride, D, x, y);
  const NormShape r = stream_shape(D, x_type, vec ? STREAM_THREADS : SHIFTED_THREADS, vec);
  int how = vec ? STREAM_PIECES : (norm_words(x_type, row_stride, D, r, x, y) ? STREAM_WORDS : STREAM_VALUES);
  int smem = stream_smem(r, x_type, how == STREAM_WORDS ? 4 : 2, 1, vec ? STREAM_STAGES : SHIFTED_STAGES, 0);
  if (how == STREAM_WORDS && smem > STREAM_SMEM) {
    how = STREAM_VALUES;
    smem = stream_smem(r, x_type, 2, 1, SHIFTED_STAGES, 0);
  }
  if (streams(rows, r, smem)) {
    return with_type(x_type, [&](auto tag) {
      return forward_stream<decltype(tag)>(how, x, row_stride, weight, w_type, bias, b_type, rows, D, eps, r, smem, y, mean, rstd,
                                           static_cast<cudaStream_t>(stream));
    });
  }
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
  const bool vectors = norm_vectors(x_type, row_stride, D, dy, x, dx);
  const NormShape r = stream_shape(D, x_type, vectors ? STREAM_BACK_THREADS : SHIFTED_BACK_THREADS, vectors);
  const int sums = r.threads * STREAM_CHUNKS * (16 / type_bytes(x_type)) * 2 * static_cast<int>(sizeof(float));
  int how = vectors ? STREAM_PIECES : (norm_words(x_type, row_stride, D, r, x, dy, dx) ? STREAM_WORDS : STREAM_VALUES);
  int stages = STREAM_BACK_STAGES;
  int smem = stream_smem(r, x_type, how == STREAM_WORDS ? 2 : 1, 2, vectors ? STREAM_BACK_STAGES : SHIFTED_STAGES, sums);
  if (how == STREAM_WORDS && smem > STREAM_SMEM) {
    how = STREAM_VALUES;
    smem = stream_smem(r, x_type, 1, 2, SHIFTED_STAGES, sums);
  }
  if (vectors && smem > STREAM_SMEM) {
    stages = STREAM_STAGES;
    smem = stream_smem(r, x_type, 1, 2, STREAM_STAGES, sums);
  }
  const bool stream_rows = streams(rows, r, smem);
  const int blocks = stream_rows ? num_sms() : backward_blocks(rows, D, x_type);
  float* part_w = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  float* part_b = dbias != nullptr ? static_cast<float*>(workspace) + static_cast<size_t>(blocks) * D : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = stream_rows ? with_type(x_type, [&](auto tag) {
    return backward_stream<decltype(tag)>(how, stages, dy, x, row_stride, weight, w_type, mean, rstd, rows, D, r, smem, dx, part_w, part_b, st);
  }) : dispatch_norm(x_type, s, vectors, [&](auto tag, auto ch, auto vec, auto threads) {
    return backward_as<decltype(tag), decltype(ch)::value, decltype(vec)::value, decltype(threads)::value>(
        dy, x, row_stride, weight, w_type, mean, rstd, rows, D, s, dx, part_w, part_b, blocks, st);
  });
  if (rc != FFM_OK || !parts) return rc;
  layer_norm_sum_kernel<<<dim3((D + 31) / 32, 2), 256, 0, st>>>(part_w, part_b, blocks, D, dweight, w_type, dbias, b_type);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}
