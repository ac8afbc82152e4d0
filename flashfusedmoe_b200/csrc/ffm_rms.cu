// Root-mean-square norm over the last dimension with the residual's addition in front of it, an output in x's type or in e4m3 with a
// scale for every 128 columns, and its backward pass.
//
//   h = x + residual, rounded to x's type: the residual stream that is handed on, and what is normalised
//   r = 1 / sqrt(mean(h^2) + eps), xh = h r, y = xh w          (w: weight + offset)
//   e4m3: s = max |y| / 448 over a block of 128 columns, q = y / s
//   g = dy w:  dx = r (g - xh mean(g xh)) + dh      dw = sum over rows of dy xh
//
// HBM-bound: forward reads x and the residual and writes h and y, backward reads dy, dh and h and writes dx, the gradient of both
// inputs. One sum over a row is all that stands between reading and writing it. bf16 with a residual: 16384 x 1024 forward 23 us, backward 27 + 3 (4.5 to
// 5.9 TB/s; 7 rows a team), 8192 x 7168 with 8 bits out 76 us (5.4 TB/s; instructions for a scale, a quotient and a rounding a value).
#include "ffm_device.h"
#include "ffm_e4m3.cuh"
#include "ffm_internal.h"
#include "ffm_norm_common.cuh"

namespace ffm {

namespace {

constexpr int RMS_THREADS = 256;    // of a block, about, unless one row takes more
constexpr int RMS_TEAM = 1024;      // threads of a row at most
constexpr int RMS_CHUNKS_MAX = 4;   // chunks of 16 bytes of a row that a thread holds at most
// backward: threads of a block of the kernel for any rows (80 registers with two chunks) and of the streaming one (128 registers)
constexpr int RMS_BACK_TEAM = 512, RMS_BACK_SM_THREADS = 768, RMS_STREAM_THREADS = 512;
constexpr int RMS_STREAM_SMEM = 226 << 10;

// h, packed as the row lies in memory. Two 16-bit values at a time: the sum in fp32 rounded to 16 bits is the sum rounded once (24 bits hold twice 11 and 2).
template <typename T>
__device__ __forceinline__ uint4 add_packed(const uint4& a, const uint4& b) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(__uint_as_float(a.x) + __uint_as_float(b.x)), __float_as_uint(__uint_as_float(a.y) + __uint_as_float(b.y)),
                      __float_as_uint(__uint_as_float(a.z) + __uint_as_float(b.z)), __float_as_uint(__uint_as_float(a.w) + __uint_as_float(b.w)));
  } else {
    using T2 = std::conditional_t<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>;
    auto add = [](uint32_t u, uint32_t v) {
      const T2 sum = __hadd2(*reinterpret_cast<const T2*>(&u), *reinterpret_cast<const T2*>(&v));
      return *reinterpret_cast<const uint32_t*>(&sum);
    };
    return make_uint4(add(a.x, b.x), add(a.y, b.y), add(a.z, b.z), add(a.w, b.w));
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_packed(T* p, const Place<T, VEC>& at, int c, const uint4& raw) {
  if constexpr (VEC) {
    if (at.has(c, 0)) *reinterpret_cast<uint4*>(p + at.column(c, 0)) = raw;
  } else {
    float v[VALUES<T>];
    unpack<T>(raw, v);
    store_chunk(p, at, c, v);
  }
}

// y of a thread's chunks as e4m3, and the scales of the blocks of 128 columns that 16 (fp32: 32) neighbouring lanes hold; chunks from `chunks` on are past
// the row's end, which may lie inside a block
template <typename T, int CH>
__device__ __forceinline__ void store_e4m3(const float2 (&v)[CH][VALUES<T> / 2], int chunks, const Place<T, true>& at, uint8_t* y, float* y_scale) {
  constexpr int V = VALUES<T>;
  float top[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    top[c] = 0.0f;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) top[c] = fmaxf(top[c], c < chunks ? fmaxf(fabsf(v[c][j].x), fabsf(v[c][j].y)) : 0.0f);
#pragma unroll
    for (int o = E4M3_BLOCK / V / 2; o > 0; o >>= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
  }
  quantize_chunks(v, top, [&](int c, const uint32_t(&word)[V / 4], float s) {
    if (c >= chunks) return;
    const int col = at.column(c, 0);
    store_words(y + col, word);
    if (col % E4M3_BLOCK == 0) y_scale[col / E4M3_BLOCK] = s;
  });
}

// A team of threads for every row, each holding CH chunks of 16 bytes in registers. E4M3: y and y_scale [rows, ceil(D / 128)] instead of y in T;
// the 16 (fp32: 32) neighbours that hold a block's columns meet in a butterfly.
template <typename T, int CH, bool VEC, bool E4M3>
__global__ void __launch_bounds__(RMS_TEAM)
rms_norm_forward_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ residual, long long residual_stride,
                        const void* __restrict__ weight, int w_type, float offset, long long rows, int D, float eps, int team,
                        T* __restrict__ h, void* __restrict__ y, float* __restrict__ y_scale, float* __restrict__ rstd) {
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>;
  const Place<T, VEC> all(team, D);
  const int teams = blockDim.x / team;
  // single values: the weight's stay in registers for all rows of a thread, or they would be fetched one by one
  constexpr bool HELD = !VEC && CH == 1;
  float held[V];
  if (HELD) load_vector<T, VEC>(weight, w_type, all, 0, 1.0f, held);
  int parity = 0;
  for (long long base = static_cast<long long>(blockIdx.x) * teams; base < rows; base += static_cast<long long>(gridDim.x) * teams, parity ^= 1) {
    const long long row = base + threadIdx.x / team;
    Place<T, VEC> at = all;
    if (row >= rows) at.count = 0;  // goes along for the sums
    uint4 raw[CH];
    load_row(x + (row < rows ? row : 0) * x_stride, at, raw);
    if (residual != nullptr) {
      uint4 more[CH];
      load_row(residual + (row < rows ? row : 0) * residual_stride, at, more);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        raw[c] = add_packed<T>(raw[c], more[c]);
        store_packed(h + row * D, at, c, raw[c]);
      }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V];
      unpack<T>(raw[c], v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] = fmaf(v[j], v[j], s[0]);
    }
    team_sum(s, team, part[parity]);
    stay_packed(raw);
    const float r = rsqrtf(s[0] / static_cast<float>(D) + eps);
    if (rstd != nullptr && at.t == 0 && row < rows) rstd[row] = r;
    [[maybe_unused]] float2 pairs[E4M3 ? CH : 1][V / 2];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], w[V];
      unpack<T>(raw[c], v);
      if constexpr (HELD) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = held[j];
      } else {
        load_vector<T, VEC>(weight, w_type, at, c, 1.0f, w);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] * r * (w[j] + offset);
      if constexpr (!E4M3) {
        store_chunk(static_cast<T*>(y) + row * D, at, c, v);
      } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) pairs[c][j] = make_float2(v[2 * j], v[2 * j + 1]);
      }
    }
    if constexpr (E4M3) store_e4m3<T, CH>(pairs, at.count, at, static_cast<uint8_t*>(y) + row * D, y_scale + row * ((D + E4M3_BLOCK - 1) / E4M3_BLOCK));
  }
}

// dx (skipped where null), and for every block one row of partial sums of dw. dh: null
// where no residual stream was handed on. Any rows.
template <typename T, int CH, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1)
rms_norm_backward_kernel(const T* __restrict__ dy, const T* __restrict__ dh, const T* __restrict__ h, long long h_stride,
                         const void* __restrict__ weight, int w_type, float offset, const float* __restrict__ rstd, long long rows, int D,
                         int team, T* __restrict__ dx, float* __restrict__ parts) {
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>;
  const Place<T, VEC> at(team, D);
  const int teams = blockDim.x / team;
  const long long step = static_cast<long long>(gridDim.x) * teams;
  float aw[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) aw[c][j] = 0.0f;
  }
  // single values: the weight's stay in registers (8 of 85), or they would be fetched one by one twice a row
  constexpr bool HELD = !VEC && CH == 1;
  float held[V];
  if (HELD) load_vector<T, VEC>(weight, w_type, at, 0, 1.0f, held);
  auto weights = [&](int c, const Place<T, VEC>& here, float(&w)[V]) {
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = held[j];
    } else {
      load_vector<T, VEC>(weight, w_type, here, c, 1.0f, w);
    }
  };
  int parity = 0;
  // all teams of a block go through their rows in step
  for (long long base = static_cast<long long>(blockIdx.x) * teams; base < rows; base += step, parity ^= 1) {
    const long long row = base + threadIdx.x / team;
    Place<T, VEC> here = at;
    if (row >= rows) here.count = 0;
    const long long from = row < rows ? row : 0;
    const float r = rstd[from];
    uint4 v_raw[CH], g_raw[CH];
    load_row(h + from * h_stride, here, v_raw);
    load_row(dy + from * D, here, g_raw);
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], g[V], w[V];
      unpack<T>(v_raw[c], v);
      unpack<T>(g_raw[c], g);
      weights(c, here, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = here.has(c, VEC ? 0 : j) ? v[j] * r : 0.0f;
        aw[c][j] = fmaf(g[j], xh, aw[c][j]);
        s[0] = fmaf(g[j] * (w[j] + offset), xh, s[0]);
      }
    }
    team_sum(s, team, part[parity]);
    if (dx == nullptr) continue;
    stay_packed(v_raw);
    stay_packed(g_raw);
    const float c2 = -r * (s[0] / static_cast<float>(D));
    uint4 more[CH];
    if (dh != nullptr) load_row(dh + from * D, here, more);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[V], g[V], w[V], m[V];
      unpack<T>(v_raw[c], v);
      unpack<T>(g_raw[c], g);
      weights(c, here, w);
#pragma unroll
      for (int j = 0; j < V; ++j) m[j] = 0.0f;
      if (dh != nullptr) unpack<T>(more[c], m);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf(v[j] * r, c2, fmaf(g[j] * (w[j] + offset), r, m[j]));
      store_chunk(dx + row * D, here, c, v);
    }
  }
  if (parts == nullptr) return;
  for (int o = team; o < 32; o <<= 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) aw[c][j] += __shfl_xor_sync(0xffffffffu, aw[c][j], o);
    }
  }
  // one row of sums a block: its teams (of a warp or more) add theirs one after the other
  extern __shared__ float sums[];
  const int wide = team < 32 ? 32 : team, groups = blockDim.x / wide;
  float* to = parts + static_cast<long long>(blockIdx.x) * D;
  for (int g = 0; g < groups; ++g) {
    if (threadIdx.x / wide == g && threadIdx.x % wide < team) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (!at.has(c, VEC ? 0 : j)) continue;
          const int col = at.column(c, j);
          const float total = g > 0 ? sums[col] + aw[c][j] : aw[c][j];
          if (g + 1 < groups) {
            sums[col] = total;
          } else {
            to[col] = total;
          }
        }
      }
    }
    if (g + 1 < groups) __syncthreads();
  }
}

// The weight (and offset) in shared memory in fp32, four neighbours of every thread side by side: threads read 16 bytes each without a bank in
// common. Filled by the whole block.
template <typename T>
__device__ __forceinline__ void fill_weight(float* to, const void* weight, int type, float offset, int D, int team) {
  constexpr int V = VALUES<T>, PARTS = V / 4;
  for (int i = threadIdx.x; i < team * RMS_CHUNKS_MAX * V; i += blockDim.x) {
    const int j = i & 3, quad = i >> 2, t = quad % team, p = quad / team;
    const int col = (p / PARTS * team + t) * V + p % PARTS * 4 + j;
    to[i] = offset + (weight != nullptr && col < D ? load1_as(weight, type, col) : 1.0f);
  }
}

template <typename T>
__device__ __forceinline__ void read_weight(uint32_t thread_base, int c, int team, float2 (&w)[VALUES<T> / 2]) {
  constexpr int PARTS = VALUES<T> / 4;
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    const uint4 u = read_shared_16(thread_base + (c * PARTS + p) * team * 16);
    w[2 * p] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    w[2 * p + 1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
}

// Rows of a team: its own, and how often its loop runs (teams of less than a warp go in step with their warp's first).
struct RmsTrips {
  long long first, step;
  int mine, all;
  __device__ __forceinline__ RmsTrips(long long rows, int team) {
    const int teams = blockDim.x / team;
    first = static_cast<long long>(blockIdx.x) * teams + threadIdx.x / team;
    step = static_cast<long long>(gridDim.x) * teams;
    auto count = [&](long long from) { return from < rows ? static_cast<int>((rows - from + step - 1) / step) : 0; };
    mine = count(first);
    all = team < 32 ? count(first - (threadIdx.x & 31) / team) : mine;
  }
};

// Many rows of 16-byte boundaries: every thread copies its chunks of the next rows to shared memory (S rows ahead; it reads back what it copied
// itself), the weight lies there in fp32, and teams of one block go their own way. A row waits for the next ones' copies to be on their way, not
// for its own sum (8192 x 7168 bf16 in 8 bits with a team a row and nothing ahead: 98 us).
template <typename T, int S, bool RESIDUAL, bool E4M3>
__global__ void __launch_bounds__(RMS_STREAM_THREADS, 1)
rms_norm_forward_stream_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ residual, long long residual_stride,
                               const void* __restrict__ weight, int w_type, float offset, long long rows, int D, float eps, int team,
                               T* __restrict__ h, void* __restrict__ y, float* __restrict__ y_scale, float* __restrict__ rstd) {
  extern __shared__ __align__(16) float scale[];  // weight, ring
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>, CH = RMS_CHUNKS_MAX, IN = RESIDUAL ? 2 : 1;
  const Place<T, true> at(team, D);
  const uint32_t my_scale = smem_u32(scale) + at.t * 16;
  const uint32_t ring = smem_u32(scale + team * CH * V) + threadIdx.x * 16, slot = blockDim.x * 16, row_bytes = IN * CH * slot;
  const float inv = 1.0f / static_cast<float>(D);
  const int across = (D + E4M3_BLOCK - 1) / E4M3_BLOCK;
  const RmsTrips trips(rows, team);
  const T *source = x + trips.first * x_stride + at.t * V, *source_r = RESIDUAL ? residual + trips.first * residual_stride + at.t * V : nullptr;
  auto fetch = [&](int k, uint32_t to) {
    const int chunks = k < trips.mine ? at.count : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      copy_async_16(to + c * slot, source + c * team * V, c < chunks, x);
      if (RESIDUAL) copy_async_16(to + (CH + c) * slot, source_r + c * team * V, c < chunks, x);
    }
    copy_async_commit();
    source += trips.step * x_stride;
    if (RESIDUAL) source_r += trips.step * residual_stride;
  };
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, ring + s * row_bytes);
  fill_weight<T>(scale, weight, w_type, offset, D, team);
  __syncthreads();
  int parity = 0;
  uint32_t here = ring;  // the row's stage
  for (int k = 0; k < trips.all; ++k, parity ^= 1) {
    const long long row = trips.first + k * trips.step;
    const int chunks = k < trips.mine ? at.count : 0;  // to write
    copy_async_wait<S - 1>();
    uint4 raw[CH];
    float2 s2 = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw[c] = read_shared_16(here + c * slot);
      if (RESIDUAL) {
        raw[c] = add_packed<T>(raw[c], read_shared_16(here + (CH + c) * slot));
        if (c < chunks) *reinterpret_cast<uint4*>(h + row * D + at.column(c, 0)) = raw[c];
      }
      float2 v[V / 2];
      unpack2<T>(raw[c], v);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) s2 = fma2(v[j], v[j], s2);
    }
    fetch(k + S, here);  // this thread's chunks have been read
    here = here == ring + (S - 1) * row_bytes ? ring : here + row_bytes;
    float s[1] = {s2.x + s2.y};
    own_team_sum<1>(s, team, part[parity]);
    const float r = rsqrtf(fmaf(s[0], inv, eps));
    if (rstd != nullptr && at.t == 0 && chunks > 0) rstd[row] = r;
    [[maybe_unused]] float2 pairs[E4M3 ? CH : 1][V / 2];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], w[V / 2];
      unpack2<T>(raw[c], v);
      read_weight<T>(my_scale, c, team, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[j] = mul2(mul2(v[j], both(r)), w[j]);
      if constexpr (E4M3) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) pairs[c][j] = v[j];
      } else {
        if (c < chunks) store2<T>(static_cast<T*>(y) + row * D + at.column(c, 0), v);
      }
    }
    if constexpr (E4M3) store_e4m3<T, CH>(pairs, chunks, at, static_cast<uint8_t*>(y) + row * D, y_scale + row * across);
  }
  copy_async_wait<0>();
}

// The backward pass in the same way. A block leaves one row of partial sums of dw.
template <typename T, int S, bool DH>
__global__ void __launch_bounds__(RMS_STREAM_THREADS, 1)
rms_norm_backward_stream_kernel(const T* __restrict__ dy, const T* __restrict__ dh, const T* __restrict__ h, long long h_stride,
                                const void* __restrict__ weight, int w_type, float offset, const float* __restrict__ rstd, long long rows,
                                int D, int team, T* __restrict__ dx, float* __restrict__ parts) {
  extern __shared__ __align__(16) float scale[];  // weight, ring; the ring's place then holds the teams' sums
  __shared__ float part[2][1][32];
  constexpr int V = VALUES<T>, CH = RMS_CHUNKS_MAX, PARTS = V / 4, IN = DH ? 3 : 2;
  const Place<T, true> at(team, D);
  const uint32_t my_scale = smem_u32(scale) + at.t * 16;
  const uint32_t ring = smem_u32(scale + team * CH * V) + threadIdx.x * 16, slot = blockDim.x * 16;
  const int teams = blockDim.x / team;
  const float inv = 1.0f / static_cast<float>(D);
  const RmsTrips trips(rows, team);
  const long long first = trips.first, step = trips.step;
  const int mine = trips.mine, all = trips.all;
  const T *source = h + first * h_stride + at.t * V, *source_dy = dy + first * D + at.t * V, *source_dh = DH ? dh + first * D + at.t * V : nullptr;
  auto fetch = [&](int k, uint32_t to) {
    const int chunks = k < mine ? at.count : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      copy_async_16(to + c * slot, source + c * team * V, c < chunks, h);
      copy_async_16(to + (CH + c) * slot, source_dy + c * team * V, c < chunks, h);
      if (DH) copy_async_16(to + (2 * CH + c) * slot, source_dh + c * team * V, c < chunks, h);
    }
    copy_async_commit();
    source += step * h_stride;
    source_dy += step * D;
    if (DH) source_dh += step * D;
  };
  const uint32_t row_bytes = IN * CH * slot;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, ring + s * row_bytes);
  fill_weight<T>(scale, weight, w_type, offset, D, team);
  __syncthreads();
  float2 aw[CH][V / 2];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) aw[c][j] = both(0.0f);
  }
  int parity = 0;
  uint32_t here = ring;  // the row's stage
  const float* rstd_next = rstd + first;
  float r_next = mine > 0 ? *rstd_next : 0.0f;
  T* out = dx + first * D + at.t * V;
  for (int k = 0; k < all; ++k, parity ^= 1, out += step * D) {
    // a row past the end has r = 0 and dy = 0: nothing in any sum
    const float r = r_next;
    rstd_next += step;
    r_next = k + 1 < mine ? *rstd_next : 0.0f;
    copy_async_wait<S - 1>();
    float2 s2 = both(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], g[V / 2], w[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
      unpack2<T>(read_shared_16(here + (CH + c) * slot), g);
      read_weight<T>(my_scale, c, team, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 xh = mul2(v[j], both(r));
        aw[c][j] = fma2(g[j], xh, aw[c][j]);
        s2 = fma2(mul2(g[j], w[j]), xh, s2);
      }
    }
    float s[1] = {s2.x + s2.y};
    own_team_sum<1>(s, team, part[parity]);
    const int chunks = dx != nullptr && k < mine ? at.count : 0;  // to write
    const float2 c2 = both(-r * (s[0] * inv));  // times v r: r^2 leaves fp32 where rows are below 2^-64 and eps is 0
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float2 v[V / 2], g[V / 2], w[V / 2];
      unpack2<T>(read_shared_16(here + c * slot), v);
      unpack2<T>(read_shared_16(here + (CH + c) * slot), g);
      read_weight<T>(my_scale, c, team, w);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[j] = fma2(mul2(v[j], both(r)), c2, mul2(mul2(g[j], w[j]), both(r)));
      if (DH) {
        unpack2<T>(read_shared_16(here + (2 * CH + c) * slot), g);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) v[j] = add2(v[j], g[j]);
      }
      if (c < chunks) store2<T>(out + c * team * V, v);
    }
    fetch(k + S, here);  // this thread's chunks have been read
    here = here == ring + (S - 1) * row_bytes ? ring : here + row_bytes;
  }
  copy_async_wait<0>();
  if (parts == nullptr) return;
  __syncthreads();
  // every thread leaves its sums in the ring's place, [team][chunk and quarter][thread], and the block adds up the teams
  float4* sums = reinterpret_cast<float4*>(scale + team * CH * V);
  const int quads = CH * PARTS * team;
  float4* my_sums = sums + threadIdx.x / team * quads + at.t;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) my_sums[(c * PARTS + p) * team] = make_float4(aw[c][2 * p].x, aw[c][2 * p].y, aw[c][2 * p + 1].x, aw[c][2 * p + 1].y);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < quads; i += blockDim.x) {
    const int col = (i / team / PARTS * team + i % team) * V + i / team % PARTS * 4;
    if (col >= D) continue;
    float4 total = sums[i];
    for (int n = 1; n < teams; ++n) {
      const float4 f = sums[n * quads + i];
      total.x += f.x, total.y += f.y, total.z += f.z, total.w += f.w;
    }
    *reinterpret_cast<float4*>(parts + static_cast<long long>(blockIdx.x) * D + col) = total;
  }
}

// out[col] = sum over p of parts[p][col], in an order that depends on the number of parts alone: 32 columns a block, 32 warps that take
// every 32nd part.
__global__ void __launch_bounds__(1024)
rms_norm_sum_kernel(const float* __restrict__ parts, int count, int D, void* __restrict__ out, int type) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (col < D) {
    for (int p = warp; p < count; p += 128) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (p + 32 * u < count) a[u] += parts[static_cast<long long>(p + 32 * u) * D + col];
      }
    }
  }
  s[warp][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  const float total = warp_sum(s[lane][warp]);
  if (lane == 0 && blockIdx.x * 32 + warp < D) store1_as(out, type, blockIdx.x * 32 + warp, total);
}

// ---- host side --------------------------------------------------------------------------------------------------

int rms_columns(int type) { return RMS_TEAM * RMS_CHUNKS_MAX * (16 / type_bytes(type)); }

struct RmsShape {
  int team, chunks, threads, teams;
};

// `least` threads a row: up to a warp a power of two, beyond that whole warps; `threads` of a block, about
RmsShape rms_shape(int D, int type, int chunks, int least, int threads) {
  const int values = 16 / type_bytes(type), pieces = (D + values - 1) / values;
  RmsShape s;
  s.chunks = chunks;
  s.team = least;
  while (s.team < 32 && s.team * chunks < pieces) s.team *= 2;
  if (s.team * chunks < pieces) s.team = (pieces + 32 * chunks - 1) / (32 * chunks) * 32;
  s.teams = s.team < threads ? threads / s.team : 1;
  s.threads = s.team * s.teams;
  return s;
}

// Few rows leave SMs idle, and a row then takes as many threads as it has chunks; many rows take few threads each, up to a warp, which
// needs no barrier.
RmsShape rms_forward_shape(int64_t rows, int D, int type, bool e4m3, bool vec) {
  const int pieces = (D + 16 / type_bytes(type) - 1) / (16 / type_bytes(type));
  const int least = e4m3 ? 32 : 1;
  if (rows <= num_sms() && pieces <= RMS_TEAM) return rms_shape(D, type, 1, least, RMS_THREADS);
  // Single values: with four chunks (32 loads) a thread's registers spill; with one of 16-bit values the weight's stay in them (4093 x 2051 bf16 with a
  // residual: 30 us, with two chunks 49; fp32 61 and 41).
  if (!vec && pieces <= 2 * RMS_TEAM) return rms_shape(D, type, type != FFM_TYPE_FP32 && pieces <= RMS_TEAM ? 1 : 2, least, RMS_THREADS);
  return rms_shape(D, type, RMS_CHUNKS_MAX, least, RMS_THREADS);
}

// Single values: one chunk, whose weights stay in registers (4093 x 2051 fp16: 27 us; fetched for every row 50, with two chunks, which spill, 64)
RmsShape rms_backward_shape(int D, int type, bool vec) {
  const RmsShape s = rms_shape(D, type, vec ? 2 : 1, 1, RMS_THREADS);
  return s.team <= (vec ? RMS_BACK_TEAM : RMS_TEAM) ? s : rms_shape(D, type, RMS_CHUNKS_MAX, 1, RMS_THREADS);
}

// Blocks of the backward kernel for any rows, each with a row of partial sums
int rms_backward_blocks(int64_t rows, const RmsShape& s) {
  const int on_sm = s.chunks <= 2 && s.threads <= RMS_BACK_SM_THREADS ? RMS_BACK_SM_THREADS / s.threads : 1;
  const int64_t want = (rows + s.teams - 1) / s.teams, most = static_cast<int64_t>(num_sms()) * on_sm;
  return static_cast<int>(want < most ? (want > 0 ? want : 1) : most);
}
struct RmsStream {
  RmsShape shape;
  int stages, smem;
};

// The ring of so many inputs as deep as shared memory allows, over as many teams as go into a block; shape.teams == 0: it does not fit. Rows that fit
// once only are fetched when the one before has been read: 4096 x 16384 bf16 backward 116 us, held in registers, which spill, 307.
RmsStream rms_stream(int D, int type, int inputs, int least) {
  const int row_values = 16 / type_bytes(type);
  RmsStream r;
  auto fits = [&](const RmsShape& s, int stages) {
    const int ring = stages * inputs * RMS_CHUNKS_MAX * s.threads * 16, sums = s.threads * RMS_CHUNKS_MAX * row_values * 4;
    r.stages = stages;
    r.smem = s.team * RMS_CHUNKS_MAX * row_values * 4 + (ring > sums ? ring : sums);
    r.shape = s;
    return r.smem <= RMS_STREAM_SMEM;
  };
  for (int threads = RMS_STREAM_THREADS; threads >= 128; threads /= 2) {
    const RmsShape s = rms_shape(D, type, RMS_CHUNKS_MAX, least, threads);
    if (s.threads <= threads && (fits(s, 3) || fits(s, 2))) return r;
  }
  const RmsShape s = rms_shape(D, type, RMS_CHUNKS_MAX, least, RMS_STREAM_THREADS);
  if (s.threads <= RMS_STREAM_THREADS && fits(s, 1)) return r;
  r.shape.teams = 0;
  return r;
}

template <typename F>
int rms_with_type(int type, F&& f) {
  if (type == FFM_TYPE_BF16) return f(bf16{});
  if (type == FFM_TYPE_FP16) return f(fp16{});
  return f(float{});
}

bool rms_vectors(int type, int D, int64_t stride_a, int64_t stride_b) {
  return static_cast<int64_t>(D) * type_bytes(type) % 16 == 0 && (stride_a * type_bytes(type)) % 16 == 0 && (stride_b * type_bytes(type)) % 16 == 0;
}

// A ring pays where a team has several rows to go through.
bool rms_streams(int64_t rows, const RmsStream& r) { return r.shape.teams > 0 && rows > 2ll * num_sms() * r.shape.teams && rows < 1ll << 31; }

template <typename K>
bool rms_room(K kernel, PerDevice& room) {
  return room.get([&] {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RMS_STREAM_SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return 1;
  }) > 0;
}

template <typename T, int S, bool RESIDUAL, bool E4M3>
int launch_rms_forward_stream(const ffm_rms_norm_args& a, const RmsStream& r, cudaStream_t stream) {
  auto kernel = rms_norm_forward_stream_kernel<T, S, RESIDUAL, E4M3>;
  static PerDevice room;
  if (!rms_room(kernel, room)) return FFM_ERR_LAUNCH;
  kernel<<<num_sms(), r.shape.threads, r.smem, stream>>>(static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.residual), a.residual_stride,
                                                        a.weight, static_cast<int>(a.w_type), static_cast<float>(a.offset), a.rows,
                                                        static_cast<int>(a.D), static_cast<float>(a.eps), r.shape.team, static_cast<T*>(a.h), a.y,
                                                        a.y_scale, a.rstd);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

template <typename T, int S, bool DH>
int launch_rms_stream(const ffm_rms_norm_args& a, const RmsStream& r, float* parts, cudaStream_t stream) {
  auto kernel = rms_norm_backward_stream_kernel<T, S, DH>;
  static PerDevice room;
  if (!rms_room(kernel, room)) return FFM_ERR_LAUNCH;
  kernel<<<num_sms(), r.shape.threads, r.smem, stream>>>(static_cast<const T*>(a.dy), static_cast<const T*>(a.dh), static_cast<const T*>(a.x), a.x_stride,
                                                        a.weight, static_cast<int>(a.w_type), static_cast<float>(a.offset), a.rstd, a.rows,
                                                        static_cast<int>(a.D), r.shape.team, static_cast<T*>(a.dx), parts);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

bool rms_arguments(const ffm_rms_norm_args* a) {
  return a != nullptr && is_type(static_cast<int>(a->x_type)) && a->rows >= 0 && a->D > 0 && (a->x_stride >= a->D || a->rows <= 1) && a->eps >= 0.0 &&
         a->offset - a->offset == 0.0 && (a->weight == nullptr || is_type(static_cast<int>(a->w_type)));
}

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" int ffm_rms_norm_forward(const ffm_rms_norm_args* args, ffm_stream_t stream) {
  if (!rms_arguments(args)) return FFM_ERR_BAD_ARG;
  const ffm_rms_norm_args& a = *args;
  const int type = static_cast<int>(a.x_type);
  const bool e4m3 = a.y_scale != nullptr;
  if (a.residual != nullptr && (a.h == nullptr || (a.residual_stride < a.D && a.rows > 1))) return FFM_ERR_BAD_ARG;
  if (a.D > rms_columns(type) || (e4m3 && a.D % 16 != 0)) return FFM_ERR_UNSUPPORTED;
  if (a.rows == 0) return FFM_OK;
  if (!a.x || !a.y) return FFM_ERR_BAD_ARG;
  const int D = static_cast<int>(a.D);
  const bool vec = rms_vectors(type, D, a.x_stride, a.residual != nullptr ? a.residual_stride : 0) && !off_16_bytes(a.x, a.residual, a.h, a.weight) &&
                   (e4m3 || !off_16_bytes(a.y));
  if (e4m3 && (!vec || (reinterpret_cast<uintptr_t>(a.y) & 7u) != 0)) return FFM_ERR_UNSUPPORTED;
  const RmsStream ring = rms_stream(D, type, a.residual != nullptr ? 2 : 1, e4m3 ? 32 : 1);
  if (vec && rms_streams(a.rows, ring)) {
    return rms_with_type(type, [&](auto tag) {
      using T = decltype(tag);
      cudaStream_t st = static_cast<cudaStream_t>(stream);
      auto launch = [&](auto stages, auto residual) {
        constexpr int S = decltype(stages)::value;
        constexpr bool R = decltype(residual)::value;
        return e4m3 ? launch_rms_forward_stream<T, S, R, true>(a, ring, st) : launch_rms_forward_stream<T, S, R, false>(a, ring, st);
      };
      auto with = [&](auto stages) { return a.residual != nullptr ? launch(stages, std::true_type{}) : launch(stages, std::false_type{}); };
      return ring.stages == 3 ? with(std::integral_constant<int, 3>{}) : with(std::integral_constant<int, 2>{});  // two inputs go in twice
    });
  }
  const RmsShape s = rms_forward_shape(a.rows, D, type, e4m3, vec);
  const int64_t each = (a.rows + s.teams - 1) / s.teams, resident = static_cast<int64_t>(num_sms()) * (RMS_TEAM / s.threads);
  const int64_t blocks = !vec && s.chunks == 1 && each > resident ? resident : each;
  if (blocks > 0x7fffffffll) return FFM_ERR_UNSUPPORTED;
  return rms_with_type(type, [&](auto tag) {
    using T = decltype(tag);
    auto launch = [&](auto kernel) {
      kernel<<<static_cast<unsigned>(blocks), s.threads, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.residual), a.residual_stride, a.weight, static_cast<int>(a.w_type),
          static_cast<float>(a.offset), a.rows, D, static_cast<float>(a.eps), s.team, static_cast<T*>(a.h), a.y, a.y_scale, a.rstd);
      return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
    };
    if (e4m3) return s.chunks == 1 ? launch(rms_norm_forward_kernel<T, 1, true, true>) : launch(rms_norm_forward_kernel<T, RMS_CHUNKS_MAX, true, true>);
    if (vec) return s.chunks == 1 ? launch(rms_norm_forward_kernel<T, 1, true, false>) : launch(rms_norm_forward_kernel<T, RMS_CHUNKS_MAX, true, false>);
    return s.chunks == 1   ? launch(rms_norm_forward_kernel<T, 1, false, false>)
           : s.chunks == 2 ? launch(rms_norm_forward_kernel<T, 2, false, false>)
                           : launch(rms_norm_forward_kernel<T, RMS_CHUNKS_MAX, false, false>);
  });
}

extern "C" size_t ffm_rms_norm_workspace_bytes(int64_t rows, int D, int x_type) {
  if (rows < 0 || !is_type(x_type) || D <= 0 || D > rms_columns(x_type)) return 0;
  int most = num_sms();  // a streaming kernel's
  for (const bool vec : {false, true}) {
    const RmsShape s = rms_backward_shape(D, x_type, vec);
    const int blocks = rms_backward_blocks(rows, s);
    most = blocks > most ? blocks : most;
  }
  return sizeof(float) * static_cast<size_t>(D) * most;
}

extern "C" int ffm_rms_norm_backward(const ffm_rms_norm_args* args, ffm_stream_t stream) {
  if (!rms_arguments(args)) return FFM_ERR_BAD_ARG;
  const ffm_rms_norm_args& a = *args;
  const int type = static_cast<int>(a.x_type), D = static_cast<int>(a.D);
  if (a.dweight != nullptr && a.weight == nullptr) return FFM_ERR_BAD_ARG;
  if (a.D > rms_columns(type)) return FFM_ERR_UNSUPPORTED;
  if (a.rows > 0 && (!a.dy || !a.x || !a.rstd)) return FFM_ERR_BAD_ARG;
  if (a.dweight != nullptr && (!a.workspace || static_cast<size_t>(a.workspace_bytes) < ffm_rms_norm_workspace_bytes(a.rows, D, type))) return FFM_ERR_WORKSPACE;
  if (a.dweight == nullptr && (a.dx == nullptr || a.rows == 0)) return FFM_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* parts = a.dweight != nullptr ? static_cast<float*>(a.workspace) : nullptr;
  const bool vec = rms_vectors(type, D, a.x_stride, 0) && !off_16_bytes(a.x, a.dy, a.dh, a.dx);
  const RmsStream r = rms_stream(D, type, a.dh != nullptr ? 3 : 2, 1);
  int count, rc;
  if (vec && rms_streams(a.rows, r)) {
    count = num_sms();
    rc = rms_with_type(type, [&](auto tag) {
      using T = decltype(tag);
      auto with = [&](auto dh) {
        constexpr bool DH = decltype(dh)::value;
        if (r.stages == 1) return launch_rms_stream<T, 1, DH>(a, r, parts, st);
        return r.stages == 3 ? launch_rms_stream<T, 3, DH>(a, r, parts, st) : launch_rms_stream<T, 2, DH>(a, r, parts, st);
      };
      return a.dh != nullptr ? with(std::true_type{}) : with(std::false_type{});
    });
  } else {
    const bool wide = vec && !off_16_bytes(a.weight);
    const RmsShape s = rms_backward_shape(D, type, wide);
    const int blocks = count = rms_backward_blocks(a.rows, s);
    // for the teams' sums; several teams have rows of up to 2048 (fp32: 1024) values
    const size_t smem = s.threads > (s.team < 32 ? 32 : s.team) ? D * sizeof(float) : 0;
    rc = rms_with_type(type, [&](auto tag) {
      using T = decltype(tag);
      auto launch = [&](auto kernel) {
        kernel<<<blocks, s.threads, smem, st>>>(static_cast<const T*>(a.dy), static_cast<const T*>(a.dh), static_cast<const T*>(a.x), a.x_stride, a.weight,
                                             static_cast<int>(a.w_type), static_cast<float>(a.offset), a.rstd, a.rows, D, s.team, static_cast<T*>(a.dx),
                                             parts);
        return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
      };
      if (s.chunks == 1 && s.threads > RMS_BACK_SM_THREADS) return launch(rms_norm_backward_kernel<T, 1, false, RMS_TEAM>);
      if (s.chunks == 1) return launch(rms_norm_backward_kernel<T, 1, false, RMS_BACK_SM_THREADS>);
      if (s.chunks == 2) return launch(rms_norm_backward_kernel<T, 2, true, RMS_BACK_SM_THREADS>);
      return wide ? launch(rms_norm_backward_kernel<T, RMS_CHUNKS_MAX, true, RMS_TEAM>) : launch(rms_norm_backward_kernel<T, RMS_CHUNKS_MAX, false, RMS_TEAM>);
    });
  }
  if (rc != FFM_OK || a.dweight == nullptr) return rc;
  rms_norm_sum_kernel<<<(D + 31) / 32, 1024, 0, st>>>(parts, count, D, a.dweight, static_cast<int>(a.w_type));
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}
