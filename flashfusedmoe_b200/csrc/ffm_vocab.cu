// Linear cross entropy: softmax cross entropy of hidden [N, D] against a vocabulary weight [V, D], with its gradients.
//
//   l = h w^T    lse = log sum_v exp(l_v)    nll = lse - l_t + z lse^2
//   dl_v = g (p_v (1 + 2 z lse) - [v = t]),  p_v = exp(l_v - lse)        dh = dl w        dw = dl^T h
//
// The logits never exist: the product's epilogue (EPI_SOFTMAX, ffm_gemm_sm100.cu) leaves the maximum and the sum of exponentials of
// every 128 entries of a row, 8 bytes in place of 512, and the target's logit. For the gradients it also leaves the exponentials
// against those maxima in fp16, times 2^15, for one piece of the rows at a time. They become dl in bf16 in the same place once the row's lse is known: a
// multiplication by exp(maximum - lse), which costs 4 bytes an entry; taking the product again instead would cost 2 D
// operations an entry, more from D = 650 on (at 1.45 PFLOP/s and 6.4 TB/s). Every logit is computed once, and the three
// products are all that is left: 6 N V D operations. Statistics, sums and the target's entry (p - 1, from expm1, since
// differences from a rounded p have nothing left where p is close to 1) are fp32.
#include "ffm_types.cuh"

#include "ffm_gemm_common.cuh"
#include "ffm_internal.h"

namespace ffm {

namespace {

constexpr int HALF = 128;         // entries with one maximum
constexpr int LOSS_THREADS = 1024;

__device__ __forceinline__ double block_sum(double v, double* part) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += part[i];
  return s;
}

// a failure that some kernel before reported goes to the caller's mapped host word
__device__ __forceinline__ void report(const int32_t* status, volatile int32_t* status_host) {
  if (status_host != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    const int32_t code = *status;
    if (code != 0) *status_host = code;
  }
}

// share[0] = 1 / number of rows that count (infinite without any: the mean is NaN then), share[1] the same for the gradients (0 then)
__global__ void __launch_bounds__(LOSS_THREADS)
loss_count_kernel(const long long* __restrict__ targets, long long rows, long long ignore, float* __restrict__ share) {
  __shared__ double part[32];
  int n = 0;
  for (long long i = threadIdx.x; i < rows; i += LOSS_THREADS) n += targets[i] != ignore;
  const double count = block_sum(n, part);
  if (threadIdx.x == 0) {
    share[0] = static_cast<float>(1.0 / count);
    share[1] = count > 0.0 ? share[0] : 0.0f;
  }
}

__device__ __forceinline__ void join(float& top, float& sum, float other_top, float other_sum) {
  const float m = fmaxf(top, other_top);
  // nothing yet (-inf), or nothing but NaN: nothing to scale
  sum = (top == -INFINITY ? sum : sum * expf(top - m)) + (other_top == -INFINITY ? other_sum : other_sum * expf(other_top - m));
  top = m;
}

// From a row's maxima and sums to its loss, and (with `factor`) to what its pieces of 128 exponentials are multiplied by for the
// gradient, exp(maximum - lse) times the row's factor, over what they are stored times of. A row has TEAM threads: a warp, or a block where there are few rows.
//
// The tensor core's sums lose some of their last bits over a long D (4096: 3e-6 of a logit). That hardly shows in lse, which is over
// many entries, but in the target's logit it does; so that one is taken again here in fp32, and replaces the other in the
// row's sum as well, where it may be nearly everything (2 N D multiply-adds and 4 bytes: 0.1 % of the products).
template <int TEAM>
__global__ void __launch_bounds__(256)
loss_rows_kernel(const float2* __restrict__ stats, const float* __restrict__ target_logits, const long long* __restrict__ targets,
                 const bf16* __restrict__ hidden, const bf16* __restrict__ weight, int D, long long rows, int pieces, int V,
                 long long ignore, float z, const float* __restrict__ row_grad, float* __restrict__ nll, float* __restrict__ factor, float* __restrict__ target_entry, int32_t* status,
                 volatile int32_t* status_host) {
  report(status, status_host);
  __shared__ float part[3][8];
  const int t = threadIdx.x % TEAM, warp = threadIdx.x >> 5;
  const long long row = static_cast<long long>(blockIdx.x) * (256 / TEAM) + threadIdx.x / TEAM;
  if (row >= rows) return;  // whole teams
  const long long target = targets[row];
  const bool counts = target != ignore, known = target >= 0 && target < V;
  float top = -INFINITY, sum = 0.0f, dot = 0.0f;
  const float2* mine = stats + row * pieces;
  for (int h = t; h < pieces; h += 4 * TEAM) {
    float2 s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = h + u * TEAM < pieces ? mine[h + u * TEAM] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int u = 0; u < 4; ++u) join(top, sum, s[u].x, s[u].y);
  }
  if (counts && known) {
    const bf16 *x = hidden + row * D, *w = weight + target * D;
    for (int c = t * 8; c < D; c += TEAM * 8) {
      float a[8], b[8];
      load8(x + c, a);
      load8(w + c, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot = fmaf(a[j], b[j], dot);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other_top = __shfl_xor_sync(0xffffffffu, top, o), other_sum = __shfl_xor_sync(0xffffffffu, sum, o);
    join(top, sum, other_top, other_sum);
    dot += __shfl_xor_sync(0xffffffffu, dot, o);
  }
  if (TEAM > 32) {
    if ((threadIdx.x & 31) == 0) {
      part[0][warp] = top;
      part[1][warp] = sum;
      part[2][warp] = dot;
    }
    __syncthreads();
    top = part[0][0], sum = part[1][0], dot = part[2][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      join(top, sum, part[0][w], part[1][w]);
      dot += part[2][w];
    }
  }
  if (counts && known) {
    const float rest = sum - expf(target_logits[row] - top);
    sum = (rest < 0.0f ? 0.0f : rest) + expf(dot - top);  // (a maximum with zero would lose a NaN that some other logit brought)
  }
  // The loss and p - 1 come from the margin: lse itself is rounded at the size of the logits, which may be far above their
  // differences.
  const float log_sum = logf(sum), lse = log_sum + top, margin = log_sum + (top - dot);
  float scale = 0.0f;
  // a row with a target that is none has no gradient; its loss is NaN
  if (counts && known && factor != nullptr) {
    // One over the number of rows is not in dl but multiplies its products: as a factor of every target's entry (-1, where the model
    // has no idea) its rounding would be the same in all of them, up to 2^-8 of the whole gradient.
    const float g = row_grad != nullptr ? row_grad[row] : 1.0f;
    scale = g * fmaf(2.0f * z, lse, 1.0f);
    if (t == 0) target_entry[row] = g * fmaf(expf(-margin), 2.0f * z * lse, expm1f(-margin));
  }
  if (t == 0) {
    nll[row] = counts ? (known ? fmaf(z * lse, lse, margin) : NAN) : 0.0f;
    if (counts && !known) atomicCAS(status, 0, FFM_STATUS_BAD_INDEX);
  }
  if (factor == nullptr) return;
  float* out = factor + row * pieces;
  for (int h = t; h < pieces; h += TEAM) {
    out[h] = scale != 0.0f ? expf((mine[h].x - top) - log_sum) * scale * (1.0f / SOFTMAX_STORED_SCALE) : 0.0f;
  }
}

// e (fp16) to dl (bf16) in place: eight entries a thread, 2048 a block, GRADIENT_ROWS rows of them at a time (a row a block took
// 1.9 times as long).
constexpr int GRADIENT_ROWS = 4;

__global__ void __launch_bounds__(256)
loss_gradient_kernel(uint16_t* __restrict__ e, long long ld, int V, int pieces, const float* __restrict__ factor,
                     const long long* __restrict__ targets, const float* __restrict__ target_entry, long long ignore, long long rows) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= V) return;
  for (long long row0 = static_cast<long long>(blockIdx.y) * GRADIENT_ROWS; row0 < rows; row0 += static_cast<long long>(gridDim.y) * GRADIENT_ROWS) {
    uint4 raw[GRADIENT_ROWS];
    float f[GRADIENT_ROWS];
    long long t[GRADIENT_ROWS];
#pragma unroll
    for (int u = 0; u < GRADIENT_ROWS; ++u) {
      const long long row = row0 + u < rows ? row0 + u : rows - 1;
      raw[u] = *reinterpret_cast<const uint4*>(e + row * ld + col);
      f[u] = factor[row * pieces + col / HALF];
      t[u] = targets[row];
    }
#pragma unroll
    for (int u = 0; u < GRADIENT_ROWS; ++u) {
      const long long row = row0 + u;
      if (row >= rows) break;
      const __half2 h[4] = {*reinterpret_cast<__half2*>(&raw[u].x), *reinterpret_cast<__half2*>(&raw[u].y),
                            *reinterpret_cast<__half2*>(&raw[u].z), *reinterpret_cast<__half2*>(&raw[u].w)};
      float v[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 x = __half22float2(h[q]);
        v[2 * q] = f[u] != 0.0f ? x.x * f[u] : 0.0f;  // rows that do not count: zero whatever e is
        v[2 * q + 1] = f[u] != 0.0f ? x.y * f[u] : 0.0f;
      }
      if (t[u] >= col && t[u] < col + 8 && t[u] < V && t[u] != ignore) {
        const float entry = target_entry[row];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (t[u] == col + j) v[j] = entry;
        }
      }
      store8(reinterpret_cast<bf16*>(e + row * ld + col), v);
    }
  }
}

// loss = sum of nll (times *share), in double, in an order of its own
__global__ void __launch_bounds__(LOSS_THREADS)
loss_sum_kernel(const float* __restrict__ nll, long long rows, const float* __restrict__ share, float* __restrict__ loss,
                const int32_t* status, volatile int32_t* status_host) {
  report(status, status_host);
  __shared__ double part[32];
  double s = 0.0;
  for (long long i = threadIdx.x; i < rows; i += LOSS_THREADS) s += nll[i];
  s = block_sum(s, part);
  if (threadIdx.x == 0) *loss = static_cast<float>(share != nullptr ? s * *share : s);
}

// out = sum of `parts` fp32 matrices of n values, to bf16
__global__ void __launch_bounds__(256)
loss_join_kernel(const float* __restrict__ in, int parts, long long n, bf16* __restrict__ out) {
  for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += static_cast<long long>(gridDim.x) * 2048) {
    float v[8];
    load8(in + i, v);
    for (int k = 1; k < parts; ++k) {
      float w[8];
      load8(in + k * n + i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
    store8(out + i, v);
  }
}

struct ScaleJob {
  void* x[FFM_CAST_MAX];
  long long chunks_end[FFM_CAST_MAX];  // 8-value chunks of this tensor and all before it
  int type[FFM_CAST_MAX];
  int count;
};

// x *= *factor in place, nothing at all where that is 1
__global__ void __launch_bounds__(256)
loss_scale_kernel(const __grid_constant__ ScaleJob job, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  const long long total = job.chunks_end[job.count - 1];
  for (long long c = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; c < total; c += static_cast<long long>(gridDim.x) * 256) {
    int i = 0;
    while (c >= job.chunks_end[i]) ++i;
    const long long e = (c - (i > 0 ? job.chunks_end[i - 1] : 0)) * 8;
    float v[8];
    load8_as(job.x[i], job.type[i], e, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    store8_as(job.x[i], job.type[i], e, v);
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
//
// Scoring a handful of rows is reading the weight once (V D 2 bytes). The tiles of 256 entries do that at 6.0 TB/s where there are
// many of them (33 rows, D = 2048, 100352 entries: 70 us), but a few hundred do not share out over 148 SMs: 50257 entries are 197
// tiles, and a third of the SMs has two (D = 1024: 27 us; 2000 entries, D = 2048: 16 us).
// Here a warp takes 16 entries at a time, and up to 8 warps share their contraction (22 us and 5.4 us; where tiles share out
// evenly it is the slower one, 161 us for 137 at D = 4096, 100352 entries: 5.1 TB/s). The entries go straight from memory into the
// registers of mma.sync's A operand: which k a lane's eight neighbours count as does not matter as long as the rows, in shared
// memory as B, are read the same way, so a lane loads 16 bytes where the instruction's layout has pairs. The tensor pipe
// idles either way. Every warp that sums keeps a running maximum and sum for its entries and leaves one pair for each row.
constexpr int FEW_WARPS = 8;
constexpr int FEW_BATCH = 4;           // 32-deep steps loaded together; two batches at a time
constexpr int FEW_SMEM = 128 << 10;    // for the rows

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// NT: groups of 8 rows; `split` warps (1, 2, 4 or 8) share a group of 16 entries. stats[n][piece], one piece a group of warps.
template <int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2)
loss_few_kernel(const bf16* __restrict__ hidden, const bf16* __restrict__ weight, int rows, int D, int V, int split,
                const long long* __restrict__ targets, float* __restrict__ target_logits, float2* __restrict__ stats) {
  extern __shared__ __align__(16) uint8_t few_smem[];  // the rows, `ld` bytes apart
  __shared__ float partial[2][FEW_WARPS][NT * 4][32];
  __shared__ long long goal[NT * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int groups = FEW_WARPS / split, group = warp / split, member = warp % split;
  const int steps = (D + 31) / 32, mine = (steps + split - 1) / split, first = member * mine;
  const int ld = steps * 64 + 64;
  // rows to shared memory, zero past their end and in rows that are not there
  for (int i = threadIdx.x; i < NT * 8 * (ld / 16); i += FEW_WARPS * 32) {
    const int n = i / (ld / 16), c = i % (ld / 16) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n < rows && c < D) v = *reinterpret_cast<const uint4*>(hidden + static_cast<long long>(n) * D + c);
    *reinterpret_cast<uint4*>(few_smem + n * ld + c * 2) = v;
  }
  if (threadIdx.x < NT * 8) goal[threadIdx.x] = threadIdx.x < rows ? targets[threadIdx.x] : -1;
  __syncthreads();
  const uint32_t row_base = smem_u32(few_smem) + g * ld + q * 16;
  float top[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;
  const int units = (V + 15) / 16, stride = gridDim.x * groups;
  // A warp has a batch of steps in flight while it multiplies the one before, across its entries as well.
  struct Batch {
    uint4 low[FEW_BATCH], high[FEW_BATCH];  // entries g and g + 8
  };
  auto load = [&](int unit, int s0, Batch& b) {
    const int v0 = (unit + group) * 16;
    const bf16* low = weight + static_cast<long long>(min(v0 + g, V - 1)) * D + q * 8;
    const bf16* high = weight + static_cast<long long>(min(v0 + g + 8, V - 1)) * D + q * 8;
#pragma unroll
    for (int u = 0; u < FEW_BATCH; ++u) {
      const int k = (first + s0 + u) * 32;
      const bool any = unit < units && s0 + u < mine && k + q * 8 < D;
      b.low[u] = any ? load_stream(low + k) : make_uint4(0, 0, 0, 0);
      b.high[u] = any ? load_stream(high + k) : make_uint4(0, 0, 0, 0);
    }
  };
  auto multiply = [&](int s0, const Batch& b, float (&c)[NT][4]) {
#pragma unroll
    for (int u = 0; u < FEW_BATCH; ++u) {
      if (s0 + u >= mine || first + s0 + u >= steps) break;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint4 x;
        ld_shared_v4(row_base + n * 8 * ld + (first + s0 + u) * 64, x);
        mma_16x8x16(c[n], b.low[u].x, b.high[u].x, b.low[u].y, b.high[u].y, x.x, x.y);
        mma_16x8x16(c[n], b.low[u].z, b.high[u].z, b.low[u].w, b.high[u].w, x.z, x.w);
      }
    }
  };
  Batch early, later;
  load(blockIdx.x * groups, 0, early);
  int parity = 0;
  // every warp of a block goes round as often as its first group
  for (int unit0 = blockIdx.x * groups; unit0 < units; unit0 += stride, parity ^= 1) {
    const int v0 = (unit0 + group) * 16;
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
    for (int s0 = 0; s0 < mine; s0 += 2 * FEW_BATCH) {
      load(unit0, s0 + FEW_BATCH, later);
      multiply(s0, early, c);
      // the next steps of these entries, or the first ones of the warp's next
      const bool more = s0 + 2 * FEW_BATCH < mine;
      load(more ? unit0 : unit0 + stride, more ? s0 + 2 * FEW_BATCH : 0, early);
      multiply(s0 + FEW_BATCH, later, c);
    }
    if (split > 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) partial[parity][warp][n * 4 + j][lane] = c[n][j];
      }
      __syncthreads();  // one a round: the other buffer was read before the round's own
      if (member != 0) continue;
      for (int w = 1; w < split; ++w) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) c[n][j] += partial[parity][warp + w][n * 4 + j][lane];
        }
      }
    }
    // entries v0 + g (values 0, 1) and v0 + g + 8 (2, 3) of rows 8 n + 2 q (0, 2) and 8 n + 2 q + 1 (1, 3)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int v = v0 + g + (j >> 1) * 8, r = 8 * n + 2 * q + (j & 1);
        if (v < V) {
          if (c[n][j] != -INFINITY) join(top[n][j & 1], sum[n][j & 1], c[n][j], 1.0f);
          if (goal[r] == v) target_logits[r] = c[n][j];
        }
      }
    }
  }
  if (member != 0) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        const float other_top = __shfl_xor_sync(0xffffffffu, top[n][j], o), other_sum = __shfl_xor_sync(0xffffffffu, sum[n][j], o);
        join(top[n][j], sum[n][j], other_top, other_sum);
      }
      const int r = 8 * n + 2 * q + j;
      if (g == 0 && r < rows) stats[static_cast<long long>(r) * stride + blockIdx.x * groups + group] = make_float2(top[n][j], sum[n][j]);
    }
  }
}

struct Few {
  int tiles, split, blocks, pieces, smem;
};

// How loss_few_kernel runs for these sizes; tiles = 0 where it does not: for more than 16 rows (32: 52 us for 27), or where the
// product's tiles keep three quarters of the SMs busy.
Few few_rows(long long rows, int D, int V) {
  Few f = {};
  const int steps = (D + 31) / 32, sms = num_sms();
  const int tiles = rows <= 8 ? 1 : 2;
  const long long product_tiles = (static_cast<long long>(V) + 255) / 256, rounds = (product_tiles + sms - 1) / sms;
  f.smem = tiles * 8 * (steps * 64 + 64);
  if (rows > 16 || f.smem > FEW_SMEM || 4 * product_tiles > 3 * rounds * sms) return f;
  f.tiles = tiles;
  f.split = 1;
  while (f.split < FEW_WARPS && steps / (2 * f.split) >= 2 * FEW_BATCH) f.split *= 2;
  const int groups = FEW_WARPS / f.split, units = (V + 15) / 16;
  const int want = (units + groups - 1) / groups, most = sms * (f.smem <= FEW_SMEM / 2 ? 2 : 1);
  f.blocks = want < most ? want : most;
  f.pieces = f.blocks * groups;
  return f;
}

template <int NT>
int launch_few(const Few& f, const void* hidden, const void* weight, int rows, int D, int V, const long long* targets, float* target_logits,
               float* stats, cudaStream_t stream) {
  static PerDevice room;
  const int allowed = room.get([&] {
    if (cudaFuncSetAttribute(loss_few_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return FEW_SMEM;
  });
  if (f.smem > allowed) return FFM_ERR_LAUNCH;
  loss_few_kernel<NT><<<f.blocks, FEW_WARPS * 32, f.smem, stream>>>(static_cast<const bf16*>(hidden), static_cast<const bf16*>(weight), rows, D,
                                                                    V, f.split, targets, target_logits, reinterpret_cast<float2*>(stats));
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

int streaming_blocks(long long n) {
  const long long want = (n + 2047) / 2048, cap = static_cast<long long>(num_sms()) * 8;
  return static_cast<int>(want < 1 ? 1 : (want < cap ? want : cap));
}

// Into how many pieces the contraction over the vocabulary is split for dh: with few output tiles most of the CTA pairs would
// stand idle, and a last round of tiles that is not full costs a whole one. In units of the time of a tile's whole contraction
// (V / 64 steps of about 0.29 us), with fp32 results to be written and read again at 6 TB/s. Measured, loss and dh alone, unsplit, as chosen here,
// and the best of 1 to 16: 256 x 1024 rows, 50257 entries 300, 108 and 108 us; 256 x 4096 366, 222, 222; 1024 x 1024 373, 224, 224; 2048 x 1024,
// 32003 entries 366, 308, 302. From about as many output tiles as CTA pairs on no split is more than 3 % off another, which is within noise.
int contraction_splits(long long rows, int D, int V) {
  const long long tiles = ((rows + 255) / 256) * ((D + 255) / 256), pairs = num_sms() / 2;
  const double tile = 0.29 * (V / 64 + 1);
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 16; ++s) {
    if (s > 1 && V / s < 2048) break;
    const double time = ((tiles * s + pairs - 1) / pairs) * tile / s + (s > 1 ? 3.0 + 8.0e-6 * rows * D * s / 6.0 : 0.0);
    if (s == 1 || time < 0.97 * least) {
      least = time;
      best = s;
    }
  }
  return best;
}

struct Layout {
  int64_t e, stats, factor, target_entry, target_logits, share, parts, wide, bytes;
  int64_t ld;
  int pieces, splits;
  Few few;
};

Layout lay_out(const ffm_loss_args& a) {
  Layout l;
  const int64_t n = a.piece_rows < a.N ? a.piece_rows : a.N;
  const bool grads = a.d_hidden != nullptr || a.d_weight != nullptr;
  l.pieces = static_cast<int>((a.V + HALF - 1) / HALF);
  l.few = grads || n < a.N ? Few{} : few_rows(n, static_cast<int>(a.D), static_cast<int>(a.V));
  if (l.few.tiles > 0) l.pieces = l.few.pieces;
  l.ld = (a.V + 63) / 64 * 64;
  l.splits = a.d_hidden != nullptr ? contraction_splits(n, static_cast<int>(a.D), static_cast<int>(a.V)) : 1;
  int64_t end = 0;
  auto next = [&](int64_t bytes) {
    const int64_t here = end;
    end += (bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t rows = n;
  l.share = next(8);
  l.target_logits = next(rows * 4);
  l.stats = next(rows * l.pieces * 8);
  l.target_entry = next(grads ? rows * 4 : 0);
  l.factor = next(grads ? rows * l.pieces * 4 : 0);
  l.e = next(grads ? rows * l.ld * 2 : 0);
  l.parts = next(l.splits > 1 ? l.splits * n * a.D * 4 : 0);
  // a bf16 gradient of the weight over several pieces of rows is summed in fp32
  l.wide = next(a.d_weight != nullptr && !a.d_weight_f32 && n < a.N ? a.V * a.D * 4 : 0);
  l.bytes = end;
  return l;
}

bool loss_arguments(const ffm_loss_args& a) {
  return a.N >= 0 && a.D > 0 && a.V > 0 && a.D < (1ll << 31) && a.V < (1ll << 31) - 256 && a.piece_rows > 0 && a.hidden && a.weight && a.targets &&
         a.nll && a.status && (!a.mean || a.loss) && !(a.mean && a.row_grad);
}

int launch_ok() { return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH; }

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" size_t ffm_linear_cross_entropy_workspace_bytes(const ffm_loss_args* args) {
  if (args == nullptr || args->N < 0 || args->D <= 0 || args->V <= 0 || args->piece_rows <= 0) return 0;
  return static_cast<size_t>(lay_out(*args).bytes);
}

extern "C" int ffm_linear_cross_entropy(const ffm_loss_args* args, ffm_stream_t stream) {
  if (args == nullptr || !loss_arguments(*args)) return FFM_ERR_BAD_ARG;
  const ffm_loss_args& a = *args;
  if (a.D % 8 != 0) return FFM_ERR_UNSUPPORTED;
  if (off_16_bytes(static_cast<const char*>(a.hidden), static_cast<const char*>(a.weight), static_cast<const char*>(a.d_hidden),
                   static_cast<const char*>(a.d_weight), static_cast<const char*>(a.workspace))) {
    return FFM_ERR_UNSUPPORTED;
  }
  const Layout l = lay_out(a);
  if (a.workspace == nullptr || a.workspace_bytes < l.bytes) return FFM_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int D = static_cast<int>(a.D), V = static_cast<int>(a.V);
  const float z = static_cast<float>(a.z);
  char* w = static_cast<char*>(a.workspace);
  auto at = [&](int64_t offset) { return reinterpret_cast<float*>(w + offset); };
  const long long* targets = reinterpret_cast<const long long*>(a.targets);
  float* share = a.mean ? at(l.share) : nullptr;
  const float* factor = a.mean ? share + 1 : nullptr;
  const bool grads = a.d_hidden != nullptr || a.d_weight != nullptr;
  int64_t launched = 0;
  int rc = FFM_OK;
  if (a.mean) {
    loss_count_kernel<<<1, LOSS_THREADS, 0, s>>>(targets, a.N, a.ignore_index, share);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
  }
  const int64_t step = a.piece_rows < a.N ? a.piece_rows : a.N;
  for (int64_t r0 = 0; r0 < a.N; r0 += step) {
    const int64_t n = a.N - r0 < step ? a.N - r0 : step;
    const char* hidden = static_cast<const char*>(a.hidden) + r0 * a.D * 2;
    void* e = grads ? static_cast<void*>(w + l.e) : nullptr;
    if (l.few.tiles > 0) {
      const auto few = l.few.tiles == 1 ? launch_few<1> : launch_few<2>;
      rc = few(l.few, hidden, a.weight, static_cast<int>(n), D, V, targets, at(l.target_logits), at(l.stats), s);
    } else {
      rc = softmax_logits(hidden, a.weight, n, D, V, a.targets + r0, at(l.target_logits), at(l.stats), e, l.ld, a.status, stream);
    }
    if (rc != FFM_OK) return rc;
    // a block a row where that does not fill the device with warps
    const bool wide = n <= 8ll * num_sms();
    (wide ? loss_rows_kernel<256> : loss_rows_kernel<32>)<<<static_cast<unsigned>(wide ? n : (n + 7) / 8), 256, 0, s>>>(
        reinterpret_cast<const float2*>(at(l.stats)), at(l.target_logits), targets + r0, reinterpret_cast<const bf16*>(hidden),
        static_cast<const bf16*>(a.weight), D, n, l.pieces, V, a.ignore_index, z, a.row_grad != nullptr ? a.row_grad + r0 : nullptr,
        a.nll + r0, grads ? at(l.factor) : nullptr, at(l.target_entry), a.status, a.status_host);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    launched += 2;
    if (!grads) continue;
    const int64_t row_groups = (n + GRADIENT_ROWS - 1) / GRADIENT_ROWS;
    loss_gradient_kernel<<<dim3((V + 2047) / 2048, static_cast<unsigned>(row_groups < 65535 ? row_groups : 65535)), 256, 0, s>>>(
        static_cast<uint16_t*>(e), l.ld, V, l.pieces, at(l.factor), targets + r0, at(l.target_entry), a.ignore_index, n);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
    if (a.d_hidden != nullptr) {
      char* dh = static_cast<char*>(a.d_hidden) + r0 * a.D * 2;
      const int splits = l.splits;
      if ((rc = dense_rows(e, l.ld, n, V, a.weight, D, splits, factor, splits > 1 ? static_cast<void*>(at(l.parts)) : dh, a.status, stream)) != FFM_OK) return rc;
      ++launched;
      if (splits > 1) {
        loss_join_kernel<<<streaming_blocks(n * a.D), 256, 0, s>>>(at(l.parts), splits, n * a.D, reinterpret_cast<bf16*>(dh));
        if ((rc = launch_ok()) != FFM_OK) return rc;
        ++launched;
      }
    }
    if (a.d_weight != nullptr) {
      const bool wide = a.d_weight_f32 || step < a.N;
      void* to = a.d_weight_f32 || !wide ? a.d_weight : static_cast<void*>(at(l.wide));
      if ((rc = dense_transposed(e, l.ld, hidden, n, V, D, wide, r0 > 0, factor, to, a.status, stream)) != FFM_OK) return rc;
      ++launched;
    }
  }
  if (a.d_weight != nullptr && !a.d_weight_f32 && step < a.N) {
    loss_join_kernel<<<streaming_blocks(a.V * a.D), 256, 0, s>>>(at(l.wide), 1, a.V * a.D, static_cast<bf16*>(a.d_weight));
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
  }
  if (a.N == 0 && a.d_weight != nullptr &&
      cudaMemsetAsync(a.d_weight, 0, static_cast<size_t>(a.V) * a.D * (a.d_weight_f32 ? 4 : 2), s) != cudaSuccess) {
    cudaGetLastError();
    return FFM_ERR_LAUNCH;
  }
  if (a.loss != nullptr) {
    loss_sum_kernel<<<1, LOSS_THREADS, 0, s>>>(a.nll, a.N, share, a.loss, a.status, a.status_host);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
  }
  if (a.launched != nullptr) *a.launched += launched;
  return FFM_OK;
}

extern "C" int ffm_scale_many(int count, void* const* x, const int64_t* types, const int64_t* elements, const float* factor, ffm_stream_t stream) {
  if (count < 0 || count > FFM_CAST_MAX || !factor || (count > 0 && (!x || !types || !elements))) return FFM_ERR_BAD_ARG;
  ScaleJob job = {};
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (elements[i] < 0 || !is_type(static_cast<int>(types[i]))) return FFM_ERR_BAD_ARG;
    if (elements[i] == 0) continue;
    if (!x[i]) return FFM_ERR_BAD_ARG;
    if (elements[i] % 8 != 0 || off_16_bytes(static_cast<const char*>(x[i]))) return FFM_ERR_UNSUPPORTED;
    chunks += elements[i] / 8;
    job.x[job.count] = x[i];
    job.type[job.count] = static_cast<int>(types[i]);
    job.chunks_end[job.count++] = chunks;
  }
  if (job.count == 0) return FFM_OK;
  loss_scale_kernel<<<streaming_blocks(chunks * 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(job, factor);
  return launch_ok();
}
