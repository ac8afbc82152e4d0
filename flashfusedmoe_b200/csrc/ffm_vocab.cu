// Linear cross entropy: softmax cross entropy of hidden [N, D] against a vocabulary weight [V, D], with its gradients.
//
//   l = h w^T    lse = log sum_v exp(l_v)    nll = lse - l_t + z lse^2
//   dl_v = g (p_v (1 + 2 z lse) - [v = t]),  p_v = exp(l_v - lse)        dh = dl w        dw = dl^T h
//
// The logits never exist: the product's epilogue (EPI_SOFTMAX, ffm_gemm_sm100.cu) leaves the maximum and the sum of exponentials of
// every 128 entries of a row, 8 bytes in place of 512, and the target's logit. For the gradients it also leaves the exponentials
// against those maxima in fp16, for one piece of the rows at a time. They become dl in bf16 in the same place once the row's lse is known: a
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
constexpr int ROW_GROUP = 32;     // rows of a block of loss_rows_kernel
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

// *share = 1 / number of rows that count (infinite without any: the mean is NaN then). A target outside of the vocabulary is reported.
__global__ void __launch_bounds__(LOSS_THREADS)
loss_count_kernel(const long long* __restrict__ targets, long long rows, long long ignore, int V, float* __restrict__ share,
                  int32_t* status) {
  __shared__ double part[32];
  int n = 0;
  bool bad = false;
  for (long long i = threadIdx.x; i < rows; i += LOSS_THREADS) {
    const long long t = targets[i];
    if (t != ignore) {
      ++n;
      bad |= t < 0 || t >= V;
    }
  }
  if (bad) atomicCAS(status, 0, FFM_STATUS_BAD_INDEX);
  const double count = block_sum(n, part);
  if (threadIdx.x == 0) *share = static_cast<float>(1.0 / count);
}

// 32 rows a block, one a lane; the warps share the row's pieces of 128 entries. First pass: the row's largest logit and sum
// (warps join in shared memory). Second pass (with `factor`): exp(maximum of a piece - lse) times the row's gradient, transposed
// to [row][piece] on the way, since the next kernel goes along rows.
__global__ void __launch_bounds__(1024)
loss_rows_kernel(const float2* __restrict__ stats, const float* __restrict__ target_logits, const long long* __restrict__ targets,
                 long long rows, int pieces, int V, long long ignore, float z, const float* __restrict__ share,
                 const float* __restrict__ row_grad, float* __restrict__ nll, float* __restrict__ factor,
                 float* __restrict__ target_entry, const int32_t* status, volatile int32_t* status_host) {
  report(status, status_host);
  __shared__ float top_part[32][33], sum_part[32][33];
  __shared__ float row_lse[ROW_GROUP], row_scale[ROW_GROUP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = static_cast<long long>(blockIdx.x) * ROW_GROUP, row = row0 + lane;
  const bool active = row < rows;
  float top = -INFINITY, sum = 0.0f;
  for (int h = warp; h < pieces; h += 4 * 32) {
    float2 s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool any = active && h + 32 * u < pieces;
      s[u] = any ? stats[(h + 32 * u) * rows + row] : make_float2(-INFINITY, 0.0f);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float m = fmaxf(top, s[u].x);
      // nothing yet (-inf), or nothing but NaN: nothing to scale
      sum = (top == -INFINITY ? sum : sum * expf(top - m)) + (s[u].x == -INFINITY ? s[u].y : s[u].y * expf(s[u].x - m));
      top = m;
    }
  }
  top_part[warp][lane] = top;
  sum_part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < 32; ++w) top = fmaxf(top, top_part[w][lane]);
    sum = 0.0f;
    for (int w = 0; w < 32; ++w) {
      const float m = top_part[w][lane];
      sum += m == -INFINITY ? sum_part[w][lane] : sum_part[w][lane] * expf(m - top);
    }
    const float lse = logf(sum) + top;
    float scale = 0.0f;
    if (active) {
      const long long t = targets[row];
      const bool counts = t != ignore, known = t >= 0 && t < V;
      const float logit = counts && known ? target_logits[row] : NAN;
      nll[row] = counts ? fmaf(z * lse, lse, lse - logit) : 0.0f;
      // a row with a target that is none has no gradient; its loss is NaN
      if (counts && known && factor != nullptr) {
        const float g = (share != nullptr ? *share : 1.0f) * (row_grad != nullptr ? row_grad[row] : 1.0f);
        const float less = logit - lse;
        scale = g * fmaf(2.0f * z, lse, 1.0f);
        target_entry[row] = g * fmaf(expf(less), 2.0f * z * lse, expm1f(less));
      }
    }
    row_lse[lane] = lse;
    row_scale[lane] = scale;
  }
  if (factor == nullptr) return;
  __syncthreads();
  const float lse = row_lse[lane], scale = row_scale[lane];
  for (int h0 = 0; h0 < pieces; h0 += 32) {
    const int h = h0 + warp;
    float f = 0.0f;
    if (active && h < pieces && scale != 0.0f) f = expf(stats[h * rows + row].x - lse) * scale;
    __syncthreads();  // the tile before has been written out
    top_part[warp][lane] = f;
    __syncthreads();
    if (row0 + warp < rows && h0 + lane < pieces) factor[(row0 + warp) * pieces + h0 + lane] = top_part[lane][warp];
  }
}

// e (fp16) to dl (bf16) in place: eight entries a thread, 2048 a block and row.
__global__ void __launch_bounds__(256)
loss_gradient_kernel(uint16_t* __restrict__ e, long long ld, int V, int pieces, const float* __restrict__ factor,
                     const long long* __restrict__ targets, const float* __restrict__ target_entry, long long ignore, long long rows) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= V) return;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    uint16_t* at = e + row * ld + col;
    const float f = factor[row * pieces + col / HALF];
    float v[8];
    load8(reinterpret_cast<const fp16*>(at), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f != 0.0f ? v[j] * f : 0.0f;  // rows that do not count: zero whatever e is
    const long long t = targets[row];
    if (t >= col && t < col + 8 && t < V && t != ignore) {
      const float entry = target_entry[row];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (t == col + j) v[j] = entry;
      }
    }
    store8(reinterpret_cast<bf16*>(at), v);
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

// x *= *factor in place (n a multiple of 8), nothing at all where that is 1
template <typename T>
__global__ void __launch_bounds__(256)
loss_scale_kernel(T* __restrict__ x, long long n, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += static_cast<long long>(gridDim.x) * 2048) {
    float v[8];
    load8(x + i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    store8(x + i, v);
  }
}

int streaming_blocks(long long n) {
  const long long want = (n + 2047) / 2048, cap = static_cast<long long>(num_sms()) * 8;
  return static_cast<int>(want < 1 ? 1 : (want < cap ? want : cap));
}

// Into how many pieces the contraction over the vocabulary is split for dh: with few output tiles most of the CTA pairs would
// stand idle, and a last round of tiles that is not full costs a whole one. In units of the time of a tile's whole contraction
// (V / 64 steps of about 0.29 us), with fp32 results to be written and read again at 6 TB/s.
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
};

Layout lay_out(const ffm_loss_args& a) {
  Layout l;
  const int64_t n = a.piece_rows < a.N ? a.piece_rows : a.N;
  const bool grads = a.d_hidden != nullptr || a.d_weight != nullptr;
  l.pieces = static_cast<int>((a.V + HALF - 1) / HALF);
  l.ld = (a.V + 63) / 64 * 64;
  l.splits = a.d_hidden != nullptr ? contraction_splits(n, static_cast<int>(a.D), static_cast<int>(a.V)) : 1;
  int64_t end = 0;
  auto next = [&](int64_t bytes) {
    const int64_t here = end;
    end += (bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t rows = grads ? n : a.N;
  l.share = next(4);
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
  const bool grads = a.d_hidden != nullptr || a.d_weight != nullptr;
  int64_t launched = 0;
  int rc = FFM_OK;
  if (a.N > 0) {
    // without a mean only the targets are looked over
    loss_count_kernel<<<1, LOSS_THREADS, 0, s>>>(targets, a.N, a.ignore_index, V, at(l.share), a.status);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
  }
  const int64_t step = grads ? (a.piece_rows < a.N ? a.piece_rows : a.N) : a.N;
  for (int64_t r0 = 0; r0 < a.N; r0 += step) {
    const int64_t n = a.N - r0 < step ? a.N - r0 : step;
    const char* hidden = static_cast<const char*>(a.hidden) + r0 * a.D * 2;
    void* e = grads ? static_cast<void*>(w + l.e) : nullptr;
    if ((rc = softmax_logits(hidden, a.weight, n, D, V, a.targets + r0, at(l.target_logits), at(l.stats), e, l.ld, a.status, stream)) !=
        FFM_OK) {
      return rc;
    }
    loss_rows_kernel<<<static_cast<unsigned>((n + ROW_GROUP - 1) / ROW_GROUP), 1024, 0, s>>>(
        reinterpret_cast<const float2*>(at(l.stats)), at(l.target_logits), targets + r0, n, l.pieces, V, a.ignore_index, z, share,
        a.row_grad != nullptr ? a.row_grad + r0 : nullptr, a.nll + r0, grads ? at(l.factor) : nullptr, at(l.target_entry),
        a.status, a.status_host);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    launched += 2;
    if (!grads) continue;
    const unsigned rows_at_once = static_cast<unsigned>(n < 65535 ? n : 65535);
    loss_gradient_kernel<<<dim3((V + 2047) / 2048, rows_at_once), 256, 0, s>>>(
        static_cast<uint16_t*>(e), l.ld, V, l.pieces, at(l.factor), targets + r0, at(l.target_entry), a.ignore_index, n);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
    if (a.d_hidden != nullptr) {
      char* dh = static_cast<char*>(a.d_hidden) + r0 * a.D * 2;
      const int splits = l.splits;
      if ((rc = dense_rows(e, l.ld, n, V, a.weight, D, splits, splits > 1 ? static_cast<void*>(at(l.parts)) : dh, a.status, stream)) != FFM_OK) return rc;
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
      if ((rc = dense_transposed(e, l.ld, hidden, n, V, D, wide, r0 > 0, to, a.status, stream)) != FFM_OK) return rc;
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
    if (a.N == 0 && share != nullptr) {  // the mean of nothing
      loss_count_kernel<<<1, LOSS_THREADS, 0, s>>>(targets, 0, a.ignore_index, V, share, a.status);
      ++launched;
    }
    loss_sum_kernel<<<1, LOSS_THREADS, 0, s>>>(a.nll, a.N, share, a.loss, a.status, a.status_host);
    if ((rc = launch_ok()) != FFM_OK) return rc;
    ++launched;
  }
  if (a.launched != nullptr) *a.launched += launched;
  return FFM_OK;
}

extern "C" int ffm_scale_in_place(void* x, int x_type, int64_t elements, const float* factor, ffm_stream_t stream) {
  if (!is_type(x_type) || elements < 0 || !factor) return FFM_ERR_BAD_ARG;
  if (elements == 0) return FFM_OK;
  if (!x) return FFM_ERR_BAD_ARG;
  if (elements % 8 != 0 || off_16_bytes(static_cast<const char*>(x))) return FFM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = streaming_blocks(elements);
  if (x_type == FFM_TYPE_BF16) {
    loss_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<bf16*>(x), elements, factor);
  } else if (x_type == FFM_TYPE_FP16) {
    loss_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<fp16*>(x), elements, factor);
  } else {
    loss_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<float*>(x), elements, factor);
  }
  return launch_ok();
}
