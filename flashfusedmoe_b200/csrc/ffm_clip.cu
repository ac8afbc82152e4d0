// The norm of many tensors together (of all gradients), the coefficient that brings it down to a bound, and their scaling by it.
//
//   norm = sqrt(sum x^2) or max |x|,   coefficient = min(1, max_norm / (norm + 1e-6)),   x = x * coefficient
//
// HBM-bound: the norm reads every value once (208 M bf16 values 68 us, 6.1 TB/s), clipping reads and writes it again. Squares of eight values are
// added in fp32 and those sums in fp64 (one such addition for eight values costs nothing beside their bytes); where fp32 would not hold them (gradients
// beyond 10^18 or all below 10^-13) the eight are squared in fp64. A block leaves one sum, and the last block to come adds them in the
// order of the blocks.
#include "ffm_device.h"
#include "ffm_internal.h"
#include "ffm_norm_common.cuh"

namespace ffm {

namespace {

constexpr int CLIP_THREADS = 512;
constexpr int CLIP_UNROLL = 4;  // groups of eight values that a thread reads at once
constexpr int CLIP_CHUNK = CLIP_THREADS * CLIP_UNROLL * 8;
constexpr int CLIP_BLOCKS = 4;  // on an SM at most

struct ClipTensor {
  void* x;
  long long n;
  long long chunks_end;  // chunks of this tensor and those before it
  int type;
  int wide;  // on a 16-byte boundary
};

template <int MAX>
struct ClipJob {
  ClipTensor tensor[MAX];
  int count;
};

struct NormEnd {
  int parts;     // of all launches
  int first;     // of this launch's
  int last;      // this is the last launch
  double max_norm;
  const double* other;
  double* part;
  double* total;
  float* norm;
  float* coefficient;
  unsigned int* ticket;
};

// magnitudes as bits compare as numbers do, and NaN is above all
__device__ __forceinline__ unsigned int magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ double squares(const float (&v)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
  // squares that matter lie far from both ends of fp32: what is lost below 2^-126 is nothing beside 2^-86
  if (s > 1.3e-26f && s < 1e37f) return s;
  unsigned int any = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) any |= magnitude(v[j]);
  if (any == 0) return 0.0;  // as in much of an embedding's gradient
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), d);
  return d;
}

__device__ __forceinline__ double join(int kind, double a, double b) {
  if (kind == 0) return a + b;
  return a != a || b != b ? a + b : (a > b ? a : b);
}

// one value of the block's, the same for any order in which blocks run
__device__ __forceinline__ double join_block(int kind, double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(kind, v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < CLIP_THREADS / 32; ++w) v = join(kind, v, shared[w]);
  return v;
}

// What a thread's groups of eight add to the block's value
template <int KIND>
__device__ __forceinline__ void take(const float (&v)[8], double& sum, unsigned int& top) {
  if (KIND == 0) {
    sum += squares(v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[j]));
  }
}

// A whole chunk on 16 bytes: all loads before the first value is used (behind a switch over the types for every eight they followed one another:
// 208 M bf16 values took 124 us, so 67)
template <typename T, int KIND>
__device__ __forceinline__ void take_chunk(const T* x, double& sum, unsigned int& top) {
  constexpr int V = VALUES<T>, STEPS = CLIP_CHUNK / V / CLIP_THREADS;
  uint4 raw[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) raw[u] = __ldcs(reinterpret_cast<const uint4*>(x) + u * CLIP_THREADS + threadIdx.x);
#pragma unroll
  for (int u = 0; u < STEPS; u += 8 / V) {
    float v[8];
    unpack<T>(raw[u], reinterpret_cast<float(&)[V]>(v));
    if constexpr (V == 4) unpack<T>(raw[u + 1], reinterpret_cast<float(&)[V]>(v[4]));
    take<KIND>(v, sum, top);
  }
}

template <int MAX, int KIND>
__global__ void __launch_bounds__(CLIP_THREADS)
grad_norm_kernel(const __grid_constant__ ClipJob<MAX> job, const __grid_constant__ NormEnd end) {
  __shared__ double shared[CLIP_THREADS / 32];
  __shared__ bool last;
  const long long chunks = job.count > 0 ? job.tensor[job.count - 1].chunks_end : 0;
  double sum = 0.0;
  unsigned int top = 0;
  int i = 0;
  for (long long chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    while (chunk >= job.tensor[i].chunks_end) ++i;  // the chunk's tensor, for the whole block alike
    const ClipTensor& a = job.tensor[i];
    const long long c0 = (chunk - (i > 0 ? job.tensor[i - 1].chunks_end : 0)) * CLIP_CHUNK;
    if (a.wide && c0 + CLIP_CHUNK <= a.n) {
      if (a.type == FFM_TYPE_BF16) {
        take_chunk<bf16, KIND>(static_cast<const bf16*>(a.x) + c0, sum, top);
      } else if (a.type == FFM_TYPE_FP16) {
        take_chunk<fp16, KIND>(static_cast<const fp16*>(a.x) + c0, sum, top);
      } else {
        take_chunk<float, KIND>(static_cast<const float*>(a.x) + c0, sum, top);
      }
    } else {
#pragma unroll
      for (int u = 0; u < CLIP_UNROLL; ++u) {
        // neighbours in neighbouring threads; zeros past the tensor's end
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const long long e = c0 + (u * 8 + j) * CLIP_THREADS + threadIdx.x;
          v[j] = e < a.n ? load1_as(a.x, a.type, e) : 0.0f;
        }
        take<KIND>(v, sum, top);
      }
    }
  }
  if (KIND != 0) sum = __uint_as_float(top);
  sum = join_block(KIND, sum, shared);
  if (threadIdx.x == 0) {
    end.part[end.first + blockIdx.x] = sum;
    if (end.last) {
      __threadfence();
      last = atomicAdd(end.ticket, 1u) == gridDim.x - 1;
      if (last) *end.ticket = 0;
      __threadfence();
    }
  }
  if (!end.last) return;
  __syncthreads();
  if (!last) return;
  double v = 0.0;
  for (int k = threadIdx.x; k < end.parts; k += CLIP_THREADS) v = join(KIND, v, __ldcg(end.part + k));
  v = join_block(KIND, v, shared);
  if (threadIdx.x == 0) {
    if (end.other != nullptr) v = join(KIND, v, *end.other);
    if (end.total != nullptr) *end.total = v;
    const double norm = KIND == 0 ? sqrt(v) : v;
    if (end.norm != nullptr) *end.norm = static_cast<float>(norm);
    if (end.coefficient != nullptr) {
      const double c = end.max_norm / (norm + 1e-6);
      *end.coefficient = c >= 1.0 ? 1.0f : static_cast<float>(c);
    }
  }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(T* x, float f) {
  constexpr int V = VALUES<T>, STEPS = CLIP_CHUNK / V / CLIP_THREADS;
  uint4* at = reinterpret_cast<uint4*>(x) + threadIdx.x;
  uint4 raw[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) raw[u] = at[u * CLIP_THREADS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    float2 v[V / 2];
    unpack2<T>(raw[u], v);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = mul2(v[j], both(f));
    store2<T>(reinterpret_cast<T*>(at + u * CLIP_THREADS), v);
  }
}

// The last chunks first: of what the norm has read they are still in L2.
template <int MAX>
__global__ void __launch_bounds__(CLIP_THREADS)
scale_tensors_kernel(const __grid_constant__ ClipJob<MAX> job, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  const long long chunks = job.tensor[job.count - 1].chunks_end;
  int i = job.count - 1;
  for (long long chunk = chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    while (i > 0 && chunk < job.tensor[i - 1].chunks_end) --i;
    const ClipTensor& a = job.tensor[i];
    const long long c0 = (chunk - (i > 0 ? job.tensor[i - 1].chunks_end : 0)) * CLIP_CHUNK;
    if (a.wide && c0 + CLIP_CHUNK <= a.n) {
      if (a.type == FFM_TYPE_BF16) {
        scale_chunk(static_cast<bf16*>(a.x) + c0, f);
      } else if (a.type == FFM_TYPE_FP16) {
        scale_chunk(static_cast<fp16*>(a.x) + c0, f);
      } else {
        scale_chunk(static_cast<float*>(a.x) + c0, f);
      }
    } else {
      // neighbours in neighbouring threads
      for (long long e = c0 + threadIdx.x; e < a.n && e < c0 + CLIP_CHUNK; e += CLIP_THREADS) {
        store1_as(a.x, a.type, e, load1_as(a.x, a.type, e) * f);
      }
    }
  }
}

constexpr int CLIP_FEW = 32;  // up to so many, a smaller argument block is launched

int clip_blocks() { return CLIP_BLOCKS * num_sms(); }

// blocks that `count` tensors are worked on by, in one launch; the job is filled in
template <int MAX>
int fill_job(ClipJob<MAX>& job, const ffm_clip_tensor* t, int count) {
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    ClipTensor& a = job.tensor[i];
    a.x = t[i].x;
    a.n = t[i].elements;
    a.type = static_cast<int>(t[i].type);
    a.wide = !off_16_bytes(a.x);
    chunks += (a.n + CLIP_CHUNK - 1) / CLIP_CHUNK;
    a.chunks_end = chunks;
  }
  job.count = count;
  return static_cast<int>(chunks < clip_blocks() ? (chunks > 0 ? chunks : 1) : clip_blocks());
}

template <int MAX, int KIND>
int launch_norm(const ffm_clip_tensor* t, int count, NormEnd& end, cudaStream_t stream) {
  ClipJob<MAX> job;
  const int blocks = fill_job(job, t, count);
  end.parts = end.first + blocks;
  grad_norm_kernel<MAX, KIND><<<blocks, CLIP_THREADS, 0, stream>>>(job, end);
  end.first += blocks;
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

template <int MAX>
int launch_scale(const ffm_clip_tensor* t, int count, const float* factor, cudaStream_t stream) {
  ClipJob<MAX> job;
  const int blocks = fill_job(job, t, count);
  scale_tensors_kernel<MAX><<<blocks, CLIP_THREADS, 0, stream>>>(job, factor);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

bool clip_arguments(const ffm_clip_tensor* tensors, int count) {
  if (count < 0 || (count > 0 && tensors == nullptr)) return false;
  for (int i = 0; i < count; ++i) {
    const ffm_clip_tensor& t = tensors[i];
    if (t.elements < 0 || !is_type(static_cast<int>(t.type)) || (t.elements > 0 && t.x == nullptr)) return false;
  }
  return true;
}

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" size_t ffm_grad_norm_workspace_bytes(int count) {
  if (count < 0) return 0;
  const size_t launches = count > 0 ? (static_cast<size_t>(count) + FFM_CLIP_MAX - 1) / FFM_CLIP_MAX : 1;
  return launches * clip_blocks() * sizeof(double);
}

extern "C" int ffm_grad_norm(const ffm_clip_tensor* tensors, int count, const ffm_grad_norm_args* args, ffm_stream_t stream) {
  if (!clip_arguments(tensors, count) || args == nullptr || !args->ticket || (args->kind != 0 && args->kind != 1)) return FFM_ERR_BAD_ARG;
  if (!(args->max_norm >= 0.0)) return FFM_ERR_BAD_ARG;
  if (!args->workspace || static_cast<size_t>(args->workspace_bytes) < ffm_grad_norm_workspace_bytes(count)) return FFM_ERR_WORKSPACE;
  NormEnd end = {};
  end.max_norm = args->max_norm;
  end.other = args->other;
  end.part = static_cast<double*>(args->workspace);
  end.total = args->total;
  end.norm = args->norm;
  end.coefficient = args->coefficient;
  end.ticket = static_cast<unsigned int*>(args->ticket);
  for (int from = 0; from == 0 || from < count; from += FFM_CLIP_MAX) {
    const int n = count - from < FFM_CLIP_MAX ? count - from : FFM_CLIP_MAX;
    end.last = from + n == count;
    auto launch = [&](auto most) {
      return args->kind == 0 ? launch_norm<decltype(most)::value, 0>(tensors + from, n, end, static_cast<cudaStream_t>(stream))
                             : launch_norm<decltype(most)::value, 1>(tensors + from, n, end, static_cast<cudaStream_t>(stream));
    };
    const int rc = n <= CLIP_FEW ? launch(std::integral_constant<int, CLIP_FEW>{}) : launch(std::integral_constant<int, FFM_CLIP_MAX>{});
    if (rc != FFM_OK) return rc;
    if (args->launched != nullptr) ++*args->launched;
  }
  return FFM_OK;
}

extern "C" int ffm_scale_tensors(const ffm_clip_tensor* tensors, int count, const float* factor, int64_t* launched, ffm_stream_t stream) {
  if (!clip_arguments(tensors, count) || (count > 0 && factor == nullptr)) return FFM_ERR_BAD_ARG;
  for (int from = 0; from < count; from += FFM_CLIP_MAX) {
    const int n = count - from < FFM_CLIP_MAX ? count - from : FFM_CLIP_MAX;
    const int rc = n <= CLIP_FEW ? launch_scale<CLIP_FEW>(tensors + from, n, factor, static_cast<cudaStream_t>(stream))
                                 : launch_scale<FFM_CLIP_MAX>(tensors + from, n, factor, static_cast<cudaStream_t>(stream));
    if (rc != FFM_OK) return rc;
    if (launched != nullptr) ++*launched;
  }
  return FFM_OK;
}
