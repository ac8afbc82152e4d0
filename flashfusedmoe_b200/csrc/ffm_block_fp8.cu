// 8-bit operands (e4m3) with a scale for every 128 values: quantising rows and weights, and products of them, dense or grouped by expert.
//
//   x [rows, K] with x_scale [rows, ceil(K / 128)], w [experts, N, K] with w_scale [experts, ceil(N / 128), ceil(K / 128)]:
//   out[m, n] = sum over blocks b of 128 k's of x_scale[m, b] w_scale[e, n / 128, b] sum over the k's of block b of x[m, k] w[e, n, k]
//   for the expert e with ends[e - 1] <= m < ends[e]; 0 for rows from the last end on.
//
// The sum over a block is what the tensor core accumulates in TMEM (exactly enough: 128 products of 8 bits in fp32). The scales change from block
// to block, so eight warps take each block's sums out of TMEM while the tensor core is at the next one (two accumulators in turn) and add them,
// scaled, to fp32 sums in registers.
#include "ffm_e4m3.cuh"
#include "ffm_gemm_common.cuh"
#include "ffm_internal.h"
#include "ffm_norm_common.cuh"

namespace ffm {

namespace {

// ---- quantising -------------------------------------------------------------------------------------------------

constexpr int QB_THREADS = 256;
constexpr int QB_CHUNKS = 2;  // of 16 bytes, of a block of a row, that a thread holds

// The largest magnitude of 16 bytes; 16-bit values are compared in pairs as they are. NaN does not count.
template <typename T>
__device__ __forceinline__ float largest(const uint4& raw) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(raw.x)), fabsf(__uint_as_float(raw.y))), fmaxf(fabsf(__uint_as_float(raw.z)), fabsf(__uint_as_float(raw.w))));
  } else {
    using T2 = std::conditional_t<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>;
    const uint32_t zero = 0, word[4] = {raw.x, raw.y, raw.z, raw.w};
    T2 top = *reinterpret_cast<const T2*>(&zero);
#pragma unroll
    for (int q = 0; q < 4; ++q) top = __hmax2(top, __habs2(*reinterpret_cast<const T2*>(&word[q])));
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&top);
    return fmaxf(to_float(bits_as<T>(bits & 0xffffu)), to_float(bits_as<T>(bits >> 16)));
  }
}

// A scale for 128 values of a row: eight (fp32: 16) neighbouring lanes hold a block, two chunks of 16 bytes each, which share what the scale costs.
// HBM-bound: 32768 x 7168 bf16 125 us (5.7 TB/s), with 16 lanes a block and a chunk each 150; 61 x 7168 1.5 us in a graph.
template <typename T>
__global__ void __launch_bounds__(QB_THREADS)
quantize_row_blocks_kernel(const T* __restrict__ x, long long stride, long long blocks, int across, int K, uint8_t* __restrict__ q,
                           float* __restrict__ scale) {
  constexpr int V = VALUES<T>, LANES = E4M3_BLOCK / V / QB_CHUNKS, TEAMS = QB_THREADS / LANES;
  const int t = threadIdx.x % LANES;
  const long long at = static_cast<long long>(blockIdx.x) * TEAMS + threadIdx.x / LANES;
  const long long row = (at >> 32) == 0 ? static_cast<uint32_t>(at) / static_cast<uint32_t>(across) : at / across;
  const int first = static_cast<int>(at - row * across) * E4M3_BLOCK + t * V;
  bool has[QB_CHUNKS];  // in the row, and the row there
  uint4 raw[QB_CHUNKS];
#pragma unroll
  for (int c = 0; c < QB_CHUNKS; ++c) {
    const int col = first + c * LANES * V;
    has[c] = at < blocks && col < K;
    raw[c] = has[c] ? *reinterpret_cast<const uint4*>(x + row * stride + col) : make_uint4(0, 0, 0, 0);
  }
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < QB_CHUNKS; ++c) top = fmaxf(top, largest<T>(raw[c]));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float2 v[1][QB_CHUNKS * V / 2];
#pragma unroll
  for (int c = 0; c < QB_CHUNKS; ++c) unpack2<T>(raw[c], reinterpret_cast<float2(&)[V / 2]>(v[0][c * V / 2]));
  quantize_chunks(v, {top}, [&](int, const uint32_t(&word)[QB_CHUNKS * V / 4], float s) {
#pragma unroll
    for (int c = 0; c < QB_CHUNKS; ++c) {
      if (has[c]) store_words(q + row * K + first + c * LANES * V, reinterpret_cast<const uint32_t(&)[V / 4]>(word[c * V / 4]));
    }
    if (t == 0 && has[0]) scale[at] = s;
  });
}

// A scale for 128 x 128 values of a matrix: one thread block for each, its values in registers in between. Three blocks of 16-bit values on an SM:
// 8 x 14336 x 4096 bf16 214 us (6.6 TB/s), fp16 214 (243 with the largest of converted values), 4 x 14336 x 4096 fp32 184 (6.4 TB/s). With products in
// place of quotients two blocks took 261 us, four 226.
template <typename T>
__global__ void __launch_bounds__(QB_THREADS, sizeof(T) == 2 ? 3 : 2)
quantize_tiles_kernel(const T* __restrict__ x, int N, int K, int down, int across, uint8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int V = VALUES<T>, LANES = E4M3_BLOCK / V, TEAMS = QB_THREADS / LANES, STEPS = E4M3_BLOCK / TEAMS;
  __shared__ float part[QB_THREADS / 32];
  const long long tile = blockIdx.x;
  const int bn = static_cast<int>(tile / across % down), bk = static_cast<int>(tile % across);
  const int col = bk * E4M3_BLOCK + threadIdx.x % LANES * V, n0 = bn * E4M3_BLOCK + threadIdx.x / LANES;
  const int left = col < K ? N - n0 : 0;  // rows from this thread's first on
  const long long first = tile / (static_cast<long long>(down) * across) * N * K + static_cast<long long>(n0) * K + col, step = static_cast<long long>(TEAMS) * K;
  uint4 raw[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) raw[i] = i * TEAMS < left ? *reinterpret_cast<const uint4*>(x + first + i * step) : make_uint4(0, 0, 0, 0);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) top = fmaxf(top, largest<T>(raw[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < QB_THREADS / 32; ++w) top = fmaxf(top, part[w]);
  auto store = [&](int i, const uint4& u, auto&& pack) {
    float2 v[V / 2];
    unpack2<T>(u, v);
    uint32_t word[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) word[j] = pack(v[2 * j], v[2 * j + 1]);
    store_words(q + first + i * step, word);
  };
  if (e4m3_by_division(top)) {
    const float s = e4m3_scale_divided(top);
    if (threadIdx.x == 0) scale[tile] = s;
#pragma unroll 1
    for (int i = 0; i < STEPS && i * TEAMS < left; ++i) {  // rare: read again, so that it takes no registers from the other way
      store(i, *reinterpret_cast<const uint4*>(x + first + i * step), [&](float2 a, float2 b) { return pack_divided(a, b, s); });
    }
  } else {
    const float s = e4m3_scale(top), y = -reciprocal(s);
    if (threadIdx.x == 0) scale[tile] = s;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i * TEAMS < left) store(i, raw[i], [&](float2 a, float2 b) { return pack_quotients(a, b, s, y); });
    }
  }
}

// ---- products ---------------------------------------------------------------------------------------------------

constexpr int BLOCK_THREADS = 384;
constexpr int MAX_EXPERTS = 1024;
constexpr int A_ROWS = 128;
constexpr int UMMA_K8 = 32;  // e4m3 values of the contraction in an instruction

struct BlockParams {
  const float* x_scale;
  const float* w_scale;
  const int32_t* ends;  // null: one expert takes all rows
  int experts;
  int rows;
  int N;
  int k_blocks;
  int out_type;
  int out_wide;  // rows of out lie on 16 bytes
  int box_rows;  // few rows: of x in a load
  void* out;
  int32_t* status;
  volatile int32_t* status_host;
  long long wait_cycles;
};

// Row ranges of the experts, and behind them as one more group the rows that belong to none; tiles before each. Read by the whole block.
struct Groups {
  int begin[MAX_EXPERTS + 2];
  int items[MAX_EXPERTS + 2];
};

// Filled by one warp. An end below the one before it or past the rows would have tiles read and written out of place: such ends are
// moved into place, and reported.
__device__ __forceinline__ void fill_groups(Groups& g, const BlockParams& p, int tile_rows, int tiles_across) {
  const int lane = threadIdx.x & 31;
  int last = 0, run = 0;
  bool bad = false;
  for (int base = 0; base < p.experts; base += 32) {
    const int e = base + lane;
    int end = p.rows;
    if (p.ends != nullptr && e < p.experts) {
      end = __ldg(p.ends + e);
      bad |= end < 0 || end > p.rows;
      end = min(max(end, 0), p.rows);
    }
    int reach = e < p.experts ? max(end, last) : last;  // the largest end so far
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, reach, d);
      if (lane >= d) reach = max(reach, before);
    }
    int begin = __shfl_up_sync(0xffffffffu, reach, 1);
    if (lane == 0) begin = last;
    bad |= e < p.experts && end < begin;
    const int mine = e < p.experts ? (reach - begin + tile_rows - 1) / tile_rows * tiles_across : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += before;
    }
    if (e < p.experts) {
      g.begin[e] = begin;
      g.items[e] = run + sum - mine;
    }
    last = __shfl_sync(0xffffffffu, reach, 31);
    run += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) {
    g.begin[p.experts] = last;
    g.items[p.experts] = run;
    g.begin[p.experts + 1] = p.rows;
    g.items[p.experts + 1] = run + (p.rows - last + tile_rows - 1) / tile_rows * tiles_across;
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) {
    atomicCAS(p.status, 0, FFM_STATUS_BAD_INDEX);
    if (p.status_host != nullptr) *p.status_host = FFM_STATUS_BAD_INDEX;
  }
}

struct BlockTile {
  int group;     // p.experts: rows of no expert
  int across;    // tile of output features
  int row0;      // first row
  int rows;      // valid rows, 1..tile_rows
  int k_blocks;  // 0 for rows of no expert
};

// Tiles by expert and feature tile, row tile fastest: the row tiles of an expert share its weights through L2.
struct BlockWalker {
  const Groups* groups;
  int experts, tile_rows, k_blocks, cur, step, g;

  __device__ BlockWalker(const Groups* groups_, const BlockParams& p, int tile_rows_, int first, int step_)
      : groups(groups_), experts(p.experts), tile_rows(tile_rows_), k_blocks(p.k_blocks), cur(first), step(step_), g(0) {}
  __device__ bool next(BlockTile& t) {
    if (cur >= groups->items[experts + 1]) return false;
    while (cur >= groups->items[g + 1]) ++g;
    const int begin = groups->begin[g], count = groups->begin[g + 1] - begin, down = (count + tile_rows - 1) / tile_rows;
    const int r = cur - groups->items[g], first = r % down * tile_rows;
    t.group = g;
    t.across = r / down;
    t.row0 = begin + first;
    t.rows = min(tile_rows, count - first);
    t.k_blocks = g < experts ? k_blocks : 0;
    cur += step;
    return true;
  }
};

__device__ __forceinline__ uint32_t pack_out(int type, float a, float b) {
  if (type == FFM_TYPE_BF16) return pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- many rows: 128 rows x BN features, rows on the M side -------------------------------------------------------

template <int BN>
struct ManyRows {
  static constexpr int COLS = BN / 2;  // features of a warp: the eight warps are two halves of a tile by four lane quarters
  static constexpr int STAGE_BYTES = (A_ROWS + BN) * 128;
  static constexpr int STAGES = 147456 / STAGE_BYTES;
  static constexpr int STORE_WARP = 2 * 32 * 128;  // two boxes of 32 rows x 128 bytes (128-byte swizzle) on their way out
  static constexpr int STORE_BYTES = 8 * STORE_WARP;
  static constexpr int SLOTS = 8;  // blocks whose scales are there or on their way
  struct Ctrl {
    unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full_bar[2], acc_empty_bar[2], scale_full_bar[SLOTS], scale_empty_bar[SLOTS], drain_bar;
    uint32_t tmem_base;
    int abort_flag;
    int filled;
    alignas(16) float scale[SLOTS][A_ROWS + 4];  // of the rows, and of the two halves' features
    Groups groups;
  };
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + STORE_BYTES + static_cast<int>(sizeof(Ctrl)) + 1024;
  static_assert(SMEM_BYTES <= 232448, "tile shape does not fit in shared memory");
};

__device__ __forceinline__ void copy_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// arrives once this thread's copies so far have landed; the barrier's count has an arrival for it
__device__ __forceinline__ void copy_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void st_shared_v2(uint32_t addr, float2 v) {
  asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// A value in front of the first whole word of a row of 16-bit values
__device__ __forceinline__ int head_of(const uint8_t* row) { return (reinterpret_cast<uintptr_t>(row) >> 1) & 1; }

// The launch's 168 registers a thread go from the four warps of the first group to the eight that hold sums: 128 x 72 + 256 x 216 = 384 x 168.
constexpr int ISSUE_REGISTERS = 72, SUM_REGISTERS = 216;
static_assert(128 * ISSUE_REGISTERS + 256 * SUM_REGISTERS <= BLOCK_THREADS * 168, "more registers than the launch has");

// 991 cycles a block of the contraction, where the MMAs take 512: the way of the sums through two loads from TMEM and 128 FMAs a lane bounds it, and back to
// back the board's power. 8192 x 4096 x 4096 133 us (2.06 PFLOP/s), 32768 x 4096 x 4096 on eight experts 560 us, back to back 630 (1.75). A pair of CTAs with a
// tile of 256 x 256 is no faster, twice as many warps for the sums slower (167 us).
//
//   warp 0      TMA producer          warp 1   MMA issuer, TMEM owner          warp 2   row ranges, scales          warp 3   nothing
//   warps 4..11 take a block's sums out of TMEM, scale and add them, store the tile
template <int BN, int OUT_BYTES>
__global__ void __launch_bounds__(BLOCK_THREADS, 1)
block_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_out,
                  const __grid_constant__ BlockParams p) {
  using S = ManyRows<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw), pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t smem_base = raw_addr + pad, staging = smem_base + S::STAGES * S::STAGE_BYTES;
  auto* ctrl = reinterpret_cast<typename S::Ctrl*>(smem_raw + pad + S::STAGES * S::STAGE_BYTES + S::STORE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(smem_u32(&ctrl->full_bar[s]), 1);
      mbar_init(smem_u32(&ctrl->empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&ctrl->acc_full_bar[a]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty_bar[a]), 8);
    }
    for (int i = 0; i < S::SLOTS; ++i) {
      mbar_init(smem_u32(&ctrl->scale_full_bar[i]), 32);
      mbar_init(smem_u32(&ctrl->scale_empty_bar[i]), 8);
    }
    mbar_init(smem_u32(&ctrl->drain_bar), 1);
    ctrl->abort_flag = 0;
    ctrl->filled = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 2) fill_groups(ctrl->groups, p, A_ROWS, (p.N + BN - 1) / BN);
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const uint32_t tmem_base = ctrl->tmem_base;
  volatile int* abort_flag = &ctrl->abort_flag;
  bool issuer = false;
  BlockWalker walker(&ctrl->groups, p, A_ROWS, blockIdx.x, gridDim.x);
  BlockTile t;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ISSUE_REGISTERS));
    if (warp == 0 && elect_one()) {
      int stage = 0, filled = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && walker.next(t)) {
        for (int kb = 0; kb < t.k_blocks; ++kb) {
          ok = mbar_wait_bounded(smem_u32(&ctrl->empty_bar[stage]), phase ^ 1u, abort_flag, p.status, FFM_STATUS_WAIT_PRODUCER, p.wait_cycles);
          if (!ok) break;
          const uint32_t full = smem_u32(&ctrl->full_bar[stage]), a_dst = smem_base + stage * S::STAGE_BYTES;
          mbar_expect_tx(full, S::STAGE_BYTES);
          tma_load_2d(a_dst, &tm_x, full, kb * E4M3_BLOCK, t.row0);
          tma_load_3d(a_dst + A_ROWS * 128, &tm_w, full, kb * E4M3_BLOCK, t.across * BN, t.group);
          ++filled;
          if (++stage == S::STAGES) stage = 0, phase ^= 1u;
        }
      }
      ctrl->filled = filled;
    }
    if (warp == 1 && elect_one()) {
      issuer = true;
      constexpr uint32_t idesc = make_idesc_e4m3(A_ROWS, BN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      while (ok && walker.next(t)) {
        for (int kb = 0; kb < t.k_blocks; ++kb) {
          ok = mbar_wait_bounded(smem_u32(&ctrl->acc_empty_bar[acc]), acc_phase ^ 1u, abort_flag, p.status, FFM_STATUS_WAIT_MMA, p.wait_cycles) &&
               mbar_wait_bounded(smem_u32(&ctrl->full_bar[stage]), phase, abort_flag, p.status, FFM_STATUS_WAIT_MMA, p.wait_cycles);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_src = smem_base + stage * S::STAGE_BYTES, b_src = a_src + A_ROWS * 128;
#pragma unroll
          for (int kk = 0; kk < E4M3_BLOCK / UMMA_K8; ++kk) {
            umma_f8(tmem_base + acc * BN, make_smem_desc_sw128(a_src + kk * UMMA_K8, 16, 1024), make_smem_desc_sw128(b_src + kk * UMMA_K8, 16, 1024),
                    idesc, kk > 0 ? 1u : 0u);
          }
          umma_commit(smem_u32(&ctrl->empty_bar[stage]));
          umma_commit(smem_u32(&ctrl->acc_full_bar[acc]));
          if (++stage == S::STAGES) stage = 0, phase ^= 1u;
          if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
      }
    }
    if (warp == 2) {
      // the scales of the tile's rows and features, block by block, ahead of the sums that they belong to
      const int scale_rows = (p.N + E4M3_BLOCK - 1) / E4M3_BLOCK;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && walker.next(t)) {
        // rows past the tile's last: any
        const float* xs = p.x_scale + static_cast<long long>(t.row0) * p.k_blocks;
        const int f = min(t.across * (BN / E4M3_BLOCK) + (BN > E4M3_BLOCK ? lane & 1 : 0), scale_rows - 1);
        const float* ws = p.w_scale + (static_cast<long long>(t.group) * scale_rows + f) * p.k_blocks;
        for (int kb = 0; kb < t.k_blocks; ++kb) {
          ok = mbar_wait_bounded(smem_u32(&ctrl->scale_empty_bar[slot]), phase ^ 1u, abort_flag, p.status, FFM_STATUS_WAIT_PRODUCER, p.wait_cycles);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t to = smem_u32(ctrl->scale[slot]);
#pragma unroll
          for (int r = 0; r < A_ROWS; r += 32) copy_async_4(to + (r + lane) * 4, xs + static_cast<long long>(min(r + lane, t.rows - 1)) * p.k_blocks + kb);
          if (lane < 2) copy_async_4(to + (A_ROWS + lane) * 4, ws + kb);
          copy_async_arrive(smem_u32(&ctrl->scale_full_bar[slot]));
          if (++slot == S::SLOTS) slot = 0, phase ^= 1u;
        }
      }
      copy_async_wait<0>();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SUM_REGISTERS));
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * S::COLS;
    const uint32_t mine = staging + (warp - 4) * S::STORE_WARP;  // this warp's rows on their way out
    uint32_t blocks = 0;  // so far
    bool ok = true;
    while (ok && walker.next(t)) {
      float2 sum[S::COLS / 2];
#pragma unroll
      for (int j = 0; j < S::COLS / 2; ++j) sum[j] = both(0.0f);
      uint32_t v[2][32];
      for (int kb = 0; kb < t.k_blocks; ++kb, ++blocks) {
        const uint32_t acc = blocks & 1, slot = blocks % S::SLOTS;
        ok = mbar_wait_bounded(smem_u32(&ctrl->acc_full_bar[acc]), (blocks >> 1) & 1, abort_flag, p.status, FFM_STATUS_WAIT_EPILOGUE, p.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        // 64 columns at a time: with 32 and the next 32 on their way the two warps of a scheduler waited together (8192 x 4096 x 4096 without
        // the stores: 137 us, so 122)
        tmem_ld_32x32(taddr + acc * BN, v[0]);
        tmem_ld_32x32(taddr + acc * BN + 32, v[1]);
        ok = mbar_wait_bounded(smem_u32(&ctrl->scale_full_bar[slot]), (blocks / S::SLOTS) & 1, abort_flag, p.status, FFM_STATUS_WAIT_EPILOGUE, p.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        const float2 s = both(ctrl->scale[slot][quarter * 32 + lane] * ctrl->scale[slot][A_ROWS + half]);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctrl->scale_empty_bar[slot]));
#pragma unroll
        for (int c = 0; c < S::COLS / 64; ++c) {
          tmem_ld_wait();
          if (c + 1 == S::COLS / 64) {
            tc_fence_before();
            if (lane == 0) mbar_arrive(smem_u32(&ctrl->acc_empty_bar[acc]));
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            sum[c * 32 + j] = fma2(make_float2(__uint_as_float(v[j >> 4][2 * (j & 15)]), __uint_as_float(v[j >> 4][2 * (j & 15) + 1])), s, sum[c * 32 + j]);
          }
          if (c + 1 < S::COLS / 64) {
            tmem_ld_32x32(taddr + acc * BN + (c + 1) * 64, v[0]);
            tmem_ld_32x32(taddr + acc * BN + (c + 1) * 64 + 32, v[1]);
          }
        }
        if (!ok) break;
      }
      if (!ok) break;
      // 128 bytes of every row at a time through one of two boxes in shared memory. 32 whole rows on 16 bytes go out by themselves, while the next
      // tile's sums begin; others are stored from here.
      constexpr int STEP = 128 / OUT_BYTES;
      const int limit = min(t.rows - quarter * 32, 32);  // of this warp's rows
      const long long pitch = static_cast<long long>(p.N) * OUT_BYTES;
#pragma unroll
      for (int c = 0; c < S::COLS / STEP; ++c) {
        const int first = t.across * BN + half * S::COLS + c * STEP, count = min(STEP, p.N - first);
        const uint32_t box = mine + (c & 1) * 4096;
        if (lane == 0) bulk_wait_read<S::COLS / STEP % 2 == 0 ? 1 : 0>();  // what was sent from this box has been read
        __syncwarp();
        uint8_t* out = static_cast<uint8_t*>(p.out) + (t.row0 + quarter * 32) * pitch + static_cast<long long>(first) * OUT_BYTES;
        // 16-bit rows off 16 bytes are staged as the words that memory has them in, without the value in front of the first
        const bool shift = OUT_BYTES == 2 && !p.out_wide && head_of(out + lane * pitch);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t at = box + box_offset(lane, q);
          if constexpr (OUT_BYTES == 2) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = c * (STEP / 2) + q * 4 + i;
              const float after = q * 4 + i + 1 < STEP / 2 ? sum[j + 1 < S::COLS / 2 ? j + 1 : j].x : 0.0f;
              u[i] = pack_out(p.out_type, shift ? sum[j].y : sum[j].x, shift ? after : sum[j].y);
            }
            st_shared_v4(at, u[0], u[1], u[2], u[3]);
          } else {
            const float2* f = sum + c * (STEP / 2) + q * 2;
            // by pairs, as the sums lie: stored by fours they would be moved in every block of the contraction (8192 x 4096 x 4096: 162 us, so 143)
            st_shared_v2(at, f[0]);
            st_shared_v2(at + 8, f[1]);
          }
        }
        if (count > 0 && limit == 32 && p.out_wide) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) tma_store_3d(&tm_out, box, first, t.row0 + quarter * 32, 0);
        } else if (count > 0 && limit > 0 && p.out_wide) {
          __syncwarp();
          for (int i = lane; i < limit * 8; i += 32) {  // 16 bytes each
            const int r = i >> 3, q = i & 7;
            uint4 u;
            ld_shared_v4(box + box_offset(r, q), u);
            if (q * (16 / OUT_BYTES) < count) *reinterpret_cast<uint4*>(out + r * pitch + q * 16) = u;
          }
        } else if (count > 0 && limit > 0) {
          if constexpr (OUT_BYTES == 2) {
            // what is not in a whole word: the first value, and the last
            uint16_t* row = reinterpret_cast<uint16_t*>(out + lane * pitch);
            const int left = count - (shift ? 1 : 0);
            if (lane < limit && shift) row[0] = static_cast<uint16_t>(pack_out(p.out_type, sum[c * (STEP / 2)].x, 0.0f));
            if (lane < limit && (left & 1)) {
              row[count - 1] = static_cast<uint16_t>(ld_shared_u32(box + box_offset(lane, left >> 3) + (left >> 1 & 3) * 4));
            }
          }
          __syncwarp();
          // a row's words, one a lane
          for (int r0 = 0; r0 < limit; r0 += 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = r0 + i;
              uint8_t* row = out + r * pitch;
              const int head = OUT_BYTES == 2 ? head_of(row) : 0, words = r < limit ? (OUT_BYTES == 2 ? (count - head) >> 1 : count) : 0;
              const uint32_t from = box + r * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4;
              if (lane < words) reinterpret_cast<uint32_t*>(row + head * 2)[lane] = ld_shared_u32(from);
            }
          }
        }
        if (lane == 0) bulk_commit();  // empty where nothing was sent
      }
    }
    bulk_wait0();  // its stores have landed before the CTA's shared memory goes away
  }

  // ---- common exit: every role reaches this point, also after an abort
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // loads and MMAs that nobody waited for must not land in shared memory or TMEM that the CTA has given back
    if (threadIdx.x == 0) {
      for (int f = max(ctrl->filled - S::STAGES, 0); f < ctrl->filled; ++f) mbar_drain(smem_u32(&ctrl->full_bar[f % S::STAGES]), (f / S::STAGES) & 1);
      if (p.status_host != nullptr) *p.status_host = *p.status;
    } else if (issuer) {
      umma_commit(smem_u32(&ctrl->drain_bar));
      mbar_drain(smem_u32(&ctrl->drain_bar), 0);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ---- few rows an expert: 128 features x up to 64 rows, features on the M side -------------------------------------

// The weights are streamed once and everything else should cost nothing: a tile loads and computes the boxes (of 16, 32 or 64 rows) that hold rows.
// Bound by the weights' stream: 288 rows on 64 experts of 2816 x 2048 63 us (369 MB, 5.9 TB/s). A call of no size takes 5.4 us (launch, set-up, a
// block's way through TMA, MMA and TMEM, the cluster's meeting), two rows against 4096 x 7168 9.3.
constexpr int FEW_ROWS = 64;

// ONE: a cluster's CTAs share one tile's contraction, and so do the two groups of warps of each; else a CTA goes through tiles.
template <bool ONE>
struct FewRows {
  static constexpr int ROWS = FEW_ROWS;
  static constexpr int STAGE_BYTES = (A_ROWS + ROWS) * 128;
  static constexpr int STAGES = ONE ? 6 : 8;
  static constexpr int PART = ONE ? 2 * ROWS * A_ROWS * 4 : 0;  // the two groups' sums
  static constexpr int SLOTS = 8;  // blocks of a group whose scales are there or on their way
  struct Ctrl {
    unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full_bar[4], acc_empty_bar[4], scale_full_bar[2 * SLOTS], scale_empty_bar[2 * SLOTS], drain_bar;
    uint32_t tmem_base;
    int abort_flag;
    int filled;
    alignas(16) float scale[2 * SLOTS][ROWS + 4];  // of the rows, and of the features; a ring for each group
    Groups groups;
  };
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + PART + static_cast<int>(sizeof(Ctrl)) + 1024;
  static_assert(SMEM_BYTES <= 232448, "tile shape does not fit in shared memory");
};
constexpr int FEW_THREADS = 384;  // four warps as above, and two groups of a warp for each lane quarter, which take tiles in turn
constexpr int MAX_SPLIT = 8;

__device__ __forceinline__ float4 ld_shared_cluster(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}

// a feature's sums, rows `pitch` apart
template <typename T>
__device__ __forceinline__ void store_rows(T* out, long long pitch, int rows, const float (&sum)[FEW_ROWS]) {
#pragma unroll
  for (int j = 0; j < FEW_ROWS; ++j) {
    if (j < rows) out[j * pitch] = from_float<T>(sum[j]);
  }
}

// Sums of COLS rows from TMEM, scaled, added to those in registers
template <int COLS>
__device__ __forceinline__ void add_rows(uint32_t taddr, const float* scale, float w, float (&sum)[FEW_ROWS]) {
  uint32_t v[COLS];
  if constexpr (COLS == 16) {
    tmem_ld_32x16(taddr, v);
  } else {
#pragma unroll
    for (int c = 0; c < COLS; c += 32) tmem_ld_32x32(taddr + c, reinterpret_cast<uint32_t(&)[32]>(v[c]));
  }
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < COLS; j += 4) {
    const float4 s = *reinterpret_cast<const float4*>(scale + j);
    sum[j] = fmaf(__uint_as_float(v[j]), s.x * w, sum[j]);
    sum[j + 1] = fmaf(__uint_as_float(v[j + 1]), s.y * w, sum[j + 1]);
    sum[j + 2] = fmaf(__uint_as_float(v[j + 2]), s.z * w, sum[j + 2]);
    sum[j + 3] = fmaf(__uint_as_float(v[j + 3]), s.w * w, sum[j + 3]);
  }
}

//   warp 0      TMA producer          warp 1   MMA issuer, TMEM owner          warp 2   row ranges, scales          warp 3   nothing
//   warps 4..7, 8..11   take every other tile: while one group stores, the other has the next tile's sums
// ONE: they take every other block of the one tile. The groups' and the CTAs' sums meet in shared memory and are added in their order, row j by
// rank j % split. What runs once has little code: unrolled over the rows, with divisions and every output type, it cost 3 us of instruction fetches.
template <bool ONE>
__global__ void __launch_bounds__(FEW_THREADS, 1)
block_gemm_few_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ BlockParams p,
                      int split) {
  using S = FewRows<ONE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw), pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t smem_base = raw_addr + pad, part = smem_base + S::STAGES * S::STAGE_BYTES;
  auto* ctrl = reinterpret_cast<typename S::Ctrl*>(smem_raw + pad + S::STAGES * S::STAGE_BYTES + S::PART);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = ONE ? static_cast<int>(cluster_ctarank()) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(smem_u32(&ctrl->full_bar[s]), 1);
      mbar_init(smem_u32(&ctrl->empty_bar[s]), 1);
    }
    for (int a = 0; a < 4; ++a) {
      mbar_init(smem_u32(&ctrl->acc_full_bar[a]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty_bar[a]), 4);
    }
    for (int i = 0; i < 2 * S::SLOTS; ++i) {
      mbar_init(smem_u32(&ctrl->scale_full_bar[i]), 32);
      mbar_init(smem_u32(&ctrl->scale_empty_bar[i]), 4);
    }
    mbar_init(smem_u32(&ctrl->drain_bar), 1);
    ctrl->abort_flag = 0;
    ctrl->filled = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 2) fill_groups(ctrl->groups, p, S::ROWS, (p.N + A_ROWS - 1) / A_ROWS);
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), 4 * S::ROWS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const uint32_t tmem_base = ctrl->tmem_base;
  volatile int* abort_flag = &ctrl->abort_flag;
  bool issuer = false;
  const int total = ctrl->groups.items[p.experts + 1], scale_rows = (p.N + E4M3_BLOCK - 1) / E4M3_BLOCK;
  // a cluster has one tile: no second one to step to
  BlockWalker walker(&ctrl->groups, p, S::ROWS, ONE ? blockIdx.x / split : blockIdx.x, ONE ? total : gridDim.x);
  BlockTile t;
  // this CTA's blocks of a tile's contraction
  auto from = [&] { return ONE ? t.k_blocks * rank / split : 0; };
  auto to = [&] { return ONE ? t.k_blocks * (rank + 1) / split : t.k_blocks; };

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, filled = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && walker.next(t)) {
        const int boxed = (t.rows + p.box_rows - 1) / p.box_rows * p.box_rows;
        for (int kb = from(); kb < to(); ++kb) {
          ok = mbar_wait_bounded(smem_u32(&ctrl->empty_bar[stage]), phase ^ 1u, abort_flag, p.status, FFM_STATUS_WAIT_PRODUCER, p.wait_cycles);
          if (!ok) break;
          const uint32_t full = smem_u32(&ctrl->full_bar[stage]), w_dst = smem_base + stage * S::STAGE_BYTES;
          mbar_expect_tx(full, (A_ROWS + boxed) * 128);
          tma_load_3d(w_dst, &tm_w, full, kb * E4M3_BLOCK, t.across * A_ROWS, t.group);
          for (int r = 0; r < boxed; r += p.box_rows) tma_load_2d(w_dst + (A_ROWS + r) * 128, &tm_x, full, kb * E4M3_BLOCK, t.row0 + r);
          ++filled;
          if (++stage == S::STAGES) stage = 0, phase ^= 1u;
        }
      }
      ctrl->filled = filled;
    }
  } else if (warp == 1) {
    if (elect_one()) {
      issuer = true;
      int stage = 0, group = 0;
      uint32_t phase = 0, count[2] = {0, 0};  // accumulators that a group was given so far
      bool ok = true;
      for (; ok && walker.next(t); group ^= 1) {
        const uint32_t idesc = make_idesc_e4m3(A_ROWS, (t.rows + 15) & ~15);
        for (int kb = from(); kb < to(); ++kb) {
          if (ONE) group = (kb - from()) & 1;
          const int acc = group * 2 + (count[group] & 1);
          ok = mbar_wait_bounded(smem_u32(&ctrl->acc_empty_bar[acc]), ((count[group] >> 1) & 1) ^ 1u, abort_flag, p.status, FFM_STATUS_WAIT_MMA,
                                 p.wait_cycles) &&
               mbar_wait_bounded(smem_u32(&ctrl->full_bar[stage]), phase, abort_flag, p.status, FFM_STATUS_WAIT_MMA, p.wait_cycles);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_src = smem_base + stage * S::STAGE_BYTES, b_src = a_src + A_ROWS * 128;
#pragma unroll
          for (int kk = 0; kk < E4M3_BLOCK / UMMA_K8; ++kk) {
            umma_f8(tmem_base + acc * S::ROWS, make_smem_desc_sw128(a_src + kk * UMMA_K8, 16, 1024),
                    make_smem_desc_sw128(b_src + kk * UMMA_K8, 16, 1024), idesc, kk > 0 ? 1u : 0u);
          }
          umma_commit(smem_u32(&ctrl->empty_bar[stage]));
          umma_commit(smem_u32(&ctrl->acc_full_bar[acc]));
          ++count[group];
          if (++stage == S::STAGES) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 2) {
    // the scales of the tile's rows and features, block by block, ahead of the sums that they belong to. Each group has a ring of its own and so
    // waits for every round of it: on a ring of both, one that has skipped the other's tile would take the round before for its own.
    int group = 0;
    uint32_t count[2] = {0, 0};  // blocks that a group was given so far
    bool ok = true;
    for (; ok && walker.next(t); group ^= 1) {
      const float* ws = p.w_scale + (static_cast<long long>(t.group) * scale_rows + t.across) * p.k_blocks;
      const float* xs0 = p.x_scale + static_cast<long long>(t.row0 + min(lane, t.rows - 1)) * p.k_blocks;
      const float* xs1 = p.x_scale + static_cast<long long>(t.row0 + min(lane + 32, t.rows - 1)) * p.k_blocks;
      for (int kb = from(); kb < to(); ++kb) {
        if (ONE) group = (kb - from()) & 1;
        const uint32_t slot = group * S::SLOTS + count[group] % S::SLOTS;
        ok = mbar_wait_bounded(smem_u32(&ctrl->scale_empty_bar[slot]), ((count[group] / S::SLOTS) & 1) ^ 1u, abort_flag, p.status,
                               FFM_STATUS_WAIT_PRODUCER, p.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t dst = smem_u32(ctrl->scale[slot]);
        copy_async_4(dst + lane * 4, xs0 + kb);
        if (t.rows > 32) copy_async_4(dst + (lane + 32) * 4, xs1 + kb);
        if (lane == 0) copy_async_4(dst + S::ROWS * 4, ws + kb);
        copy_async_arrive(smem_u32(&ctrl->scale_full_bar[slot]));
        ++count[group];
      }
    }
    copy_async_wait<0>();
  } else if (warp >= 4) {
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + group * 2 * S::ROWS;
    uint32_t count = 0;  // blocks that this group was given so far
    bool ok = true;
    for (int turn = 0; ok && walker.next(t); turn ^= 1) {
      if (!ONE && turn != group) continue;
      float sum[S::ROWS];
#pragma unroll
      for (int j = 0; j < S::ROWS; ++j) sum[j] = 0.0f;
      for (int kb = from() + (ONE ? group : 0); kb < to(); kb += ONE ? 2 : 1, ++count) {
        const uint32_t acc = count & 1, slot = group * S::SLOTS + count % S::SLOTS;
        ok = mbar_wait_bounded(smem_u32(&ctrl->scale_full_bar[slot]), (count / S::SLOTS) & 1, abort_flag, p.status, FFM_STATUS_WAIT_EPILOGUE,
                               p.wait_cycles) &&
             mbar_wait_bounded(smem_u32(&ctrl->acc_full_bar[group * 2 + acc]), (count >> 1) & 1, abort_flag, p.status, FFM_STATUS_WAIT_EPILOGUE,
                               p.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const float* scale = ctrl->scale[slot];
        const float w = scale[S::ROWS];
        if (t.rows <= 16) {
          add_rows<16>(taddr + acc * S::ROWS, scale, w, sum);
        } else if (t.rows <= 32) {
          add_rows<32>(taddr + acc * S::ROWS, scale, w, sum);
        } else {
          add_rows<64>(taddr + acc * S::ROWS, scale, w, sum);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&ctrl->acc_empty_bar[group * 2 + acc]));
          mbar_arrive(smem_u32(&ctrl->scale_empty_bar[slot]));
        }
      }
      if (!ok) break;
      const int feature = quarter * 32 + lane, n = t.across * A_ROWS + feature;
      if constexpr (ONE) {
        const uint32_t at = part + (group * S::ROWS * A_ROWS + feature) * 4;
#pragma unroll
        for (int j = 0; j < S::ROWS; ++j) {
          if (j < t.rows) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + j * (A_ROWS * 4)), "f"(sum[j]) : "memory");
        }
      } else if (n < p.N) {
        const long long out = static_cast<long long>(t.row0) * p.N + n;
        if (p.out_type == FFM_TYPE_BF16) {
          store_rows(static_cast<bf16*>(p.out) + out, p.N, t.rows, sum);
        } else if (p.out_type == FFM_TYPE_FP16) {
          store_rows(static_cast<fp16*>(p.out) + out, p.N, t.rows, sum);
        } else {
          store_rows(static_cast<float*>(p.out) + out, p.N, t.rows, sum);
        }
      }
    }
  }
  if constexpr (ONE) {
    __syncwarp();
    cluster_sync_all();
    BlockWalker again(&ctrl->groups, p, S::ROWS, blockIdx.x / split, total);
    if (warp >= 4 && again.next(t)) {
      // a warp has a row, a lane four features of it
      const int n = t.across * A_ROWS + lane * 4;
      for (int j = rank + (warp - 4) * split; j < t.rows; j += 8 * split) {
        float4 v[2 * MAX_SPLIT];
#pragma unroll
        for (int r = 0; r < MAX_SPLIT; ++r) {
          if (r < split) {
            const uint32_t at = map_to_cta(part + (j * A_ROWS + lane * 4) * 4, r);
            v[2 * r] = ld_shared_cluster(at);
            v[2 * r + 1] = ld_shared_cluster(at + S::ROWS * A_ROWS * 4);
          }
        }
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < 2 * MAX_SPLIT; ++r) {
          if (r < 2 * split) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
        }
        const long long out = static_cast<long long>(t.row0 + j) * p.N + n;
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          if (n + i < p.N) store1_as(p.out, p.out_type, out + i, i == 0 ? f[0] : i == 1 ? f[1] : i == 2 ? f[2] : f[3]);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // this CTA's sums have been read
  }

  // ---- common exit, as above
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    if (threadIdx.x == 0) {
      for (int f = max(ctrl->filled - S::STAGES, 0); f < ctrl->filled; ++f) mbar_drain(smem_u32(&ctrl->full_bar[f % S::STAGES]), (f / S::STAGES) & 1);
      if (p.status_host != nullptr) *p.status_host = *p.status;
    } else if (issuer) {
      umma_commit(smem_u32(&ctrl->drain_bar));
      mbar_drain(smem_u32(&ctrl->drain_bar), 0);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 4 * S::ROWS);
  }
}

// ---- one row ----------------------------------------------------------------------------------------------------

// The products of one row on the CUDA cores: a stream of the weights, without the way through TMA, MMA, TMEM and a cluster's meeting that a tile takes.
// Bound by its instructions (eight conversions of two values to fp16 and sixteen on to fp32 for 16 weights): 4096 x 4096 6.9 us, a call of no size 2.6. A block has `features` of them and its warps equal shares of their 512-byte chunks; every share of a feature leaves one sum, added in their order.
constexpr int ROW_THREADS = 512, ROW_WARPS = ROW_THREADS / 32;
constexpr int ROW_AHEAD = 2;        // chunks that a warp works on, with as many on their way: instructions bound it, with more it is slower
constexpr int ROW_K_MAX = 16384;    // the row lies in shared memory in fp32, and two blocks on an SM
constexpr int ROW_FEATURES = 256;   // of a block at most: they lie in up to three blocks of weights' scales

// four e4m3 values
__device__ __forceinline__ float4 unpack_e4m3x4(uint32_t u) {
  const __half2_raw low = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(u & 0xffffu), __NV_E4M3);
  const __half2_raw high = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(u >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(low)), b = __half22float2(__half2(high));
  return make_float4(a.x, a.y, b.x, b.y);
}

__global__ void __launch_bounds__(ROW_THREADS, 2)
block_row_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w, int K, int features, const __grid_constant__ BlockParams p) {
  extern __shared__ __align__(16) float4 row[];  // [quarter of 16 values][piece of 16 values]: neighbouring lanes read neighbouring 16 bytes
  __shared__ float parts[ROW_FEATURES][ROW_WARPS + 1], scale[3][ROW_K_MAX / E4M3_BLOCK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = K / 16, chunks = (pieces + 31) / 32, first = blockIdx.x * features, count = min(features, p.N - first);
  // this warp's chunks of all features' together; the first of them are on their way while the row is laid out
  const int all = count * chunks, begin = all * warp / ROW_WARPS, end = all * (warp + 1) / ROW_WARPS;
  int feature = begin / chunks, chunk = begin % chunks, next_chunk = chunk, ahead = begin;
  const uint8_t* next_row = w + static_cast<long long>(first + feature) * K;
  auto fetch = [&](uint4 (&u)[ROW_AHEAD]) {
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      const int piece = next_chunk * 32 + lane;
      u[i] = ahead < end && piece < pieces ? *reinterpret_cast<const uint4*>(next_row + piece * 16) : make_uint4(0, 0, 0, 0);
      ++ahead;
      if (++next_chunk == chunks) next_chunk = 0, next_row += K;
    }
  };
  uint4 u[ROW_AHEAD];
  fetch(u);
  for (int i = threadIdx.x; i < pieces; i += ROW_THREADS) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + i * 16);
    row[i] = unpack_e4m3x4(v.x);
    row[pieces + i] = unpack_e4m3x4(v.y);
    row[2 * pieces + i] = unpack_e4m3x4(v.z);
    row[3 * pieces + i] = unpack_e4m3x4(v.w);
  }
  const int band = first / E4M3_BLOCK, bands = (first + count - 1) / E4M3_BLOCK - band + 1;
  for (int i = threadIdx.x; i < bands * p.k_blocks; i += ROW_THREADS) {
    const int b = i / p.k_blocks, kb = i % p.k_blocks;
    scale[b][kb] = __ldg(p.x_scale + kb) * __ldg(p.w_scale + static_cast<long long>(band + b) * p.k_blocks + kb);
  }
  for (int i = threadIdx.x; i < count * ROW_WARPS; i += ROW_THREADS) parts[i / ROW_WARPS][i % ROW_WARPS] = 0.0f;
  __syncthreads();
  float sum = 0.0f;
  auto leave = [&](int f) {
    const float total = warp_sum(sum);
    if (lane == 0) parts[f][warp] = total;
    sum = 0.0f;
  };
  for (int at = begin; at < end; at += ROW_AHEAD) {
    uint4 now[ROW_AHEAD];
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) now[i] = u[i];
    fetch(u);
#pragma unroll
    for (int i = 0; i < ROW_AHEAD; ++i) {
      if (at + i >= end) break;
      const int piece = chunk * 32 + lane;
      if (piece < pieces) {
        const uint32_t word[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
        float2 a = both(0.0f), b = both(0.0f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 v = unpack_e4m3x4(word[q]), r = row[q * pieces + piece];
          a = fma2(make_float2(v.x, v.y), make_float2(r.x, r.y), a);
          b = fma2(make_float2(v.z, v.w), make_float2(r.z, r.w), b);
        }
        sum = fmaf((a.x + a.y) + (b.x + b.y), scale[(first + feature) / E4M3_BLOCK - band][piece / (E4M3_BLOCK / 16)], sum);
      }
      if (++chunk == chunks) {
        leave(feature);
        chunk = 0;
        ++feature;
      }
    }
  }
  if (end > begin && chunk != 0) leave(feature);
  __syncthreads();
  for (int f = threadIdx.x; f < count; f += ROW_THREADS) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < ROW_WARPS; ++i) total += parts[f][i];
    store1_as(p.out, p.out_type, first + f, total);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------

// bytes [groups, rows, cols], rows `ld` bytes apart, boxes of 128 bytes x box_rows, 128-byte swizzle, zeros out of bounds
int make_byte_map(CUtensorMap* map, const void* base, long long groups, long long rows, long long cols, long long ld, int box_rows) {
  EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) return FFM_ERR_NO_DRIVER;
  if ((reinterpret_cast<uintptr_t>(base) & 15u) != 0 || ld % 16 != 0) return FFM_ERR_UNSUPPORTED;
  const bool flat = groups == 0;  // two dimensions
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(groups)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld), static_cast<cuuint64_t>(ld) * rows};
  cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, flat ? 2 : 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FFM_OK : FFM_ERR_LAUNCH;
}

template <typename K>
bool allow_smem(K kernel, int bytes, PerDevice& room) {
  return room.get([&] {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return 1;
  }) > 0;
}

template <int BN, int OUT_BYTES>
int launch_many(const CUtensorMap& tm_x, const CUtensorMap& tm_w, const CUtensorMap& tm_out, const BlockParams& p, long long tiles, cudaStream_t stream) {
  static PerDevice room;
  auto kernel = block_gemm_kernel<BN, OUT_BYTES>;
  if (!allow_smem(kernel, ManyRows<BN>::SMEM_BYTES, room)) return FFM_ERR_LAUNCH;
  kernel<<<static_cast<unsigned>(tiles < num_sms() ? tiles : num_sms()), BLOCK_THREADS, ManyRows<BN>::SMEM_BYTES, stream>>>(tm_x, tm_w, tm_out, p);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

template <bool ONE>
bool few_config(cudaLaunchConfig_t& config, cudaLaunchAttribute& attribute, int split) {
  static PerDevice room;
  if (!allow_smem(block_gemm_few_kernel<ONE>, FewRows<ONE>::SMEM_BYTES, room)) return false;
  config.blockDim = dim3(FEW_THREADS);
  config.dynamicSmemBytes = FewRows<ONE>::SMEM_BYTES;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(split);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = ONE ? 1 : 0;
  return true;
}

// Clusters of `split` CTAs that run at once: fewer than their SMs (148 give 74 of 2, 33 of 4, 22 of 6, 15 of 8).
int clusters_at_once(int split) {
  static PerDevice found[MAX_SPLIT + 1];
  return found[split].get([&] {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attribute = {};
    int n = 0;
    if (!few_config<true>(config, attribute, split)) return 0;
    config.gridDim = dim3(split);
    if (cudaOccupancyMaxActiveClusters(&n, block_gemm_few_kernel<true>, &config) != cudaSuccess) cudaGetLastError();
    return n;
  });
}

template <bool ONE>
int launch_few(const CUtensorMap& tm_x, const CUtensorMap& tm_w, const BlockParams& p, long long tiles, int split, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attribute = {};
  if (!few_config<ONE>(config, attribute, split)) return FFM_ERR_LAUNCH;
  config.gridDim = dim3(static_cast<unsigned>(ONE ? tiles * split : (tiles < num_sms() ? tiles : num_sms())));
  config.stream = stream;
  const cudaError_t rc = cudaLaunchKernelEx(&config, block_gemm_few_kernel<ONE>, tm_x, tm_w, p, split);
  if (rc != cudaSuccess) cudaGetLastError();
  return rc == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

int launch_row(const ffm_linear_blocks_args& a, const BlockParams& p, cudaStream_t stream) {
  static PerDevice room;
  if (!allow_smem(block_row_kernel, ROW_K_MAX * static_cast<int>(sizeof(float)), room)) return FFM_ERR_LAUNCH;
  const int64_t even = (a.N + 2 * num_sms() - 1) / (2 * num_sms());
  const int features = static_cast<int>(even < ROW_FEATURES ? even : ROW_FEATURES);
  block_row_kernel<<<static_cast<unsigned>((a.N + features - 1) / features), ROW_THREADS, static_cast<size_t>(a.K) * sizeof(float), stream>>>(
      static_cast<const uint8_t*>(a.x), static_cast<const uint8_t*>(a.w), static_cast<int>(a.K), features, p);
  return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
}

}  // namespace

}  // namespace ffm

using namespace ffm;

extern "C" int ffm_quantize_blocks_e4m3(const void* x, int x_type, int64_t matrices, int64_t rows, int64_t row_stride, int K, int block_rows, void* q,
                                        float* scale, ffm_stream_t stream) {
  if (!is_type(x_type) || matrices < 0 || rows < 0 || K <= 0 || (block_rows != 1 && block_rows != E4M3_BLOCK)) return FFM_ERR_BAD_ARG;
  if ((row_stride < K && rows > 1) || (block_rows == 1 && matrices > 1)) return FFM_ERR_BAD_ARG;
  if (K % 16 != 0 || rows > 0x7fffffffll || (block_rows > 1 && matrices * rows > 0 && row_stride != K)) return FFM_ERR_UNSUPPORTED;
  if (matrices == 0 || rows == 0) return FFM_OK;
  if (!x || !q || !scale) return FFM_ERR_BAD_ARG;
  if (off_16_bytes(x) || (row_stride * type_bytes(x_type)) % 16 != 0 || (reinterpret_cast<uintptr_t>(q) & 7u) != 0) return FFM_ERR_UNSUPPORTED;
  const int across = (K + E4M3_BLOCK - 1) / E4M3_BLOCK, down = static_cast<int>((rows + block_rows - 1) / block_rows);
  const long long blocks = block_rows == 1 ? rows * across : matrices * down * across;
  const int per = block_rows == 1 ? QB_CHUNKS * QB_THREADS / (x_type == FFM_TYPE_FP32 ? 32 : 16) : 1;
  const long long grid = (blocks + per - 1) / per;
  if (grid > 0x7fffffffll) return FFM_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto tag) {
    using T = decltype(tag);
    if (block_rows == 1) {
      quantize_row_blocks_kernel<T><<<static_cast<unsigned>(grid), QB_THREADS, 0, st>>>(static_cast<const T*>(x), row_stride, blocks, across, K,
                                                                                      static_cast<uint8_t*>(q), scale);
    } else {
      quantize_tiles_kernel<T><<<static_cast<unsigned>(grid), QB_THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<int>(rows), K, down, across,
                                                                                 static_cast<uint8_t*>(q), scale);
    }
    return cudaGetLastError() == cudaSuccess ? FFM_OK : FFM_ERR_LAUNCH;
  };
  if (x_type == FFM_TYPE_BF16) return launch(bf16{});
  if (x_type == FFM_TYPE_FP16) return launch(fp16{});
  return launch(float{});
}

extern "C" int ffm_linear_blocks_e4m3(const ffm_linear_blocks_args* args, ffm_stream_t stream) {
  if (args == nullptr) return FFM_ERR_BAD_ARG;
  const ffm_linear_blocks_args& a = *args;
  if (a.rows < 0 || a.N < 1 || a.K < 1 || a.experts < 1 || !is_type(static_cast<int>(a.out_type)) || (a.x_stride < a.K && a.rows > 1)) return FFM_ERR_BAD_ARG;
  if (a.ends == nullptr && a.experts != 1) return FFM_ERR_BAD_ARG;
  if (a.rows == 0) return FFM_OK;
  if (!a.x || !a.x_scale || !a.w || !a.w_scale || !a.out || !a.status) return FFM_ERR_BAD_ARG;
  if (a.K % 16 != 0 || a.x_stride % 16 != 0 || a.experts > MAX_EXPERTS || a.rows > (1ll << 30) || a.N > (1ll << 30) || a.K > (1ll << 30)) return FFM_ERR_UNSUPPORTED;
  BlockParams p = {};
  p.x_scale = a.x_scale;
  p.w_scale = a.w_scale;
  p.ends = a.ends;
  p.experts = static_cast<int>(a.experts);
  p.rows = static_cast<int>(a.rows);
  p.N = static_cast<int>(a.N);
  p.k_blocks = static_cast<int>((a.K + E4M3_BLOCK - 1) / E4M3_BLOCK);
  p.out_type = static_cast<int>(a.out_type);
  p.out_wide = a.N * type_bytes(p.out_type) % 16 == 0 && !off_16_bytes(a.out);
  p.out = a.out;
  p.status = a.status;
  p.status_host = a.status_host;
  p.wait_cycles = gemm_wait_cycles();
  const bool grouped = a.ends != nullptr;
  // One row: us against a cluster a tile, weights in L2 (from memory): 256 x 512 2.6 / 5.1, 2048 x 2048 3.9 / 5.8 (4.3 / 6.7), 4096 x 4096 6.5 / 7.3
  // (7.3 / 8.8), 24 M weights 8.0 / 9.4 (9.0 / 10.9), 28 M 9.1 / 9.2 (10.1 / 10.8), 32 M 9.7 / 9.6 (10.7 / 11.5), 40 M 10240 x 4096 11.5 / 13.9 (12.7 / 15.0),
  // but 2560 x 16384 11.9 / 11.2 (13.2 / 12.9), 44 M 13.3 / 11.2 (14.7 / 13.1), 56 M 14.8 / 13.9 (16.4 / 15.7).
  if (!grouped && a.rows == 1 && a.K <= ROW_K_MAX && a.N * a.K <= 32ll << 20) {
    if (off_16_bytes(a.x, a.w)) return FFM_ERR_UNSUPPORTED;
    return launch_row(a, p, static_cast<cudaStream_t>(stream));
  }
  const int64_t average = a.rows / a.experts;
  // Tiles at most: every expert may end inside of one, and so may the rows behind the last. And about: half of the experts' ends cost one.
  auto tiles = [&](int64_t tile_rows, int64_t width) {
    const int64_t ends = grouped ? (a.experts < a.rows ? a.experts : a.rows) + 1 : (a.rows % tile_rows != 0);
    return (a.rows / tile_rows + ends) * ((a.N + width - 1) / width);
  };
  auto rounds = [&](int64_t width) {
    const int64_t down = a.rows / A_ROWS + (grouped ? (a.experts + 1) / 2 : (a.rows % A_ROWS != 0));
    return (down * ((a.N + width - 1) / width) + num_sms() - 1) / num_sms();
  };
  // One tile a cluster, where all fit at once: its contraction is split over as many CTAs as that leaves.
  const int64_t few_tiles = tiles(FEW_ROWS, A_ROWS);
  int split = 1;
  for (int s = MAX_SPLIT; s > 1 && split == 1; --s) {
    if (p.k_blocks >= 2 * s && few_tiles * s <= num_sms() && few_tiles <= clusters_at_once(s)) split = s;
  }
  // The weights' stream bounds few rows. us, few against many rows a tile: 64 experts of 2816 x 2048, rows each 4: 62 / 67, 16: 65 / 70, 32: 73 / 71, 64:
  // 123 / 72; dense 4096 x 4096, 16 rows 8 / 13, 64 rows 10.5 / 13, 128 rows 17 / 13; where the contraction is not split, 32 x 14336 x 4096 18 / 14;
  // 64 x 1024 x 1024 7.6 / 6.1.
  const bool few = grouped ? average <= 24 : a.rows <= 16 || (a.rows <= FEW_ROWS && split > 1 && p.k_blocks >= 16);
  // an expert's rows in one load of x for the most part
  p.box_rows = average <= (grouped ? 8 : 16) ? 16 : (average <= (grouped ? 24 : 32) ? 32 : FEW_ROWS);
  // A tile of 256 features takes 1.65 times as long as one of 128 (1024 x 4096 x 4096: one round of it 23 us, two of 128 27; 512 x 4096 x 4096: 21 and 15).
  const int box_n = few || rounds(256) * 165 > rounds(128) * 100 ? A_ROWS : 256, box_m = few ? p.box_rows : A_ROWS;
  const int64_t most = few ? few_tiles : tiles(A_ROWS, box_n);
  if (most > 0x3fffffff) return FFM_ERR_UNSUPPORTED;
  CUtensorMap tm_x, tm_w;
  int rc = make_byte_map(&tm_x, a.x, 0, a.rows, a.K, a.rows > 1 ? a.x_stride : a.K, box_m);
  if (rc == FFM_OK) rc = make_byte_map(&tm_w, a.w, a.experts, a.N, a.K, a.K, box_n);
  if (rc != FFM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool four = p.out_type == FFM_TYPE_FP32;
  if (few) return most <= num_sms() ? launch_few<true>(tm_x, tm_w, p, most, split, st) : launch_few<false>(tm_x, tm_w, p, most, 1, st);
  CUtensorMap tm_out = {};  // read only where rows lie on 16 bytes
  if (p.out_wide) {
    rc = make_box_map(&tm_out, a.out, 1, a.rows, a.N, a.N, type_bytes(p.out_type));
    if (rc != FFM_OK) return rc;
  }
  if (box_n == 256) return four ? launch_many<256, 4>(tm_x, tm_w, tm_out, p, most, st) : launch_many<256, 2>(tm_x, tm_w, tm_out, p, most, st);
  return four ? launch_many<128, 4>(tm_x, tm_w, tm_out, p, most, st) : launch_many<128, 2>(tm_x, tm_w, tm_out, p, most, st);
}
