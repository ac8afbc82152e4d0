// Entry points shared by the translation units of the library: the C ABI's routing functions with the small per-call
// values (losses, their gradients) read and written on the device, as the layer driver (ffm_layer.cu) uses them.
#pragma once

#include "../../include/ffmoe.h"

namespace ffm {

// True where an address does not lie on a 16-byte boundary. The row and routing kernels load and store 16 bytes at a time, and an
// access off that boundary ends the context; the GEMMs' tensor maps refuse such operands themselves.
template <typename... P>
bool off_16_bytes(const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 15u) != 0;
}

// ffm_route_forward; aux = aux_scale * stats[E + 1], z = z_scale * stats[E], *zero = 0 (each skipped when null).
int route_forward_losses(const void* hidden, const void* gate_w, const float* expert_bias, int64_t N, int D, int E,
                         int top_k, int gating, float weight_scale, int pre_softmax, int n_group, int topk_group,
                         void* logits, float* topk_w, int32_t* topk_idx, float* lse, int32_t* counts,
                         int32_t* tile_start, int32_t* pos, int32_t* src, int64_t rows_cap, float* stats, float* aux,
                         float aux_scale, float* z, float z_scale, int32_t* zero, void* workspace,
                         size_t workspace_bytes, int32_t* status, ffm_stream_t stream);

// Gradients of the two losses: either the arrays of ffm_route_backward (gaux [E], gz scalar), or the upstream scalars
// (grad_aux, grad_z; null = no such term) with gaux[e] = counts[e] * (*grad_aux * aux_coef), gz = *grad_z * z_coef.
struct LossGrads {
  const float* gaux;
  const float* gz;
  const int32_t* counts;
  const float* grad_aux;
  const float* grad_z;
  float aux_coef;
  float z_coef;
};

int route_backward_losses(const float* gw, const float* topk_w, const int32_t* topk_idx, const void* logits,
                          const float* lse, const LossGrads& lg, const void* hidden, const void* gate_w, int64_t N,
                          int D, int E, int top_k, int gating, int accumulate, void* dH, void* dGate, void* workspace,
                          size_t workspace_bytes, int32_t* status, ffm_stream_t stream);

// ffm_grouped_gemm_wgrad_rows; with tile_start null the groups are equal ranges (in 128-row tiles) of the rows, a split of
// one dense contraction.
int grouped_wgrad(const void* A, const void* B, int groups, const int32_t* tile_start, const int32_t* counts,
                  int64_t rows_cap, int M, int Nout, float scale, void* dW, int32_t* status, ffm_stream_t stream);

// ffm_combine_forward_add2; with status_host (host memory the device can write) a non-zero *status is stored there.
int combine_forward_status(const void* Y, const int32_t* pos, const float* w, const void* addend, const void* addend2,
                           int64_t N, int top_k, int D, void* out, const int32_t* status, int32_t* status_host,
                           ffm_stream_t stream);

// out = a + b, bf16 values added in fp32 (n elements, a multiple of 8)
int add_bf16(const void* a, const void* b, int64_t n, void* out, ffm_stream_t stream);

// ---- products of the linear cross entropy (ffm_gemm_sm100.cu) ----

// What softmax_logits' exponentials are stored times of: the largest of 128 is 2^15 then, and fp16 holds all of its 11 bits down to 2^-29 of
// that one in place of 2^-14 (and something down to 2^-40 in place of 2^-25).
constexpr float SOFTMAX_STORED_SCALE = 32768.0f;

// Logits hidden [rows, D] weight [V, D]^T, a tile at a time and never stored: stats[n * ceil(V / 128) + h] = (largest,
// sum of exp(logit - largest)) (pairs of floats) over row n's entries 128 h .. 128 h + 127, target_logits[n] the logit of targets[n] where that is
// an entry; with `e` the exponentials times SOFTMAX_STORED_SCALE in fp16, rows ld_e apart (a multiple of 8). D % 8 == 0.
int softmax_logits(const void* hidden, const void* weight, int64_t rows, int D, int V, const int64_t* targets,
                   float* target_logits, float* stats, void* e, int64_t ld_e, int32_t* status, ffm_stream_t stream);

// A [rows, K] (rows ld_a apart) B [K, Nout]: bf16 out [rows, Nout], or with splits > 1 fp32 out [splits, rows, Nout] of as many
// pieces of the contraction. Nout % 8 == 0, any K. scale: device scalar that multiplies the result before it is rounded, or null.
int dense_rows(const void* A, int64_t ld_a, int64_t rows, int K, const void* B, int Nout, int splits, const float* scale, void* out,
               int32_t* status, ffm_stream_t stream);

// A [rows, M]^T (rows ld_a apart) B [rows, Nout]: out [M, Nout] in bf16, or in fp32, with `add` added to what is there.
// Nout % 8 == 0, any M. scale as above.
int dense_transposed(const void* A, int64_t ld_a, const void* B, int64_t rows, int M, int Nout, int f32, int add, const float* scale,
                     void* out, int32_t* status, ffm_stream_t stream);

}  // namespace ffm
