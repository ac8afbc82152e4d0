// The operators beside the layer for torch tensors: argument checks, outputs, scratch and the call into libffmoe. A call from
// Python costs these few checks; the torch operations that they would be there (views, contiguity, empty) take longer than
// the kernels of a small call.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <limits>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "../../include/ffmoe.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

decltype(&ffm_error_string) error_string = nullptr;
decltype(&ffm_layer_norm_forward) norm_forward = nullptr;
decltype(&ffm_layer_norm_workspace_bytes) norm_workspace = nullptr;
decltype(&ffm_layer_norm_backward) norm_backward = nullptr;
decltype(&ffm_adamw_step) adamw = nullptr;
decltype(&ffm_linear_cross_entropy) cross_entropy = nullptr;
decltype(&ffm_linear_cross_entropy_workspace_bytes) cross_entropy_workspace = nullptr;
decltype(&ffm_scale_many) scale_many = nullptr;
decltype(&ffm_capture_id) capture_id = nullptr;
decltype(&ffm_rms_norm_forward) rms_forward = nullptr;
decltype(&ffm_rms_norm_workspace_bytes) rms_workspace = nullptr;
decltype(&ffm_rms_norm_backward) rms_backward = nullptr;
decltype(&ffm_quantize_blocks_e4m3) quantize_blocks = nullptr;
decltype(&ffm_linear_blocks_e4m3) linear_blocks = nullptr;
decltype(&ffm_grad_norm_workspace_bytes) grad_norm_workspace = nullptr;
decltype(&ffm_grad_norm) grad_norm = nullptr;
decltype(&ffm_scale_tensors) scale_tensors = nullptr;

void bind_ops(const std::unordered_map<std::string, uintptr_t>& at) {
  auto take = [&](const char* name, auto& f) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at.at(name)); };
  take("ffm_error_string", error_string);
  take("ffm_layer_norm_forward", norm_forward);
  take("ffm_layer_norm_workspace_bytes", norm_workspace);
  take("ffm_layer_norm_backward", norm_backward);
  take("ffm_adamw_step", adamw);
  take("ffm_linear_cross_entropy", cross_entropy);
  take("ffm_linear_cross_entropy_workspace_bytes", cross_entropy_workspace);
  take("ffm_scale_many", scale_many);
  take("ffm_capture_id", capture_id);
  take("ffm_rms_norm_forward", rms_forward);
  take("ffm_rms_norm_workspace_bytes", rms_workspace);
  take("ffm_rms_norm_backward", rms_backward);
  take("ffm_quantize_blocks_e4m3", quantize_blocks);
  take("ffm_linear_blocks_e4m3", linear_blocks);
  take("ffm_grad_norm_workspace_bytes", grad_norm_workspace);
  take("ffm_grad_norm", grad_norm);
  take("ffm_scale_tensors", scale_tensors);
}

void check(int rc, const char* what) {
  if (rc != FFM_OK) {
    throw std::runtime_error(std::string("libffmoe ") + what + " failed: " + std::to_string(rc) + " (" + error_string(rc) + ")");
  }
}

// The device of `t` is current and its current stream is the call's.
class On {
 public:
  explicit On(const Tensor& t) : guard_(t.device()), device_(t.device()) {}
  ffm_stream_t stream() const {
    return c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getStream(device_).native_handle();
  }

 private:
  c10::DeviceGuard guard_;
  c10::Device device_;
};

// What goes past torch's dispatcher: a tangent would be dropped, and a trace would record an output that nothing fills.
void no_tangent(const Tensor& t, const char* name) {
  if (t.defined() && t._fw_grad(0).defined()) {
    throw std::runtime_error(std::string(name) + " carries a forward-mode tangent: there are no forward-mode derivatives here");
  }
}
void not_traced(const char* what) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value()) {
    throw std::runtime_error(std::string(what) + " cannot be traced");
  }
}

void on_gpu(const Tensor& t, const char* name) {
  no_tangent(t, name);
  if (!t.is_cuda()) {
    throw std::runtime_error(std::string(name) + " must be a CUDA tensor: flashfusedmoe_b200 has no CPU path");
  }
  if (t.layout() != at::kStrided) throw py::value_error(std::string(name) + " must be a dense tensor");
}

void same_device(const Tensor& t, const Tensor& other, const char* name) {
  on_gpu(t, name);
  if (t.device() != other.device()) throw py::value_error("All tensors must be on same device");
}

int element_type(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FFM_TYPE_BF16;
    case at::kHalf: return FFM_TYPE_FP16;
    case at::kFloat: return FFM_TYPE_FP32;
    default:
      throw py::type_error(std::string(name) + " must be bfloat16, float16 or float32, got " + c10::toString(t.scalar_type()));
  }
}

// A leaf's gradient is added to it on the stream where the oldest graph that still lives first took the leaf. Where that is the
// default stream, which takes no part in a capture, a captured backward pass ends the process: refused while nothing has happened.
void capturable(std::initializer_list<const Tensor*> operands) {
  for (const Tensor* t : operands) {
    if (!t->defined() || !t->is_cuda() || !t->requires_grad() || !t->is_leaf()) continue;
    const c10::impl::VirtualGuardImpl cuda(c10::DeviceType::CUDA);
    if (cuda.getStream(t->device()) == cuda.getDefaultStream(t->device())) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (node == nullptr || node->stream() != cuda.getDefaultStream(t->device())) continue;
    const py::gil_scoped_acquire held;
    if (py::module_::import("torch.cuda").attr("is_current_stream_capturing")().cast<bool>()) {
      throw std::runtime_error("an autograd graph that was made on the default stream before the capture still holds an operand: let go of what "
                               "came from it (a loss, an output) before the capture");
    }
  }
}

// values in memory, one after the other, with no negation pending
Tensor plain(const Tensor& t) { return t.contiguous().resolve_neg(); }

// ---- layer norm ---------------------------------------------------------------------------------------------

struct Rows {
  Tensor x;  // keeps the memory
  int64_t rows, stride;
};

// x as rows of its last dimension: as it lies where its rows are one distance apart, else a copy
Rows as_rows(const Tensor& t) {
  Tensor x = t.is_neg() ? t.resolve_neg() : t;
  const int64_t D = x.size(-1), rows = D > 0 ? x.numel() / D : 0;
  bool fits = x.stride(-1) == 1 || D == 1;
  int64_t stride = 0, expected = 0;  // distance of two rows; of two neighbours in the dimension looked at
  for (int64_t d = x.dim() - 2; d >= 0 && fits; --d) {
    if (x.size(d) == 1) continue;
    if (stride == 0) {
      stride = x.stride(d);
      fits = stride >= D;
    } else {
      fits = x.stride(d) == expected;
    }
    expected = x.stride(d) * x.size(d);
  }
  if (!fits) {
    x = x.contiguous();
    stride = D;
  }
  return {x, rows, stride == 0 ? D : stride};
}

void check_vector(const Tensor& v, const Tensor& x, const char* name) {
  if (!v.defined()) return;
  same_device(v, x, name);
  if (v.dim() != 1 || v.size(0) != x.size(-1)) {
    throw py::value_error(std::string(name) + " must be [" + std::to_string(x.size(-1)) + "], got " + c10::str(v.sizes()));
  }
  element_type(v, name);
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::atomic<int64_t> launches{0};  // of these operators' kernels so far

struct NormResult {
  Tensor y, mean, rstd;
};

NormResult norm_forward_of(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool stats) {
  on_gpu(x, "x");
  if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error("x must have a last dimension to normalise, got " + c10::str(x.sizes()));
  if (x.size(-1) > std::numeric_limits<int>::max()) throw py::value_error("x has rows of " + std::to_string(x.size(-1)) + " values");
  if (!(eps >= 0.0)) throw py::value_error("eps must not be negative, got " + std::to_string(eps));
  const int type = element_type(x, "x");
  check_vector(weight, x, "weight");
  check_vector(bias, x, "bias");
  const On device(x);
  const Rows r = as_rows(x);
  const Tensor w = weight.defined() ? plain(weight) : Tensor(), b = bias.defined() ? plain(bias) : Tensor();
  NormResult out;
  out.y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (stats) {
    const Tensor both = at::empty({2, r.rows}, x.options().dtype(at::kFloat));
    out.mean = both.select(0, 0);
    out.rstd = both.select(0, 1);
  }
  check(norm_forward(r.x.data_ptr(), type, r.rows, r.stride, static_cast<int>(x.size(-1)), address(w),
                     w.defined() ? element_type(w, "weight") : 0, address(b), b.defined() ? element_type(b, "bias") : 0,
                     static_cast<float>(eps), out.y.data_ptr(), stats ? out.mean.data_ptr<float>() : nullptr,
                     stats ? out.rstd.data_ptr<float>() : nullptr, device.stream()),
        "ffm_layer_norm_forward");
  launches += r.rows > 0;
  return out;
}

struct NormGradients {
  Tensor dx, dweight, dbias;
};

NormGradients norm_backward_of(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& mean, const Tensor& rstd,
                               bool want_x, bool want_weight, bool want_bias, at::ScalarType bias_type) {
  const On device(x);
  const int type = element_type(x, "x");
  const int64_t D = x.size(-1);
  const Rows r = as_rows(x);
  // saved-tensor hooks may have handed back other tensors than were saved
  for (const Tensor* t : {&mean, &rstd}) {
    if (t->numel() != r.rows || t->scalar_type() != at::kFloat || !t->is_cuda()) throw py::value_error("saved statistics do not belong to x");
  }
  const Tensor m = plain(mean), s = plain(rstd);
  const Tensor g = plain(dy.scalar_type() == x.scalar_type() ? dy : dy.to(x.scalar_type()));
  same_device(g, x, "the gradient of y");
  if (g.sizes() != x.sizes()) throw py::value_error("the gradient of y has another shape than x");
  const Tensor w = weight.defined() ? plain(weight) : Tensor();
  NormGradients out;
  Tensor workspace;
  if (want_x) out.dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (want_weight) out.dweight = at::empty({D}, w.options());
  if (want_bias) out.dbias = at::empty({D}, x.options().dtype(bias_type));
  size_t bytes = 0;
  if (want_weight || want_bias) {
    bytes = norm_workspace(r.rows, static_cast<int>(D), type);
    workspace = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  }
  check(norm_backward(g.data_ptr(), r.x.data_ptr(), type, r.rows, r.stride, static_cast<int>(D), address(w),
                      w.defined() ? element_type(w, "weight") : 0, m.data_ptr<float>(), s.data_ptr<float>(), address(out.dx),
                      address(out.dweight), address(out.dbias), want_bias ? element_type(out.dbias, "bias") : 0, address(workspace),
                      bytes, device.stream()),
        "ffm_layer_norm_backward");
  launches += want_weight || want_bias ? 2 : want_x && r.rows > 0;
  return out;
}

using torch::autograd::variable_list;

// What a backward pass hands out when it is itself recorded (create_graph): gradients that refuse to be differentiated.
variable_list once(variable_list gradients) {
  if (!at::GradMode::is_enabled()) return gradients;
  for (Tensor& g : gradients) {
    if (g.defined()) g = g.detach().set_requires_grad(true);
  }
  auto refuses = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that can be differentiated once", static_cast<int64_t>(gradients.size()));
  return (*refuses)(std::move(gradients));
}

// The graph's node in C++: from Python, the engine's thread takes the interpreter's lock and a training step of a small norm
// took 92 us of host time.
class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight_or_none, const OptTensor& bias_or_none,
                        double eps) {
    const Tensor weight = weight_or_none.value_or(Tensor()), bias = bias_or_none.value_or(Tensor());
    NormResult r = norm_forward_of(x, weight, bias, eps, true);
    ctx->save_for_backward({x, weight, r.mean, r.rstd});
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["bias_type"] = static_cast<int64_t>(bias.defined() ? bias.scalar_type() : x.scalar_type());
    return r.y;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grad) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(4);
    {
      const at::AutoGradMode no_grad(false);
      // an operand that is not there has no edge, and those after it move up
      const bool weight = saved[1].defined(), bias = ctx->saved_data["bias"].toBool();
      NormGradients g = norm_backward_of(grad[0], saved[0], saved[1], saved[2], saved[3], ctx->needs_input_grad(0),
                                         weight && ctx->needs_input_grad(1), bias && ctx->needs_input_grad(weight ? 2 : 1),
                                         static_cast<at::ScalarType>(ctx->saved_data["bias_type"].toInt()));
      out[0] = g.dx;
      out[1] = g.dweight;
      out[2] = g.dbias;
    }
    return once(std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  not_traced("layer_norm");
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  no_tangent(x, "x");
  no_tangent(w, "weight");
  no_tangent(b, "bias");
  const py::gil_scoped_release released;
  if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()))) {
    capturable({&x, &w, &b});
    return LayerNorm::apply(x, weight, bias, eps);
  }
  return norm_forward_of(x, w, b, eps, false).y;
}

// ---- linear cross entropy -------------------------------------------------------------------------------------

// Scratch for the entries of a piece of rows, in bytes: 1 % of the device's memory. More pieces are more launches, and traffic for the sum of the
// weight's gradient: 16384 x 1024 rows, 50257 entries take 4.5 ms in one piece, 4.6-5.2 in two and 5.2 in four; 8192 x 4096 rows, 131072 entries,
// at the power cap, 22.1 in one and 21.5 in two.
constexpr int64_t PIECE_BYTES = int64_t{2} << 30;

enum Reduction { REDUCE_NONE = 0, REDUCE_MEAN = 1, REDUCE_SUM = 2 };

struct LossCall {
  int64_t ignore_index = 0;
  int64_t reduction = REDUCE_MEAN;
  double z = 0.0;
  int64_t piece_rows = 0;  // 0: as many as PIECE_BYTES hold
  int64_t status = 0, status_host = 0;
};

struct LossResult {
  Tensor nll, loss, d_hidden, d_weight;
};

// hidden [N, D] and weight [V, D] in bf16, contiguous
LossResult loss_pass(const Tensor& hidden, const Tensor& weight, const Tensor& target, const LossCall& call, const Tensor& row_grad,
                     bool want_hidden, bool want_weight, bool weight_f32) {
  const On device(hidden);
  const auto f32 = hidden.options().dtype(at::kFloat);
  LossResult out;
  ffm_loss_args a = {};
  a.N = hidden.size(0);
  a.D = hidden.size(1);
  a.V = weight.size(0);
  a.ignore_index = call.ignore_index;
  a.mean = call.reduction == REDUCE_MEAN;
  a.d_weight_f32 = weight_f32;
  a.z = call.z;
  a.piece_rows = call.piece_rows;
  if (a.piece_rows <= 0) {
    // two bytes an entry, or without gradients (8 bytes for 128 entries) as many rows as would take a quarter of it
    const int64_t row_bytes = want_hidden || want_weight ? (a.V + 63) / 64 * 128 : (a.V + 127) / 128 * 32, most = std::max<int64_t>(PIECE_BYTES / row_bytes / 256 * 256, 256);
    const int64_t pieces = std::max<int64_t>((a.N + most - 1) / most, 1);
    a.piece_rows = std::max<int64_t>(((a.N + pieces - 1) / pieces + 255) / 256 * 256, 256);
  }
  out.nll = at::empty({a.N}, f32);
  if (call.reduction != REDUCE_NONE) out.loss = at::empty({}, f32);
  if (want_hidden) out.d_hidden = at::empty_like(hidden, at::MemoryFormat::Contiguous);
  if (want_weight) out.d_weight = at::empty_like(weight, weight.options().dtype(weight_f32 ? at::kFloat : at::kBFloat16), at::MemoryFormat::Contiguous);
  a.hidden = hidden.data_ptr();
  a.weight = weight.data_ptr();
  a.targets = target.data_ptr<int64_t>();
  a.row_grad = row_grad.defined() ? row_grad.data_ptr<float>() : nullptr;
  a.nll = out.nll.data_ptr<float>();
  a.loss = static_cast<float*>(address(out.loss));
  a.d_hidden = address(out.d_hidden);
  a.d_weight = address(out.d_weight);
  if (a.N == 0) {  // nothing to read, and empty tensors have no address
    if (out.loss.defined()) out.loss.fill_(a.mean ? std::numeric_limits<double>::quiet_NaN() : 0.0);
    if (want_weight) out.d_weight.zero_();
    return out;
  }
  a.workspace_bytes = static_cast<int64_t>(cross_entropy_workspace(&a));
  const Tensor workspace = at::empty({a.workspace_bytes}, hidden.options().dtype(at::kByte));
  a.workspace = workspace.data_ptr();
  a.status = reinterpret_cast<int32_t*>(call.status);
  a.status_host = reinterpret_cast<int32_t*>(call.status_host);
  int64_t launched = 0;
  a.launched = &launched;
  check(cross_entropy(&a, device.stream()), "ffm_linear_cross_entropy");
  launches += launched;
  return out;
}

void scale_gradients(const Tensor& a, const Tensor& b, const Tensor& factor) {
  void* x[2];
  int64_t types[2], elements[2];
  int n = 0;
  for (const Tensor* t : {&a, &b}) {
    if (!t->defined() || t->numel() == 0) continue;
    x[n] = t->data_ptr();
    types[n] = element_type(*t, "gradient");
    elements[n++] = t->numel();
  }
  if (n == 0) return;
  const On device(factor);
  check(scale_many(n, x, types, elements, factor.data_ptr<float>(), device.stream()), "ffm_scale_many");
  ++launches;
}

Tensor as_bf16(const Tensor& t) { return plain(t.scalar_type() == at::kBFloat16 ? t : t.to(at::kBFloat16)); }

// Where the loss is one number, its gradients are computed with it, while the exponentials of a piece of rows are there: with them
// taken again in the backward pass a step would have four large products instead of three. The backward pass multiplies them by
// its factor, in place, which does nothing where that is 1. It hands them out once; a second backward pass over the same graph
// computes them again. A backward pass that is not in the loss's own capture may run more often than the loss (a graph of its own,
// replayed): it takes a copy, or computes the gradients again where the loss was not captured and is not there to be read by replays. With a value
// for each row the factors come with the backward pass, and so do the products.
class LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& target,
                        int64_t ignore_index, int64_t reduction, double z, int64_t piece_rows, int64_t status, int64_t status_host) {
    const LossCall call{ignore_index, reduction, z, piece_rows, status, status_host};
    const bool now = reduction != REDUCE_NONE;
    const Tensor flat = hidden.reshape({-1, hidden.size(-1)});
    LossResult r = loss_pass(as_bf16(flat), as_bf16(weight), target, call, Tensor(), now && hidden.requires_grad(), now && weight.requires_grad(),
                             weight.scalar_type() == at::kFloat);
    ctx->save_for_backward({hidden, weight, target});
    ctx->saved_data["call"] = std::vector<int64_t>{ignore_index, reduction, piece_rows, status, status_host};
    ctx->saved_data["z"] = z;
    if (now) ctx->saved_data["capture"] = static_cast<int64_t>(capture_id(On(hidden).stream()));
    if (r.d_hidden.defined()) ctx->saved_data["d_hidden"] = r.d_hidden;
    if (r.d_weight.defined()) ctx->saved_data["d_weight"] = r.d_weight;
    return now ? r.loss : r.nll.view(target.sizes());
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grad) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &weight = saved[1], &target = saved[2];
    const std::vector<int64_t> c = ctx->saved_data["call"].toIntVector();
    const LossCall call{c[0], c[1], ctx->saved_data["z"].toDouble(), c[2], c[3], c[4]};
    variable_list out(9);
    {
      const at::AutoGradMode no_grad(false);
      const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
      no_tangent(grad[0], "the gradient of the loss");
      const Tensor factor = plain(grad[0].to(at::kFloat));
      Tensor dh, dw;
      const int64_t now = static_cast<int64_t>(capture_id(On(hidden).stream()));
      const auto made = ctx->saved_data.find("capture");
      const int64_t then = made == ctx->saved_data.end() ? 0 : made->second.toInt();
      auto take = [&](const char* name, bool want, Tensor& to) {
        auto it = ctx->saved_data.find(name);
        if (it == ctx->saved_data.end() || (then == 0 && now != 0)) return;
        if (want) to = now == then ? it->second.toTensor() : it->second.toTensor().clone();
        if (now == then) ctx->saved_data.erase(it);
      };
      take("d_hidden", want_hidden, dh);
      take("d_weight", want_weight, dw);
      if (want_hidden != dh.defined() || want_weight != dw.defined()) {
        const bool rows = call.reduction == REDUCE_NONE;
        LossResult r = loss_pass(as_bf16(hidden.reshape({-1, hidden.size(-1)})), as_bf16(weight), target, call, rows ? factor.view(-1) : Tensor(),
                                 want_hidden, want_weight, weight.scalar_type() == at::kFloat);
        dh = r.d_hidden;
        dw = r.d_weight;
      }
      if (call.reduction != REDUCE_NONE) scale_gradients(dh, dw, factor);
      if (dh.defined()) out[0] = dh.view(hidden.sizes()).to(hidden.scalar_type());
      if (dw.defined()) out[1] = dw.to(weight.scalar_type());
    }
    return once(std::move(out));
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t ignore_index, int64_t reduction, double z,
                            int64_t piece_rows, int64_t status, int64_t status_host) {
  not_traced("linear_cross_entropy");
  no_tangent(hidden, "hidden");
  no_tangent(weight, "weight");
  const py::gil_scoped_release released;
  const Tensor t = plain(target);
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad())) {
    capturable({&hidden, &weight});
    return LinearCrossEntropy::apply(hidden, weight, t, ignore_index, reduction, z, piece_rows, status, status_host);
  }
  const LossCall call{ignore_index, reduction, z, piece_rows, status, status_host};
  LossResult r = loss_pass(as_bf16(hidden.reshape({-1, hidden.size(-1)})), as_bf16(weight), t, call, Tensor(), false, false, false);
  return reduction != REDUCE_NONE ? r.loss : r.nll.view(t.sizes());
}

// A contiguous tensor beside `like`, from the allocator itself: through the dispatcher it takes 0.5 us more, which a call of a few us
// has several of.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// ---- RMS norm -------------------------------------------------------------------------------------------------

struct RmsCall {
  double eps = 0.0, offset = 0.0;
  bool e4m3 = false;
};

struct RmsResult {
  Tensor y, y_scale, h, rstd;
};

// rows as they lie, or copied where 8-bit outputs ask for 16-byte boundaries that they are not on
Rows as_rows_for(const Tensor& t, bool on_16) {
  Rows r = as_rows(t);
  if (on_16 && (reinterpret_cast<uintptr_t>(r.x.data_ptr()) % 16 != 0 || r.stride * static_cast<int64_t>(t.element_size()) % 16 != 0)) {
    r.x = r.x.clone(at::MemoryFormat::Contiguous);
    r.stride = t.size(-1);
  }
  return r;
}

RmsResult rms_forward_of(const Tensor& x, const Tensor& weight, const Tensor& residual, const RmsCall& call, bool stats) {
  on_gpu(x, "x");
  if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error("x must have a last dimension to normalise, got " + c10::str(x.sizes()));
  if (x.size(-1) > std::numeric_limits<int>::max()) throw py::value_error("x has rows of " + std::to_string(x.size(-1)) + " values");
  if (!(call.eps >= 0.0)) throw py::value_error("eps must not be negative, got " + std::to_string(call.eps));
  if (!(std::abs(call.offset) <= std::numeric_limits<float>::max())) throw py::value_error("weight_offset must be finite, got " + std::to_string(call.offset));
  ffm_rms_norm_args a = {};
  a.x_type = element_type(x, "x");
  check_vector(weight, x, "weight");
  if (residual.defined()) {
    same_device(residual, x, "residual");
    if (residual.sizes() != x.sizes()) throw py::value_error("residual must be " + c10::str(x.sizes()) + ", got " + c10::str(residual.sizes()));
    if (residual.scalar_type() != x.scalar_type()) {
      throw py::type_error(std::string("residual must be of x's type, got ") + c10::toString(residual.scalar_type()) + " and " + c10::toString(x.scalar_type()));
    }
  }
  const int64_t D = x.size(-1);
  if (call.e4m3 && D % 16 != 0) throw py::value_error("an 8-bit output has rows of a multiple of 16 values, got " + std::to_string(D));
  const On device(x);
  const Rows r = as_rows_for(x, call.e4m3);
  Rows more;
  Tensor w = weight.defined() ? plain(weight) : Tensor();
  if (call.e4m3 && w.defined() && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 != 0) w = w.clone();
  RmsResult out;
  if (residual.defined()) {
    more = as_rows_for(residual, call.e4m3);
    out.h = fresh(x.sizes(), x.scalar_type(), x);
  }
  if (call.e4m3) {
    std::vector<int64_t> sizes = x.sizes().vec();
    out.y = fresh(sizes, at::kFloat8_e4m3fn, x);
    sizes.back() = (D + 127) / 128;
    out.y_scale = fresh(sizes, at::kFloat, x);
  } else {
    out.y = fresh(x.sizes(), x.scalar_type(), x);
  }
  if (stats) out.rstd = fresh({r.rows}, at::kFloat, x);
  a.rows = r.rows;
  a.D = D;
  a.x_stride = r.stride;
  a.eps = call.eps;
  a.offset = call.offset;
  a.x = r.x.data_ptr();
  if (residual.defined()) {
    a.residual = more.x.data_ptr();
    a.residual_stride = more.stride;
    a.h = out.h.data_ptr();
  }
  a.weight = address(w);
  a.w_type = w.defined() ? element_type(w, "weight") : 0;
  a.y = out.y.data_ptr();
  a.y_scale = static_cast<float*>(address(out.y_scale));
  a.rstd = static_cast<float*>(address(out.rstd));
  check(rms_forward(&a, device.stream()), "ffm_rms_norm_forward");
  launches += r.rows > 0;
  return out;
}

struct RmsGradients {
  Tensor dx, dweight;
};

RmsGradients rms_backward_of(const Tensor& dy, const Tensor& dh, const Tensor& h, const Tensor& weight, const Tensor& rstd, const RmsCall& call,
                             bool want_x, bool want_weight) {
  const On device(h);
  on_gpu(h, "x");
  ffm_rms_norm_args a = {};
  a.x_type = element_type(h, "x");
  const int64_t D = h.size(-1);
  const Rows r = as_rows(h);
  // saved-tensor hooks may have handed back other tensors than were saved
  if (rstd.numel() != r.rows || rstd.scalar_type() != at::kFloat || rstd.device() != h.device()) throw py::value_error("saved statistics do not belong to x");
  check_vector(weight, h, "weight");
  const Tensor s = plain(rstd), w = weight.defined() ? plain(weight) : Tensor();
  auto gradient = [&](const Tensor& t, const char* name) {
    if (!t.defined()) return Tensor();
    const Tensor g = plain(t.scalar_type() == h.scalar_type() ? t : t.to(h.scalar_type()));
    same_device(g, h, name);
    if (g.sizes() != h.sizes()) throw py::value_error(std::string(name) + " has another shape than x");
    return g;
  };
  Tensor g = gradient(dy, "the gradient of y");
  const Tensor m = gradient(dh, "the gradient of the sum");
  RmsGradients out;
  if (!g.defined()) {  // only the sum was used
    if (want_x && m.defined()) out.dx = m;
    if (want_weight) out.dweight = at::zeros_like(w);
    return out;
  }
  Tensor workspace;
  if (want_x) out.dx = fresh(h.sizes(), h.scalar_type(), h);
  if (want_weight) {
    out.dweight = fresh({D}, w.scalar_type(), w);
    a.workspace_bytes = static_cast<int64_t>(rms_workspace(r.rows, static_cast<int>(D), static_cast<int>(a.x_type)));
    workspace = fresh({a.workspace_bytes}, at::kByte, h);
    a.workspace = workspace.data_ptr();
  }
  a.rows = r.rows;
  a.D = D;
  a.x_stride = r.stride;
  a.eps = call.eps;
  a.offset = call.offset;
  a.x = r.x.data_ptr();
  a.weight = address(w);
  a.w_type = w.defined() ? element_type(w, "weight") : 0;
  a.rstd = s.data_ptr<float>();
  a.dy = g.data_ptr();
  a.dh = address(m);
  a.dx = address(out.dx);
  a.dweight = address(out.dweight);
  check(rms_backward(&a, device.stream()), "ffm_rms_norm_backward");
  launches += want_weight ? 2 : want_x && r.rows > 0;
  return out;
}

class RmsNorm : public torch::autograd::Function<RmsNorm> {
 public:
  static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight_or_none, const OptTensor& residual_or_none,
                               double eps, double offset) {
    const Tensor weight = weight_or_none.value_or(Tensor()), residual = residual_or_none.value_or(Tensor());
    RmsResult r = rms_forward_of(x, weight, residual, {eps, offset, false}, true);
    ctx->save_for_backward({residual.defined() ? r.h : x, weight, r.rstd});
    ctx->saved_data["residual"] = residual.defined();
    ctx->saved_data["call"] = std::vector<double>{eps, offset};
    ctx->set_materialize_grads(false);
    return residual.defined() ? variable_list{r.y, r.h} : variable_list{r.y};
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grad) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(5);
    {
      const at::AutoGradMode no_grad(false);
      // an operand that is not there has no edge, and those after it move up
      const bool weight = saved[1].defined(), residual = ctx->saved_data["residual"].toBool();
      const std::vector<double> call = ctx->saved_data["call"].toDoubleVector();
      const bool want_x = ctx->needs_input_grad(0), want_residual = residual && ctx->needs_input_grad(weight ? 2 : 1);
      RmsGradients g = rms_backward_of(grad[0], residual ? grad[1] : Tensor(), saved[0], saved[1], saved[2], {call[0], call[1], false},
                                       want_x || want_residual, weight && ctx->needs_input_grad(1));
      if (want_x) out[0] = g.dx;
      out[1] = g.dweight;
      if (want_residual) out[2] = g.dx;
    }
    return once(std::move(out));
  }
};

py::object rms_norm(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual, double offset, bool e4m3) {
  not_traced("rms_norm");
  const Tensor w = weight.value_or(Tensor()), more = residual.value_or(Tensor());
  no_tangent(x, "x");
  no_tangent(w, "weight");
  no_tangent(more, "residual");
  const bool grads = at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (more.defined() && more.requires_grad()));
  if (grads && e4m3) throw std::runtime_error("an 8-bit output is not differentiable: call under torch.no_grad()");
  RmsResult r;
  {
    const py::gil_scoped_release released;
    if (grads) {
      capturable({&x, &w, &more});
      const variable_list out = RmsNorm::apply(x, weight, residual, eps, offset);
      r.y = out[0];
      if (more.defined()) r.h = out[1];
    } else {
      r = rms_forward_of(x, w, more, {eps, offset, e4m3}, false);
    }
  }
  if (e4m3) return more.defined() ? py::object(py::make_tuple(r.y, r.y_scale, r.h)) : py::object(py::make_tuple(r.y, r.y_scale));
  return more.defined() ? py::object(py::make_tuple(r.y, r.h)) : py::cast(r.y);
}

// ---- 8-bit operands with a scale for every 128 values -----------------------------------------------------------

void no_gradient(const Tensor& t, const char* name, const char* what) {
  no_tangent(t, name);
  if (at::GradMode::is_enabled() && t.requires_grad()) {
    throw std::runtime_error(std::string(what) + " is not differentiable, and " + name + " requires a gradient: call under torch.no_grad()");
  }
}

py::tuple quantize_e4m3(const Tensor& x, int64_t block_rows) {
  not_traced("quantize_e4m3");
  no_gradient(x, "x", "quantize_e4m3");
  on_gpu(x, "x");
  if (block_rows != 1 && block_rows != 128) throw py::value_error("block_rows must be 1 or 128, got " + std::to_string(block_rows));
  if (x.dim() < (block_rows == 1 ? 1 : 2)) throw py::value_error("x must have rows" + std::string(block_rows == 1 ? "" : " and columns") + ", got " + c10::str(x.sizes()));
  const int type = element_type(x, "x");
  const int64_t K = x.size(-1);
  if (K < 1 || K % 16 != 0 || K > std::numeric_limits<int>::max()) throw py::value_error("rows must have a multiple of 16 values, got " + std::to_string(K));
  const int64_t rows = block_rows == 1 ? x.numel() / K : x.size(-2), matrices = block_rows == 1 ? 1 : (rows > 0 ? x.numel() / K / rows : 0);
  Tensor q, scale;
  {
    const py::gil_scoped_release released;
    const On device(x);
    Rows r;
    if (block_rows == 1) {
      r = as_rows_for(x, true);
    } else {
      r.x = plain(x);
      if (reinterpret_cast<uintptr_t>(r.x.data_ptr()) % 16 != 0) r.x = r.x.clone();
      r.stride = K;
    }
    std::vector<int64_t> sizes = x.sizes().vec();
    q = fresh(sizes, at::kFloat8_e4m3fn, x);
    sizes.back() = (K + 127) / 128;
    if (block_rows > 1) sizes[sizes.size() - 2] = (rows + 127) / 128;
    scale = fresh(sizes, at::kFloat, x);
    check(quantize_blocks(r.x.data_ptr(), type, matrices, rows, r.stride, static_cast<int>(K), static_cast<int>(block_rows), q.data_ptr(),
                          scale.data_ptr<float>(), device.stream()),
          "ffm_quantize_blocks_e4m3");
    launches += matrices > 0 && rows > 0;
  }
  return py::make_tuple(q, scale);
}

void check_scale(const Tensor& scale, const Tensor& of, std::vector<int64_t> sizes, const char* name) {
  same_device(scale, of, name);
  no_gradient(scale, name, "linear_e4m3");
  if (scale.scalar_type() != at::kFloat) throw py::type_error(std::string(name) + " must be float32, got " + c10::toString(scale.scalar_type()));
  if (scale.sizes() != at::IntArrayRef(sizes)) throw py::value_error(std::string(name) + " must be " + c10::str(at::IntArrayRef(sizes)) + ", got " + c10::str(scale.sizes()));
}

Tensor linear_e4m3(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale, const OptTensor& ends_or_none,
                   at::ScalarType out_type, int64_t status, int64_t status_host) {
  not_traced("linear_e4m3");
  on_gpu(x, "x");
  same_device(weight, x, "weight");
  for (const auto& [t, name] : {std::pair<const Tensor*, const char*>{&x, "x"}, {&weight, "weight"}}) {
    no_gradient(*t, name, "linear_e4m3");
    if (t->scalar_type() != at::kFloat8_e4m3fn) throw py::type_error(std::string(name) + " must be float8_e4m3fn, got " + c10::toString(t->scalar_type()));
  }
  const bool grouped = ends_or_none.has_value();
  if (weight.dim() != (grouped ? 3 : 2)) throw py::value_error(std::string("weight must be ") + (grouped ? "[experts, N, K]" : "[N, K]") + ", got " + c10::str(weight.sizes()));
  const int64_t K = weight.size(-1), N = weight.size(-2), experts = grouped ? weight.size(0) : 1;
  if (x.dim() < 1 || x.size(-1) != K) throw py::value_error("x must end in " + std::to_string(K) + ", got " + c10::str(x.sizes()));
  if (grouped && x.dim() != 2) throw py::value_error("x must be [rows, K] where rows belong to experts, got " + c10::str(x.sizes()));
  if (K < 1 || K % 16 != 0 || N < 1) throw py::value_error("K must be a multiple of 16 and N positive, got " + c10::str(weight.sizes()));
  if (experts < 1 || experts > 1024) throw py::value_error("there are 1 to 1024 experts, got " + std::to_string(experts));
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = (K + 127) / 128;
  check_scale(x_scale, x, sizes, "x_scale");
  std::vector<int64_t> w_sizes = weight.sizes().vec();
  w_sizes.back() = (K + 127) / 128;
  w_sizes[w_sizes.size() - 2] = (N + 127) / 128;
  check_scale(weight_scale, x, w_sizes, "weight_scale");
  Tensor ends;
  if (grouped) {
    ends = *ends_or_none;
    same_device(ends, x, "ends");
    if (ends.scalar_type() != at::kInt) throw py::type_error(std::string("ends must be int32, got ") + c10::toString(ends.scalar_type()));
    if (ends.dim() != 1 || ends.size(0) != experts) throw py::value_error("ends must be [" + std::to_string(experts) + "], got " + c10::str(ends.sizes()));
  }
  if (out_type != at::kBFloat16 && out_type != at::kHalf && out_type != at::kFloat) {
    throw py::type_error(std::string("out_dtype must be bfloat16, float16 or float32, got ") + c10::toString(out_type));
  }
  const py::gil_scoped_release released;
  const On device(x);
  const Rows r = as_rows_for(x, true);
  const Tensor xs = plain(x_scale), ws = plain(weight_scale);
  Tensor w = plain(weight);
  if (reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 != 0) w = w.clone();
  if (grouped) ends = ends.contiguous();
  sizes.back() = N;
  const Tensor out = fresh(sizes, out_type, x);
  ffm_linear_blocks_args a = {};
  a.rows = r.rows;
  a.N = N;
  a.K = K;
  a.experts = experts;
  a.x_stride = r.stride;
  a.out_type = element_type(out, "out");
  a.x = r.x.data_ptr();
  a.x_scale = xs.data_ptr<float>();
  a.w = w.data_ptr();
  a.w_scale = ws.data_ptr<float>();
  a.ends = grouped ? ends.data_ptr<int32_t>() : nullptr;
  a.out = out.data_ptr();
  a.status = reinterpret_cast<int32_t*>(status);
  a.status_host = reinterpret_cast<int32_t*>(status_host);
  check(linear_blocks(&a, device.stream()), "ffm_linear_blocks_e4m3");
  launches += r.rows > 0;
  return out;
}

// ---- AdamW --------------------------------------------------------------------------------------------------

// A zero word per device and stream that the kernel leaves zero: calls on one stream follow one another. A captured call gets
// one of its own, zeroed in the graph: replays of two graphs may overlap.
Tensor ticket_for(const Tensor& like, const void* stream, bool capturing) {
  const auto options = like.options().dtype(at::kInt).requires_grad(false);
  if (capturing) return at::zeros({1}, options);
  static std::mutex mutex;
  static std::unordered_map<std::string, Tensor>* kept = new std::unordered_map<std::string, Tensor>();  // never destroyed: outlives CUDA
  const std::string key = std::to_string(like.device().index()) + ":" + std::to_string(reinterpret_cast<uintptr_t>(stream));
  const std::lock_guard<std::mutex> lock(mutex);
  Tensor& t = (*kept)[key];
  if (!t.defined()) t = at::zeros({1}, options);
  return t;
}

using Tensors = std::vector<Tensor>;

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
                   const Tensors& steps, const std::optional<Tensors>& masters, const std::optional<Tensors>& exp_avg_scales,
                   const std::optional<Tensors>& exp_avg_sq_scales, const py::object& lr, double beta1, double beta2, double eps,
                   double weight_decay, const OptTensor& grad_scale, int64_t seed, bool capturing) {
  not_traced("adamw_step");
  const size_t n = params.size();
  const bool eight = exp_avg_scales.has_value();
  auto length = [n](size_t other, const char* name) {
    if (other != n) throw py::value_error(std::string(name) + " must have one tensor for each parameter: " + std::to_string(other) + " for " + std::to_string(n));
  };
  length(grads.size(), "grads");
  length(exp_avgs.size(), "exp_avgs");
  length(exp_avg_sqs.size(), "exp_avg_sqs");
  length(steps.size(), "steps");
  if (masters.has_value()) length(masters->size(), "masters");
  if (eight != exp_avg_sq_scales.has_value()) throw py::value_error("8-bit states have scales for both moments");
  if (eight) {
    length(exp_avg_scales->size(), "exp_avg_scales");
    length(exp_avg_sq_scales->size(), "exp_avg_sq_scales");
  }
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) throw py::value_error("betas must be in [0, 1)");
  if (!(eps >= 0.0)) throw py::value_error("eps must not be negative");
  if (!(weight_decay >= 0.0)) throw py::value_error("weight_decay must not be negative");
  if (n == 0) return;

  const Tensor& first = params[0];
  on_gpu(first, "param");
  ffm_adamw_args h = {};
  Tensor lr_device;
  if (THPVariable_Check(lr.ptr())) {
    const Tensor t = lr.cast<Tensor>();
    if (t.numel() != 1) throw py::value_error("lr must be a number or a tensor of one element");
    if (t.is_cuda()) {
      same_device(t, first, "lr");
      if (t.scalar_type() != at::kFloat) throw py::type_error("lr on the device must be float32");
      lr_device = t.resolve_neg();
      h.lr_device = lr_device.data_ptr<float>();
    } else {
      h.lr = t.item<double>();
    }
  } else {
    h.lr = lr.cast<double>();
  }
  if (h.lr_device == nullptr && !(h.lr >= 0.0)) throw py::value_error("lr must not be negative");
  h.beta1 = beta1;
  h.beta2 = beta2;
  h.eps = eps;
  h.weight_decay = weight_decay;
  h.bits = eight ? 8 : 32;
  h.seed = seed;
  Tensor scale;
  if (grad_scale.has_value()) {
    same_device(*grad_scale, first, "grad_scale");
    if (grad_scale->numel() != 1 || grad_scale->scalar_type() != at::kFloat) throw py::type_error("grad_scale must be one float32 value");
    scale = grad_scale->resolve_neg();
    h.grad_scale = scale.data_ptr<float>();
  }

  // written in place: one after the other in memory, no negation pending, and no two on the same memory, nor on a gradient's
  struct Range {
    const char *from, *to;
    const char* name;
    bool written;
  };
  std::vector<Range> ranges;
  ranges.reserve(n * 8 + 2);
  auto range = [&](const Tensor& t, const char* name, bool written) {
    const char* from = static_cast<const char*>(t.data_ptr());
    if (t.numel() > 0) ranges.push_back({from, from + t.numel() * t.element_size(), name, written});
  };
  auto state = [&](const Tensor& t, int64_t elements, const char* name) {
    same_device(t, first, name);
    if (!t.is_contiguous() || t.is_neg()) throw py::value_error(std::string(name) + " must be contiguous");
    if (t.numel() != elements) throw py::value_error(std::string(name) + " must have " + std::to_string(elements) + " elements, got " + std::to_string(t.numel()));
    range(t, name, true);
    return t.data_ptr();
  };
  std::vector<ffm_adamw_tensor> table(n);
  std::vector<Tensor> held;
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    ffm_adamw_tensor& a = table[i];
    const int64_t elements = p.numel();
    a.elements = elements;
    a.param = state(p, elements, "param");
    a.param_type = element_type(p, "param");
    Tensor g = grads[i];
    same_device(g, first, "grad");
    if (g.sizes() != p.sizes()) throw py::value_error("grad must have its parameter's shape: " + c10::str(g.sizes()) + " for " + c10::str(p.sizes()));
    a.grad_type = element_type(g, "grad");
    if (!g.is_contiguous() || g.is_neg()) {
      g = plain(g);
      held.push_back(g);
    }
    a.grad = g.data_ptr();
    range(g, "grad", false);
    if (eight) {
      for (const Tensor* t : {&exp_avgs[i], &exp_avg_sqs[i]}) {
        if (t->scalar_type() != at::kFloat8_e4m3fn) throw py::type_error("8-bit states must be float8_e4m3fn, got " + std::string(c10::toString(t->scalar_type())));
      }
      const int64_t blocks = (elements + 127) / 128;
      for (const Tensor* t : {&(*exp_avg_scales)[i], &(*exp_avg_sq_scales)[i]}) {
        if (t->scalar_type() != at::kByte) throw py::type_error("scales of 8-bit states must be uint8, got " + std::string(c10::toString(t->scalar_type())));
      }
      a.exp_avg_scale = state((*exp_avg_scales)[i], blocks, "exp_avg_scale");
      a.exp_avg_sq_scale = state((*exp_avg_sq_scales)[i], blocks, "exp_avg_sq_scale");
    } else {
      for (const Tensor* t : {&exp_avgs[i], &exp_avg_sqs[i]}) {
        if (t->scalar_type() != at::kFloat) throw py::type_error("states must be float32 (or float8_e4m3fn with scales), got " + std::string(c10::toString(t->scalar_type())));
      }
    }
    a.exp_avg = state(exp_avgs[i], elements, "exp_avg");
    a.exp_avg_sq = state(exp_avg_sqs[i], elements, "exp_avg_sq");
    if (masters.has_value()) {
      if ((*masters)[i].scalar_type() != at::kFloat) throw py::type_error("masters must be float32");
      a.master = state((*masters)[i], elements, "master");
    }
    if (steps[i].scalar_type() != at::kInt) throw py::type_error("steps must be int32, got " + std::string(c10::toString(steps[i].scalar_type())));
    a.step = static_cast<int32_t*>(state(steps[i], 1, "step"));
  }

  if (lr_device.defined()) range(lr_device, "lr", false);
  if (scale.defined()) range(scale, "grad_scale", false);
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  // what was written or read so far, up to its furthest end
  const char *written_to = nullptr, *read_to = nullptr;
  for (const Range& r : ranges) {
    if (r.from < written_to || (r.written && r.from < read_to)) {
      throw py::value_error(std::string(r.name) + " appears twice in one call, or lies on another of its tensors");
    }
    (r.written ? written_to : read_to) = std::max(r.written ? written_to : read_to, r.to);
  }

  const On device(first);
  const ffm_stream_t stream = device.stream();
  const Tensor ticket = ticket_for(first, stream, capturing);
  h.ticket = ticket.data_ptr();
  int64_t launched = 0;
  h.launched = &launched;
  int rc;
  {
    py::gil_scoped_release released;
    rc = adamw(table.data(), static_cast<int>(n), &h, stream);
  }
  check(rc, "ffm_adamw_step");
  // what was read before (a saved operand, a cast or quantised copy) is not current any more
  auto changed = [](const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (const Tensors* list : {&params, &exp_avgs, &exp_avg_sqs, &steps}) {
    for (const Tensor& t : *list) changed(t);
  }
  for (const std::optional<Tensors>* list : {&masters, &exp_avg_scales, &exp_avg_sq_scales}) {
    if (list->has_value()) {
      for (const Tensor& t : **list) changed(t);
    }
  }
  launches += launched;
}

// ---- gradient norm ----------------------------------------------------------------------------------------------

// One after the other in memory in some order of the dimensions, each value once: then any pass over the memory is one over the tensor.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense() && !t.is_neg(); }

struct ClipTable {
  std::vector<ffm_clip_tensor> entries;
  std::vector<Tensor> held;

  void add(const Tensor& t, const Tensor& like, const char* name) {
    same_device(t, like, name);
    ffm_clip_tensor e = {};
    e.type = element_type(t, name);
    held.push_back(dense(t) ? t : t.contiguous().resolve_neg());
    e.x = held.back().data_ptr();
    e.elements = t.numel();
    if (e.elements > 0) entries.push_back(e);
  }
  int count() const {
    if (entries.size() > static_cast<size_t>(std::numeric_limits<int>::max())) throw py::value_error("too many tensors");
    return static_cast<int>(entries.size());
  }
};

struct ClipNorm {
  Tensor norm, coefficient, workspace;  // the workspace begins with the sum of squares (the magnitude), float64
};

// The norm of `grads` and of what `other` (float64 [1], a sum of squares or a magnitude) stands for
ClipNorm norm_of(const ClipTable& table, const Tensor& like, const On& device, double max_norm, bool largest, const Tensor& other) {
  ffm_grad_norm_args a = {};
  a.kind = largest ? 1 : 0;
  a.max_norm = max_norm;
  a.other = static_cast<const double*>(address(other));
  ClipNorm out;
  out.norm = fresh({}, at::kFloat, like);
  out.coefficient = fresh({}, at::kFloat, like);
  const int64_t doubles = static_cast<int64_t>(grad_norm_workspace(table.count())) / 8;
  out.workspace = fresh({1 + doubles}, at::kDouble, like);
  a.total = out.workspace.data_ptr<double>();
  a.norm = out.norm.data_ptr<float>();
  a.coefficient = out.coefficient.data_ptr<float>();
  a.workspace = a.total + 1;
  a.workspace_bytes = doubles * 8;
  const Tensor ticket = ticket_for(like, device.stream(), capture_id(device.stream()) != 0);
  a.ticket = ticket.data_ptr();
  int64_t launched = 0;
  a.launched = &launched;
  check(grad_norm(table.entries.data(), table.count(), &a, device.stream()), "ffm_grad_norm");
  launches += launched;
  return out;
}

void check_norm(const Tensors& grads, const Tensor& like, double max_norm) {
  not_traced("gradient clipping");
  on_gpu(like, "grad");
  if (!(max_norm >= 0.0)) throw py::value_error("max_norm must not be negative, got " + std::to_string(max_norm));
  for (const Tensor& t : grads) on_gpu(t, "grad");
}

// (float64 [n] that begins with the total, norm, coefficient)
py::tuple gradient_norm(const Tensors& grads, const Tensor& like, double max_norm, bool largest, const OptTensor& other) {
  check_norm(grads, like, max_norm);
  const On device(like);
  ClipTable table;
  for (const Tensor& t : grads) table.add(t, like, "grad");
  Tensor more;
  if (other.has_value()) {
    same_device(*other, like, "other");
    if (other->numel() != 1 || other->scalar_type() != at::kDouble) throw py::type_error("other must be one float64 value");
    more = other->resolve_neg();
  }
  const ClipNorm r = norm_of(table, like, device, max_norm, largest, more);
  return py::make_tuple(r.workspace, r.norm, r.coefficient);
}

// grads *= factor (one float32 on the device), in place
void scale_by(const Tensors& grads, const ClipTable& table, const Tensor& factor, const On& device) {
  int64_t launched = 0;
  check(scale_tensors(table.entries.data(), table.count(), factor.data_ptr<float>(), &launched, device.stream()), "ffm_scale_tensors");
  launches += launched;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& t = grads[i];
    if (!table.held[i].is_same(t)) {
      const at::NoGradGuard no_grad;
      t.copy_(table.held[i]);  // it lies in a way that the kernel does not take
    } else if (!t.is_inference()) {
      t.unsafeGetTensorImpl()->bump_version();
    }
  }
}

// Refuses tensors of which one, or two of which, share memory: scaling in place would multiply twice. What does not lie dense is scaled as a copy, made
// before anything is, and so only once.
void check_separate(const Tensors& grads) {
  std::vector<std::pair<const char*, const char*>> ranges;
  for (const Tensor& t : grads) {
    if (t.numel() == 0) continue;
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) > 1 && t.stride(d) == 0) throw py::value_error("a gradient that was expanded cannot be scaled in place");
    }
    if (!dense(t)) continue;
    const char* from = static_cast<const char*>(t.data_ptr());
    ranges.emplace_back(from, from + t.numel() * t.element_size());
  }
  std::sort(ranges.begin(), ranges.end());
  const char* end = nullptr;
  for (const auto& r : ranges) {
    if (r.first < end) throw py::value_error("a gradient appears twice in one call, or lies on another");
    end = std::max(end, r.second);
  }
}

void scale_gradients_by(const Tensors& grads, const Tensor& factor) {
  not_traced("gradient clipping");
  on_gpu(factor, "factor");
  if (factor.numel() != 1 || factor.scalar_type() != at::kFloat) throw py::type_error("factor must be one float32 value");
  check_separate(grads);
  const On device(factor);
  ClipTable table;
  for (const Tensor& t : grads) table.add(t, factor, "grad");
  scale_by(grads, table, factor, device);
}

// The gradients of `parameters` scaled in place to a norm of max_norm at most: their norm, or nothing where there is no gradient
OptTensor clip_grad_norm(const Tensors& parameters, double max_norm, bool largest) {
  Tensors grads;
  grads.reserve(parameters.size());
  for (const Tensor& p : parameters) {
    if (p.grad().defined()) grads.push_back(p.grad());
  }
  if (grads.empty()) return std::nullopt;
  check_norm(grads, grads[0], max_norm);
  check_separate(grads);
  const On device(grads[0]);
  ClipTable table;
  for (const Tensor& t : grads) table.add(t, grads[0], "grad");
  const ClipNorm r = norm_of(table, grads[0], device, max_norm, largest, Tensor());
  scale_by(grads, table, r.coefficient, device);
  return r.norm;
}

}  // namespace

void define_ops(py::module_& m) {
  m.def("bind_ops", &bind_ops);
  m.def("launches", [] { return launches.load(); });
  m.def("layer_norm", &layer_norm);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("adamw_step", &adamw_step);
  m.def("rms_norm", &rms_norm);
  m.def("quantize_e4m3", &quantize_e4m3);
  m.def("linear_e4m3", [](const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale, const OptTensor& ends,
                          const py::object& out_type, int64_t status, int64_t status_host) {
    return linear_e4m3(x, x_scale, weight, weight_scale, ends, torch::python::detail::py_object_to_dtype(out_type), status, status_host);
  });
  m.def("gradient_norm", &gradient_norm);
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("scale_gradients", &scale_gradients_by);
}
