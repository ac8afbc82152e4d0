// The operators beside the layer for torch tensors: argument checks, outputs, scratch and the call into libffmoe. A call from
// Python costs these few checks; the torch operations that they would be there (views, contiguity, empty) take longer than
// the kernels of a small call.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

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

}  // namespace

void define_ops(py::module_& m) {
  m.def("bind_ops", &bind_ops);
  m.def("launches", [] { return launches.load(); });
  m.def("layer_norm", &layer_norm);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("adamw_step", &adamw_step);
}
