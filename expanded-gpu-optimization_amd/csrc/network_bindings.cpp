// fused_hoad._C: the torch-facing boundary of the operators of fused_hoad_networks.h. Each call
// validates its tensors, makes non-contiguous ones contiguous, allocates outputs and workspace with
// the torch caching allocator, and enqueues on the current stream of the inputs' device. No host
// synchronization.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>
#include <vector>

#include "fused_hoad_networks.h"

namespace {

using torch::Tensor;
using OptionalTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_status(int status) {
  TORCH_CHECK(status == FHOAD_SUCCESS, "fused_hoad kernel error (", fhoad_status_string(status),
              "): ", fhoad_net_last_error());
}

void* current_stream(const Tensor& tensor) {
  return static_cast<void*>(at::hip::getCurrentHIPStreamMasqueradingAsCUDA(tensor.get_device()).stream());
}

int dtype_of(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, what,
              " must use float32 or bfloat16");
  return t.scalar_type() == torch::kFloat32 ? FHOAD_FLOAT32 : FHOAD_BFLOAT16;
}

void check_like(const Tensor& t, const Tensor& other, const char* what, const char* of) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == other.scalar_type(), what, " must have ", of, "'s dtype");
  TORCH_CHECK(t.device() == other.device(), what, " must be on ", of, "'s device");
}

void check_vector(const OptionalTensor& t, int64_t size, const Tensor& other, const char* what,
                  const char* of) {
  if (!t.has_value()) return;
  check_like(*t, other, what, of);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == size, what, " must have shape [", size, "]");
}

const void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* writable(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor contiguous(const OptionalTensor& t) { return t.has_value() ? t->contiguous() : Tensor(); }

Tensor workspace_for(size_t bytes, const Tensor& like) {
  return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

// The kernels' gradients carry no graph of their own: asking for one has to be an error, not zero
// second derivatives.
void check_once(const char* what) {
  TORCH_CHECK(!torch::GradMode::is_enabled(), what,
              " is differentiable once: create_graph=True is not supported");
}

// Forward-mode automatic differentiation has to be an error as well: the kernels read a dual tensor's
// values alone, and what they write would carry no tangent, a derivative of zero to what follows.
void check_no_tangent(std::initializer_list<const Tensor*> tensors, const char* what) {
  for (const Tensor* t : tensors) {
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                " has no forward-mode derivative: a dual tensor is not supported");
  }
}

// A trace would hold the allocations of a call and not its kernels, and replay uninitialised memory.
void check_not_traced(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be recorded by torch.jit.trace");
}

const Tensor* maybe(const OptionalTensor& t) { return t.has_value() ? &*t : nullptr; }

// ---- gated linear -------------------------------------------------------------------------------

int activation_of(const std::string& name) {
  if (name == "silu") return FHOAD_SILU;
  if (name == "tanh") return FHOAD_TANH;
  if (name == "gelu") return FHOAD_GELU;
  if (name == "sigmoid") return FHOAD_SIGMOID;
  TORCH_CHECK(false, "activation must be 'silu', 'tanh', 'gelu' or 'sigmoid', got '", name, "'");
}

std::vector<int64_t> with_last(c10::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> shape(sizes.begin(), sizes.end());
  shape.back() = last;
  return shape;
}

// The forward; with a context it saves what the backward reads.
struct GatedLinear : public torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate_weight,
                        const Tensor& up_weight, const OptionalTensor& gate_bias,
                        const OptionalTensor& up_bias, int64_t activation) {
    const bool save = ctx != nullptr;
    const int dtype = dtype_of(x, "x");
    const int64_t width = x.size(-1), hidden = gate_weight.size(0);
    const int64_t rows = x.numel() / width;
    const c10::DeviceGuard device_guard(x.device());
    const Tensor xc = x.contiguous(), gw = gate_weight.contiguous(), uw = up_weight.contiguous();
    const Tensor gb = contiguous(gate_bias), ub = contiguous(up_bias);
    Tensor h = torch::empty(with_last(x.sizes(), hidden), xc.options());
    Tensor pre;
    if (save) {
      pre = torch::empty({static_cast<int64_t>(fhoad_gated_linear_saved_size(rows, hidden) / sizeof(float))},
                         xc.options().dtype(torch::kFloat32));
    }
    const size_t bytes = fhoad_gated_linear_forward_workspace_size(rows, width, hidden, dtype);
    const Tensor workspace = bytes ? workspace_for(bytes, xc) : Tensor();
    check_status(fhoad_gated_linear_forward(
        pointer(xc), pointer(gw), pointer(uw), pointer(gb), pointer(ub), writable(h),
        rows == 0 || !save ? nullptr : pre.data_ptr<float>(), writable(workspace), bytes, rows, width, hidden,
        static_cast<int>(activation), dtype, current_stream(xc)));
    if (save) {
      ctx->save_for_backward({xc, gw, uw, pre});
      ctx->saved_data["activation"] = activation;
      ctx->saved_data["gate_bias"] = gate_bias.has_value();
      ctx->saved_data["up_bias"] = up_bias.has_value();
    }
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gated_linear");
    variable_list result(6);
    if (!grads[0].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate_weight = saved[1], &up_weight = saved[2], &pre = saved[3];
    const int64_t width = x.size(-1), hidden = gate_weight.size(0), rows = x.numel() / width;
    const int dtype = dtype_of(x, "x");
    const c10::DeviceGuard device_guard(x.device());
    const Tensor grad = grads[0].contiguous();
    // Differentiable inputs, in order: x, the two weights, and the biases that are there.
    const bool has_gate_bias = ctx->saved_data["gate_bias"].toBool(), has_up_bias = ctx->saved_data["up_bias"].toBool();
    const bool weights = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dx, dgw, duw, dgb, dub;
    if (ctx->needs_input_grad(0)) dx = torch::empty_like(x);
    if (weights) {
      dgw = torch::empty_like(gate_weight);
      duw = torch::empty_like(up_weight);
    }
    if (has_gate_bias && ctx->needs_input_grad(3)) dgb = torch::empty({hidden}, x.options());
    if (has_up_bias && ctx->needs_input_grad(has_gate_bias ? 4 : 3)) dub = torch::empty({hidden}, x.options());
    const size_t bytes = fhoad_gated_linear_backward_workspace_size(rows, width, hidden, dtype);
    const Tensor workspace = workspace_for(bytes, x);
    check_status(fhoad_gated_linear_backward(
        pointer(x), pointer(gate_weight), pointer(up_weight), static_cast<const float*>(pointer(pre)),
        pointer(grad), writable(dx), writable(dgw), writable(duw), writable(dgb), writable(dub),
        workspace.data_ptr(), bytes, rows, width, hidden,
        static_cast<int>(ctx->saved_data["activation"].toInt()), dtype, current_stream(x)));
    result[0] = dx;
    if (ctx->needs_input_grad(1)) result[1] = dgw;
    if (ctx->needs_input_grad(2)) result[2] = duw;
    result[3] = dgb;
    result[4] = dub;
    return result;
  }
};

bool needs_grad(std::initializer_list<const Tensor*> tensors) {
  if (!torch::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors) {
    if (t && t->defined() && t->requires_grad()) return true;
  }
  return false;
}

Tensor gated_linear(const Tensor& x, const Tensor& gate_weight, const Tensor& up_weight,
                    const OptionalTensor& gate_bias, const OptionalTensor& up_bias,
                    const std::string& activation) {
  check_not_traced("gated_linear");
  const int64_t kind = activation_of(activation);
  dtype_of(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have shape [..., width] with width > 0");
  check_like(gate_weight, x, "gate_weight", "x");
  check_like(up_weight, x, "up_weight", "x");
  TORCH_CHECK(gate_weight.dim() == 2 && gate_weight.size(0) > 0 && gate_weight.size(1) == x.size(-1),
              "gate_weight must have shape [hidden, ", x.size(-1), "] with hidden > 0");
  TORCH_CHECK(up_weight.sizes() == gate_weight.sizes(), "up_weight must have gate_weight's shape");
  check_vector(gate_bias, gate_weight.size(0), x, "gate_bias", "x");
  check_vector(up_bias, gate_weight.size(0), x, "up_bias", "x");
  check_no_tangent({&x, &gate_weight, &up_weight, maybe(gate_bias), maybe(up_bias)}, "gated_linear");
  const bool save = needs_grad({&x, &gate_weight, &up_weight, maybe(gate_bias), maybe(up_bias)});
  if (!save) return GatedLinear::forward(nullptr, x, gate_weight, up_weight, gate_bias, up_bias, kind);
  return GatedLinear::apply(x, gate_weight, up_weight, gate_bias, up_bias, kind);
}

// ---- residual norm ------------------------------------------------------------------------------

int norm_of(const std::string& name) {
  if (name == "rms") return FHOAD_RMS_NORM;
  if (name == "layer") return FHOAD_LAYER_NORM;
  TORCH_CHECK(false, "kind must be 'rms' or 'layer', got '", name, "'");
}

// Rows of x that share a gate row: the gate's shape is x's up to some dimension, and one from
// there to the last.
int64_t rows_per_gate(const Tensor& x, const Tensor& gate) {
  TORCH_CHECK(gate.dim() >= 1 && gate.dim() <= x.dim() && gate.size(-1) == x.size(-1),
              "gate must broadcast to residual's shape and have its width");
  int64_t shared = 1;
  bool sharing = true;  // from the last row dimension to the first
  for (int64_t back = 2; back <= x.dim(); ++back) {
    const int64_t extent = x.size(-back), own = back <= gate.dim() ? gate.size(-back) : 1;
    TORCH_CHECK(own == extent || own == 1, "gate must broadcast to residual's shape");
    if (extent == 1) continue;
    if (own == extent) {
      sharing = false;
    } else {
      TORCH_CHECK(sharing, "gate must have residual's first dimensions and be shared over the others");
      shared *= extent;
    }
  }
  return shared;
}

// As GatedLinear.
struct ResidualNorm : public torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const OptionalTensor& block,
                               const OptionalTensor& gate, const Tensor& weight, const OptionalTensor& bias,
                               const OptionalTensor& post_weight, const OptionalTensor& post_bias,
                               double scale, int64_t kind, double eps) {
    const bool save = ctx != nullptr;
    const int dtype = dtype_of(residual, "residual");
    const int64_t width = residual.size(-1), rows = residual.numel() / width;
    const int64_t shared = gate.has_value() && rows > 0 ? rows_per_gate(residual, *gate) : 1;
    const c10::DeviceGuard device_guard(residual.device());
    const Tensor r = residual.contiguous(), b = contiguous(block), g = contiguous(gate);
    const Tensor w = weight.contiguous(), wb = contiguous(bias);
    const Tensor pw = contiguous(post_weight), pb = contiguous(post_bias);
    Tensor hidden, statistics;
    if (block.has_value()) hidden = torch::empty_like(r);
    Tensor normed = torch::empty_like(r);
    if (save) statistics = torch::empty({rows, 4}, r.options().dtype(torch::kFloat32));
    if (rows > 0) {
      check_status(fhoad_residual_norm_forward(
          pointer(r), pointer(b), pointer(g), pointer(w), pointer(wb), pointer(pw), pointer(pb),
          writable(hidden), writable(normed), static_cast<float*>(writable(statistics)), rows, width, shared,
          static_cast<int>(kind), dtype, scale, eps, current_stream(r)));
    }
    if (save) {
      ctx->save_for_backward({r, b, g, w, pw, pb, statistics});
      ctx->set_materialize_grads(false);
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["kind"] = kind;
      ctx->saved_data["shared"] = shared;
      ctx->saved_data["bias"] = bias.has_value();
    }
    if (!block.has_value()) return {normed};
    return {hidden, normed};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("residual_norm");
    variable_list result(10);
    bool any = false;
    for (const Tensor& g : grads) any |= g.defined();
    if (!any) return result;
    const auto saved = ctx->get_saved_variables();
    const Tensor &r = saved[0], &b = saved[1], &g = saved[2], &w = saved[3], &pw = saved[4], &pb = saved[5];
    const Tensor& statistics = saved[6];
    const int64_t width = r.size(-1), rows = r.numel() / width, shared = ctx->saved_data["shared"].toInt();
    const int dtype = dtype_of(r, "residual");
    const c10::DeviceGuard device_guard(r.device());
    const Tensor grad_hidden = b.defined() && grads[0].defined() ? grads[0].contiguous() : Tensor();
    const Tensor& last = grads[b.defined() ? 1 : 0];
    const Tensor grad_normed = last.defined() ? last.contiguous() : Tensor();
    // Differentiable inputs in order, those that are there.
    const bool there[] = {true, b.defined(), g.defined(), true, ctx->saved_data["bias"].toBool(), pw.defined(), pb.defined()};
    const Tensor like[] = {r, b, g, w, w, pw, pb};
    Tensor out[7];
    size_t input = 0;
    for (int k = 0; k < 7; ++k) {
      if (!there[k]) continue;
      if (ctx->needs_input_grad(input++)) out[k] = rows == 0 ? torch::zeros_like(like[k]) : torch::empty_like(like[k]);
    }
    if (rows > 0) {
      const size_t bytes = fhoad_residual_norm_backward_workspace_size(rows, width, g.defined() ? shared : rows);
      const Tensor workspace = workspace_for(bytes, r);
      check_status(fhoad_residual_norm_backward(
          pointer(r), pointer(b), pointer(g), pointer(w), pointer(pw), pointer(pb),
          statistics.data_ptr<float>(), pointer(grad_hidden), pointer(grad_normed), writable(out[0]),
          writable(out[1]), writable(out[2]), writable(out[3]), writable(out[4]), writable(out[5]),
          writable(out[6]), workspace.data_ptr(), bytes, rows, width, shared,
          static_cast<int>(ctx->saved_data["kind"].toInt()), dtype, ctx->saved_data["scale"].toDouble(),
          current_stream(r)));
    }
    for (int k = 0; k < 7; ++k) result[k] = out[k];
    return result;
  }
};

variable_list residual_norm(const Tensor& residual, const OptionalTensor& block, const OptionalTensor& gate,
                            const Tensor& weight, const OptionalTensor& bias, const OptionalTensor& post_weight,
                            const OptionalTensor& post_bias, double residual_scale, const std::string& kind,
                            double eps) {
  check_not_traced("residual_norm");
  const int64_t norm = norm_of(kind);
  dtype_of(residual, "residual");
  TORCH_CHECK(residual.dim() >= 1 && residual.size(-1) > 0, "residual must have shape [..., width] with width > 0");
  const int64_t width = residual.size(-1);
  TORCH_CHECK(width <= FHOAD_NORM_MAX_WIDTH, "width must be at most ", FHOAD_NORM_MAX_WIDTH);
  TORCH_CHECK(eps >= 0.0, "eps must be non-negative");
  check_vector(weight, width, residual, "weight", "residual");
  check_vector(bias, width, residual, "bias", "residual");
  check_vector(post_weight, width, residual, "post_weight", "residual");
  check_vector(post_bias, width, residual, "post_bias", "residual");
  if (block.has_value()) {
    check_like(*block, residual, "block", "residual");
    TORCH_CHECK(block->sizes() == residual.sizes(), "block must have residual's shape");
  } else {
    TORCH_CHECK(!gate.has_value() && !post_weight.has_value() && !post_bias.has_value() && residual_scale == 1.0,
                "gate, post_weight, post_bias and residual_scale need a block");
  }
  TORCH_CHECK(!post_bias.has_value() || post_weight.has_value(), "post_bias needs post_weight");
  if (gate.has_value()) {
    check_like(*gate, residual, "gate", "residual");
    rows_per_gate(residual, *gate);
  }
  check_no_tangent({&residual, maybe(block), maybe(gate), &weight, maybe(bias), maybe(post_weight), maybe(post_bias)},
                   "residual_norm");
  const bool save = needs_grad({&residual, maybe(block), maybe(gate), &weight, maybe(bias), maybe(post_weight),
                                maybe(post_bias)});
  variable_list out =
      save ? ResidualNorm::apply(residual, block, gate, weight, bias, post_weight, post_bias, residual_scale, norm, eps)
           : ResidualNorm::forward(nullptr, residual, block, gate, weight, bias, post_weight, post_bias,
                                   residual_scale, norm, eps);
  if (!block.has_value()) return {residual, out[0]};
  return out;
}

// ---- AdamW --------------------------------------------------------------------------------------

int64_t span_of(int64_t numel) { return (numel + FHOAD_ADAMW_BLOCK - 1) / FHOAD_ADAMW_BLOCK * FHOAD_ADAMW_BLOCK; }

void check_state(const Tensor& t, torch::ScalarType type, int64_t size, const Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.scalar_type() == type, what, " must be a contiguous ",
              c10::toString(type), " CUDA tensor");
  TORCH_CHECK(t.numel() == size, what, " must have ", size, " values");
  TORCH_CHECK(t.device() == like.device(), what, " must be on the parameters' device");
}

void adamw_step(const std::vector<Tensor>& parameters, const std::vector<OptionalTensor>& gradients,
                const Tensor& exp_avg, const Tensor& exp_avg_sq, const Tensor& steps, double lr, double beta1,
                double beta2, double eps, double weight_decay, const OptionalTensor& exp_avg_scale,
                const OptionalTensor& exp_avg_sq_scale, int64_t seed) {
  check_not_traced("adamw_step");
  TORCH_CHECK(parameters.size() == gradients.size(), "parameters and gradients must be as many");
  TORCH_CHECK(lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0, "lr, eps and weight_decay must be non-negative");
  TORCH_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "the betas must lie in [0, 1)");
  TORCH_CHECK(seed >= 0 && seed <= 0xffffffffll, "seed must fit 32 bits");
  TORCH_CHECK(exp_avg_scale.has_value() == exp_avg_sq_scale.has_value(), "the scales come together");
  if (parameters.empty()) return;
  const bool eight = exp_avg_scale.has_value();
  std::vector<fhoad_adamw_tensor> tensors[2];
  std::vector<Tensor> copies;  // of gradients that are not contiguous, until the launch
  int64_t offset = 0;
  for (size_t k = 0; k < parameters.size(); ++k) {
    const Tensor& p = parameters[k];
    const int dtype = dtype_of(p, "parameters");
    TORCH_CHECK(p.is_contiguous(), "parameters must be contiguous (parameter ", k, ")");
    TORCH_CHECK(p.device() == parameters[0].device(), "parameters must be on one device");
    check_no_tangent({&p, maybe(gradients[k])}, "adamw_step");
    const int64_t numel = p.numel();
    if (gradients[k].has_value()) {
      const Tensor& g = *gradients[k];
      check_like(g, p, "a gradient", "its parameter");
      TORCH_CHECK(g.layout() == torch::kStrided && g.sizes() == p.sizes(),
                  "a gradient must be dense and have its parameter's shape (parameter ", k, ")");
      const void* from = g.is_contiguous() ? g.data_ptr() : copies.emplace_back(g.contiguous()).data_ptr();
      tensors[dtype].push_back({p.data_ptr(), from, numel, offset, static_cast<int64_t>(k)});
    }
    offset += span_of(numel);
  }
  const Tensor& first = parameters[0];
  const torch::ScalarType type = eight ? torch::kUInt8 : torch::kFloat32;
  check_state(exp_avg, type, offset, first, "exp_avg");
  check_state(exp_avg_sq, type, offset, first, "exp_avg_sq");
  check_state(steps, torch::kInt32, static_cast<int64_t>(parameters.size()), first, "steps");
  if (eight) {
    check_state(*exp_avg_scale, torch::kFloat32, offset / FHOAD_ADAMW_BLOCK, first, "exp_avg_scale");
    check_state(*exp_avg_sq_scale, torch::kFloat32, offset / FHOAD_ADAMW_BLOCK, first, "exp_avg_sq_scale");
  }
  const c10::DeviceGuard device_guard(first.device());
  for (int dtype : {FHOAD_FLOAT32, FHOAD_BFLOAT16}) {
    const auto& some = tensors[dtype];
    if (some.empty()) continue;
    const size_t bytes = fhoad_adamw_workspace_size(static_cast<int64_t>(some.size()));
    const Tensor workspace = workspace_for(bytes, first);
    check_status(fhoad_adamw_step(some.data(), static_cast<int64_t>(some.size()), dtype, eight ? 8 : 32,
                                  exp_avg.data_ptr(), exp_avg_sq.data_ptr(),
                                  eight ? exp_avg_scale->data_ptr<float>() : nullptr,
                                  eight ? exp_avg_sq_scale->data_ptr<float>() : nullptr, steps.data_ptr<int32_t>(),
                                  workspace.data_ptr(), bytes, lr, beta1, beta2, eps, weight_decay,
                                  static_cast<uint32_t>(seed), current_stream(first)));
  }
  // In-place updates that autograd's check of saved tensors has to see.
  for (size_t k = 0; k < parameters.size(); ++k) {
    if (gradients[k].has_value()) parameters[k].unsafeGetTensorImpl()->bump_version();
  }
  for (const Tensor* t : {&exp_avg, &exp_avg_sq, &steps, maybe(exp_avg_scale), maybe(exp_avg_sq_scale)}) {
    if (t) t->unsafeGetTensorImpl()->bump_version();
  }
}

std::vector<Tensor> decode_moments(const Tensor& exp_avg, const Tensor& exp_avg_sq, const Tensor& exp_avg_scale,
                                   const Tensor& exp_avg_sq_scale) {
  check_not_traced("decode_moments");
  const int64_t count = exp_avg.numel();
  TORCH_CHECK(count % FHOAD_ADAMW_BLOCK == 0, "packed states hold a multiple of ", FHOAD_ADAMW_BLOCK, " values");
  check_state(exp_avg, torch::kUInt8, count, exp_avg, "exp_avg");
  check_state(exp_avg_sq, torch::kUInt8, count, exp_avg, "exp_avg_sq");
  check_state(exp_avg_scale, torch::kFloat32, count / FHOAD_ADAMW_BLOCK, exp_avg, "exp_avg_scale");
  check_state(exp_avg_sq_scale, torch::kFloat32, count / FHOAD_ADAMW_BLOCK, exp_avg, "exp_avg_sq_scale");
  const c10::DeviceGuard device_guard(exp_avg.device());
  const auto options = exp_avg.options().dtype(torch::kFloat32);
  std::vector<Tensor> out{torch::empty({count}, options), torch::empty({count}, options)};
  check_status(fhoad_adamw_decode(exp_avg.data_ptr<uint8_t>(), exp_avg_scale.data_ptr<float>(),
                                  out[0].data_ptr<float>(), count, 0, current_stream(exp_avg)));
  check_status(fhoad_adamw_decode(exp_avg_sq.data_ptr<uint8_t>(), exp_avg_sq_scale.data_ptr<float>(),
                                  out[1].data_ptr<float>(), count, 1, current_stream(exp_avg)));
  return out;
}

// Whether the members of `lists` and then the values of the dicts in `entries` are the very objects of
// `seen`, in order. An optimizer asks this each step: 108 tensors and their state take 10 us in Python.
bool same_objects(const pybind11::list& lists, const pybind11::dict& entries, const pybind11::list& seen) {
  const Py_ssize_t count = PyList_GET_SIZE(seen.ptr());
  Py_ssize_t at = 0;
  for (const pybind11::handle list : lists) {
    if (!PyList_Check(list.ptr())) return false;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(list.ptr()); ++k, ++at) {
      if (at == count || PyList_GET_ITEM(list.ptr(), k) != PyList_GET_ITEM(seen.ptr(), at)) return false;
    }
  }
  PyObject *key, *entry, *value;
  for (Py_ssize_t outer = 0; PyDict_Next(entries.ptr(), &outer, &key, &entry);) {
    if (!PyDict_Check(entry)) return false;
    for (Py_ssize_t inner = 0; PyDict_Next(entry, &inner, &key, &value); ++at) {
      if (at == count || value != PyList_GET_ITEM(seen.ptr(), at)) return false;
    }
  }
  return at == count;
}

}  // namespace

void register_network_operators(pybind11::module_& module) {
  namespace py = pybind11;
  module.def("gated_linear", &gated_linear,
             "activation(x Wg^T + bg) * (x Wu^T + bu), differentiable (MI355X HIP kernels)", py::arg("x"),
             py::arg("gate_weight"), py::arg("up_weight"), py::arg("gate_bias") = py::none(),
             py::arg("up_bias") = py::none(), py::arg("activation") = "silu");
  module.def("residual_norm", &residual_norm,
             "(hidden, normed) of a scaled residual, a gated block and the norms around it, differentiable "
             "(MI355X HIP kernels)",
             py::arg("residual"), py::arg("block"), py::arg("gate"), py::arg("weight"), py::arg("bias"),
             py::arg("post_weight"), py::arg("post_bias"), py::arg("residual_scale"), py::arg("kind"),
             py::arg("eps"));
  module.def("adamw_step", &adamw_step, "One AdamW step over many tensors, in place (MI355X HIP kernels)",
             py::arg("parameters"), py::arg("gradients"), py::arg("exp_avg"), py::arg("exp_avg_sq"),
             py::arg("steps"), py::arg("lr"), py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
             py::arg("weight_decay"), py::arg("exp_avg_scale"), py::arg("exp_avg_sq_scale"), py::arg("seed"));
  module.def("decode_moments", &decode_moments, "Values of packed 8-bit AdamW moments (MI355X HIP kernel)",
             py::arg("exp_avg"), py::arg("exp_avg_sq"), py::arg("exp_avg_scale"), py::arg("exp_avg_sq_scale"));
  module.def("same_objects", &same_objects, "Whether lists and then dicts' values hold exactly these objects",
             py::arg("lists"), py::arg("entries"), py::arg("seen"));
  module.attr("ADAMW_BLOCK") = FHOAD_ADAMW_BLOCK;
}
