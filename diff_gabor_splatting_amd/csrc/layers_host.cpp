// Host side of the surfel decoder's layers (include/gabor_layers.h): checks
// of arguments, allocation, launches on the current stream, and first-order
// autograd, in C++ because a layer over a few rows is mostly host time.
//
// Rows may have any stride as long as their features are contiguous and the
// leading dimensions collapse into one; other inputs are copied first.

#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "gabor_layers.h"
#include "host.hpp"

namespace gs_host {
namespace {

struct Api {
  decltype(&gs_last_error) last_error = nullptr;
  decltype(&gs_checkpoint8_write) checkpoint_write = nullptr;
  decltype(&gs_checkpoint8_read) checkpoint_read = nullptr;
  decltype(&gs_activation_forward) activation_forward = nullptr;
  decltype(&gs_activation_backward) activation_backward = nullptr;
  decltype(&gs_layer_norm_forward) layer_norm_forward = nullptr;
  decltype(&gs_layer_norm_backward_workspace_size) layer_norm_workspace = nullptr;
  decltype(&gs_layer_norm_backward) layer_norm_backward = nullptr;
  decltype(&gs_linear_forward) linear_forward = nullptr;
  decltype(&gs_linear_backward_input) linear_backward_input = nullptr;
  decltype(&gs_linear_backward_weight_workspace_size) linear_workspace = nullptr;
  decltype(&gs_linear_backward_weight) linear_backward_weight = nullptr;
};

Api api;

void check(int status) {
  if (status == 0) return;
  const char* message = api.last_error ? api.last_error() : nullptr;
  if (message && *message) fail(message);
  fail("gabor HIP call failed with status " + std::to_string(status));
}

constexpr int64_t kGroup = 32;

// What is kept of an input: bytes and exponents (empty where nothing is).
struct Kept {
  at::Tensor values, exponents;

  static Kept empty(int64_t rows, int64_t features, const at::Device& device) {
    const int64_t groups = (features + kGroup - 1) / kGroup;
    return {at::empty({rows, groups * kGroup}, on(device, at::kChar)),
            at::empty({rows, groups}, on(device, at::kByte))};
  }
};

int32_t type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GS_FLOAT32;
    case at::kBFloat16: return GS_BFLOAT16;
    case at::kHalf: return GS_FLOAT16;
    default: return -1;
  }
}

void check_input(const at::Tensor& x) {
  if (!x.is_cuda() || type_of(x) < 0)
    throw py::value_error("x must be float32, bfloat16 or float16 on a HIP device");
  if (x.dim() < 1 || x.size(-1) < 1)
    throw py::value_error("x must have a last dimension of at least one feature");
}

// `t`, which has a default of none, of shape `shape` beside x.
void check_parameter(const char* name, const at::Tensor& t, c10::IntArrayRef shape,
                     const at::Tensor& x, bool or_float) {
  if (!t.defined()) return;
  if (t.device() != x.device())
    throw py::value_error(std::string(name) + " must be on the device of x");
  if (t.scalar_type() != x.scalar_type() && !(or_float && t.scalar_type() == at::kFloat))
    throw py::value_error(std::string(name) + (or_float ? " must have the type of x or float32"
                                                        : " must have the type of x"));
  if (!t.sizes().equals(shape)) {
    std::string text = std::string(name) + " must have shape (";
    for (size_t i = 0; i < shape.size(); ++i) text += (i ? ", " : "") + std::to_string(shape[i]);
    throw py::value_error(text + (shape.size() == 1 ? ",)" : ")"));
  }
}

// The values themselves where `t` is a view that negates them lazily (what
// torch.imag gives of a conjugate): the kernels read memory as it is.
at::Tensor in_memory(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A parameter as the kernels read it.
at::Tensor dense(const at::Tensor& t) { return t.defined() ? in_memory(t).contiguous() : t; }

// A tensor as rows of its last dimension.
struct RowsOf {
  at::Tensor held;  // keeps a copy alive, where one was made
  int64_t rows, features, stride;

  explicit RowsOf(const at::Tensor& t) : held(in_memory(t)) {
    features = t.size(-1);
    rows = t.numel() / features;
    if (!collapses(held)) held = held.contiguous();
    const int64_t last = t.dim() - 2;
    stride = rows > 1 && held.dim() >= 2 ? row_stride(held, last) : features;
  }
  const void* data() const { return held.data_ptr(); }

 private:
  // The stride between rows: that of the innermost leading dimension of
  // more than one entry.
  static int64_t row_stride(const at::Tensor& t, int64_t last) {
    for (int64_t i = last; i >= 0; --i)
      if (t.size(i) > 1) return t.stride(i);
    return t.size(-1);
  }
  static bool collapses(const at::Tensor& t) {
    if (t.numel() == 0) return true;
    const int64_t features = t.size(-1);
    if (features > 1 && t.stride(-1) != 1) return false;
    int64_t expected = -1;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      if (t.size(i) == 1) continue;
      if (expected < 0) {
        if (t.stride(i) < features) return false;
      } else if (t.stride(i) != expected) {
        return false;
      }
      expected = t.stride(i) * t.size(i);
    }
    return true;
  }
};

const void* data_of(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// First derivatives only: with create_graph, gradients of the gradients
// raise when they are asked for.
torch::autograd::variable_list once(torch::autograd::variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<size_t> at;
  torch::autograd::variable_list given;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      at.push_back(i);
      given.push_back(grads[i].detach().requires_grad_());
    }
  if (given.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once", int64_t(given.size()));
  given = (*error)(std::move(given));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = given[i];
  return grads;
}

// The kernels write into tensors that torch sees as empty, so what follows
// its operators and not these calls would get that for a result: a tracer
// (torch.jit.trace; make_fx and torch.export, whose mode is PROXY or the
// pre-dispatch key) would record the allocation alone, and forward mode would
// find no tangent. Both are refused, in the backward pass too.
void check_calls(const char* name, std::initializer_list<const at::Tensor*> inputs) {
  using c10::impl::TorchDispatchModeTLS;
  if (at::tracer::impl::is_dispatch_enabled() ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
      TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    fail(std::string(name) + " cannot be traced");
  for (const at::Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      fail(std::string(name) + " has no forward-mode derivative");
}

bool grad_wanted(std::initializer_list<const at::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// --------------------------------------------------------------------------
// Checkpoints

std::vector<at::Tensor> checkpoint8_write(const at::Tensor& x) {
  check_calls("quantize", {&x});
  check_input(x);
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  Kept kept = Kept::empty(r.rows, r.features, x.device());
  check(api.checkpoint_write(type_of(x), r.data(), r.stride, r.rows, r.features,
                             kept.values.data_ptr(), kept.exponents.data_ptr(),
                             stream_of(x.device())));
  return {kept.values, kept.exponents};
}

at::Tensor checkpoint8_read(const at::Tensor& values, const at::Tensor& exponents,
                            std::vector<int64_t> shape, at::ScalarType type) {
  check_calls("dequantize", {});
  if (shape.empty() || shape.back() < 1) throw py::value_error("invalid checkpoint shape");
  const int64_t features = shape.back(), groups = (features + kGroup - 1) / kGroup;
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
  if (!(values.is_cuda() && exponents.device() == values.device() &&
        values.scalar_type() == at::kChar && exponents.scalar_type() == at::kByte &&
        values.is_contiguous() && exponents.is_contiguous() && values.dim() == 2 &&
        exponents.dim() == 2 && rows >= 0 && values.size(0) == rows &&
        exponents.size(0) == rows && values.size(1) == groups * kGroup &&
        exponents.size(1) == groups))
    throw py::value_error("values and exponents do not hold a checkpoint of that shape");
  const c10::DeviceGuard guard(values.device());
  at::Tensor out = at::empty(shape, on(values.device(), type));
  if (type_of(out) < 0)
    throw py::value_error("a checkpoint reads back as float32, bfloat16 or float16");
  check(api.checkpoint_read(type_of(out), values.data_ptr(), exponents.data_ptr(), rows, features,
                            out.data_ptr(), stream_of(values.device())));
  return out;
}

// --------------------------------------------------------------------------
// Activations

at::Tensor activation_rows(const at::Tensor& x, int64_t kind, double omega, Kept* kept) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (kept) *kept = Kept::empty(r.rows, r.features, x.device());
  check(api.activation_forward(type_of(x), int32_t(kind), float(omega), r.data(), r.stride,
                               r.rows, r.features, y.data_ptr(),
                               kept ? kept->values.data_ptr() : nullptr,
                               kept ? kept->exponents.data_ptr() : nullptr,
                               stream_of(x.device())));
  return y;
}

struct Activation : torch::autograd::Function<Activation> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            int64_t kind, double omega) {
    Kept kept;
    at::Tensor y = activation_rows(x, kind, omega, &kept);
    ctx->save_for_backward({kept.values, kept.exponents});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["omega"] = omega;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("activation", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const c10::DeviceGuard guard(grads[0].device());
    const RowsOf g(grads[0]);
    at::Tensor dx = at::empty(grads[0].sizes(), grads[0].options());
    check(api.activation_backward(type_of(dx), int32_t(ctx->saved_data["kind"].toInt()),
                                  float(ctx->saved_data["omega"].toDouble()), g.data(), g.stride,
                                  saved[0].data_ptr(), saved[1].data_ptr(), g.rows, g.features,
                                  dx.data_ptr(), stream_of(dx.device())));
    return once({dx, at::Tensor(), at::Tensor()}, "activation");
  }
};

at::Tensor activation(const at::Tensor& x, int64_t kind, double omega) {
  check_calls("activation", {&x});
  check_input(x);
  if (!grad_wanted({&x})) return activation_rows(x, kind, omega, nullptr);
  return Activation::apply(x, kind, omega);
}

// --------------------------------------------------------------------------
// Layer norm

at::Tensor norm_rows(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
                     double eps, at::Tensor* statistics, Kept* kept) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  const at::Tensor w = dense(weight), b = dense(bias);
  const int32_t parameters =
      w.defined() ? type_of(w) : b.defined() ? type_of(b) : type_of(x);
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (statistics) *statistics = at::empty({r.rows, 2}, on(x.device(), at::kFloat));
  if (kept) *kept = Kept::empty(r.rows, r.features, x.device());
  check(api.layer_norm_forward(type_of(x), parameters, r.data(), r.stride, data_of(w), data_of(b),
                               float(eps), r.rows, r.features, y.data_ptr(),
                               statistics ? statistics->data_ptr() : nullptr,
                               kept ? kept->values.data_ptr() : nullptr,
                               kept ? kept->exponents.data_ptr() : nullptr,
                               stream_of(x.device())));
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const std::optional<at::Tensor>& weight,
                            const std::optional<at::Tensor>& bias, double eps, bool eight) {
    at::Tensor statistics;
    Kept kept;
    at::Tensor y = norm_rows(x, weight.value_or(at::Tensor()), bias.value_or(at::Tensor()), eps,
                             &statistics, eight ? &kept : nullptr);
    ctx->save_for_backward({eight ? at::Tensor() : x, weight.value_or(at::Tensor()), statistics,
                            kept.values, kept.exponents});
    const at::Tensor parameter = weight ? *weight : bias ? *bias : x;
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["type"] = int64_t(parameter.scalar_type());
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("layer_norm", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const bool has_weight = ctx->saved_data["weight"].toBool();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const auto type = at::ScalarType(ctx->saved_data["type"].toInt());
    const at::Tensor& grad = grads[0];
    const c10::DeviceGuard guard(grad.device());
    const RowsOf g(grad);
    at::Tensor x = saved[0], w, dx, dw, db, space;
    int64_t stride = g.features;
    std::optional<RowsOf> rows;
    if (x.defined()) {
      rows.emplace(x);
      stride = rows->stride;
    }
    if (has_weight) w = dense(saved[1]);
    dx = at::empty(grad.sizes(), grad.options());
    if (has_weight && ctx->needs_input_grad(1))
      dw = at::empty({g.features}, on(grad.device(), type));
    if (has_bias && ctx->needs_input_grad(has_weight ? 2 : 1))
      db = at::empty({g.features}, on(grad.device(), type));
    const int32_t parameters = type == at::kFloat ? GS_FLOAT32 : type_of(grad);
    if (dw.defined() || db.defined())
      space = workspace(api.layer_norm_workspace(g.rows, g.features), grad.device());
    check(api.layer_norm_backward(
        type_of(grad), parameters, g.data(), g.stride, rows ? rows->data() : nullptr, stride,
        data_of(saved[3]), data_of(saved[4]), saved[2].data_ptr(), data_of(w), g.rows, g.features,
        dx.data_ptr(), const_cast<void*>(data_of(dw)), const_cast<void*>(data_of(db)),
        const_cast<void*>(data_of(space)), space.defined() ? size_t(space.numel()) : 0,
        stream_of(grad.device())));
    return once({dx, dw, db, at::Tensor(), at::Tensor()}, "layer_norm");
  }
};

at::Tensor layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                      const std::optional<at::Tensor>& bias, double eps, bool eight) {
  const at::Tensor w = weight.value_or(at::Tensor()), b = bias.value_or(at::Tensor());
  check_calls("layer_norm", {&x, &w, &b});
  check_input(x);
  check_parameter("weight", w, {x.size(-1)}, x, true);
  check_parameter("bias", b, {x.size(-1)}, x, true);
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    throw py::value_error("weight and bias must have one type");
  if (!grad_wanted({&x, &w, &b})) return norm_rows(x, w, b, eps, nullptr, nullptr);
  return LayerNorm::apply(x, weight, bias, eps, eight);
}

// --------------------------------------------------------------------------
// Linear layers

at::Tensor linear_rows(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
                       Kept* kept) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  const at::Tensor w = dense(weight), b = dense(bias);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.size(0);
  at::Tensor y = at::empty(shape, x.options());
  if (kept) *kept = Kept::empty(r.rows, r.features, x.device());
  check(api.linear_forward(type_of(x), r.data(), r.stride, w.data_ptr(), data_of(b), r.rows,
                           r.features, w.size(0), y.data_ptr(),
                           kept ? kept->values.data_ptr() : nullptr,
                           kept ? kept->exponents.data_ptr() : nullptr, stream_of(x.device())));
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& weight, const std::optional<at::Tensor>& bias) {
    const bool keep = weight.requires_grad() || (bias && bias->requires_grad());
    Kept kept;
    at::Tensor y = linear_rows(x, weight, bias.value_or(at::Tensor()), keep ? &kept : nullptr);
    ctx->save_for_backward({weight, kept.values, kept.exponents});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("linear", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const at::Tensor& grad = grads[0];
    const c10::DeviceGuard guard(grad.device());
    const RowsOf g(grad);
    const at::Tensor w = dense(saved[0]);
    const int64_t outputs = w.size(0), features = w.size(1);
    const int32_t type = type_of(grad);
    void* const stream = stream_of(grad.device());
    at::Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) {
      dx = at::empty(ctx->saved_data["shape"].toIntVector(), grad.options());
      check(api.linear_backward_input(type, g.data(), g.stride, w.data_ptr(), g.rows, features,
                                      outputs, dx.data_ptr(), stream));
    }
    if (ctx->needs_input_grad(1)) dw = at::empty_like(w);
    if (has_bias && ctx->needs_input_grad(2)) db = at::empty({outputs}, grad.options());
    if (dw.defined() || db.defined()) {
      const at::Tensor space =
          workspace(api.linear_workspace(type, g.rows, features, outputs), grad.device());
      check(api.linear_backward_weight(
          type, g.data(), g.stride, data_of(saved[1]), data_of(saved[2]), g.rows, features,
          outputs, const_cast<void*>(data_of(dw)), const_cast<void*>(data_of(db)),
          space.data_ptr(), size_t(space.numel()), stream));
    }
    return once({dx, dw, db}, "linear");
  }
};

at::Tensor linear(const at::Tensor& x, const at::Tensor& weight,
                  const std::optional<at::Tensor>& bias) {
  const at::Tensor b = bias.value_or(at::Tensor());
  check_calls("linear", {&x, &weight, &b});
  check_input(x);
  if (weight.dim() != 2 || weight.size(0) < 1)
    throw py::value_error("weight must have shape (outputs, features)");
  check_parameter("weight", weight, {weight.size(0), x.size(-1)}, x, false);
  check_parameter("bias", b, {weight.size(0)}, x, false);
  if (!grad_wanted({&x, &weight, &b})) return linear_rows(x, weight, b, nullptr);
  return Linear::apply(x, weight, bias);
}

}  // namespace

void bind_layers(const py::dict& table) {
  Api next;
  take(table, "gs_last_error", next.last_error);
  take(table, "gs_checkpoint8_write", next.checkpoint_write);
  take(table, "gs_checkpoint8_read", next.checkpoint_read);
  take(table, "gs_activation_forward", next.activation_forward);
  take(table, "gs_activation_backward", next.activation_backward);
  take(table, "gs_layer_norm_forward", next.layer_norm_forward);
  take(table, "gs_layer_norm_backward_workspace_size", next.layer_norm_workspace);
  take(table, "gs_layer_norm_backward", next.layer_norm_backward);
  take(table, "gs_linear_forward", next.linear_forward);
  take(table, "gs_linear_backward_input", next.linear_backward_input);
  take(table, "gs_linear_backward_weight_workspace_size", next.linear_workspace);
  take(table, "gs_linear_backward_weight", next.linear_backward_weight);
  api = next;
}

std::vector<std::string> layer_entry_points() {
  return {"gs_checkpoint8_write", "gs_checkpoint8_read", "gs_activation_forward",
          "gs_activation_backward", "gs_layer_norm_forward",
          "gs_layer_norm_backward_workspace_size", "gs_layer_norm_backward", "gs_linear_forward",
          "gs_linear_backward_input", "gs_linear_backward_weight_workspace_size",
          "gs_linear_backward_weight"};
}

void define_layers(py::module_& m) {
  m.def("checkpoint8_write", &checkpoint8_write, py::arg("x"));
  m.def("checkpoint8_read", [](const at::Tensor& values, const at::Tensor& exponents,
                               std::vector<int64_t> shape, const py::object& type) {
    return checkpoint8_read(values, exponents, std::move(shape),
                            torch::python::detail::py_object_to_dtype(type));
  });
  m.def("activation", &activation, py::arg("x"), py::arg("kind"), py::arg("omega"));
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"),
        py::arg("eps"), py::arg("eight"));
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"));
}

}  // namespace gs_host
