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
  decltype(&gs_dropout) dropout = nullptr;
  decltype(&gs_row_groups_workspace_size) row_groups_workspace = nullptr;
  decltype(&gs_row_groups) row_groups = nullptr;
  decltype(&gs_grouped_linear_forward) grouped_forward = nullptr;
  decltype(&gs_grouped_linear_backward_input) grouped_backward_input = nullptr;
  decltype(&gs_grouped_linear_backward_weight_workspace_size) grouped_workspace = nullptr;
  decltype(&gs_grouped_linear_backward_weight) grouped_backward_weight = nullptr;
  decltype(&gs_adapted_linear_inner_size) adapted_inner = nullptr;
  decltype(&gs_adapted_linear_forward) adapted_forward = nullptr;
  decltype(&gs_adapted_linear_backward_input) adapted_backward_input = nullptr;
  decltype(&gs_adapted_linear_backward_adapters_workspace_size) adapted_workspace = nullptr;
  decltype(&gs_adapted_linear_backward_adapters) adapted_backward_adapters = nullptr;
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
    Kept kept;  // the bias's gradient takes none
    at::Tensor y = linear_rows(x, weight, bias.value_or(at::Tensor()),
                               weight.requires_grad() ? &kept : nullptr);
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

// --------------------------------------------------------------------------
// Dropout

at::Tensor masked(const at::Tensor& x, double p, int64_t seed, const at::Tensor& seed_at) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  at::Tensor y = at::empty(x.sizes(), x.options());
  check(api.dropout(type_of(x), p, seed, data_of(seed_at), r.data(), r.stride, r.rows, r.features,
                    y.data_ptr(), stream_of(x.device())));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, double p,
                            int64_t seed, const std::optional<at::Tensor>& seed_at) {
    // A seed on the device is saved as it is: one that is changed before the
    // backward pass raises there, by torch's own check.
    ctx->save_for_backward({seed_at.value_or(at::Tensor())});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    return masked(x, p, seed, seed_at.value_or(at::Tensor()));
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("dropout", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    return once({masked(grads[0], ctx->saved_data["p"].toDouble(),
                        ctx->saved_data["seed"].toInt(), saved[0]),
                 at::Tensor(), at::Tensor(), at::Tensor()},
                "dropout");
  }
};

at::Tensor dropout(const at::Tensor& x, double p, int64_t seed,
                   const std::optional<at::Tensor>& seed_at) {
  const at::Tensor word = seed_at.value_or(at::Tensor());
  check_calls("dropout", {&x, &word});
  check_input(x);
  if (word.defined() &&
      (word.device() != x.device() || word.scalar_type() != at::kLong || word.numel() != 1))
    throw py::value_error("seed must be an integer, or one int64 on the device of x");
  if (!grad_wanted({&x})) return masked(x, p, seed, word);
  return Dropout::apply(x, p, seed, seed_at);
}

// --------------------------------------------------------------------------
// Rows in groups

std::vector<at::Tensor> row_groups(const at::Tensor& index, int64_t groups) {
  check_calls("row_groups", {&index});
  const bool wide = index.scalar_type() == at::kLong;
  if (!index.is_cuda() || !(wide || index.scalar_type() == at::kInt))
    throw py::value_error("index must be int32 or int64 on a HIP device");
  const c10::DeviceGuard guard(index.device());
  const at::Tensor rows = index.contiguous();
  at::Tensor order = at::empty({rows.numel()}, on(index.device(), at::kInt));
  at::Tensor offsets = at::empty({groups + 1}, on(index.device(), at::kInt));
  const size_t bytes = api.row_groups_workspace(rows.numel(), groups);
  at::Tensor space;
  if (bytes) space = workspace(bytes, index.device());
  check(api.row_groups(wide, rows.data_ptr(), rows.numel(), groups, order.data_ptr<int32_t>(),
                       offsets.data_ptr<int32_t>(), const_cast<void*>(data_of(space)), bytes,
                       stream_of(index.device())));
  return {offsets, order};
}

// How rows are grouped, as the entry points take it.
struct Groups {
  at::Tensor offsets, order;  // no order: the rows lie by group

  const int32_t* begins() const { return offsets.data_ptr<int32_t>(); }
  const int32_t* places() const { return order.defined() ? order.data_ptr<int32_t>() : nullptr; }
  int64_t count() const { return offsets.numel() - 1; }

  void check(const at::Tensor& x, int64_t groups) const {
    if (offsets.device() != x.device() || (order.defined() && order.device() != x.device()))
      throw py::value_error("groups must be on the device of x");
    if (count() != groups)
      throw py::value_error("groups has offsets of " + std::to_string(count()) + " groups, not " +
                            std::to_string(groups));
    const int64_t rows = x.numel() / x.size(-1);
    if (rows > 0x7ffff000) throw py::value_error("x has more than 2^31 - 4096 rows");
    if (order.defined() && order.numel() != rows)
      throw py::value_error("groups has an order of " + std::to_string(order.numel()) +
                            " rows, x has " + std::to_string(rows));
  }
};

at::Tensor grouped_rows(const at::Tensor& x, const at::Tensor& weight, const Groups& groups,
                        const at::Tensor& bias) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  const at::Tensor w = dense(weight), b = dense(bias);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.size(1);
  at::Tensor y = at::empty(shape, x.options());
  check(api.grouped_forward(type_of(x), r.data(), r.stride, w.data_ptr(), data_of(b),
                            groups.places(), groups.begins(), r.rows, groups.count(), r.features,
                            w.size(1), y.data_ptr(), stream_of(x.device())));
  return y;
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& weight, const at::Tensor& offsets,
                            const std::optional<at::Tensor>& order,
                            const std::optional<at::Tensor>& bias) {
    const Groups groups{offsets, order.value_or(at::Tensor())};
    at::Tensor y = grouped_rows(x, weight, groups, bias.value_or(at::Tensor()));
    // The bias's gradient takes no rows of x.
    ctx->save_for_backward(
        {weight.requires_grad() ? x : at::Tensor(), weight, offsets, groups.order});
    ctx->saved_data["order"] = order.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("grouped_linear", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const bool has_order = ctx->saved_data["order"].toBool();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const at::Tensor& grad = grads[0];
    const c10::DeviceGuard guard(grad.device());
    const RowsOf g(grad);
    const at::Tensor w = dense(saved[1]);
    const Groups groups{saved[2], saved[3]};
    const int64_t outputs = w.size(1), features = w.size(2);
    const int32_t type = type_of(grad);
    void* const stream = stream_of(grad.device());
    at::Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) {
      dx = at::empty(ctx->saved_data["shape"].toIntVector(), grad.options());
      check(api.grouped_backward_input(type, g.data(), g.stride, w.data_ptr(), groups.places(),
                                       groups.begins(), g.rows, groups.count(), features, outputs,
                                       dx.data_ptr(), stream));
    }
    // A tensor that is not there is no input of the function's graph.
    const size_t bias_at = has_order ? 4 : 3;
    if (ctx->needs_input_grad(1)) dw = at::empty(w.sizes(), grad.options());
    if (has_bias && ctx->needs_input_grad(bias_at))
      db = at::empty({groups.count(), outputs}, grad.options());
    if (dw.defined() || db.defined()) {
      std::optional<RowsOf> r;
      if (dw.defined()) r.emplace(saved[0]);
      const at::Tensor space = workspace(
          api.grouped_workspace(type, g.rows, groups.count(), features, outputs), grad.device());
      check(api.grouped_backward_weight(
          type, g.data(), g.stride, r ? r->data() : nullptr, r ? r->stride : features,
          groups.places(), groups.begins(), g.rows, groups.count(), features, outputs,
          const_cast<void*>(data_of(dw)), const_cast<void*>(data_of(db)), space.data_ptr(),
          size_t(space.numel()), stream));
    }
    return once({dx, dw, at::Tensor(), at::Tensor(), db}, "grouped_linear");
  }
};

at::Tensor grouped_linear(const at::Tensor& x, const at::Tensor& weight,
                          const at::Tensor& offsets, const std::optional<at::Tensor>& order,
                          const std::optional<at::Tensor>& bias) {
  const at::Tensor b = bias.value_or(at::Tensor());
  const Groups groups{offsets, order.value_or(at::Tensor())};
  check_calls("grouped_linear", {&x, &weight, &b});
  check_input(x);
  if (weight.dim() != 3 || weight.size(0) < 1 || weight.size(1) < 1)
    throw py::value_error("weight must have shape (groups, outputs, features)");
  check_parameter("weight", weight, {weight.size(0), weight.size(1), x.size(-1)}, x, false);
  check_parameter("bias", b, {weight.size(0), weight.size(1)}, x, false);
  groups.check(x, weight.size(0));
  if (!grad_wanted({&x, &weight, &b})) return grouped_rows(x, weight, groups, b);
  return GroupedLinear::apply(x, weight, offsets, order, bias);
}

// --------------------------------------------------------------------------
// Linear layers with low-rank adapters

at::Tensor adapted_rows(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& down,
                        const at::Tensor& up, const Groups& groups, const at::Tensor& bias,
                        double scale, at::Tensor* kept) {
  const c10::DeviceGuard guard(x.device());
  const RowsOf r(x);
  const at::Tensor w = dense(weight), b = dense(bias), a = dense(down), u = dense(up);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.size(0);
  at::Tensor y = at::empty(shape, x.options());
  at::Tensor inner = workspace(api.adapted_inner(r.rows, a.size(1)), x.device());
  check(api.adapted_forward(type_of(x), r.data(), r.stride, w.data_ptr(), data_of(b),
                            a.data_ptr(), u.data_ptr(), float(scale), groups.places(),
                            groups.begins(), r.rows, groups.count(), r.features, w.size(0),
                            a.size(1), inner.data_ptr(), size_t(inner.numel()), y.data_ptr(),
                            stream_of(x.device())));
  if (kept) *kept = inner;
  return y;
}

struct AdaptedLinear : torch::autograd::Function<AdaptedLinear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& weight, const at::Tensor& down,
                            const at::Tensor& up, const at::Tensor& offsets,
                            const std::optional<at::Tensor>& order,
                            const std::optional<at::Tensor>& bias, double scale) {
    const Groups groups{offsets, order.value_or(at::Tensor())};
    // The bias's gradient takes no rows of x.
    const bool keep = weight.requires_grad() || down.requires_grad();
    at::Tensor inner;
    at::Tensor y = adapted_rows(x, weight, down, up, groups, bias.value_or(at::Tensor()), scale,
                                up.requires_grad() ? &inner : nullptr);
    ctx->save_for_backward({keep ? x : at::Tensor(), weight, down, up, offsets, groups.order,
                            inner});
    ctx->saved_data["order"] = order.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    check_calls("adapted_linear", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const bool has_order = ctx->saved_data["order"].toBool();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const at::Tensor& grad = grads[0];
    const c10::DeviceGuard guard(grad.device());
    const RowsOf g(grad);
    const at::Tensor w = dense(saved[1]), a = dense(saved[2]), u = dense(saved[3]);
    const Groups groups{saved[4], saved[5]};
    const int64_t outputs = w.size(0), features = w.size(1), rank = a.size(1);
    const int32_t type = type_of(grad);
    void* const stream = stream_of(grad.device());
    at::Tensor dx, dw, da, du, db, back;
    std::optional<RowsOf> x;
    if (saved[0].defined()) x.emplace(saved[0]);
    if (ctx->needs_input_grad(0))
      dx = at::empty(ctx->saved_data["shape"].toIntVector(), grad.options());
    if (ctx->needs_input_grad(2)) da = at::empty(a.sizes(), grad.options());
    if (ctx->needs_input_grad(3)) du = at::empty(u.sizes(), grad.options());
    if (dx.defined() || da.defined()) {
      back = workspace(api.adapted_inner(g.rows, rank), grad.device());
      check(api.adapted_backward_input(
          type, g.data(), g.stride, w.data_ptr(), a.data_ptr(), u.data_ptr(),
          float(ctx->saved_data["scale"].toDouble()), groups.places(), groups.begins(), g.rows,
          groups.count(), features, outputs, rank, back.data_ptr(), size_t(back.numel()),
          const_cast<void*>(data_of(dx)), stream));
    }
    if (da.defined() || du.defined()) {
      const at::Tensor space = workspace(
          api.adapted_workspace(g.rows, groups.count(), features, outputs, rank), grad.device());
      check(api.adapted_backward_adapters(
          type, g.data(), g.stride, x ? x->data() : nullptr, x ? x->stride : features,
          data_of(saved[6]), data_of(back), groups.places(), groups.begins(), g.rows,
          groups.count(), features, outputs, rank, const_cast<void*>(data_of(da)),
          const_cast<void*>(data_of(du)), space.data_ptr(), size_t(space.numel()), stream));
    }
    // The shared layer's gradients are linear's, of the input in 8 bits.
    if (ctx->needs_input_grad(1)) dw = at::empty(w.sizes(), grad.options());
    if (has_bias && ctx->needs_input_grad(has_order ? 6 : 5))
      db = at::empty({outputs}, grad.options());
    if (dw.defined() || db.defined()) {
      Kept kept;
      if (dw.defined()) {
        kept = Kept::empty(g.rows, features, grad.device());
        check(api.checkpoint_write(type, x->data(), x->stride, g.rows, features,
                                   kept.values.data_ptr(), kept.exponents.data_ptr(), stream));
      }
      const at::Tensor space =
          workspace(api.linear_workspace(type, g.rows, features, outputs), grad.device());
      check(api.linear_backward_weight(
          type, g.data(), g.stride, data_of(kept.values), data_of(kept.exponents), g.rows,
          features, outputs, const_cast<void*>(data_of(dw)), const_cast<void*>(data_of(db)),
          space.data_ptr(), size_t(space.numel()), stream));
    }
    return once({dx, dw, da, du, at::Tensor(), at::Tensor(), db, at::Tensor()},
                "adapted_linear");
  }
};

at::Tensor adapted_linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& down,
                          const at::Tensor& up, const at::Tensor& offsets,
                          const std::optional<at::Tensor>& order,
                          const std::optional<at::Tensor>& bias, double scale) {
  const at::Tensor b = bias.value_or(at::Tensor());
  const Groups groups{offsets, order.value_or(at::Tensor())};
  check_calls("adapted_linear", {&x, &weight, &down, &up, &b});
  check_input(x);
  if (weight.dim() != 2 || weight.size(0) < 1)
    throw py::value_error("weight must have shape (outputs, features)");
  check_parameter("weight", weight, {weight.size(0), x.size(-1)}, x, false);
  check_parameter("bias", b, {weight.size(0)}, x, false);
  if (down.dim() != 3 || down.size(0) < 1 || down.size(1) < 1 || down.size(1) > 64)
    throw py::value_error("down must have shape (groups, rank, features), rank at most 64");
  check_parameter("down", down, {down.size(0), down.size(1), x.size(-1)}, x, false);
  check_parameter("up", up, {down.size(0), weight.size(0), down.size(1)}, x, false);
  groups.check(x, down.size(0));
  if (!grad_wanted({&x, &weight, &down, &up, &b}))
    return adapted_rows(x, weight, down, up, groups, b, scale, nullptr);
  return AdaptedLinear::apply(x, weight, down, up, offsets, order, bias, scale);
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
  take(table, "gs_dropout", next.dropout);
  take(table, "gs_row_groups_workspace_size", next.row_groups_workspace);
  take(table, "gs_row_groups", next.row_groups);
  take(table, "gs_grouped_linear_forward", next.grouped_forward);
  take(table, "gs_grouped_linear_backward_input", next.grouped_backward_input);
  take(table, "gs_grouped_linear_backward_weight_workspace_size", next.grouped_workspace);
  take(table, "gs_grouped_linear_backward_weight", next.grouped_backward_weight);
  take(table, "gs_adapted_linear_inner_size", next.adapted_inner);
  take(table, "gs_adapted_linear_forward", next.adapted_forward);
  take(table, "gs_adapted_linear_backward_input", next.adapted_backward_input);
  take(table, "gs_adapted_linear_backward_adapters_workspace_size", next.adapted_workspace);
  take(table, "gs_adapted_linear_backward_adapters", next.adapted_backward_adapters);
  api = next;
}

std::vector<std::string> layer_entry_points() {
  return {"gs_checkpoint8_write", "gs_checkpoint8_read", "gs_activation_forward",
          "gs_activation_backward", "gs_layer_norm_forward",
          "gs_layer_norm_backward_workspace_size", "gs_layer_norm_backward", "gs_linear_forward",
          "gs_linear_backward_input", "gs_linear_backward_weight_workspace_size",
          "gs_linear_backward_weight", "gs_dropout", "gs_row_groups_workspace_size",
          "gs_row_groups", "gs_grouped_linear_forward", "gs_grouped_linear_backward_input",
          "gs_grouped_linear_backward_weight_workspace_size",
          "gs_grouped_linear_backward_weight", "gs_adapted_linear_inner_size",
          "gs_adapted_linear_forward", "gs_adapted_linear_backward_input",
          "gs_adapted_linear_backward_adapters_workspace_size",
          "gs_adapted_linear_backward_adapters"};
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
  m.def("dropout", &dropout, py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("seed_at"));
  m.def("row_groups", &row_groups, py::arg("index"), py::arg("groups"));
  m.def("grouped_linear", &grouped_linear, py::arg("x"), py::arg("weight"), py::arg("offsets"),
        py::arg("order"), py::arg("bias"));
  m.def("adapted_linear", &adapted_linear, py::arg("x"), py::arg("weight"), py::arg("down"),
        py::arg("up"), py::arg("offsets"), py::arg("order"), py::arg("bias"), py::arg("scale"));
}

}  // namespace gs_host
