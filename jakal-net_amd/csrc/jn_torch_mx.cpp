// PyTorch operators over the microscaled entry points of the C ABI (jn_mx_*,
// jn_gelu_*, jn_column_sums), built like those of jn_torch.cpp: the public ones
// (mx_quantize, mx_dequantize, mx_linear, linear_saved, gelu_saved,
// stabilize_saved, layer_norm_saved) check, set up their autograd nodes and call
// inner ones, which have a kernel for GPU tensors and one for tensors without
// memory.  What a node keeps of an activation is its e4m3 codes and scales.
#include "jn_torch.hpp"

#include <ATen/ops/linear.h>
#include <ATen/ops/mm.h>

namespace {

constexpr int64_t kRun = 32;

c10::SymInt runs_of(const c10::SymInt& dim) { return (dim + (kRun - 1)) / kRun; }
// bytes of a row's codes
c10::SymInt pitch_of(const c10::SymInt& dim, int64_t form) { return runs_of(dim) * (form == JN_E4M3 ? kRun : kRun / 2); }

// t as it lies in memory, starting on 16 bytes.
Tensor aligned(const Tensor& t) {
  const Tensor p = plain(t);
  return p.numel() && reinterpret_cast<uintptr_t>(p.data_ptr()) % 16 ? p.clone() : p;
}

void check_width(const char* what, const c10::SymInt& size) {
  TORCH_CHECK_NOT_IMPLEMENTED(size < (int64_t(1) << 31), what, " takes rows of up to 2^31 - 1 elements, got ", size, ".");
}

void check_rows(const char* what, const Tensor& x) {
  type_code(what, x);
  TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1, what, " needs a last axis of at least one element, got shape ",
              x.sym_sizes(), ".");
  check_width(what, x.sym_size(-1));
  check_gpu(x, x);
}
void check_form(const char* what, int64_t form) {
  TORCH_CHECK(form == JN_E4M3 || form == JN_E2M1, what, ": unknown format code ", form, ".");
}

// codes [..., pitch] and scales [..., runs] of rows of `size` elements.
void check_packed(const char* what, const Tensor& codes, const Tensor& scales, int64_t form, const c10::SymInt& size) {
  check_form(what, form);
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what,
              ": codes and scales are uint8 tensors, got ", codes.scalar_type(), " and ", scales.scalar_type(), ".");
  TORCH_CHECK(size >= 1 && codes.dim() >= 1 && scales.dim() == codes.dim() &&
                  codes.sym_sizes().slice(0, codes.dim() - 1) == scales.sym_sizes().slice(0, codes.dim() - 1) &&
                  codes.sym_size(-1) == pitch_of(size, form) && scales.sym_size(-1) == runs_of(size),
              what, ": rows of ", size, " elements have no codes of shape ", codes.sym_sizes(), " and scales of shape ",
              scales.sym_sizes(), ".");
  check_gpu(codes, codes);
  check_gpu(scales, codes);
}

Tensor bytes_like(const Tensor& t, int64_t count) { return at::empty({count}, t.options().dtype(at::kByte)); }

// Sizes with the last one replaced.
std::vector<c10::SymInt> with_last(c10::SymIntArrayRef sizes, const c10::SymInt& last) {
  std::vector<c10::SymInt> out(sizes.begin(), sizes.end());
  out.back() = last;
  return out;
}

// ---- quantising and dequantising ----------------------------------------------
using Packed = std::tuple<Tensor, Tensor>;  // codes, scales

Packed packed_outputs(const Tensor& x, int64_t form) {
  const auto bytes = x.options().dtype(at::kByte);
  return {at::empty_symint(with_last(x.sym_sizes(), pitch_of(x.sym_size(-1), form)), bytes),
          at::empty_symint(with_last(x.sym_sizes(), runs_of(x.sym_size(-1))), bytes)};
}

Packed mx_codes_meta(const Tensor& x, int64_t form) { return packed_outputs(x, form); }

Packed mx_codes(const Tensor& x_in, int64_t form) {
  check_rows("mx_quantize", x_in);
  check_form("mx_quantize", form);
  const Tensor x = plain(x_in);
  const c10::DeviceGuard guard(x.device());
  const Packed out = packed_outputs(x, form);
  if (x.numel()) {
    check(jn_mx_quantize(ptr(x), x.numel() / x.size(-1), x.size(-1), type_code("mx_quantize", x), (int32_t)form,
                         ptr(std::get<0>(out)), ptr(std::get<1>(out)), stream_of(x)));
  }
  return out;
}

Tensor mx_values_meta(const Tensor& codes, const Tensor&, int64_t, c10::SymInt size, at::ScalarType type) {
  return at::empty_symint(with_last(codes.sym_sizes(), size), codes.options().dtype(type));
}

Tensor mx_values(const Tensor& codes_in, const Tensor& scales_in, int64_t form, c10::SymInt size, at::ScalarType type) {
  check_packed("mx_dequantize", codes_in, scales_in, form, size);
  const Tensor codes = aligned(codes_in), scales = plain(scales_in);
  const c10::DeviceGuard guard(codes.device());
  const Tensor out = mx_values_meta(codes, scales, form, size, type);
  const int32_t code = type_code("mx_dequantize", out);
  if (out.numel()) {
    const int64_t dim = out.size(-1);
    check(jn_mx_dequantize(ptr(codes), ptr(scales), out.numel() / dim, dim, (int32_t)form, code, ptr(out),
                           stream_of(out)));
  }
  return out;
}

using Codes = Packed(const Tensor&, int64_t);
using Values = Tensor(const Tensor&, const Tensor&, int64_t, c10::SymInt, at::ScalarType);

Packed call_codes(const Tensor& x, int64_t form) {
  static const auto op = inner<Codes>("jakal_net_hip::mx_codes");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, form);
}

Packed mx_quantize(const Tensor& x, int64_t form) {
  check_rows("mx_quantize", x);
  check_form("mx_quantize", form);
  return call_codes(x, form);
}

Tensor mx_dequantize(const Tensor& codes, const Tensor& scales, int64_t form, c10::SymInt size, at::ScalarType type) {
  check_packed("mx_dequantize", codes, scales, form, size);
  check_width("mx_dequantize", size);
  type_code("mx_dequantize", type);
  static const auto op = inner<Values>("jakal_net_hip::mx_values");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(codes, scales, form, std::move(size), type);
}

// ---- sums over rows -----------------------------------------------------------
Tensor column_sums_meta(const Tensor& x) { return at::empty_symint({x.sym_size(-1)}, x.options()); }

Tensor column_sums(const Tensor& x_in) {
  check_rows("column_sums", x_in);
  const Tensor x = plain(x_in);
  const c10::DeviceGuard guard(x.device());
  const Tensor out = column_sums_meta(x);
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  if (rows == 0) return out.zero_();
  const size_t bytes = jn_column_sums_workspace_bytes(rows, dim);
  const Tensor ws = bytes_like(x, (int64_t)bytes);
  check(jn_column_sums(ptr(x), rows, dim, type_code("column_sums", x), ptr(out), ptr(ws), bytes, stream_of(x)));
  return out;
}

Tensor call_column_sums(const Tensor& x) {
  static const auto op = inner<Tensor(const Tensor&)>("jakal_net_hip::column_sums");
  return op.call(x);
}

// What the library's products of x [..., inputs] and their gradients take.
void check_product(const char* what, const Tensor& x, const c10::SymInt& out) {
  constexpr int64_t kRows = int64_t(1) << 31, kWidth = int64_t(1) << 24;
  TORCH_CHECK_NOT_IMPLEMENTED(x.sym_size(-1) < kWidth && out < kWidth && x.sym_numel() < x.sym_size(-1) * kRows, what,
                              " takes up to 2^31 - 1 rows and 2^24 - 1 inputs and outputs, got shape ", x.sym_sizes(),
                              " and ", out, " outputs.");
}

// ---- products by 4-bit weights ------------------------------------------------
void check_linear(const char* what, const Tensor& x, const Tensor& weight, const Tensor& bias, const c10::SymInt& out) {
  check_rows(what, x);
  check_gpu(weight, x);
  if (!bias.defined()) return;
  TORCH_CHECK(bias.dim() == 1 && bias.sym_size(0) == out, what, ": a bias for ", out, " outputs is shaped [", out,
              "], got ", bias.sym_sizes(), ".");
  TORCH_CHECK(bias.scalar_type() == x.scalar_type(), what, ": x is ", x.scalar_type(), " but the bias ",
              bias.scalar_type(), ".");
  check_gpu(bias, x);
}

void check_mx_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, const Tensor& bias, int64_t acts) {
  TORCH_CHECK(acts == JN_E2M1 || acts == JN_PLAIN, "mx_linear: unknown activations code ", acts, ".");
  TORCH_CHECK(codes.dim() == 2, "mx_linear: the weight is a matrix [outputs, inputs], got codes of shape ",
              codes.sym_sizes(), ".");
  check_linear("mx_linear", x, codes, bias, codes.sym_size(0));
  check_packed("mx_linear", codes, scales, JN_E2M1, x.sym_size(-1));
  TORCH_CHECK(codes.sym_size(0) >= 1, "mx_linear: a weight without outputs.");
  check_product("mx_linear", x, codes.sym_size(0));
}

using Product = Tensor(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, int64_t);
using InputGrad = Tensor(const Tensor&, const Tensor&, const Tensor&, c10::SymInt);

Tensor mx_product_meta(const Tensor& x, const Tensor& codes, const Tensor&, const std::optional<Tensor>&, int64_t) {
  return at::empty_symint(with_last(x.sym_sizes(), codes.sym_size(0)), x.options());
}

Tensor mx_product(const Tensor& x_in, const Tensor& codes_in, const Tensor& scales_in,
                  const std::optional<Tensor>& bias_in, int64_t acts) {
  check_mx_linear(x_in, codes_in, scales_in, given(bias_in), acts);
  const Tensor x = aligned(x_in), codes = aligned(codes_in), scales = aligned(scales_in), bias = plain(given(bias_in));
  const c10::DeviceGuard guard(x.device());
  const Tensor y = mx_product_meta(x, codes, scales, bias_in, acts);
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  if (rows == 0) return y;
  const int32_t type = type_code("mx_linear", x);
  const size_t bytes = jn_mx_linear_forward_workspace_bytes(rows, dim, codes.size(0), type, (int32_t)acts);
  const Tensor ws = bytes_like(x, (int64_t)bytes);
  check(jn_mx_linear_forward(ptr(x), ptr(codes), ptr(scales), ptr(bias), rows, dim, codes.size(0), type, (int32_t)acts, ptr(y), ptr(ws), bytes, stream_of(x)));
  return y;
}

Tensor mx_input_grad_meta(const Tensor& grad, const Tensor&, const Tensor&, c10::SymInt size) {
  return at::empty_symint(with_last(grad.sym_sizes(), size), grad.options());
}

Tensor mx_input_grad(const Tensor& grad_in, const Tensor& codes_in, const Tensor& scales_in, c10::SymInt size) {
  check_rows("mx_linear backward", grad_in);
  check_packed("mx_linear backward", codes_in, scales_in, JN_E2M1, size);
  TORCH_CHECK(codes_in.dim() == 2 && codes_in.size(0) == grad_in.size(-1),
              "mx_linear backward: gradients of another number of outputs than the weight has.");
  check_gpu(codes_in, grad_in);
  const Tensor grad = aligned(grad_in), codes = aligned(codes_in), scales = plain(scales_in);
  const c10::DeviceGuard guard(grad.device());
  const Tensor out = mx_input_grad_meta(grad, codes, scales, size);
  const int64_t dim = out.size(-1), rows = out.numel() / dim, outs = grad.size(-1);
  if (rows == 0) return out;
  const int32_t type = type_code("mx_linear", grad);
  const size_t bytes = jn_mx_linear_backward_workspace_bytes(rows, dim, outs, type);
  const Tensor ws = bytes_like(grad, (int64_t)bytes);
  check(jn_mx_linear_backward(ptr(grad), ptr(codes), ptr(scales), rows, dim, outs, type, ptr(out), ptr(ws), bytes,
                              stream_of(grad)));
  return out;
}

struct JakalMxLinearBackward : torch::autograd::Node {
  Kept codes_, scales_;
  c10::SymInt dim = 0;
  at::ScalarType type = at::kFloat;

  std::string name() const override { return "JakalMxLinearBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    codes_.reset();
    scales_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    if (!grads[0].defined()) return variable_list(2);
    const Tensor g = grads[0].to(type);
    Tensor gx, gb;
    const at::AutoDispatchBelowADInplaceOrView below;
    if (task_should_compute_output(0)) {
      static const auto op = inner<InputGrad>("jakal_net_hip::mx_input_grad");
      gx = op.call(g, codes_.get(), scales_.get(), dim);
    }
    if (task_should_compute_output(1)) gb = call_column_sums(g);
    return once_differentiable({gx, gb}, recorded);
  }
};

Tensor mx_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, const std::optional<Tensor>& bias_in,
                 int64_t acts) {
  const Tensor bias = given(bias_in);
  check_mx_linear(x, codes, scales, bias, acts);
  std::shared_ptr<JakalMxLinearBackward> node;
  if (records(x, bias)) {
    node = make_node<JakalMxLinearBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, bias));
  }
  Tensor y;
  {
    static const auto op = inner<Product>("jakal_net_hip::mx_product");
    const at::AutoDispatchBelowADInplaceOrView below;
    y = op.call(x, codes, scales, bias_in, acts);
  }
  if (node) {
    node->codes_.set(codes);
    node->scales_.set(scales);
    node->dim = x.sym_size(-1);
    node->type = x.scalar_type();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- a linear layer that keeps its input in e4m3 ------------------------------
using WeightGrad = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, c10::SymInt, bool);

std::tuple<Tensor, Tensor> mx_weight_grad_meta(const Tensor& grad, const Tensor&, const Tensor&, c10::SymInt size,
                                               bool bias) {
  const c10::SymInt out = grad.sym_size(-1);
  return {at::empty_symint({out, size}, grad.options()), bias ? at::empty_symint({out}, grad.options()) : Tensor()};
}

std::tuple<Tensor, Tensor> mx_weight_grad(const Tensor& grad_in, const Tensor& codes_in, const Tensor& scales_in,
                                          c10::SymInt size, bool bias) {
  check_rows("linear backward", grad_in);
  check_packed("linear backward", codes_in, scales_in, JN_E4M3, size);
  check_gpu(codes_in, grad_in);
  const int64_t out = grad_in.size(-1), rows = grad_in.numel() / out;
  TORCH_CHECK(scales_in.numel() == rows * scales_in.size(-1),
              "linear backward: gradients of another number of rows than were kept.");
  const Tensor grad = aligned(grad_in), codes = aligned(codes_in), scales = plain(scales_in);
  const c10::DeviceGuard guard(grad.device());
  auto [gw, gb] = mx_weight_grad_meta(grad, codes, scales, size, bias);
  if (rows == 0) {
    gw.zero_();
    if (bias) gb.zero_();
    return {gw, gb};
  }
  const int64_t dim = gw.size(1);
  const int32_t type = type_code("linear backward", grad);
  const size_t bytes = jn_mx_weight_grad_workspace_bytes(rows, dim, out, type, bias);
  const Tensor ws = bytes_like(grad, (int64_t)bytes);
  check(jn_mx_weight_grad(ptr(grad), ptr(codes), ptr(scales), rows, dim, out, type, ptr(gw), ptr(gb), ptr(ws), bytes,
                          stream_of(grad)));
  return {gw, gb};
}

Tensor linear_input_grad_meta(const Tensor& grad, const Tensor& weight) {
  return at::empty_symint(with_last(grad.sym_sizes(), weight.sym_size(1)), grad.options());
}

// grad . weight: here where the sum is short, or long over few outputs, else the library
// product that a plain linear layer's backward is.
Tensor linear_input_grad(const Tensor& grad_in, const Tensor& weight_in) {
  check_rows("linear backward", grad_in);
  TORCH_CHECK(weight_in.dim() == 2 && weight_in.size(0) == grad_in.size(-1) &&
                  weight_in.scalar_type() == grad_in.scalar_type(),
              "linear backward: a weight that does not pair with the gradients.");
  check_gpu(weight_in, grad_in);
  const int64_t out = grad_in.size(-1), rows = grad_in.numel() / out, dim = weight_in.size(1);
  const int32_t type = type_code("linear backward", grad_in);
  const c10::DeviceGuard guard(grad_in.device());
  if (rows == 0 || !jn_linear_input_grad_fits(rows, dim, out, type)) {
    const Tensor product = at::mm(grad_in.reshape({rows, out}), weight_in);
    std::vector<int64_t> sizes(grad_in.sizes().begin(), grad_in.sizes().end());
    sizes.back() = dim;
    return product.view(sizes);
  }
  const Tensor grad = aligned(grad_in), weight = aligned(weight_in);
  const Tensor gx = linear_input_grad_meta(grad, weight);
  const size_t bytes = jn_linear_input_grad_workspace_bytes(rows, dim, out, type);
  const Tensor ws = bytes_like(grad, (int64_t)bytes);
  check(jn_linear_input_grad(ptr(grad), ptr(weight), rows, dim, out, type, ptr(gx), ptr(ws), bytes, stream_of(grad)));
  return gx;
}

struct JakalLinearSavedBackward : torch::autograd::Node {
  Kept codes_, scales_, weight_;
  c10::SymInt dim = 0;
  at::ScalarType type = at::kFloat;

  std::string name() const override { return "JakalLinearSavedBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    codes_.reset();
    scales_.reset();
    weight_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    if (!grads[0].defined()) return variable_list(3);
    const Tensor g = plain(grads[0].to(type));
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
               need_b = task_should_compute_output(2);
    Tensor gx, gw, gb;
    const at::AutoDispatchBelowADInplaceOrView below;
    if (need_x) {
      static const auto op = inner<Tensor(const Tensor&, const Tensor&)>("jakal_net_hip::linear_input_grad");
      gx = op.call(g, weight_.get());
    }
    if (need_w) {
      static const auto op = inner<WeightGrad>("jakal_net_hip::mx_weight_grad");
      std::tie(gw, gb) = op.call(g, codes_.get(), scales_.get(), dim, need_b);
    } else if (need_b) {
      gb = call_column_sums(g);
    }
    return once_differentiable({gx, gw, gb}, recorded);
  }
};

Tensor linear_saved(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_in) {
  const Tensor bias = given(bias_in);
  TORCH_CHECK(weight.dim() == 2 && x.dim() >= 1 && weight.sym_size(1) == x.sym_size(-1),
              "linear: a weight of shape ", weight.sym_sizes(), " for values of shape ", x.sym_sizes(), ".");
  check_linear("linear", x, weight, bias, weight.sym_size(0));
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "linear: x is ", x.scalar_type(), " but the weight ",
              weight.scalar_type(), ".");
  TORCH_CHECK(weight.sym_size(0) >= 1, "linear: a weight without outputs.");
  std::shared_ptr<JakalLinearSavedBackward> node;
  if (records(x, weight, bias)) {
    // (the input's gradient may be the library product's)
    if (torch::autograd::compute_requires_grad(weight, bias)) check_product("linear", x, weight.sym_size(0));
    node = make_node<JakalLinearSavedBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
  }
  Tensor y, codes, scales;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    y = at::linear(x, weight, bias_in);
  }
  if (node) {
    if (torch::autograd::compute_requires_grad(weight)) {
      std::tie(codes, scales) = call_codes(x, JN_E4M3);
      node->codes_.set(codes);
      node->scales_.set(scales);
    }
    if (torch::autograd::compute_requires_grad(x)) node->weight_.set(weight);
    node->dim = x.sym_size(-1);
    node->type = x.scalar_type();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- GELU -----------------------------------------------------------------------
using Gelu = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, bool);  // y, codes, scales (or none)
using GeluBackward = Tensor(const Tensor&, const Tensor&, const Tensor&);

std::tuple<Tensor, Tensor, Tensor> gelu_forward_meta(const Tensor& x_in, bool keep) {
  const Tensor x = plain(x_in);
  Tensor codes, scales;
  if (keep) std::tie(codes, scales) = packed_outputs(x, JN_E4M3);
  return {at::empty_like(x), codes, scales};
}

std::tuple<Tensor, Tensor, Tensor> gelu_forward(const Tensor& x_in, bool keep) {
  check_rows("gelu", x_in);
  const Tensor x = plain(x_in);
  const c10::DeviceGuard guard(x.device());
  auto [y, codes, scales] = gelu_forward_meta(x, keep);
  if (x.numel()) {
    check(jn_gelu_forward(ptr(x), x.numel() / x.size(-1), x.size(-1), type_code("gelu", x), ptr(y), ptr(codes),
                          ptr(scales), stream_of(x)));
  }
  return {y, codes, scales};
}

Tensor gelu_backward_meta(const Tensor& grad, const Tensor&, const Tensor&) { return at::empty_like(plain(grad)); }

Tensor gelu_backward(const Tensor& grad_in, const Tensor& codes_in, const Tensor& scales_in) {
  check_rows("gelu backward", grad_in);
  check_packed("gelu backward", codes_in, scales_in, JN_E4M3, grad_in.size(-1));
  check_gpu(codes_in, grad_in);
  const Tensor grad = plain(grad_in), codes = aligned(codes_in), scales = plain(scales_in);
  const int64_t dim = grad.size(-1), rows = grad.numel() / dim;
  TORCH_CHECK(scales.numel() == rows * scales.size(-1), "gelu backward: gradients of another number of rows than were kept.");
  const c10::DeviceGuard guard(grad.device());
  const Tensor out = at::empty_like(grad);
  if (rows) {
    check(jn_gelu_backward(ptr(codes), ptr(scales), ptr(grad), rows, dim, type_code("gelu", grad), ptr(out),
                           stream_of(grad)));
  }
  return out;
}

struct JakalGeluSavedBackward : torch::autograd::Node {
  Kept codes_, scales_;
  at::ScalarType type = at::kFloat;

  std::string name() const override { return "JakalGeluSavedBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    codes_.reset();
    scales_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    static const auto op = inner<GeluBackward>("jakal_net_hip::gelu_backward");
    const at::AutoDispatchBelowADInplaceOrView below;
    return once_differentiable({op.call(grads[0].to(type), codes_.get(), scales_.get())}, recorded);
  }
};

Tensor gelu_saved(const Tensor& x) {
  check_rows("gelu", x);
  std::shared_ptr<JakalGeluSavedBackward> node;
  if (records(x)) {
    node = make_node<JakalGeluSavedBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
  }
  Tensor y, codes, scales;
  {
    static const auto op = inner<Gelu>("jakal_net_hip::gelu_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    std::tie(y, codes, scales) = op.call(x, node != nullptr);
  }
  if (node) {
    node->codes_.set(codes);
    node->scales_.set(scales);
    node->type = x.scalar_type();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- layer norm and stabilisation that keep their values in e4m3 --------------
// state_out (or none), y, stats, codes, scales
using KeptNorms = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
using KeptNormForward = KeptNorms(const std::optional<Tensor>&, const Tensor&, const std::optional<Tensor>&,
                                  const std::optional<Tensor>&, double, double);
using KeptNormGrads = std::tuple<Tensor, Tensor, Tensor, Tensor>;  // of state, x, weight, bias, where the mask has them
using KeptNormBackward = KeptNormGrads(const std::optional<Tensor>&, const std::optional<Tensor>&,
                                       const std::optional<Tensor>&, const Tensor&, const Tensor&,
                                       const std::optional<Tensor>&, const Tensor&, c10::SymInt, at::ScalarType,
                                       double, at::ScalarType, std::array<bool, 4>);

KeptNorms kept_norm_outputs(const Tensor& state, const Tensor& x) {
  Tensor out;
  if (state.defined()) out = at::empty_like(state);
  auto [codes, scales] = packed_outputs(x, JN_E4M3);
  return {out, at::empty_like(x), at::empty_symint({x.sym_numel() / x.sym_size(-1), 2}, x.options().dtype(at::kFloat)),
          codes, scales};
}

KeptNorms kept_norm_forward_meta(const std::optional<Tensor>& state, const Tensor& x, const std::optional<Tensor>&,
                                 const std::optional<Tensor>&, double, double) {
  return kept_norm_outputs(plain(given(state)), plain(x));
}

KeptNorms kept_norm_forward(const std::optional<Tensor>& state_in, const Tensor& x_in,
                            const std::optional<Tensor>& weight_in, const std::optional<Tensor>& bias_in, double eps,
                            double scale) {
  Tensor weight = given(weight_in), bias = given(bias_in);
  check_norm(given(state_in), x_in, weight, bias, eps);
  norm_params(x_in, weight, bias);
  const Tensor x = plain(x_in), state = plain(given(state_in));
  const c10::DeviceGuard guard(x.device());
  const KeptNorms made = kept_norm_outputs(state, x);
  const auto& [out, y, stats, codes, scales] = made;
  const Tensor& param = weight.defined() ? weight : bias;
  if (x.numel()) {
    check(jn_layer_norm_forward_kept(ptr(state), ptr(x), ptr(weight), ptr(bias), x.numel() / x.size(-1), x.size(-1),
                                     (float)scale, (float)eps, type_code("layer norm", x),
                                     state.defined() ? type_code("stabilize", state) : JN_F32,
                                     param.defined() ? type_code("layer norm", param) : JN_F32, ptr(out), ptr(y),
                                     fptr(stats), ptr(codes), ptr(scales), stream_of(x)));
  }
  return made;
}

KeptNormGrads kept_norm_grads(const Tensor& state, const Tensor& codes, const Tensor& weight, const c10::SymInt& dim,
                              at::ScalarType type, at::ScalarType bias_type, std::array<bool, 4> mask) {
  const auto options = codes.options();
  return {mask[0] ? at::empty_like(state) : Tensor(),
          mask[1] ? at::empty_symint(with_last(codes.sym_sizes(), dim), options.dtype(type)) : Tensor(),
          mask[2] ? at::empty_like(weight) : Tensor(),
          mask[3] ? at::empty_symint({dim}, options.dtype(bias_type)) : Tensor()};
}

KeptNormGrads kept_norm_backward_meta(const std::optional<Tensor>&, const std::optional<Tensor>&,
                                      const std::optional<Tensor>& state, const Tensor& codes, const Tensor&,
                                      const std::optional<Tensor>& weight, const Tensor&, c10::SymInt dim,
                                      at::ScalarType type, double, at::ScalarType bias_type, std::array<bool, 4> mask) {
  return kept_norm_grads(plain(given(state)), codes, plain(given(weight)), dim, type, bias_type, mask);
}

// codes, scales, stats as the forward gave them of x [..., size] of `type`; the mask:
// the gradients wanted, of state, x, weight and bias.
KeptNormGrads kept_norm_backward(const std::optional<Tensor>& g_state_in, const std::optional<Tensor>& g_in,
                                 const std::optional<Tensor>& state_in, const Tensor& codes_in, const Tensor& scales_in,
                                 const std::optional<Tensor>& weight_in, const Tensor& stats_in, c10::SymInt size,
                                 at::ScalarType type, double scale, at::ScalarType bias_type, std::array<bool, 4> mask) {
  check_packed("layer norm backward", codes_in, scales_in, JN_E4M3, size);
  const int64_t dim = size.expect_int();
  const Tensor state = plain(given(state_in)), codes = aligned(codes_in), scales = plain(scales_in),
               weight = plain(given(weight_in)), stats = plain(stats_in);
  const int64_t rows = scales.numel() / scales.size(-1);
  const bool sums = mask[2] || mask[3];
  Tensor g_state = given(g_state_in), g = given(g_in);
  TORCH_CHECK(!mask[0] || (state.defined() && g_state.defined() && g_state.numel() == rows && state.numel() == rows),
              "layer norm backward: a state's gradient needs the state and its output's gradient.");
  TORCH_CHECK((!mask[1] && !sums) || (g.defined() && g.numel() == rows * dim),
              "layer norm backward: the output's gradient has another size than the rows.");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows,
              "layer norm backward: statistics that no forward of these rows gave.");
  TORCH_CHECK(!mask[2] || weight.defined(), "layer norm backward: no weight to take a gradient of.");
  TORCH_CHECK(!weight.defined() || (weight.dim() == 1 && weight.size(0) == dim),
              "layer norm backward: a weight of another width than the rows.");
  const at::ScalarType param = weight.defined() ? weight.scalar_type() : bias_type;
  TORCH_CHECK((param == at::kFloat || param == type) && (!mask[3] || bias_type == param),
              "layer norm backward: parameters are fp32 or of the rows' type, and of one type.");
  if (mask[0]) check_gpu(g_state, codes), g_state = plain(g_state.to(state.scalar_type()));
  if (mask[1] || sums) check_gpu(g, codes), g = plain(g.to(type));
  check_gpu(state, codes);
  check_gpu(weight, codes);
  check_gpu(stats, codes);
  const c10::DeviceGuard guard(codes.device());
  const KeptNormGrads out = kept_norm_grads(state, codes, weight, dim, type, bias_type, mask);
  const auto& [gs, gx, gw, gb] = out;
  if (rows == 0) {
    if (mask[2]) gw.zero_();
    if (mask[3]) gb.zero_();
    return out;
  }
  size_t bytes = 0;
  Tensor ws;
  if (sums) {
    bytes = jn_layer_norm_backward_workspace_bytes(rows, dim);
    ws = bytes_like(codes, (int64_t)bytes);
  }
  const auto code = [](at::ScalarType t) { return t == at::kFloat ? JN_F32 : t == at::kBFloat16 ? JN_BF16 : JN_F16; };
  check(jn_layer_norm_backward_kept(ptr(state), ptr(codes), ptr(scales), ptr(weight), fptr(stats),
                                    mask[0] ? ptr(g_state) : nullptr, mask[1] || sums ? ptr(g) : nullptr, rows, dim,
                                    (float)scale, code(type), state.defined() ? code(state.scalar_type()) : JN_F32,
                                    code(param), ptr(gs), ptr(gx), ptr(gw), ptr(gb), ptr(ws), bytes,
                                    stream_of(codes)));
  return out;
}

struct JakalKeptNormBackward : torch::autograd::Node {
  Kept state_, codes_, scales_, weight_, stats_;
  c10::SymInt dim = 0;
  double scale = 1.0;
  int state_at = -1, y_at = -1;  // the outputs' places, or -1: no gradient comes through it
  at::ScalarType type = at::kFloat, bias_type = at::kFloat;

  std::string name() const override { return "JakalKeptNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (Kept* k : {&state_, &codes_, &scales_, &weight_, &stats_}) k->reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const Tensor g_state = state_at < 0 ? Tensor() : grads[state_at], g = y_at < 0 ? Tensor() : grads[y_at];
    std::array<bool, 4> need;
    bool any = false;
    for (int i = 0; i < 4; ++i) {
      need[i] = (i ? g : g_state).defined() && task_should_compute_output(i);
      any = any || need[i];
    }
    if (!any) return variable_list(4);
    static const auto op = inner<KeptNormBackward>("jakal_net_hip::kept_norm_backward");
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [gs, gx, gw, gb] = op.call(maybe(g_state), maybe(g), maybe(state_.get()), codes_.get(), scales_.get(),
                                    maybe(weight_.get()), stats_.get(), dim, type, scale, bias_type, need);
    return once_differentiable({gs, gx, gw, gb}, recorded);
  }
};

// (state_out, y) as the plain operators give them; without history they are called.
std::tuple<Tensor, Tensor> kept_norm(const Tensor& state_in, const Tensor& x_in, const std::optional<Tensor>& weight_in,
                                     const std::optional<Tensor>& bias_in, double eps, double scale) {
  Tensor weight = given(weight_in), bias = given(bias_in);
  check_norm(state_in, x_in, weight, bias, eps);
  norm_params(x_in, weight, bias);
  const Tensor x = plain(x_in), state = plain(state_in);
  std::shared_ptr<JakalKeptNormBackward> node;
  Tensor out, y, stats, codes, scales;
  if (!records(state, x, weight, bias)) {
    using Forward = std::tuple<Tensor, Tensor, Tensor>(const std::optional<Tensor>&, const Tensor&,
                                                       const std::optional<Tensor>&, const std::optional<Tensor>&,
                                                       double, double, bool);
    static const auto op = inner<Forward>("jakal_net_hip::row_norm_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    std::tie(out, y, stats) = op.call(maybe(state), x, maybe(weight), maybe(bias), eps, scale, false);
    return {out, y};
  }
  node = make_node<JakalKeptNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(state, x, weight, bias));
  {
    static const auto op = inner<KeptNormForward>("jakal_net_hip::kept_norm_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    std::tie(out, y, stats, codes, scales) = op.call(maybe(state), x, maybe(weight), maybe(bias), eps, scale);
  }
  node->state_.set(state);
  node->codes_.set(codes);
  node->scales_.set(scales);
  node->weight_.set(weight);
  node->stats_.set(stats);
  node->dim = x.sym_size(-1);
  node->scale = scale;
  node->type = x.scalar_type();
  if (bias.defined()) node->bias_type = bias.scalar_type();
  int places = 0;
  if (torch::autograd::compute_requires_grad(state)) {
    node->state_at = places++;
    torch::autograd::set_history(out, node);
  }
  if (torch::autograd::compute_requires_grad(x, weight, bias)) {
    node->y_at = places++;
    torch::autograd::set_history(y, node);
  }
  return {out, y};
}

Tensor layer_norm_saved(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                        double eps) {
  return std::get<1>(kept_norm(Tensor(), x, weight, bias, eps, 1.0));
}

std::tuple<Tensor, Tensor> stabilize_saved(const Tensor& state, const Tensor& val, const std::optional<Tensor>& weight,
                                           const std::optional<Tensor>& bias, double eps, double scale) {
  return kept_norm(state, val, weight, bias, eps, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(jakal_net_hip, m) {
  m.def("mx_quantize(Tensor x, int format) -> (Tensor, Tensor)", &mx_quantize);
  m.def("mx_dequantize(Tensor codes, Tensor scales, int format, SymInt size, ScalarType type) -> Tensor",
        &mx_dequantize);
  m.def("mx_linear(Tensor x, Tensor codes, Tensor scales, Tensor? bias, int activations) -> Tensor", &mx_linear);
  m.def("linear_saved(Tensor x, Tensor weight, Tensor? bias) -> Tensor", &linear_saved);
  m.def("gelu_saved(Tensor x) -> Tensor", &gelu_saved);
  m.def("layer_norm_saved(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm_saved);
  m.def("stabilize_saved(Tensor state, Tensor val, Tensor? weight, Tensor? bias, float eps, float scale)"
        " -> (Tensor, Tensor)", &stabilize_saved);

  m.def("mx_codes(Tensor x, int format) -> (Tensor, Tensor)");
  m.def("mx_values(Tensor codes, Tensor scales, int format, SymInt size, ScalarType type) -> Tensor");
  m.def("column_sums(Tensor x) -> Tensor");
  m.def("mx_product(Tensor x, Tensor codes, Tensor scales, Tensor? bias, int activations) -> Tensor");
  m.def("mx_input_grad(Tensor grad, Tensor codes, Tensor scales, SymInt size) -> Tensor");
  m.def("mx_weight_grad(Tensor grad, Tensor codes, Tensor scales, SymInt size, bool bias) -> (Tensor, Tensor)");
  m.def("linear_input_grad(Tensor grad, Tensor weight) -> Tensor");
  m.def("gelu_forward(Tensor x, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("gelu_backward(Tensor grad, Tensor codes, Tensor scales) -> Tensor");
  m.def("kept_norm_forward(Tensor? state, Tensor x, Tensor? weight, Tensor? bias, float eps, float scale)"
        " -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("kept_norm_backward(Tensor? grad_state, Tensor? grad_y, Tensor? state, Tensor codes, Tensor scales,"
        " Tensor? weight, Tensor stats, SymInt size, ScalarType type, float scale, ScalarType bias_type, bool[4] mask)"
        " -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(jakal_net_hip, CUDA, m) {
  m.impl("mx_codes", &mx_codes);
  m.impl("mx_values", &mx_values);
  m.impl("column_sums", &column_sums);
  m.impl("mx_product", &mx_product);
  m.impl("mx_input_grad", &mx_input_grad);
  m.impl("mx_weight_grad", &mx_weight_grad);
  m.impl("linear_input_grad", &linear_input_grad);
  m.impl("gelu_forward", &gelu_forward);
  m.impl("gelu_backward", &gelu_backward);
  m.impl("kept_norm_forward", &kept_norm_forward);
  m.impl("kept_norm_backward", &kept_norm_backward);
}

TORCH_LIBRARY_IMPL(jakal_net_hip, Meta, m) {
  m.impl("mx_codes", &mx_codes_meta);
  m.impl("mx_values", &mx_values_meta);
  m.impl("column_sums", &column_sums_meta);
  m.impl("mx_product", &mx_product_meta);
  m.impl("mx_input_grad", &mx_input_grad_meta);
  m.impl("mx_weight_grad", &mx_weight_grad_meta);
  m.impl("linear_input_grad", &linear_input_grad_meta);
  m.impl("gelu_forward", &gelu_forward_meta);
  m.impl("gelu_backward", &gelu_backward_meta);
  m.impl("kept_norm_forward", &kept_norm_forward_meta);
  m.impl("kept_norm_backward", &kept_norm_backward_meta);
}
