// PyTorch operators over the training-step entry points of the C ABI
// (jn_layer_norm_*, jn_cross_entropy_*, jn_grads_*): torch.ops.jakal_net_hip.*.
//
// These operators run for microseconds and a model makes many calls of them,
// so their checks, allocations and autograd nodes are C++: a Python node costs
// several times the kernels.  The C ABI stays free of torch types; this file
// only calls it, on the current stream of the tensors' device.  It holds no
// reference to the library's file: jakal_net_native loads that first, with its
// symbols global.
//
// Each public operator (layer_norm, stabilize, cross_entropy, grad_norm,
// clip_grads) checks its arguments, sets up its autograd node and calls an
// operator below autograd, as does the node's backward (row_norm_*, loss_*,
// list_*).  Those have a kernel for GPU tensors and one for tensors without
// memory, which gives the outputs' sizes and types: fake tensors, and so
// torch.compile, trace through the public ones.  What runs before the inner
// operators therefore reads sizes as symbols and never a tensor's memory.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/empty_strided.h>
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <array>
#include <cmath>
#include <limits>
#include <tuple>
#include <vector>

#include "../../include/jakal_net_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check(int rc) { TORCH_CHECK(rc == 0, "jakal_net HIP library error ", rc, ": ", jn_last_error()); }

int32_t type_code(const char* what, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return JN_F32;
    case at::kBFloat16:
      return JN_BF16;
    case at::kHalf:
      return JN_F16;
    default:
      break;
  }
  TORCH_CHECK_NOT_IMPLEMENTED(false, what, " takes fp32, bf16 and fp16 tensors, got ", t.scalar_type(), ".");
}

void check_gpu(const Tensor& t, const Tensor& first) {
  if (!t.defined()) return;
  TORCH_CHECK(t.is_cuda(), "jakal_net_native ops need GPU tensors, got a tensor on ", t.device(), ".");
  TORCH_CHECK(t.device() == first.device(), "jakal_net_native ops need all tensors on one device.");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

// t as memory holds it row by row, its lazy negation carried out (contiguous()
// alone leaves that to the reader where there is nothing to copy).
Tensor plain(const Tensor& t) {
  if (!t.defined()) return t;
  return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous();
}

Tensor given(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// An inner operator of this library by its name and signature.
template <typename F>
c10::TypedOperatorHandle<F> inner(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool transformed(const Tensor& t) {
  return t.defined() && t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::FuncTorchGradWrapper);
}

// Whether a call has to record a backward.  Forward-mode tangents and
// torch.func's gradients are refused: the operators have none to give.
template <typename... T>
bool records(const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(t) || ...),
                              "jakal_net_native: this operator has no forward-mode derivative.");
  TORCH_CHECK_NOT_IMPLEMENTED(!(transformed(t) || ...),
                              "jakal_net_native: this operator has no derivative under torch.func's transforms.");
  return torch::autograd::compute_requires_grad(t...);
}

template <typename Node>
std::shared_ptr<Node> make_node() {
  return std::shared_ptr<Node>(new Node(), torch::autograd::deleteNode);
}

// A tensor kept for the backward, or none.  Hooks on saved tensors may give back
// another than was saved; the kernels read what its type and size were.
class Kept {
 public:
  void set(const Tensor& t) {
    saved_ = SavedVariable(t, false);
    if (!t.defined()) return;
    device_ = t.device(), type_ = t.scalar_type(), count_ = t.sym_numel(), some_ = true;
  }
  Tensor get() const {
    const Tensor t = saved_.unpack();
    TORCH_CHECK(t.defined() == some_ && (!some_ || (t.device() == device_ && t.scalar_type() == type_ &&
                                                    t.sym_numel() == count_)),
                "jakal_net_native: a saved tensor came back with another device, type or size.");
    return plain(t);
  }
  void reset() { saved_.reset_data(); }

 private:
  SavedVariable saved_;
  c10::Device device_ = at::kCPU;
  at::ScalarType type_ = at::kFloat;
  c10::SymInt count_ = 0;
  bool some_ = false;
};

// The gradients of a backward that is recorded itself (create_graph) raise when
// they are differentiated: the operators have a first derivative only.
variable_list once_differentiable(variable_list grads, bool recorded) {
  if (recorded) {
    const std::shared_ptr<torch::autograd::Node> error(
        new torch::autograd::Error("jakal_net_native: this operator is differentiable once."),
        torch::autograd::deleteNode);
    for (const Tensor& g : grads) torch::autograd::set_history(g, error);
  }
  return grads;
}

// ---- layer norm and stabilisation -------------------------------------------
// weight and bias have to be of one type: x's or fp32 (norm_params sees to it).
void check_norm(const Tensor& state, const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  type_code("layer norm", x);
  if (state.defined()) type_code("stabilize", state);
  TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1 && x.sym_size(-1) < (int64_t(1) << 28),
              "layer norm needs a last axis of 1 to 2^28 - 1 elements, got shape ", x.sym_sizes(), ".");
  TORCH_CHECK(eps >= 0.0, "layer norm eps must not be negative, got ", eps, ".");
  check_gpu(x, x);
  if (state.defined()) {
    TORCH_CHECK(state.sym_sizes() == x.sym_sizes().slice(0, x.dim() - 1), "stabilize: values of shape ", x.sym_sizes(),
                " do not pair with states of shape ", state.sym_sizes(), ".");
    check_gpu(state, x);
  }
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    TORCH_CHECK(p->dim() == 1 && p->sym_size(0) == x.sym_size(-1), "layer norm parameters must be shaped [",
                x.sym_size(-1), "], got ", p->sym_sizes(), ".");
    type_code("layer norm", *p);
    check_gpu(*p, x);
  }
}

// weight and bias contiguous and of one type: x's where both are, else fp32.
void norm_params(const Tensor& x, Tensor& weight, Tensor& bias) {
  bool own = true;
  for (const Tensor* p : {&weight, &bias}) own = own && (!p->defined() || p->scalar_type() == x.scalar_type());
  for (Tensor* p : {&weight, &bias}) {
    if (p->defined()) *p = plain(own ? *p : p->to(at::kFloat));
  }
}

using Norms = std::tuple<Tensor, Tensor, Tensor>;  // state_out (or none), y, stats (or none)
using NormForward = Norms(const std::optional<Tensor>&, const Tensor&, const std::optional<Tensor>&,
                          const std::optional<Tensor>&, double, double, bool);
using NormGrads = std::tuple<Tensor, Tensor, Tensor, Tensor>;  // of state, x, weight, bias, where the mask has them
using NormBackward = NormGrads(const std::optional<Tensor>&, const std::optional<Tensor>&, const std::optional<Tensor>&,
                               const Tensor&, const std::optional<Tensor>&, const Tensor&, double, at::ScalarType,
                               std::array<bool, 4>);

Norms norm_outputs(const Tensor& state, const Tensor& x, bool train) {
  Tensor out, stats;
  if (state.defined()) out = at::empty_like(state);
  if (train) stats = at::empty_symint({x.sym_numel() / x.sym_size(-1), 2}, x.options().dtype(at::kFloat));
  return {out, at::empty_like(x), stats};
}

Norms row_norm_forward_meta(const std::optional<Tensor>& state, const Tensor& x, const std::optional<Tensor>&,
                            const std::optional<Tensor>&, double, double, bool train) {
  return norm_outputs(plain(given(state)), plain(x), train);
}

Norms row_norm_forward(const std::optional<Tensor>& state_in, const Tensor& x_in, const std::optional<Tensor>& weight_in,
                       const std::optional<Tensor>& bias_in, double eps, double scale, bool train) {
  Tensor weight = given(weight_in), bias = given(bias_in);
  check_norm(given(state_in), x_in, weight, bias, eps);
  norm_params(x_in, weight, bias);
  const Tensor x = plain(x_in), state = plain(given(state_in));
  const c10::DeviceGuard guard(x.device());
  const Norms out = norm_outputs(state, x, train);
  const Tensor& param = weight.defined() ? weight : bias;
  check(jn_layer_norm_forward(ptr(state), ptr(x), ptr(weight), ptr(bias), x.numel() / x.size(-1), x.size(-1),
                              (float)scale, (float)eps, type_code("layer norm", x),
                              state.defined() ? type_code("stabilize", state) : JN_F32,
                              param.defined() ? type_code("layer norm", param) : JN_F32, ptr(std::get<0>(out)),
                              ptr(std::get<1>(out)), fptr(std::get<2>(out)), stream_of(x)));
  return out;
}

NormGrads norm_grads(const Tensor& state, const Tensor& x, const Tensor& weight, at::ScalarType bias_type,
                     std::array<bool, 4> mask) {
  return {mask[0] ? at::empty_like(state) : Tensor(), mask[1] ? at::empty_like(x) : Tensor(),
          mask[2] ? at::empty_like(weight) : Tensor(),
          mask[3] ? at::empty_symint({x.sym_size(-1)}, x.options().dtype(bias_type)) : Tensor()};
}

NormGrads row_norm_backward_meta(const std::optional<Tensor>&, const std::optional<Tensor>&,
                                 const std::optional<Tensor>& state, const Tensor& x,
                                 const std::optional<Tensor>& weight, const Tensor&, double, at::ScalarType bias_type,
                                 std::array<bool, 4> mask) {
  return norm_grads(plain(given(state)), plain(x), plain(given(weight)), bias_type, mask);
}

// state, x, weight and stats as the forward had and gave them; the mask: the
// gradients wanted, of state, x, weight and bias.
NormGrads row_norm_backward(const std::optional<Tensor>& g_state_in, const std::optional<Tensor>& g_in,
                            const std::optional<Tensor>& state_in, const Tensor& x_in,
                            const std::optional<Tensor>& weight_in, const Tensor& stats_in, double scale,
                            at::ScalarType bias_type, std::array<bool, 4> mask) {
  const Tensor state = plain(given(state_in)), x = plain(x_in), weight = plain(given(weight_in)), stats = plain(stats_in);
  check_norm(state, x, weight, Tensor(), 0.0);
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  const bool sums = mask[2] || mask[3];
  Tensor g_state = given(g_state_in), g = given(g_in);
  TORCH_CHECK(!mask[0] || (state.defined() && g_state.defined() && g_state.numel() == rows),
              "layer norm backward: a state's gradient needs the state and its output's gradient.");
  TORCH_CHECK((!mask[1] && !sums) || (g.defined() && g.numel() == x.numel()),
              "layer norm backward: the output's gradient has another size than the rows.");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows,
              "layer norm backward: statistics that no forward of these rows gave.");
  TORCH_CHECK(!mask[2] || weight.defined(), "layer norm backward: no weight to take a gradient of.");
  const at::ScalarType param = weight.defined() ? weight.scalar_type() : bias_type;
  TORCH_CHECK((param == at::kFloat || param == x.scalar_type()) && (!mask[3] || bias_type == param),
              "layer norm backward: parameters are fp32 or of the rows' type, and of one type.");
  if (mask[0]) check_gpu(g_state, x), g_state = plain(g_state.to(state.scalar_type()));
  if (mask[1] || sums) check_gpu(g, x), g = plain(g.to(x.scalar_type()));
  check_gpu(stats, x);
  const c10::DeviceGuard guard(x.device());
  const NormGrads out = norm_grads(state, x, weight, bias_type, mask);
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
    ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  }
  const auto code = [](at::ScalarType t) { return t == at::kFloat ? JN_F32 : t == at::kBFloat16 ? JN_BF16 : JN_F16; };
  check(jn_layer_norm_backward(ptr(state), ptr(x), ptr(weight), fptr(stats), mask[0] ? ptr(g_state) : nullptr,
                               mask[1] || sums ? ptr(g) : nullptr, rows, dim, (float)scale, code(x.scalar_type()),
                               state.defined() ? code(state.scalar_type()) : JN_F32, code(param), ptr(gs), ptr(gx),
                               ptr(gw), ptr(gb), ptr(ws), bytes, stream_of(x)));
  return out;
}

struct JakalRowNormBackward : torch::autograd::Node {
  Kept state_, x_, weight_, stats_;
  double scale = 1.0;
  int state_at = -1, y_at = -1;  // the outputs' places, or -1: no gradient comes through it
  at::ScalarType bias_type = at::kFloat;

  std::string name() const override { return "JakalRowNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    state_.reset();
    x_.reset();
    weight_.reset();
    stats_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const Tensor state = state_.get(), x = x_.get(), weight = weight_.get(), stats = stats_.get();
    const Tensor g_state = state_at < 0 ? Tensor() : grads[state_at], g = y_at < 0 ? Tensor() : grads[y_at];
    // wanted: what something takes, of outputs that something used
    std::array<bool, 4> need;
    bool any = false;
    for (int i = 0; i < 4; ++i) {
      need[i] = (i ? g : g_state).defined() && task_should_compute_output(i);
      any = any || need[i];
    }
    if (!any) return variable_list(4);
    static const auto op = inner<NormBackward>("jakal_net_hip::row_norm_backward");
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [gs, gx, gw, gb] =
        op.call(maybe(g_state), maybe(g), maybe(state), x, maybe(weight), stats, scale, bias_type, need);
    return once_differentiable({gs, gx, gw, gb}, recorded);
  }
};

// (state_out, y): tanh(scale * state) where a state is given, and the layer norm of scale * x.
std::tuple<Tensor, Tensor> row_norm(const Tensor& state_in, const Tensor& x_in, const std::optional<Tensor>& weight_in,
                                    const std::optional<Tensor>& bias_in, double eps, double scale) {
  Tensor weight = given(weight_in), bias = given(bias_in);
  check_norm(state_in, x_in, weight, bias, eps);
  norm_params(x_in, weight, bias);
  const Tensor x = plain(x_in), state = plain(state_in);
  std::shared_ptr<JakalRowNormBackward> node;
  if (records(state, x, weight, bias)) {
    node = make_node<JakalRowNormBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(state, x, weight, bias));
  }
  Tensor out, y, stats;
  {
    static const auto op = inner<NormForward>("jakal_net_hip::row_norm_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    std::tie(out, y, stats) = op.call(maybe(state), x, maybe(weight), maybe(bias), eps, scale, node != nullptr);
  }
  if (node) {
    node->state_.set(state);
    node->x_.set(x);
    node->weight_.set(weight);
    node->stats_.set(stats);
    node->scale = scale;
    if (bias.defined()) node->bias_type = bias.scalar_type();
    // an output is differentiable where its own inputs are
    int places = 0;
    if (torch::autograd::compute_requires_grad(state)) {
      node->state_at = places++;
      torch::autograd::set_history(out, node);
    }
    if (torch::autograd::compute_requires_grad(x, weight, bias)) {
      node->y_at = places++;
      torch::autograd::set_history(y, node);
    }
  }
  return {out, y};
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                  double eps) {
  return std::get<1>(row_norm(Tensor(), x, weight, bias, eps, 1.0));
}

std::tuple<Tensor, Tensor> stabilize(const Tensor& state, const Tensor& val, const std::optional<Tensor>& weight,
                                     const std::optional<Tensor>& bias, double eps, double scale) {
  return row_norm(state, val, weight, bias, eps, scale);
}

// ---- cross entropy ------------------------------------------------------------
void check_loss(const Tensor& logits, const Tensor& target) {
  type_code("cross_entropy", logits);
  TORCH_CHECK(logits.dim() >= 1 && target.sym_sizes() == logits.sym_sizes().slice(0, logits.dim() - 1),
              "cross_entropy: logits [..., classes] of shape ", logits.sym_sizes(),
              " do not pair with targets of shape ", target.sym_sizes(), ".");
  TORCH_CHECK(logits.sym_size(-1) >= 1 && logits.sym_size(-1) < (int64_t(1) << 31),
              "cross_entropy needs 1 to 2^31 - 1 classes, got ", logits.sym_size(-1), ".");
  TORCH_CHECK(target.scalar_type() == at::kLong || target.scalar_type() == at::kInt,
              "cross_entropy targets are int64 or int32 class indices, got ", target.scalar_type(), ".");
  check_gpu(logits, logits);
  check_gpu(target, logits);
}

using Losses = std::tuple<Tensor, Tensor, Tensor>;  // the loss, stats (or none), count (none without a reduction)
using LossForward = Losses(const Tensor&, const Tensor&, int64_t, int64_t, bool);
using LossBackward = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&,
                            int64_t, int64_t);

Losses loss_forward_meta(const Tensor& logits, const Tensor& target, int64_t, int64_t reduction, bool train) {
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor stats, count;
  if (train) stats = at::empty_symint({target.sym_numel(), 2}, f32);
  if (reduction) count = at::empty({}, f32);
  return {reduction ? at::empty({}, f32) : at::empty_symint(target.sym_sizes(), f32), stats, count};
}

Losses loss_forward(const Tensor& logits_in, const Tensor& target_in, int64_t ignore_index, int64_t reduction,
                    bool train) {
  check_loss(logits_in, target_in);
  const Tensor logits = plain(logits_in), target = target_in.to(at::kLong).contiguous();
  const c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  const int64_t rows = target.numel();
  const Tensor loss = at::empty(target.sizes(), f32);
  Tensor reduced, stats, count;
  if (reduction) {
    reduced = rows ? at::empty({}, f32) : at::full({}, reduction == 2 ? std::nan("") : 0.0, f32);
    count = at::empty({}, f32);
  }
  if (train) stats = at::empty({rows, 2}, f32);
  if (rows) {
    // the losses of many rows are reduced by many workgroups, in a call of its own
    const size_t bytes = reduction ? jn_cross_entropy_reduce_workspace_bytes(rows) : 0;
    check(jn_cross_entropy_forward(ptr(logits), target.data_ptr<int64_t>(), rows, logits.size(-1), ignore_index,
                                   bytes ? 0 : (int32_t)reduction, type_code("cross_entropy", logits), fptr(loss),
                                   fptr(stats), fptr(reduced), fptr(count), stream_of(logits)));
    if (bytes) {
      const Tensor ws = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
      check(jn_cross_entropy_reduce(fptr(loss), target.data_ptr<int64_t>(), rows, ignore_index, (int32_t)reduction,
                                    fptr(reduced), fptr(count), ptr(ws), bytes, stream_of(logits)));
    }
  }
  return {reduction ? reduced : loss, stats, count};
}

Tensor loss_backward_meta(const Tensor&, const Tensor& logits, const Tensor&, const Tensor&,
                          const std::optional<Tensor>&, int64_t, int64_t) {
  return at::empty_like(plain(logits));
}

Tensor loss_backward(const Tensor& grad, const Tensor& logits_in, const Tensor& target_in, const Tensor& stats_in,
                     const std::optional<Tensor>& count, int64_t ignore_index, int64_t reduction) {
  check_loss(logits_in, target_in);
  const Tensor logits = plain(logits_in), target = target_in.to(at::kLong).contiguous(), stats = plain(stats_in);
  const int64_t rows = target.numel();
  TORCH_CHECK(grad.numel() == (reduction ? 1 : rows) && stats.numel() == 2 * rows &&
                  stats.scalar_type() == at::kFloat &&
                  (reduction != 2 || (count.has_value() && count->defined() && count->numel() == 1 &&
                                      count->scalar_type() == at::kFloat)),
              "cross_entropy backward: a gradient, statistics or a count that are not of these logits' loss.");
  check_gpu(grad, logits);
  check_gpu(stats, logits);
  check_gpu(given(count), logits);
  const c10::DeviceGuard guard(logits.device());
  const Tensor out = at::empty_like(logits);
  if (rows) {
    const Tensor g = plain(grad.to(at::kFloat));
    check(jn_cross_entropy_backward(ptr(logits), target.data_ptr<int64_t>(), fptr(stats), fptr(given(count)), fptr(g),
                                    rows, logits.size(-1), ignore_index, (int32_t)reduction,
                                    type_code("cross_entropy", logits), ptr(out), stream_of(logits)));
  }
  return out;
}

struct JakalCrossEntropyBackward : torch::autograd::Node {
  Kept logits_, target_, stats_, count_;
  int64_t ignore_index = 0, reduction = 0;

  std::string name() const override { return "JakalCrossEntropyBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits_.reset();
    target_.reset();
    stats_.reset();
    count_.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool recorded = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    const Tensor logits = logits_.get(), target = target_.get(), stats = stats_.get(), count = count_.get();
    static const auto op = inner<LossBackward>("jakal_net_hip::loss_backward");
    const at::AutoDispatchBelowADInplaceOrView below;
    return once_differentiable({op.call(grads[0], logits, target, stats, maybe(count), ignore_index, reduction)},
                               recorded);
  }
};

Tensor cross_entropy(const Tensor& logits_in, const Tensor& target_in, int64_t ignore_index, int64_t reduction) {
  check_loss(logits_in, target_in);
  const Tensor logits = plain(logits_in), target = target_in.to(at::kLong).contiguous();
  std::shared_ptr<JakalCrossEntropyBackward> node;
  if (records(logits)) {
    node = make_node<JakalCrossEntropyBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
  }
  Tensor loss, stats, count;
  {
    static const auto op = inner<LossForward>("jakal_net_hip::loss_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    std::tie(loss, stats, count) = op.call(logits, target, ignore_index, reduction, node != nullptr);
  }
  if (node) {
    node->logits_.set(logits);
    node->target_.set(target);
    node->stats_.set(stats);
    node->count_.set(count);
    node->ignore_index = ignore_index;
    node->reduction = reduction;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

// ---- gradient norm and clipping -----------------------------------------------
void check_list(const char* what, at::TensorList tensors, const Tensor& first) {
  for (const Tensor& t : tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == at::kStrided, what, " takes dense tensors, got layout ", t.layout(),
                                ".");
    TORCH_CHECK_NOT_IMPLEMENTED(!t.is_neg(), what, " takes tensors without a pending negation (resolve_neg).");
    type_code(what, t);
    check_gpu(t, first);
  }
}

struct ListArgs {
  std::vector<void*> at;
  std::vector<int64_t> counts;
  std::vector<int32_t> types;

  explicit ListArgs(at::TensorList tensors) {
    at.reserve(tensors.size());
    counts.reserve(tensors.size());
    types.reserve(tensors.size());
    for (const Tensor& t : tensors) {
      at.push_back(t.numel() ? t.data_ptr() : nullptr);
      counts.push_back(t.numel());
      types.push_back(type_code("a list", t));
    }
  }
};

using ListNorm = Tensor(at::TensorList, int64_t);
using ListClip = Tensor(at::TensorList, at::TensorList, double, int64_t);

Tensor list_norm_meta(at::TensorList grads, int64_t) { return at::empty({}, grads[0].options().dtype(at::kFloat)); }

// Tensors that fill their memory.
Tensor list_norm(at::TensorList grads, int64_t kind) {
  TORCH_CHECK_VALUE(!grads.empty(), "grad_norm: an empty list.");
  check_list("grad_norm", grads, grads[0]);
  for (const Tensor& t : grads) TORCH_CHECK(t.is_non_overlapping_and_dense(), "grad_norm: a tensor with gaps.");
  const c10::DeviceGuard guard(grads[0].device());
  const ListArgs in(grads);
  const size_t bytes = jn_grads_workspace_bytes((int64_t)grads.size());
  const auto options = grads[0].options();
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  check(jn_grads_norm(in.at.data(), in.counts.data(), in.types.data(), (int64_t)grads.size(), (int32_t)kind,
                      fptr(norm), ptr(ws), bytes, stream_of(norm)));
  return norm;
}

Tensor grad_norm(at::TensorList grads, int64_t kind) {
  if (grads.empty()) return at::zeros({});
  check_list("grad_norm", grads, grads[0]);
  const at::AutoGradMode off(false);
  std::vector<Tensor> reads;
  reads.reserve(grads.size());
  for (const Tensor& t : grads) reads.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
  static const auto op = inner<ListNorm>("jakal_net_hip::list_norm");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(reads, kind);
}

// g with its elements in memory in the order that o has them in.
bool same_order(const Tensor& g, const Tensor& o) {
  return (g.is_contiguous() && o.is_contiguous()) ||
         (o.is_non_overlapping_and_dense() && g.sym_strides() == o.sym_strides());
}
Tensor in_order_of(const Tensor& g, const Tensor& o) {
  if (same_order(g, o)) return g;
  TORCH_CHECK_NOT_IMPLEMENTED(o.is_non_overlapping_and_dense(),
                              "clip_grads writes tensors that fill their memory, got strides ", o.sym_strides(),
                              " for shape ", o.sym_sizes(), ".");
  Tensor copy = at::empty_strided_symint(o.sym_sizes(), o.sym_strides(), g.options().requires_grad(false));
  copy.copy_(g);
  return copy;
}

Tensor list_clip_meta(at::TensorList grads, at::TensorList, double, int64_t) { return list_norm_meta(grads, 0); }

// Pairs of one shape with their elements in one order in memory.
Tensor list_clip(at::TensorList grads, at::TensorList out, double max_norm, int64_t kind) {
  TORCH_CHECK_VALUE(grads.size() == out.size() && !grads.empty(), "clip_grads: ", grads.size(), " gradients but ",
                    out.size(), " outputs.");
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = out[i];
    check_gpu(g, grads[0]);
    if (!g.is_same(o)) check_gpu(o, grads[0]);
    TORCH_CHECK(!g.is_neg() && !o.is_neg() && g.sizes() == o.sizes() && same_order(g, o),
                "clip_grads: an output of another shape or order than its gradient, or a pending negation.");
  }
  const c10::DeviceGuard guard(grads[0].device());
  const ListArgs in(grads), to(out);
  const int64_t n = (int64_t)grads.size();
  const size_t bytes = jn_grads_workspace_bytes(n);
  const auto options = grads[0].options();
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  check(jn_grads_clip(in.at.data(), to.at.data(), in.counts.data(), in.types.data(), to.types.data(), n, max_norm,
                      (int32_t)kind, fptr(norm), ptr(ws), bytes, stream_of(norm)));
  return norm;
}

Tensor clip_grads(at::TensorList grads, at::TensorList out, double max_norm, int64_t kind) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "clip_grads: max_norm must not be negative, got ", max_norm, ".");
  TORCH_CHECK_VALUE(grads.size() == out.size(), "clip_grads: ", grads.size(), " gradients but ", out.size(),
                    " outputs.");
  if (grads.empty()) return at::zeros({});
  check_list("clip_grads", grads, grads[0]);
  check_list("clip_grads", out, grads[0]);
  const at::AutoGradMode off(false);
  std::vector<Tensor> reads;
  reads.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = out[i];
    if (!g.is_same(o)) {
      TORCH_CHECK_VALUE(o.sym_sizes() == g.sym_sizes(), "clip_grads: an output of shape ", o.sym_sizes(),
                        " for a gradient of shape ", g.sym_sizes(), ".");
      TORCH_CHECK_VALUE(!(o.requires_grad() && o.is_leaf()), "clip_grads: an output requires grad.");
    }
    reads.push_back(in_order_of(g, o));
  }
  Tensor norm;
  {
    static const auto op = inner<ListClip>("jakal_net_hip::list_clip");
    const at::AutoDispatchBelowADInplaceOrView below;
    norm = op.call(reads, out, max_norm, kind);
  }
  for (const Tensor& o : out) {
    if (!o.is_inference()) torch::autograd::impl::bump_version(o);
  }
  return norm;
}

}  // namespace

TORCH_LIBRARY(jakal_net_hip, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("stabilize(Tensor state, Tensor val, Tensor? weight, Tensor? bias, float eps, float scale)"
        " -> (Tensor, Tensor)", &stabilize);
  m.def("cross_entropy(Tensor logits, Tensor target, int ignore_index, int reduction) -> Tensor", &cross_entropy);
  m.def("grad_norm(Tensor[] grads, int kind) -> Tensor", &grad_norm);
  m.def("clip_grads(Tensor[] grads, Tensor(a!)[] out, float max_norm, int kind) -> Tensor", &clip_grads);

  m.def("row_norm_forward(Tensor? state, Tensor x, Tensor? weight, Tensor? bias, float eps, float scale, bool train)"
        " -> (Tensor, Tensor, Tensor)");
  m.def("row_norm_backward(Tensor? grad_state, Tensor? grad_y, Tensor? state, Tensor x, Tensor? weight, Tensor stats,"
        " float scale, ScalarType bias_type, bool[4] mask) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("loss_forward(Tensor logits, Tensor target, int ignore_index, int reduction, bool train)"
        " -> (Tensor, Tensor, Tensor)");
  m.def("loss_backward(Tensor grad, Tensor logits, Tensor target, Tensor stats, Tensor? count, int ignore_index,"
        " int reduction) -> Tensor");
  m.def("list_norm(Tensor[] grads, int kind) -> Tensor");
  m.def("list_clip(Tensor[] grads, Tensor(a!)[] out, float max_norm, int kind) -> Tensor");
}

TORCH_LIBRARY_IMPL(jakal_net_hip, CUDA, m) {
  m.impl("row_norm_forward", &row_norm_forward);
  m.impl("row_norm_backward", &row_norm_backward);
  m.impl("loss_forward", &loss_forward);
  m.impl("loss_backward", &loss_backward);
  m.impl("list_norm", &list_norm);
  m.impl("list_clip", &list_clip);
}

TORCH_LIBRARY_IMPL(jakal_net_hip, Meta, m) {
  m.impl("row_norm_forward", &row_norm_forward_meta);
  m.impl("row_norm_backward", &row_norm_backward_meta);
  m.impl("loss_forward", &loss_forward_meta);
  m.impl("loss_backward", &loss_backward_meta);
  m.impl("list_norm", &list_norm_meta);
  m.impl("list_clip", &list_clip_meta);
}
