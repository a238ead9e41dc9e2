// PyTorch operators over the training-step entry points of the C ABI
// (jn_layer_norm_*, jn_cross_entropy_*, jn_grads_*): torch.ops.jakal_net_hip.*.
//
// These operators run for microseconds and a model makes many calls of them,
// so their checks, allocations and autograd nodes are C++: a Python node costs
// several times the kernels.  The C ABI stays free of torch types; this file
// only calls it, on the current stream of the tensors' device.  It holds no
// reference to the library's file: jakal_net_native loads that first, with its
// symbols global.
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

// Whether a call has to record a backward.  Forward-mode tangents are refused:
// the operators have none to give.
template <typename... T>
bool records(const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(t) || ...),
                              "jakal_net_native: this operator has no forward-mode derivative.");
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
    device_ = t.device(), type_ = t.scalar_type(), count_ = t.numel();
  }
  Tensor get() const {
    const Tensor t = saved_.unpack();
    TORCH_CHECK(t.defined() ? t.device() == device_ && t.scalar_type() == type_ && t.numel() == count_ : count_ < 0,
                "jakal_net_native: a saved tensor came back with another device, type or size.");
    return plain(t);
  }
  void reset() { saved_.reset_data(); }

 private:
  SavedVariable saved_;
  c10::Device device_ = at::kCPU;
  at::ScalarType type_ = at::kFloat;
  int64_t count_ = -1;  // none
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
struct NormCall {
  int64_t rows, dim;
  float scale;
  int32_t type, state_type, param_type;
};

struct JakalRowNormBackward : torch::autograd::Node {
  Kept state_, x_, weight_, stats_;
  NormCall call{};
  bool has_state = false;
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
    Tensor g_state = has_state ? grads[0] : Tensor(), g = grads[has_state ? 1 : 0];
    // wanted: what something takes, of outputs that something used
    bool need[4];
    for (int i = 0; i < 4; ++i) need[i] = (i ? g : g_state).defined() && task_should_compute_output(i);
    const bool sums = need[2] || need[3];
    const c10::DeviceGuard guard(x.device());
    Tensor gs, gx, gw, gb, ws;
    if (need[0]) {
      gs = at::empty_like(state);
      g_state = plain(g_state.to(state.scalar_type()));
    }
    if (need[1] || sums) g = plain(g.to(x.scalar_type()));
    if (need[1]) gx = at::empty_like(x);
    if (need[2]) gw = at::empty_like(weight);
    if (need[3]) gb = at::empty({call.dim}, x.options().dtype(bias_type));
    if (call.rows == 0) {
      if (need[2]) gw.zero_();
      if (need[3]) gb.zero_();
    } else if (need[0] || need[1] || sums) {
      size_t bytes = 0;
      if (sums) {
        bytes = jn_layer_norm_backward_workspace_bytes(call.rows, call.dim);
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      }
      check(jn_layer_norm_backward(ptr(state), ptr(x), ptr(weight), fptr(stats), need[0] ? ptr(g_state) : nullptr,
                                   need[1] || sums ? ptr(g) : nullptr, call.rows, call.dim, call.scale, call.type,
                                   call.state_type, call.param_type, ptr(gs), ptr(gx), ptr(gw), ptr(gb), ptr(ws),
                                   bytes, stream_of(x)));
    }
    return once_differentiable({gs, gx, gw, gb}, recorded);
  }
};

// weight and bias contiguous and of one type: x's where both are, else fp32.
void norm_params(const Tensor& x, Tensor& weight, Tensor& bias) {
  bool own = true;
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    TORCH_CHECK(p->dim() == 1 && p->size(0) == x.size(-1), "layer norm parameters must be shaped [", x.size(-1),
                "], got ", p->sizes(), ".");
    type_code("layer norm", *p);
    check_gpu(*p, x);
    own = own && p->scalar_type() == x.scalar_type();
  }
  for (Tensor* p : {&weight, &bias}) {
    if (p->defined()) *p = plain(own ? *p : p->to(at::kFloat));
  }
}

// (state_out, y): tanh(scale * state) where a state is given, and the layer norm of scale * x.
std::tuple<Tensor, Tensor> row_norm(const Tensor& state_in, const Tensor& x_in, const std::optional<Tensor>& weight_in,
                                    const std::optional<Tensor>& bias_in, double eps, double scale) {
  NormCall call;
  call.type = type_code("layer norm", x_in);
  call.state_type = state_in.defined() ? type_code("stabilize", state_in) : JN_F32;
  TORCH_CHECK(x_in.dim() >= 1 && x_in.size(-1) >= 1 && x_in.size(-1) < (1LL << 28),
              "layer norm needs a last axis of 1 to 2^28 - 1 elements, got shape ", x_in.sizes(), ".");
  TORCH_CHECK(eps >= 0.0, "layer norm eps must not be negative, got ", eps, ".");
  check_gpu(x_in, x_in);
  if (state_in.defined()) {
    TORCH_CHECK(state_in.sizes() == x_in.sizes().slice(0, x_in.dim() - 1), "stabilize: values of shape ", x_in.sizes(),
                " do not pair with states of shape ", state_in.sizes(), ".");
    check_gpu(state_in, x_in);
  }
  Tensor weight = given(weight_in), bias = given(bias_in);
  norm_params(x_in, weight, bias);
  const Tensor x = plain(x_in), state = plain(state_in);
  call.dim = x.size(-1);
  call.rows = x.numel() / call.dim;
  call.scale = (float)scale;
  const Tensor& param = weight.defined() ? weight : bias;
  call.param_type = param.defined() ? type_code("layer norm", param) : JN_F32;

  std::shared_ptr<JakalRowNormBackward> node;
  if (records(state, x, weight, bias)) {
    node = make_node<JakalRowNormBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(state, x, weight, bias));
  }
  const c10::DeviceGuard guard(x.device());
  Tensor out, y, stats;
  {
    const at::AutoGradMode off(false);
    y = at::empty_like(x);
    if (state.defined()) out = at::empty_like(state);
    if (node) stats = at::empty({call.rows, 2}, x.options().dtype(at::kFloat));
    check(jn_layer_norm_forward(ptr(state), ptr(x), ptr(weight), ptr(bias), call.rows, call.dim, call.scale,
                                (float)eps, call.type, call.state_type, call.param_type, ptr(out), ptr(y), fptr(stats),
                                stream_of(x)));
  }
  if (node) {
    node->state_.set(state);
    node->x_.set(x);
    node->weight_.set(weight);
    node->stats_.set(stats);
    node->call = call;
    node->has_state = state.defined();
    if (bias.defined()) node->bias_type = bias.scalar_type();
    if (state.defined()) torch::autograd::set_history(out, node);
    torch::autograd::set_history(y, node);
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
    const Tensor logits = logits_.get(), target = target_.get(), stats = stats_.get(),
                 count = count_.get();
    const c10::DeviceGuard guard(logits.device());
    const Tensor out = at::empty_like(logits);
    if (target.numel()) {
      const Tensor g = plain(grads[0].to(at::kFloat));
      check(jn_cross_entropy_backward(ptr(logits), target.data_ptr<int64_t>(), fptr(stats), fptr(count), fptr(g),
                                      target.numel(), logits.size(-1), ignore_index, (int32_t)reduction,
                                      type_code("cross_entropy", logits), ptr(out), stream_of(logits)));
    }
    return once_differentiable({out}, recorded);
  }
};

Tensor cross_entropy(const Tensor& logits_in, const Tensor& target_in, int64_t ignore_index, int64_t reduction) {
  const int32_t type = type_code("cross_entropy", logits_in);
  TORCH_CHECK(logits_in.dim() >= 1 && target_in.sizes() == logits_in.sizes().slice(0, logits_in.dim() - 1),
              "cross_entropy: logits [..., classes] of shape ", logits_in.sizes(),
              " do not pair with targets of shape ", target_in.sizes(), ".");
  TORCH_CHECK(logits_in.size(-1) >= 1 && logits_in.size(-1) < (1LL << 31),
              "cross_entropy needs 1 to 2^31 - 1 classes, got ", logits_in.size(-1), ".");
  TORCH_CHECK(target_in.scalar_type() == at::kLong || target_in.scalar_type() == at::kInt,
              "cross_entropy targets are int64 or int32 class indices, got ", target_in.scalar_type(), ".");
  check_gpu(logits_in, logits_in);
  check_gpu(target_in, logits_in);
  const Tensor logits = plain(logits_in), target = target_in.to(at::kLong).contiguous();
  std::shared_ptr<JakalCrossEntropyBackward> node;
  if (records(logits)) {
    node = make_node<JakalCrossEntropyBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
  }
  const c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const int64_t rows = target.numel();
  Tensor loss, reduced, stats, count;
  {
    const at::AutoGradMode off(false);
    loss = at::empty(target.sizes(), f32);
    if (reduction) {
      reduced = rows ? at::empty({}, f32) : at::full({}, reduction == 2 ? std::nan("") : 0.0, f32);
      count = at::empty({}, f32);
    }
    if (node) stats = at::empty({rows, 2}, f32);
    if (rows) {
      // the losses of many rows are reduced by many workgroups, in a call of its own
      const size_t bytes = reduction ? jn_cross_entropy_reduce_workspace_bytes(rows) : 0;
      check(jn_cross_entropy_forward(ptr(logits), target.data_ptr<int64_t>(), rows, logits.size(-1), ignore_index,
                                     bytes ? 0 : (int32_t)reduction, type, fptr(loss), fptr(stats), fptr(reduced),
                                     fptr(count), stream_of(logits)));
      if (bytes) {
        const Tensor ws = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
        check(jn_cross_entropy_reduce(fptr(loss), target.data_ptr<int64_t>(), rows, ignore_index, (int32_t)reduction,
                                      fptr(reduced), fptr(count), ptr(ws), bytes, stream_of(logits)));
      }
    }
  }
  const Tensor& out = reduction ? reduced : loss;
  if (node) {
    node->logits_.set(logits);
    node->target_.set(target);
    node->stats_.set(stats);
    node->count_.set(count);
    node->ignore_index = ignore_index;
    node->reduction = reduction;
    torch::autograd::set_history(out, node);
  }
  return out;
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

Tensor grad_norm(at::TensorList grads, int64_t kind) {
  if (grads.empty()) return at::zeros({});
  check_list("grad_norm", grads, grads[0]);
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<Tensor> reads;
  reads.reserve(grads.size());
  for (const Tensor& t : grads) reads.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
  const ListArgs in(reads);
  const size_t bytes = jn_grads_workspace_bytes((int64_t)reads.size());
  const auto options = grads[0].options().requires_grad(false);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  check(jn_grads_norm(in.at.data(), in.counts.data(), in.types.data(), (int64_t)reads.size(), (int32_t)kind,
                      fptr(norm), ptr(ws), bytes, stream_of(norm)));
  return norm;
}

// g with its elements in memory in the order that o has them in.
Tensor in_order_of(const Tensor& g, const Tensor& o) {
  if (g.is_contiguous() && o.is_contiguous()) return g;
  TORCH_CHECK_NOT_IMPLEMENTED(o.is_non_overlapping_and_dense(),
                              "clip_grads writes tensors that fill their memory, got strides ", o.strides(),
                              " for shape ", o.sizes(), ".");
  if (g.strides() == o.strides()) return g;
  Tensor copy = at::empty_strided(o.sizes(), o.strides(), g.options().requires_grad(false));
  copy.copy_(g);
  return copy;
}

Tensor clip_grads(at::TensorList grads, at::TensorList out, double max_norm, int64_t kind) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "clip_grads: max_norm must not be negative, got ", max_norm, ".");
  TORCH_CHECK_VALUE(grads.size() == out.size(), "clip_grads: ", grads.size(), " gradients but ", out.size(),
                    " outputs.");
  if (grads.empty()) return at::zeros({});
  check_list("clip_grads", grads, grads[0]);
  check_list("clip_grads", out, grads[0]);
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<Tensor> reads;
  reads.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = out[i];
    if (!g.is_same(o)) {
      TORCH_CHECK_VALUE(o.sizes() == g.sizes(), "clip_grads: an output of shape ", o.sizes(),
                        " for a gradient of shape ", g.sizes(), ".");
      TORCH_CHECK_VALUE(!(o.requires_grad() && o.is_leaf()), "clip_grads: an output requires grad.");
    }
    reads.push_back(in_order_of(g, o));
  }
  const ListArgs in(reads), to(out);
  const int64_t n = (int64_t)reads.size();
  const size_t bytes = jn_grads_workspace_bytes(n);
  const auto options = grads[0].options().requires_grad(false);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
  check(jn_grads_clip(in.at.data(), to.at.data(), in.counts.data(), in.types.data(), to.types.data(), n, max_norm,
                      (int32_t)kind, fptr(norm), ptr(ws), bytes, stream_of(norm)));
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
}
