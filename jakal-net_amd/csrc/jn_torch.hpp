// What the PyTorch operators over the C ABI share (jn_torch.cpp, jn_torch_mx.cpp):
// checks, streams, and what their autograd nodes keep.
#pragma once

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

// What the library declines (2) is a NotImplementedError, for which callers have another form.
void check(int rc) {
  TORCH_CHECK_NOT_IMPLEMENTED(rc != 2, "jakal_net HIP library error ", rc, ": ", jn_last_error());
  TORCH_CHECK(rc == 0, "jakal_net HIP library error ", rc, ": ", jn_last_error());
}

int32_t type_code(const char* what, at::ScalarType type) {
  switch (type) {
    case at::kFloat:
      return JN_F32;
    case at::kBFloat16:
      return JN_BF16;
    case at::kHalf:
      return JN_F16;
    default:
      break;
  }
  TORCH_CHECK_NOT_IMPLEMENTED(false, what, " takes fp32, bf16 and fp16 tensors, got ", type, ".");
}
int32_t type_code(const char* what, const Tensor& t) { return type_code(what, t.scalar_type()); }

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

// ---- layer norm's arguments -----------------------------------------------------
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

}  // namespace
