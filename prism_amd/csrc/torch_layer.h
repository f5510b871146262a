// What the operators with C++ autograd nodes share (torch_layer_ops.cpp,
// torch_packed_ops.cpp): outputs, type codes, layouts, and the checks and helpers
// of their gradients.
#pragma once
#include "torch_common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <limits>

namespace {

// An operator's outputs: those that the call has, and no placeholders (an empty
// tensor costs the host 1 us of the 7 that a small call takes)
typedef std::vector<Tensor> Outputs;

int type_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return PRISM_F32;
  if (t.scalar_type() == at::kBFloat16) return PRISM_BF16;
  if (t.scalar_type() == at::kHalf) return PRISM_F16;
  TORCH_CHECK_TYPE(false, "prism: ", name, ": unsupported dtype ", t.scalar_type(), " (float32, bfloat16 or float16)");
  return -1;
}
void same_device(const Tensor& like, const OptT& t, const char* name) {
  on_gpu(t, name);
  if (t && t->defined())
    TORCH_CHECK_VALUE(t->device() == like.device(), "prism: ", name, " is on ", t->device(), ", not on ", like.device());
}
Tensor unit_rows(const Tensor& t) { return t.numel() == 0 || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
int32_t small(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n >= 0 && n <= std::numeric_limits<int32_t>::max(), "prism: ", name, " out of range");
  return (int32_t)n;
}

// x's strides where they are dense with adjacent channels, else contiguous
Tensor like_layout(const Tensor& x) {
  Tensor o = at::empty_like(x);
  return o.numel() == 0 || o.stride(3) == 1 ? o : at::empty(x.sizes(), x.options());
}

// ------------------------------------------------------------------ gradients
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// The nodes reach the kernels through the dispatcher, so that fake tensors (a
// traced or compiled program) get the operators' fake implementations.
template <class F>
auto prism_op(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define PRISM_OP(f) ([]() -> const auto& { static const auto op = prism_op("prism::" #f, &f); return op; }())

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptT& t) { return t && t->defined() && t->requires_grad(); }
// The operators have no forward-mode derivatives.  A dual tensor need not require
// gradients, and below autograd its tangent would be lost without a word: refused.
bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptT& t) { return t && t->defined() && has_tangent(*t); }
template <class... T>
void check_no_tangents(const char* op, const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), "prism: ", op,
                              " has no forward-mode derivatives (an input has a tangent)");
}
// A leaf's gradient is added on the stream on which a graph first took the leaf,
// as long as that graph lives.  If that was the default stream, a backward pass
// captured into a graph would call on a stream that may not take part in a
// capture, which ends the process: refused here, before anything is captured.
void check_captured(const OptT& t) {
  if (!wants_grad(t) || !t->is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
  if (!node) return;
  const auto s = node->stream();
  TORCH_CHECK(!s || s->id() != 0,
              "prism: an input that requires gradients is still held by a graph of eager calls on the default stream; "
              "free that graph (its outputs and losses) or pass a new leaf before capturing, or capture under "
              "torch.no_grad()");
}
template <class... T>
bool grads_wanted(const Tensor& first, const T&... t) {
  if (!at::GradMode::is_enabled() || !(wants_grad(first) || ... || wants_grad(t))) return false;
  if (!first.is_cuda() || first.unsafeGetTensorImpl()->is_python_dispatch()) return true;  // (fake tensors: nothing is launched)
  const hipStream_t stream = stream_of(first);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (stream && hipStreamIsCapturing(stream, &status) == hipSuccess && status != hipStreamCaptureStatusNone) {
    check_captured(first);
    (check_captured(t), ...);
  }
  return true;
}
OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
// gradients that cannot be differentiated again: using them so raises
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)  // (the error's node takes what requires gradients)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "prism: the gradients of this operator cannot be differentiated again", (int64_t)grads.size());
  return error->apply(std::move(grads));
}

}  // namespace
