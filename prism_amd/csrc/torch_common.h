// What the PyTorch operator files share: device and type checks, optional
// tensors, the current stream, and the C-ABI's errors as torch errors.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "../../include/prism_bsa.h"

namespace {

using at::Tensor;
using OptT = c10::optional<Tensor>;

// the C-ABI's messages start with the entry point's name
void check_rc(int rc) {
  if (rc == 1) TORCH_CHECK_VALUE(false, prism_last_error());
  TORCH_CHECK(rc == 0, prism_last_error());
}
#define PRISM_TORCH_CALL(fn, ...) check_rc(fn(__VA_ARGS__))

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.defined() && t.is_cuda(), "prism: ", name, " must be a GPU tensor (no CPU path)");
}
void on_gpu(const OptT& t, const char* name) {
  if (t && t->defined()) on_gpu(*t, name);
}

const void* p(const OptT& t) { return t && t->defined() ? t->data_ptr() : nullptr; }
OptT cont(const OptT& t) { return t && t->defined() ? OptT(t->contiguous()) : OptT(); }

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return PRISM_F32;
  if (t.scalar_type() == at::kBFloat16) return PRISM_BF16;
  TORCH_CHECK_TYPE(false, "prism: unsupported dtype ", t.scalar_type(), " (float32 or bfloat16)");
  return -1;
}
at::ScalarType dtype_of_code(int64_t c) {
  TORCH_CHECK_VALUE(c == PRISM_F32 || c == PRISM_BF16, "prism: dtype code ", c, " unknown");
  return c == PRISM_F32 ? at::kFloat : at::kBFloat16;
}
void check_dtype(const Tensor& t, at::ScalarType s, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == s, "prism: ", name, " must be ", s, ", got ", t.scalar_type());
}
void check_dtype(const OptT& t, at::ScalarType s, const char* name) {
  if (t && t->defined()) check_dtype(*t, s, name);
}
at::TensorOptions opts(const Tensor& like, at::ScalarType s) { return like.options().dtype(s); }
Tensor none_like(const Tensor& like) { return at::empty({0}, opts(like, at::kFloat)); }

}  // namespace
