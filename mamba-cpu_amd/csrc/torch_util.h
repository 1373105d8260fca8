// Helpers shared by the torch operator sources: argument checks with the
// exception types of the public API, pointers and strides for the C ABI's
// argument blocks, the caller's stream.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <optional>

#include "mamba_hip.h"

namespace mcpu_torch {
namespace {

using at::Tensor;
using std::optional;

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check_rc(int rc, const char* what) {
  if (rc == MCPU_OK) return;
  const char* msg = mcpu_last_error();
  TORCH_CHECK_VALUE(rc != MCPU_ERR_INVALID, what, ": ", msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != MCPU_ERR_UNSUPPORTED, what, ": ", msg);
  TORCH_CHECK(false, what, ": ", msg);
}

bool x_dtype(at::ScalarType s) {
  return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}

int32_t dtype_tag(at::ScalarType s) {
  return s == at::kFloat ? MCPU_F32 : (s == at::kBFloat16 ? MCPU_BF16 : MCPU_F16);
}

bool has(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
const void* ptr(const optional<Tensor>& t) { return has(t) ? t->data_ptr() : nullptr; }
const float* fptr(const optional<Tensor>& t) {
  return has(t) ? static_cast<const float*>(t->data_ptr()) : nullptr;
}

void strides3(int64_t (&s)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
void strides3(int64_t (&s)[3], const optional<Tensor>& t) {
  if (has(t)) strides3(s, *t);
  else s[0] = s[1] = s[2] = 0;
}

void check_gpu(const char* name, const optional<Tensor>& t) {
  if (has(t))
    TORCH_CHECK_VALUE(t->is_cuda(), name, " runs on ROCm GPU tensors, got a tensor on ", t->device());
}

optional<Tensor> opt(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

// Float32 copy of a parameter tensor when it is not already float32 and
// contiguous (the reference computes in float32 whatever they are stored in).
Tensor f32c(const Tensor& t) { return t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.to(at::kFloat).contiguous(); }
optional<Tensor> f32c(const optional<Tensor>& t) { return has(t) ? optional<Tensor>(f32c(*t)) : std::nullopt; }

}  // namespace
}  // namespace mcpu_torch
