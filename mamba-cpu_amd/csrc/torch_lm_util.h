// Helpers shared by the torch operators of a language model beside its scans.
#pragma once

#include "torch_util.h"

#include <initializer_list>

namespace mcpu_torch {
namespace {

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
void* ws_ptr(const Tensor& ws) { return ws.defined() ? ws.data_ptr() : nullptr; }

// Whether a call goes through its autograd function: for a backward, or with a
// forward-mode tangent, which the function refuses (none has a rule for it).
bool any_grad(std::initializer_list<optional<Tensor>> tensors) {
  for (const optional<Tensor>& t : tensors)
    if (has(t) && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
  return false;
}

// Rows the kernels take as they are: contiguous elements, any distance.
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous(); }

}  // namespace
}  // namespace mcpu_torch
