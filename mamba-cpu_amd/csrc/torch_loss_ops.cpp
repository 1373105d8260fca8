// The torch operators of the head's losses, in C++ over the C ABI of
// libmamba_hip.so, in the manner of torch_lm_ops.cpp.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include <cstring>
#include <tuple>

#include "mamba_hip.h"
#include "torch_lm_util.h"

namespace mcpu_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

mcpu_linear_loss_args loss_args(const char* name, const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                                int64_t ignore_index, double temperature, int64_t reduction) {
  for (const Tensor& t : {hidden, weight, ids}) check_gpu(name, t);
  TORCH_CHECK_VALUE(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1) &&
                        x_dtype(hidden.scalar_type()) && weight.scalar_type() == hidden.scalar_type(),
                    name, " expects hidden (tokens, dim) and weight (vocab, dim) of one type, float32, bfloat16 or "
                    "float16, got ", hidden.sizes(), " ", hidden.scalar_type(), " and ", weight.sizes(), " ",
                    weight.scalar_type());
  TORCH_CHECK_VALUE((ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) && ids.dim() == 2 &&
                        ids.size(0) == hidden.size(0) && ids.is_contiguous(),
                    name, " expects contiguous ids (tokens, k) in int32 or int64");
  for (const Tensor& t : {weight, ids})
    TORCH_CHECK_VALUE(t.device() == hidden.device(), name, " expects its tensors on one device, got ", t.device(),
                      " and ", hidden.device());
  mcpu_linear_loss_args a;
  std::memset(&a, 0, sizeof(a));
  a.hidden = hidden.data_ptr();
  a.weight = weight.data_ptr();
  a.ids = ids.data_ptr();
  a.tokens = hidden.size(0);
  a.vocab = weight.size(0);
  a.dim = hidden.size(1);
  a.k = ids.size(1);
  a.hidden_stride = hidden.stride(0);
  a.weight_stride = weight.stride(0);
  a.ignore_index = ignore_index;
  a.temperature = static_cast<float>(temperature);
  a.dtype = dtype_tag(hidden.scalar_type());
  a.ids64 = ids.scalar_type() == at::kLong ? 1 : 0;
  a.reduction = static_cast<int32_t>(reduction);
  return a;
}

const Tensor& check_like(const char* name, const char* what, const Tensor& t, at::ScalarType dtype,
                         at::IntArrayRef sizes, const Tensor& with) {
  TORCH_CHECK_VALUE(t.device() == with.device() && t.scalar_type() == dtype && t.sizes() == sizes && t.is_contiguous(),
                    name, " expects ", what, " as a contiguous ", dtype, " tensor of ", sizes, " on ", with.device());
  return t;
}

// Bytes of weight kept for the backward: not by its address, which a traced tensor does not tell. Where that alone
// keeps weight from being read in place, the backward lays it out once more.
int64_t kept_bytes(mcpu_linear_loss_args a) {
  a.weight = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(a.weight) & ~uintptr_t{255});
  return static_cast<int64_t>(mcpu_linear_loss_laid_size(&a));
}

// loss, lse, and for the backward the ids' products, the rows' statistics, the teacher's distribution
// (distillation), the rows that count and, where saved, weight as the products read it.
using Losses = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
Losses linear_loss_fwd(const Tensor& hidden_in, const Tensor& weight_in, const Tensor& ids,
                       const optional<Tensor>& teacher, int64_t ignore_index, double temperature, int64_t reduction,
                       bool save) {
  const char* name = "mamba_cpu::linear_loss_fwd";
  check_gpu(name, hidden_in);
  c10::DeviceGuard guard(hidden_in.device());
  TORCH_CHECK_VALUE(hidden_in.dim() == 2 && weight_in.dim() == 2, name, " expects hidden and weight of two dimensions");
  const Tensor hidden = rows_of(hidden_in), weight = rows_of(weight_in);
  mcpu_linear_loss_args a = loss_args(name, hidden, weight, ids, ignore_index, temperature, reduction);
  const auto f32 = hidden.options().dtype(at::kFloat);
  const int64_t tokens = a.tokens;
  if (has(teacher)) a.teacher = static_cast<const float*>(
      check_like(name, "the teacher's logits", *teacher, at::kFloat, ids.sizes(), hidden).data_ptr());
  const at::IntArrayRef all(&tokens, 1), one;
  Tensor loss = at::empty(reduction == MCPU_REDUCE_NONE ? all : one, f32), lse = at::empty({tokens}, f32);
  Tensor picked = at::empty({has(teacher) ? tokens : 0, a.k}, f32), share = at::empty_like(picked);
  Tensor stat = at::empty({4, tokens}, f32);
  Tensor rows = at::empty({tokens + 1}, hidden.options().dtype(at::kInt));
  a.loss = static_cast<float*>(loss.data_ptr());
  a.lse = static_cast<float*>(lse.data_ptr());
  a.picked = has(teacher) ? static_cast<float*>(picked.data_ptr()) : nullptr;
  a.stat = static_cast<float*>(stat.data_ptr());
  a.share = has(teacher) ? static_cast<float*>(share.data_ptr()) : nullptr;
  a.rows = static_cast<int32_t*>(rows.data_ptr());
  const int64_t kept = save ? kept_bytes(a) : 0;
  Tensor laid = at::empty({kept}, hidden.options().dtype(at::kByte));
  if (kept > 0) a.laid = laid.data_ptr();
  const size_t nws = mcpu_linear_loss_fwd_workspace_size(&a);
  Tensor ws = workspace(nws, hidden);
  check_rc(mcpu_linear_loss_fwd(&a, ws_ptr(ws), nws, stream_of(hidden)), name);
  return {loss, lse, picked, stat, share, rows, laid};
}

// Gradients of hidden and weight, each where wanted.
std::tuple<Tensor, Tensor> linear_loss_bwd(const optional<Tensor>& dloss, const optional<Tensor>& dlse,
                                           const Tensor& hidden_in, const Tensor& weight_in, const Tensor& ids,
                                           const Tensor& picked, const Tensor& stat, const Tensor& share,
                                           const Tensor& rows, const Tensor& laid, int64_t ignore_index,
                                           double temperature, int64_t reduction, bool distil, bool want_hidden,
                                           bool want_weight) {
  const char* name = "mamba_cpu::linear_loss_bwd";
  check_gpu(name, hidden_in);
  c10::DeviceGuard guard(hidden_in.device());
  TORCH_CHECK_VALUE(hidden_in.dim() == 2 && weight_in.dim() == 2, name, " expects hidden and weight of two dimensions");
  const Tensor hidden = rows_of(hidden_in), weight = rows_of(weight_in);
  mcpu_linear_loss_args a = loss_args(name, hidden, weight, ids, ignore_index, temperature, reduction);
  Tensor dh = at::empty({want_hidden ? a.tokens : 0, a.dim}, hidden.options());
  Tensor dw = at::empty({want_weight ? a.vocab : 0, a.dim}, weight.options());
  const int64_t n = a.tokens, k = a.k, last = n + 1;
  const int64_t all[2] = {n, k}, stats[2] = {4, n};
  const at::IntArrayRef per(&n, 1), both(all, 2), four(stats, 2), one;
  a.stat = static_cast<float*>(check_like(name, "stat", stat, at::kFloat, four, hidden).data_ptr());
  if (distil) a.picked = static_cast<float*>(check_like(name, "picked", picked, at::kFloat, both, hidden).data_ptr());
  if (distil) a.share = static_cast<float*>(check_like(name, "share", share, at::kFloat, both, hidden).data_ptr());
  a.rows = static_cast<int32_t*>(
      check_like(name, "rows", rows, at::kInt, at::IntArrayRef(&last, 1), hidden).data_ptr());
  const size_t kept = mcpu_linear_loss_laid_size(&a);
  // Not where weight is read in place, as of a saved weight that came back in another layout.
  if (laid.numel() > 0 && kept > 0) {
    TORCH_CHECK_VALUE(static_cast<size_t>(laid.numel()) == kept && laid.scalar_type() == at::kByte &&
                          laid.is_contiguous() && laid.device() == hidden.device(),
                      name, " expects the laid out weight that the forward left");
    a.laid = laid.data_ptr();
  }
  Tensor g, e;
  if (has(dloss)) {
    g = dloss->to(at::kFloat).contiguous();
    a.dloss = static_cast<const float*>(
        check_like(name, "dloss", g, at::kFloat, reduction == MCPU_REDUCE_NONE ? per : one, hidden).data_ptr());
  }
  if (has(dlse)) {
    e = dlse->to(at::kFloat).contiguous();
    a.dlse = static_cast<const float*>(check_like(name, "dlse", e, at::kFloat, per, hidden).data_ptr());
  }
  if (want_hidden) a.dhidden = dh.data_ptr();
  if (want_weight) a.dweight = dw.data_ptr();
  const size_t nws = mcpu_linear_loss_bwd_workspace_size(&a);
  Tensor ws = workspace(nws, hidden);
  check_rc(mcpu_linear_loss_bwd(&a, ws_ptr(ws), nws, stream_of(hidden)), name);
  return {dh, dw};
}

auto loss_fwd_below() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mamba_cpu::linear_loss_fwd", "")
                       .typed<decltype(linear_loss_fwd)>();
  return op;
}

struct LinearLossFn : public torch::autograd::Function<LinearLossFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                               const optional<Tensor>& teacher, int64_t ignore_index, double temperature,
                               int64_t reduction, bool save) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = loss_fwd_below().call(hidden, weight, ids, teacher, ignore_index, temperature, reduction, save);
    const Tensor lse = std::get<1>(r), picked = std::get<2>(r), stat = std::get<3>(r), share = std::get<4>(r),
                 rows = std::get<5>(r), laid = std::get<6>(r);
    ctx->mark_non_differentiable(has(teacher) ? variable_list{lse, picked, stat, share, rows, laid}
                                              : variable_list{picked, stat, share, rows, laid});
    ctx->save_for_backward({hidden, weight, ids, picked, stat, share, rows, laid});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["distil"] = has(teacher);
    ctx->set_materialize_grads(false);
    return {std::get<0>(r), lse, picked, stat, share, rows, laid};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t reduction = ctx->saved_data["reduction"].toInt();
    const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
    optional<Tensor> g = opt(grads[0]);
    if (!has(g) && reduction != MCPU_REDUCE_NONE) g = at::zeros({}, s[3].options());
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::linear_loss_bwd", "")
                         .typed<decltype(linear_loss_bwd)>();
    auto r = op.call(g, opt(grads[1]), s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                     ctx->saved_data["ignore"].toInt(), ctx->saved_data["temperature"].toDouble(), reduction,
                     ctx->saved_data["distil"].toBool(), want_hidden, want_weight);
    return {want_hidden ? std::get<0>(r) : Tensor(), want_weight ? std::get<1>(r) : Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Losses linear_loss_autograd(const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                            const optional<Tensor>& teacher, int64_t ignore_index, double temperature,
                            int64_t reduction, bool save) {
  TORCH_CHECK_VALUE(!any_grad({teacher}), "mamba_cpu::linear_loss_fwd has no gradient of the teacher's logits: detach "
                    "them");
  if (!any_grad({opt(hidden), opt(weight)})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return loss_fwd_below().call(hidden, weight, ids, teacher, ignore_index, temperature, reduction, save);
  }
  auto r = LinearLossFn::apply(hidden, weight, ids, teacher, ignore_index, temperature, reduction, save);
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6]};
}

}  // namespace
}  // namespace mcpu_torch

TORCH_LIBRARY_FRAGMENT(mamba_cpu, m) {
  m.def("linear_loss_fwd(Tensor hidden, Tensor weight, Tensor ids, Tensor? teacher, int ignore_index, "
        "float temperature, int reduction, bool save) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("linear_loss_bwd(Tensor? dloss, Tensor? dlse, Tensor hidden, Tensor weight, Tensor ids, Tensor picked, "
        "Tensor stat, Tensor share, Tensor rows, Tensor laid, int ignore_index, float temperature, int reduction, "
        "bool distil, bool want_hidden, bool want_weight) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mamba_cpu, CUDA, m) {
  using namespace mcpu_torch;
  m.impl("linear_loss_fwd", &linear_loss_fwd);
  m.impl("linear_loss_bwd", &linear_loss_bwd);
}

TORCH_LIBRARY_IMPL(mamba_cpu, Autograd, m) {
  using namespace mcpu_torch;
  m.impl("linear_loss_fwd", &linear_loss_autograd);
  // A gradient of the gradient raises.
  m.impl("linear_loss_bwd", torch::autograd::autogradNotImplementedFallback());
}
