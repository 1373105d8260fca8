// The torch operators of a recurrent language model beside the scans of
// torch_ops.cpp, in C++ over the C ABI of libmamba_hip.so, in the same manner:
// registered for the CUDA dispatch key (ROCm GPU tensors) with autograd as
// torch::autograd::Functions; argument errors raise ValueError or
// NotImplementedError; outputs and workspaces come from torch's caching
// allocator and launches go to the current stream, without synchronising.
// Shape functions are registered from Python (mamba_cpu/ops/*.py).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>
#include <tuple>

#include "mamba_hip.h"
#include "torch_util.h"

namespace mcpu_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

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

// ---- gated linear recurrence -----------------------------------------------------

void check_gated(const char* name, const Tensor& x, const Tensor& a_gate, const Tensor& x_gate, const Tensor& decay,
                 const optional<Tensor>& init, const optional<Tensor>& seq_idx) {
  for (const optional<Tensor>& t : {opt(x), opt(a_gate), opt(x_gate), opt(decay), init, seq_idx}) check_gpu(name, t);
  TORCH_CHECK_VALUE(x_dtype(x.scalar_type()) && a_gate.scalar_type() == x.scalar_type() &&
                        x_gate.scalar_type() == x.scalar_type(),
                    name, " expects x, a_gate and x_gate of one dtype among float32, bfloat16 and float16");
  TORCH_CHECK_VALUE(x.dim() == 3 && a_gate.sizes() == x.sizes() && x_gate.sizes() == x.sizes(), name,
                    " expects x, a_gate and x_gate of shape (batch, seqlen, dim)");
  TORCH_CHECK_VALUE(decay.scalar_type() == at::kFloat && decay.dim() == 1 && decay.size(0) == x.size(2) &&
                        decay.is_contiguous(),
                    name, " expects a contiguous float32 decay of shape (dim,)");
  TORCH_CHECK_VALUE(!has(init) || (init->scalar_type() == at::kFloat && init->dim() == 2 &&
                                   init->size(0) == x.size(0) && init->size(1) == x.size(2) && init->is_contiguous()),
                    name, " expects a contiguous float32 initial_state of shape (batch, dim)");
  TORCH_CHECK_VALUE(!has(seq_idx) || (seq_idx->scalar_type() == at::kInt && seq_idx->dim() == 2 &&
                                      seq_idx->size(0) == x.size(0) && seq_idx->size(1) == x.size(1) &&
                                      seq_idx->is_contiguous()),
                    name, " expects seq_idx as a contiguous int32 tensor of shape (batch, seqlen)");
}

// A (batch, seqlen, dim) operand within the kernels' reach (a row's channels over
// 16 steps within 4 GiB), copied where it is not.
Tensor in_reach(const Tensor& t) {
  const int64_t reach = (int64_t{1} << 32) / t.element_size(), dim = std::max<int64_t>(t.size(2), 1);
  const bool in = t.stride(2) < reach / dim && t.stride(1) < reach / 16 && dim * t.stride(2) + 16 * t.stride(1) < reach;
  return in ? t : t.contiguous();
}

mcpu_gated_scan_args gated_args(const Tensor& x, const Tensor& a_gate, const Tensor& x_gate, const Tensor& decay,
                                const optional<Tensor>& init, const optional<Tensor>& seq_idx, double c) {
  mcpu_gated_scan_args a;
  std::memset(&a, 0, sizeof(a));
  a.x = x.data_ptr();
  a.a_gate = a_gate.data_ptr();
  a.x_gate = x_gate.data_ptr();
  a.decay = static_cast<const float*>(decay.data_ptr());
  a.initial_state = fptr(init);
  a.seq_idx = has(seq_idx) ? static_cast<const int32_t*>(seq_idx->data_ptr()) : nullptr;
  a.batch = x.size(0);
  a.seqlen = x.size(1);
  a.dim = x.size(2);
  a.c = static_cast<float>(c);
  a.dtype = dtype_tag(x.scalar_type());
  strides3(a.x_stride, x);
  strides3(a.a_stride, a_gate);
  strides3(a.i_stride, x_gate);
  return a;
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_fwd(const Tensor& x_in, const Tensor& a_in, const Tensor& i_in,
                                                  const Tensor& decay, const optional<Tensor>& init,
                                                  const optional<Tensor>& seq_idx, double c, bool save) {
  const char* name = "mamba_cpu::gated_scan_fwd";
  check_gated(name, x_in, a_in, i_in, decay, init, seq_idx);
  c10::DeviceGuard guard(x_in.device());
  const Tensor x = in_reach(x_in), a_gate = in_reach(a_in), x_gate = in_reach(i_in);
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor last = at::empty({x.size(0), x.size(2)}, decay.options());
  mcpu_gated_scan_args a = gated_args(x, a_gate, x_gate, decay, init, seq_idx, c);
  const int64_t kept = save ? static_cast<int64_t>(mcpu_gated_scan_ckpt_size(&a) / sizeof(float)) : 0;
  Tensor ckpt = at::empty({kept}, decay.options());
  a.y = y.data_ptr();
  strides3(a.y_stride, y);
  a.last_state = static_cast<float*>(last.data_ptr());
  a.ckpt = kept > 0 ? static_cast<float*>(ckpt.data_ptr()) : nullptr;
  const size_t nws = mcpu_gated_scan_fwd_workspace_size(&a);
  Tensor ws = workspace(nws, x);
  check_rc(mcpu_gated_scan_fwd(&a, ws_ptr(ws), nws, stream_of(x)), name);
  return {y, last, ckpt};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_scan_bwd(
    const Tensor& dy_in, const optional<Tensor>& dlast, const Tensor& x_in, const Tensor& a_in, const Tensor& i_in,
    const Tensor& decay, const optional<Tensor>& init, const optional<Tensor>& seq_idx, double c,
    const Tensor& ckpt) {
  const char* name = "mamba_cpu::gated_scan_bwd";
  check_gated(name, x_in, a_in, i_in, decay, init, seq_idx);
  for (const optional<Tensor>& t : {opt(dy_in), dlast, opt(ckpt)}) check_gpu(name, t);
  const Tensor x = in_reach(x_in), a_gate = in_reach(a_in), x_gate = in_reach(i_in);
  TORCH_CHECK_VALUE(dy_in.sizes() == x.sizes() && dy_in.scalar_type() == x.scalar_type(), name,
                    " expects dy shaped and typed like x");
  const Tensor dy = in_reach(dy_in);
  TORCH_CHECK_VALUE(!has(dlast) || (dlast->scalar_type() == at::kFloat && dlast->dim() == 2 &&
                                    dlast->size(0) == x.size(0) && dlast->size(1) == x.size(2) &&
                                    dlast->is_contiguous()),
                    name, " expects a contiguous float32 dlast_state of shape (batch, dim)");
  c10::DeviceGuard guard(x.device());
  mcpu_gated_scan_args a = gated_args(x, a_gate, x_gate, decay, init, seq_idx, c);
  TORCH_CHECK_VALUE(ckpt.scalar_type() == at::kFloat && ckpt.is_contiguous() &&
                        ckpt.numel() * sizeof(float) == mcpu_gated_scan_ckpt_size(&a),
                    name, " expects the states that gated_scan_fwd kept");
  Tensor dx = at::empty(x.sizes(), x.options()), da = at::empty(x.sizes(), x.options()),
         di = at::empty(x.sizes(), x.options());
  Tensor ddecay = at::empty(decay.sizes(), decay.options());
  Tensor dinit = has(init) ? at::empty(init->sizes(), init->options()) : at::empty({0}, decay.options());
  a.ckpt = static_cast<float*>(ckpt.data_ptr());
  a.dy = dy.data_ptr();
  strides3(a.dy_stride, dy);
  a.dlast_state = fptr(dlast);
  a.dx = dx.data_ptr();
  strides3(a.dx_stride, dx);
  a.da_gate = da.data_ptr();
  strides3(a.da_stride, da);
  a.dx_gate = di.data_ptr();
  strides3(a.di_stride, di);
  a.ddecay = static_cast<float*>(ddecay.data_ptr());
  a.dinitial_state = has(init) ? static_cast<float*>(dinit.data_ptr()) : nullptr;
  const size_t nws = mcpu_gated_scan_bwd_workspace_size(&a);
  Tensor ws = workspace(nws, x);
  check_rc(mcpu_gated_scan_bwd(&a, ws_ptr(ws), nws, stream_of(x)), name);
  return {dx, da, di, ddecay, dinit};
}

// The states kept for the backward are an output without a gradient.
struct GatedScanFn : public torch::autograd::Function<GatedScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& a_gate, const Tensor& x_gate,
                               const Tensor& decay, const optional<Tensor>& init, const optional<Tensor>& seq_idx,
                               double c, bool save) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::gated_scan_fwd", "")
                         .typed<decltype(gated_scan_fwd)>();
    auto r = op.call(x, a_gate, x_gate, decay, init, seq_idx, c, save);
    const Tensor ckpt = std::get<2>(r);
    ctx->mark_non_differentiable({ckpt});
    ctx->save_for_backward({x, a_gate, x_gate, decay, init.value_or(Tensor()), seq_idx.value_or(Tensor()), ckpt});
    ctx->saved_data["c"] = c;
    ctx->saved_data["save"] = save;
    ctx->set_materialize_grads(false);
    return {std::get<0>(r), std::get<1>(r), ckpt};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor& x = s[0];
    const optional<Tensor> init = opt(s[4]), seq_idx = opt(s[5]);
    TORCH_CHECK_VALUE(ctx->saved_data["save"].toBool(),
                      "mamba_cpu::gated_scan_fwd kept no states (save=False), so it has no backward");
    const Tensor dy = grads[0].defined() ? grads[0].to(x.scalar_type()) : at::zeros_like(x);
    const optional<Tensor> dlast =
        grads[1].defined() ? optional<Tensor>(grads[1].to(at::kFloat).contiguous()) : std::nullopt;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::gated_scan_bwd", "")
                         .typed<decltype(gated_scan_bwd)>();
    auto g = op.call(dy, dlast, x, s[1], s[2], s[3], init, seq_idx, ctx->saved_data["c"].toDouble(), s[6]);
    return {std::get<0>(g), std::get<1>(g), std::get<2>(g), std::get<3>(g), has(init) ? std::get<4>(g) : Tensor(),
            Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> gated_scan_fwd_autograd(const Tensor& x, const Tensor& a_gate,
                                                           const Tensor& x_gate, const Tensor& decay,
                                                           const optional<Tensor>& init,
                                                           const optional<Tensor>& seq_idx, double c, bool save) {
  if (!any_grad({opt(x), opt(a_gate), opt(x_gate), opt(decay), init})) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::gated_scan_fwd", "")
                         .typed<decltype(gated_scan_fwd)>();
    return op.call(x, a_gate, x_gate, decay, init, seq_idx, c, save);
  }
  auto r = GatedScanFn::apply(x, a_gate, x_gate, decay, init, seq_idx, c, save);
  return {r[0], r[1], r[2]};
}

Tensor gated_step(Tensor& state, const Tensor& x, const Tensor& a_gate, const Tensor& x_gate, const Tensor& decay_in,
                  double c, const optional<Tensor>& state_batch_indices) {
  const char* name = "mamba_cpu::gated_step";
  for (const optional<Tensor>& t : {opt(state), opt(x), opt(a_gate), opt(x_gate), opt(decay_in), state_batch_indices})
    check_gpu(name, t);
  TORCH_CHECK_VALUE(x_dtype(x.scalar_type()) && a_gate.scalar_type() == x.scalar_type() &&
                        x_gate.scalar_type() == x.scalar_type(),
                    name, " expects x, a_gate and x_gate of one dtype among float32, bfloat16 and float16");
  TORCH_CHECK_VALUE(x.dim() == 2 && a_gate.sizes() == x.sizes() && x_gate.sizes() == x.sizes(), name,
                    " expects x, a_gate and x_gate of shape (batch, dim)");
  TORCH_CHECK_VALUE(decay_in.dim() == 1 && decay_in.size(0) == x.size(1), name, " expects decay of shape (dim,)");
  TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.dim() == 2 && state.size(1) == x.size(1) &&
                        (has(state_batch_indices) || state.size(0) == x.size(0)),
                    name, " expects a float32 state (batch, dim), or (rows, dim) with state_batch_indices");
  TORCH_CHECK_VALUE(!has(state_batch_indices) ||
                        (state_batch_indices->scalar_type() == at::kInt && state_batch_indices->dim() == 1 &&
                         state_batch_indices->size(0) == x.size(0) && state_batch_indices->is_contiguous()),
                    name, " expects state_batch_indices as a contiguous int32 tensor of shape (batch,)");
  const Tensor decay = f32c(decay_in);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  mcpu_gated_step_args a;
  std::memset(&a, 0, sizeof(a));
  a.state = static_cast<float*>(state.data_ptr());
  a.x = x.data_ptr();
  a.a_gate = a_gate.data_ptr();
  a.x_gate = x_gate.data_ptr();
  a.decay = static_cast<const float*>(decay.data_ptr());
  a.y = y.data_ptr();
  a.batch = x.size(0);
  a.dim = x.size(1);
  a.state_batch = state.size(0);
  a.c = static_cast<float>(c);
  a.dtype = dtype_tag(x.scalar_type());
  for (int i = 0; i < 2; ++i) {
    a.state_stride[i] = state.stride(i);
    a.x_stride[i] = x.stride(i);
    a.a_stride[i] = a_gate.stride(i);
    a.i_stride[i] = x_gate.stride(i);
  }
  a.state_batch_indices =
      has(state_batch_indices) ? static_cast<const int32_t*>(state_batch_indices->data_ptr()) : nullptr;
  check_rc(mcpu_gated_step(&a, stream_of(x)), name);
  return y;
}

Tensor gated_step_inplace(Tensor& state, const Tensor& x, const Tensor& a_gate, const Tensor& x_gate,
                          const Tensor& decay, double c, const optional<Tensor>& state_batch_indices) {
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::gated_step", "")
                         .typed<decltype(gated_step)>();
    y = op.call(state, x, a_gate, x_gate, decay, c, state_batch_indices);
  }
  state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// ---- residual norm -----------------------------------------------------------------

// Rows the kernels take as they are: contiguous elements, any distance.
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous(); }
// The same of a tensor of any dimensions, rows along the last.
Tensor as_rows(const Tensor& t) {
  const int64_t dim = t.size(-1);
  return rows_of(t.dim() == 2 ? t : t.reshape({dim > 0 ? t.numel() / dim : 0, dim}));
}
optional<Tensor> as_rows(const optional<Tensor>& t) { return has(t) ? optional<Tensor>(as_rows(*t)) : std::nullopt; }

void check_norm(const char* name, const Tensor& like, const Tensor& weight, const optional<Tensor>& bias,
                double eps) {
  for (const optional<Tensor>& t : {opt(like), opt(weight), bias}) check_gpu(name, t);
  TORCH_CHECK_VALUE(x_dtype(like.scalar_type()) && like.dim() >= 1, name,
                    " expects x (..., dim) in float32, bfloat16 or float16");
  for (const optional<Tensor>& t : {opt(weight), bias})
    TORCH_CHECK_VALUE(!has(t) || (t->dim() == 1 && t->size(0) == like.size(-1) && t->is_floating_point()), name,
                      " expects weight and bias of shape (dim,) = (", like.size(-1), ",)");
  TORCH_CHECK_VALUE(eps >= 0, name, ": eps must not be negative, got ", eps);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm_fwd(const Tensor& x, const Tensor& weight_in,
                                                    const optional<Tensor>& bias_in, const optional<Tensor>& residual,
                                                    double eps, bool rms, bool want_res, bool res_float32) {
  const char* name = "mamba_cpu::norm_fwd";
  check_norm(name, x, weight_in, bias_in, eps);
  check_gpu(name, residual);
  TORCH_CHECK_VALUE(!has(residual) || (residual->sizes() == x.sizes() &&
                                       (residual->scalar_type() == at::kFloat ||
                                        residual->scalar_type() == x.scalar_type())),
                    name, " expects residual shaped like x, in x's dtype or float32");
  c10::DeviceGuard guard(x.device());
  const Tensor xr = as_rows(x), weight = f32c(weight_in);
  const optional<Tensor> rr = as_rows(residual), bias = f32c(bias_in);
  const at::ScalarType rt = has(rr) ? rr->scalar_type() : (res_float32 ? at::kFloat : x.scalar_type());
  const int64_t rows = xr.size(0);
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor res = want_res ? at::empty(x.sizes(), x.options().dtype(rt)) : at::empty({0}, x.options().dtype(rt));
  Tensor rstd = at::empty({rows}, weight.options());
  Tensor mean = at::empty({rms ? 0 : rows}, weight.options());
  mcpu_norm_args a;
  std::memset(&a, 0, sizeof(a));
  a.x = xr.data_ptr();
  a.residual = ptr(rr);
  a.weight = static_cast<const float*>(weight.data_ptr());
  a.bias = fptr(bias);
  a.rows = rows;
  a.dim = xr.size(1);
  a.x_stride = xr.stride(0);
  a.res_stride = has(rr) ? rr->stride(0) : 0;
  a.y_stride = xr.size(1);
  a.eps = static_cast<float>(eps);
  a.rms = rms ? 1 : 0;
  a.dtype = dtype_tag(x.scalar_type());
  a.res_dtype = dtype_tag(rt);
  a.y = y.data_ptr();
  a.res_out = want_res ? res.data_ptr() : nullptr;
  a.mean = rms ? nullptr : static_cast<float*>(mean.data_ptr());
  a.rstd = static_cast<float*>(rstd.data_ptr());
  check_rc(mcpu_norm_fwd(&a, stream_of(x)), name);
  return {y, res, mean, rstd};
}

// The gradients from z (a float32 residual that norm_fwd returned) or from x
// and residual. `res_kind`: 0 without a residual, 1 one of x's dtype, 2 float32.
std::tuple<Tensor, Tensor, Tensor, Tensor> norm_bwd(const Tensor& dy, const optional<Tensor>& dres_out,
                                                    const optional<Tensor>& x, const optional<Tensor>& residual,
                                                    const optional<Tensor>& z, const Tensor& weight_in, bool has_bias,
                                                    int64_t res_kind, double eps, bool rms, const Tensor& mean,
                                                    const Tensor& rstd) {
  const char* name = "mamba_cpu::norm_bwd";
  check_norm(name, dy, weight_in, std::nullopt, eps);
  for (const optional<Tensor>& t : {dres_out, x, residual, z, opt(mean), opt(rstd)}) check_gpu(name, t);
  const at::ScalarType xt = dy.scalar_type();
  TORCH_CHECK_VALUE(has(x) != has(z), name, " expects either x or z");
  TORCH_CHECK_VALUE(!has(x) || (x->sizes() == dy.sizes() && x->scalar_type() == xt), name,
                    " expects dy shaped and typed like x");
  TORCH_CHECK_VALUE(!has(z) || (z->sizes() == dy.sizes() && z->scalar_type() == at::kFloat && z->is_contiguous()),
                    name, " expects z as norm_fwd returned it in float32");
  const at::ScalarType rt = res_kind == 2 || (res_kind == 0 && has(dres_out) && dres_out->scalar_type() == at::kFloat)
                                ? at::kFloat
                                : xt;
  TORCH_CHECK_VALUE(!has(residual) || (residual->sizes() == dy.sizes() && residual->scalar_type() == rt &&
                                       res_kind > 0),
                    name, " expects residual shaped like x, of the type that residual_kind says");
  TORCH_CHECK_VALUE(!has(dres_out) || (dres_out->sizes() == dy.sizes() && dres_out->scalar_type() == rt), name,
                    " expects dresidual_out shaped like x and typed like the residual");
  const Tensor g = as_rows(dy);
  const int64_t rows = g.size(0), dim = g.size(1);
  TORCH_CHECK_VALUE(rstd.numel() == rows && (rms || mean.numel() == rows) && rstd.scalar_type() == at::kFloat &&
                        mean.scalar_type() == at::kFloat && rstd.is_contiguous() && mean.is_contiguous(),
                    name, " expects the mean and rstd that norm_fwd returned");
  c10::DeviceGuard guard(dy.device());
  const Tensor weight = f32c(weight_in);
  const optional<Tensor> xr = as_rows(x), rr = as_rows(residual);
  const optional<Tensor> dr = has(dres_out) ? optional<Tensor>(dres_out->contiguous()) : std::nullopt;
  Tensor dx = at::empty(dy.sizes(), dy.options());
  Tensor dres = res_kind > 0 ? at::empty(dy.sizes(), dy.options().dtype(rt)) : at::empty({0}, dy.options());
  Tensor dw = at::empty({dim}, weight.options());
  Tensor db = at::empty({has_bias ? dim : 0}, weight.options());
  mcpu_norm_args a;
  std::memset(&a, 0, sizeof(a));
  a.x = ptr(xr);
  a.residual = ptr(rr);
  a.z = fptr(z);
  a.weight = static_cast<const float*>(weight.data_ptr());
  a.bias = has_bias ? a.weight : nullptr;  // only whether there is one
  a.rows = rows;
  a.dim = dim;
  a.x_stride = has(xr) ? xr->stride(0) : 0;
  a.res_stride = has(rr) ? rr->stride(0) : 0;
  a.eps = static_cast<float>(eps);
  a.rms = rms ? 1 : 0;
  a.dtype = dtype_tag(xt);
  a.res_dtype = dtype_tag(rt);
  a.mean = rms ? nullptr : static_cast<float*>(mean.data_ptr());
  a.rstd = static_cast<float*>(rstd.data_ptr());
  a.dy = g.data_ptr();
  a.dy_stride = g.stride(0);
  a.dres_out = ptr(dr);
  a.dx = dx.data_ptr();
  a.dres = res_kind > 0 ? dres.data_ptr() : nullptr;
  a.dweight = static_cast<float*>(dw.data_ptr());
  a.dbias = has_bias ? static_cast<float*>(db.data_ptr()) : nullptr;
  const size_t nws = mcpu_norm_bwd_workspace_size(&a);
  Tensor ws = workspace(nws, dy);
  check_rc(mcpu_norm_bwd(&a, ws_ptr(ws), nws, stream_of(dy)), name);
  return {dx, dres, dw, db};
}

auto norm_fwd_below() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mamba_cpu::norm_fwd", "")
                       .typed<decltype(norm_fwd)>();
  return op;
}

// Keeps the summed residual where it is returned in float32, x and residual
// where it is not.
struct NormFn : public torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               const optional<Tensor>& bias, const optional<Tensor>& residual, double eps, bool rms,
                               bool want_res, bool res_float32) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = norm_fwd_below().call(x, weight, bias, residual, eps, rms, want_res, res_float32);
    const Tensor res = std::get<1>(r), mean = std::get<2>(r), rstd = std::get<3>(r);
    const bool keep_z = want_res && res.scalar_type() == at::kFloat;
    ctx->mark_non_differentiable({mean, rstd});
    ctx->save_for_backward({weight, keep_z ? Tensor() : x, keep_z ? Tensor() : residual.value_or(Tensor()),
                            keep_z ? res : Tensor(), mean, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["want_res"] = want_res;
    ctx->saved_data["bias"] = has(bias);
    ctx->saved_data["kind"] = static_cast<int64_t>(!has(residual) ? 0 : residual->scalar_type() == at::kFloat ? 2 : 1);
    ctx->saved_data["dtype"] = static_cast<int64_t>(x.scalar_type());
    ctx->set_materialize_grads(false);
    return {std::get<0>(r), res, mean, rstd};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const at::ScalarType xt = static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt());
    const Tensor& like = s[1].defined() ? s[1] : s[3];
    const Tensor dy = grads[0].defined() ? grads[0].to(xt) : at::zeros(like.sizes(), like.options().dtype(xt));
    const optional<Tensor> dres_out =
        ctx->saved_data["want_res"].toBool() && grads[1].defined() ? optional<Tensor>(grads[1]) : std::nullopt;
    const int64_t kind = ctx->saved_data["kind"].toInt();
    const bool bias = ctx->saved_data["bias"].toBool();
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::norm_bwd", "")
                         .typed<decltype(norm_bwd)>();
    auto g = op.call(dy, dres_out, opt(s[1]), opt(s[2]), opt(s[3]), s[0], bias, kind,
                     ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool(), s[4], s[5]);
    return {std::get<0>(g), std::get<2>(g).to(s[0].scalar_type()), bias ? std::get<3>(g) : Tensor(),
            kind > 0 ? std::get<1>(g) : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> norm_fwd_autograd(const Tensor& x, const Tensor& weight,
                                                             const optional<Tensor>& bias,
                                                             const optional<Tensor>& residual, double eps, bool rms,
                                                             bool want_res, bool res_float32) {
  if (!any_grad({opt(x), opt(weight), bias, residual})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return norm_fwd_below().call(x, weight, bias, residual, eps, rms, want_res, res_float32);
  }
  auto r = NormFn::apply(x, weight, bias, residual, eps, rms, want_res, res_float32);
  return {r[0], r[1], r[2], r[3]};
}

// ---- embedding ------------------------------------------------------------------------

Tensor embedding_ids(const char* name, const Tensor& ids) {
  check_gpu(name, ids);
  TORCH_CHECK_VALUE((ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) && ids.dim() == 1, name,
                    " expects ids (tokens,) in int32 or int64");
  return ids.contiguous();
}

mcpu_embedding_args embedding_args(const Tensor& ids, int64_t vocab, int64_t dim, double scale,
                                   at::ScalarType dtype) {
  mcpu_embedding_args a;
  std::memset(&a, 0, sizeof(a));
  a.ids = ids.data_ptr();
  a.tokens = ids.size(0);
  a.vocab = vocab;
  a.dim = dim;
  a.scale = static_cast<float>(scale);
  a.dtype = dtype_tag(dtype);
  a.ids64 = ids.scalar_type() == at::kLong ? 1 : 0;
  return a;
}

Tensor embedding_fwd(const Tensor& ids_in, const Tensor& weight_in, double scale) {
  const char* name = "mamba_cpu::embedding_fwd";
  check_gpu(name, weight_in);
  TORCH_CHECK_VALUE(weight_in.dim() == 2 && x_dtype(weight_in.scalar_type()), name,
                    " expects weight (vocab, dim) in float32, bfloat16 or float16");
  c10::DeviceGuard guard(weight_in.device());
  const Tensor ids = embedding_ids(name, ids_in), weight = rows_of(weight_in);
  Tensor out = at::empty({ids.size(0), weight.size(1)}, weight.options());
  mcpu_embedding_args a = embedding_args(ids, weight.size(0), weight.size(1), scale, weight.scalar_type());
  a.weight = weight.data_ptr();
  a.weight_stride = weight.stride(0);
  a.out = out.data_ptr();
  check_rc(mcpu_embedding_fwd(&a, stream_of(weight)), name);
  return out;
}

Tensor embedding_bwd(const Tensor& dout_in, const Tensor& ids_in, int64_t vocab, double scale) {
  const char* name = "mamba_cpu::embedding_bwd";
  check_gpu(name, dout_in);
  TORCH_CHECK_VALUE(dout_in.dim() == 2 && dout_in.size(0) == ids_in.size(0) && x_dtype(dout_in.scalar_type()) &&
                        vocab >= 0,
                    name, " expects dout (tokens, dim) in float32, bfloat16 or float16");
  c10::DeviceGuard guard(dout_in.device());
  const Tensor ids = embedding_ids(name, ids_in), dout = rows_of(dout_in);
  Tensor dw = at::empty({vocab, dout.size(1)}, dout.options());
  mcpu_embedding_args a = embedding_args(ids, vocab, dout.size(1), scale, dout.scalar_type());
  a.dout = dout.data_ptr();
  a.dout_stride = dout.stride(0);
  a.dweight = dw.data_ptr();
  const size_t nws = mcpu_embedding_bwd_workspace_size(&a);
  Tensor ws = workspace(nws, dout);
  check_rc(mcpu_embedding_bwd(&a, ws_ptr(ws), nws, stream_of(dout)), name);
  return dw;
}

struct EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::embedding_fwd", "")
                         .typed<decltype(embedding_fwd)>();
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    return op.call(ids, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::embedding_bwd", "")
                         .typed<decltype(embedding_bwd)>();
    return {Tensor(), op.call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["vocab"].toInt(),
                              ctx->saved_data["scale"].toDouble()),
            Tensor()};
  }
};

Tensor embedding_fwd_autograd(const Tensor& ids, const Tensor& weight, double scale) {
  if (!any_grad({opt(weight)})) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_cpu::embedding_fwd", "")
                         .typed<decltype(embedding_fwd)>();
    return op.call(ids, weight, scale);
  }
  return EmbeddingFn::apply(ids, weight, scale);
}

// ---- sampling -------------------------------------------------------------------------

const Tensor& check_setting(const char* name, const char* what, const Tensor& t, at::ScalarType dtype, int64_t rows) {
  check_gpu(name, t);
  TORCH_CHECK_VALUE(t.scalar_type() == dtype && t.dim() == 1 && t.size(0) == rows && t.is_contiguous(), name,
                    " expects ", what, " per row as a contiguous ", dtype, " tensor of shape (rows,)");
  return t;
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits_in, const optional<Tensor>& noise_in, double temperature,
                                  int64_t top_k, double top_p, double min_p,
                                  const optional<Tensor>& temperature_rows, const optional<Tensor>& top_k_rows,
                                  const optional<Tensor>& top_p_rows, const optional<Tensor>& min_p_rows,
                                  bool logprobs) {
  const char* name = "mamba_cpu::sample";
  check_gpu(name, logits_in);
  check_gpu(name, noise_in);
  TORCH_CHECK_VALUE(logits_in.dim() == 2 && x_dtype(logits_in.scalar_type()), name,
                    " expects logits (rows, vocab) in float32, bfloat16 or float16");
  TORCH_CHECK_VALUE(!has(noise_in) || (noise_in->sizes() == logits_in.sizes() &&
                                       noise_in->scalar_type() == at::kFloat),
                    name, " expects float32 noise shaped like logits");
  c10::DeviceGuard guard(logits_in.device());
  const Tensor logits = rows_of(logits_in);
  const optional<Tensor> noise = has(noise_in) ? optional<Tensor>(rows_of(*noise_in)) : std::nullopt;
  const int64_t rows = logits.size(0);
  Tensor token = at::empty({rows}, logits.options().dtype(at::kLong));
  Tensor logprob = at::empty({logprobs ? rows : 0}, logits.options().dtype(at::kFloat));
  mcpu_sample_args a;
  std::memset(&a, 0, sizeof(a));
  a.logits = logits.data_ptr();
  a.noise = fptr(noise);
  a.rows = rows;
  a.vocab = logits.size(1);
  a.logits_stride = logits.stride(0);
  a.noise_stride = has(noise) ? noise->stride(0) : 0;
  a.temperature = static_cast<float>(temperature);
  a.top_p = static_cast<float>(top_p);
  a.min_p = static_cast<float>(min_p);
  a.top_k = static_cast<int32_t>(std::clamp<int64_t>(top_k, -1, INT32_MAX));  // -1: refused
  if (has(temperature_rows))
    a.temperature_rows = fptr(check_setting(name, "temperature", *temperature_rows, at::kFloat, rows));
  if (has(top_p_rows)) a.top_p_rows = fptr(check_setting(name, "top_p", *top_p_rows, at::kFloat, rows));
  if (has(min_p_rows)) a.min_p_rows = fptr(check_setting(name, "min_p", *min_p_rows, at::kFloat, rows));
  if (has(top_k_rows))
    a.top_k_rows = static_cast<const int32_t*>(check_setting(name, "top_k", *top_k_rows, at::kInt, rows).data_ptr());
  a.token = token.data_ptr<int64_t>();
  a.logprob = logprobs && rows > 0 ? static_cast<float*>(logprob.data_ptr()) : nullptr;
  a.dtype = dtype_tag(logits.scalar_type());
  const size_t nws = mcpu_sample_workspace_size(&a);
  Tensor ws = workspace(nws, logits);
  check_rc(mcpu_sample(&a, ws_ptr(ws), nws, stream_of(logits)), name);
  return {token, logprob};
}

}  // namespace
}  // namespace mcpu_torch

TORCH_LIBRARY_FRAGMENT(mamba_cpu, m) {
  m.def("gated_scan_fwd(Tensor x, Tensor a_gate, Tensor x_gate, Tensor decay, Tensor? initial_state, "
        "Tensor? seq_idx, float c, bool save) -> (Tensor, Tensor, Tensor)");
  m.def("gated_scan_bwd(Tensor dy, Tensor? dlast_state, Tensor x, Tensor a_gate, Tensor x_gate, Tensor decay, "
        "Tensor? initial_state, Tensor? seq_idx, float c, Tensor ckpt) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_step(Tensor(a!) state, Tensor x, Tensor a_gate, Tensor x_gate, Tensor decay, float c, "
        "Tensor? state_batch_indices=None) -> Tensor");
  m.def("norm_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, float eps, bool rms, bool want_residual, "
        "bool residual_float32) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("norm_bwd(Tensor dy, Tensor? dresidual_out, Tensor? x, Tensor? residual, Tensor? z, Tensor weight, "
        "bool has_bias, int residual_kind, float eps, bool rms, Tensor mean, Tensor rstd) -> "
        "(Tensor, Tensor, Tensor, Tensor)");
  m.def("embedding_fwd(Tensor ids, Tensor weight, float scale) -> Tensor");
  m.def("embedding_bwd(Tensor dout, Tensor ids, int vocab, float scale) -> Tensor");
  m.def("sample(Tensor logits, Tensor? noise, float temperature, int top_k, float top_p, float min_p, "
        "Tensor? temperature_rows, Tensor? top_k_rows, Tensor? top_p_rows, Tensor? min_p_rows, bool logprobs) -> "
        "(Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mamba_cpu, CUDA, m) {
  using namespace mcpu_torch;
  m.impl("gated_scan_fwd", &gated_scan_fwd);
  m.impl("gated_scan_bwd", &gated_scan_bwd);
  m.impl("gated_step", &gated_step);
  m.impl("norm_fwd", &norm_fwd);
  m.impl("norm_bwd", &norm_bwd);
  m.impl("embedding_fwd", &embedding_fwd);
  m.impl("embedding_bwd", &embedding_bwd);
  m.impl("sample", &sample);
}

TORCH_LIBRARY_IMPL(mamba_cpu, Autograd, m) {
  using namespace mcpu_torch;
  m.impl("gated_scan_fwd", &gated_scan_fwd_autograd);
  m.impl("norm_fwd", &norm_fwd_autograd);
  m.impl("embedding_fwd", &embedding_fwd_autograd);
  // No gradient flows through a decode step or a choice of tokens.
  m.impl("sample", torch::CppFunction::makeFallthrough());
  m.impl("gated_step", torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(mamba_cpu, ADInplaceOrView, m) {
  using namespace mcpu_torch;
  m.impl("gated_step", &gated_step_inplace);
}
