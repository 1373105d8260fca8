"""layer_norm_fn on MI355X: layer norm or RMS norm of a residual stream,
forward and backward, over the gfx950 kernels of csrc/norm.hip.

The reference has no such op; the arguments it shares with the mamba_ssm
package's function of this name (mamba_ssm/ops/triton/layer_norm.py) have that
function's order and meaning. Arithmetic is float32 for every storage type.
"""

import torch

from mamba_cpu import _C  # noqa: F401  (loads the operator library)

_X_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


# mamba_cpu::norm_fwd (autograd through mamba_cpu::norm_bwd) is defined in C++
# (csrc/torch_lm_ops.cpp, loaded by mamba_cpu._C); these are its shape
# functions for FakeTensor tracing.


@torch.library.register_fake("mamba_cpu::norm_fwd")
def _(x, weight, bias, residual, eps, rms, want_residual, residual_float32):
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    rdt = residual.dtype if residual is not None else torch.float32 if residual_float32 else x.dtype
    f32 = dict(dtype=torch.float32)
    return (x.new_empty(x.shape), x.new_empty(x.shape if want_residual else (0,), dtype=rdt),
            weight.new_empty(0 if rms else rows, **f32), weight.new_empty(rows, **f32))


@torch.library.register_fake("mamba_cpu::norm_bwd")
def _(dy, dresidual_out, x, residual, z, weight, has_bias, residual_kind, eps, rms, mean, rstd):
    rdt = torch.float32 if residual_kind == 2 else dy.dtype
    f32 = dict(dtype=torch.float32)
    return (dy.new_empty(dy.shape), dy.new_empty(dy.shape if residual_kind else (0,), dtype=rdt),
            weight.new_empty(weight.shape, **f32), weight.new_empty(weight.shape if has_bias else (0,), **f32))


def layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-5, prenorm=False, residual_in_fp32=False,
                  is_rms_norm=False):
    """
    x: (..., dim); weight, bias: (dim,); residual: optional, like x
    With z = x + residual, summed in float32, over each row of dim elements:
        layer norm: (z - mean(z)) / sqrt(var(z) + eps) * weight + bias
        RMS norm (is_rms_norm): z / sqrt(mean(z**2) + eps) * weight + bias
    Returns y like x [, z (prenorm): the new residual, in the residual's dtype;
    without a residual in float32 when residual_in_fp32, else x itself]. y is
    formed from the unrounded z. Differentiable in x, weight, bias and
    residual, through both outputs.
    """
    if x.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {x.device}")
    in_dtype, given, res = x.dtype, x, residual
    if in_dtype not in _X_DTYPES:
        x = x.float()
    if res is not None and res.dtype != x.dtype and res.dtype != torch.float32:
        res = res.float()
    wide = residual_in_fp32 and x.dtype != torch.float32
    want = prenorm and (res is not None or wide)
    # The operator takes any leading dimensions and casts the parameters
    # itself: the common call is one dispatch.
    y, z, _, _ = torch.ops.mamba_cpu.norm_fwd(x, weight, bias, res, eps, is_rms_norm, want, wide)
    y = y.to(in_dtype)
    if not prenorm:
        return y
    if not want:
        return y, x if residual_in_fp32 else given
    return y, z if residual is None else z.to(residual.dtype)
