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
    rows = x.shape[0]
    rdt = residual.dtype if residual is not None else torch.float32 if residual_float32 else x.dtype
    return (x.new_empty(x.shape), x.new_empty(x.shape if want_residual else (0,), dtype=rdt),
            weight.new_empty(0 if rms else rows), weight.new_empty(rows))


@torch.library.register_fake("mamba_cpu::norm_bwd")
def _(dy, dresidual_out, x, weight, bias, residual, eps, rms, mean, rstd):
    return (x.new_empty(x.shape), x.new_empty(0) if residual is None else residual.new_empty(x.shape),
            weight.new_empty(weight.shape), weight.new_empty(weight.shape if bias is not None else (0,)))


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
    if x.dim() < 1 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"layer_norm_fn expects x (..., dim) and weight (dim,), got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape:
        raise ValueError(f"bias must have weight's shape {tuple(weight.shape)}, got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dim, in_dtype, res = x.shape[-1], x.dtype, residual
    rows = x.numel() // dim if dim else 0
    xr = (x if in_dtype in _X_DTYPES else x.float()).reshape(rows, dim)
    if res is not None:
        res = (res if res.dtype == xr.dtype else res.float()).reshape(rows, dim)
    wide = residual_in_fp32 and xr.dtype != torch.float32
    want = prenorm and (res is not None or wide)
    y, z, _, _ = torch.ops.mamba_cpu.norm_fwd(
        xr, weight.float().contiguous(), None if bias is None else bias.float().contiguous(), res, float(eps),
        bool(is_rms_norm), want, bool(wide))
    y = y.view(x.shape).to(in_dtype)
    if not prenorm:
        return y
    if not want:
        return y, x
    return y, z.view(x.shape).to(z.dtype if residual is None else residual.dtype)
