"""Temperatures whose inverse or square float32 does not have are refused; those at the ends of what is taken give
finite losses."""

import ctypes
import math

import pytest
import torch

import mamba_cpu
from test_linear_loss import DEV, WAYS, inputs, teacher

OUT = [1e-40, 1e-30, 2.0 ** -61, 2.0 ** 61, 1e30, 3e38]


@pytest.mark.parametrize("temperature", OUT)
def test_temperatures_out_of_range_are_refused(temperature):
    from mamba_cpu import _C

    with pytest.raises(ValueError, match="temperature"):
        mamba_cpu.linear_distillation_fn(torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.long),
                                         torch.zeros(2, 3), temperature=temperature)
    a = _C.LinearLossArgs()
    for name in ("hidden", "weight", "ids", "teacher", "loss", "lse", "picked", "stat", "share", "rows", "dloss"):
        setattr(a, name, 4096)
    a.tokens, a.vocab, a.dim, a.k, a.hidden_stride, a.weight_stride = 300, 500, 64, 3, 64, 64
    a.temperature, a.dtype, a.ids64, a.reduction = temperature, _C.MCPU_BF16, 1, 2
    for name in ("fwd", "bwd"):
        assert getattr(_C.lib, f"mcpu_linear_loss_{name}")(ctypes.byref(a), 4096, 2 ** 60, None) == _C.MCPU_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [2.0 ** -60, 2.0 ** 60])
@pytest.mark.parametrize("t,v", WAYS)
def test_the_ends_of_the_range(temperature, t, v):
    """Hardest: the divergence is the gap between the largest logit and the id's, times the temperature. Softest: both
    are uniform, so it is temperature^2 log(v / k)."""
    h, w, _, g = inputs("f32", t, v, 64)
    ids, tl = teacher(t, v, 5, g)
    loss = mamba_cpu.linear_distillation_fn(h.to(DEV), w.to(DEV), ids.to(DEV), tl.to(DEV), temperature=temperature,
                                            reduction="none").double().cpu()
    if temperature > 1:
        want = torch.full((t,), temperature ** 2 * math.log(v / 5), dtype=torch.double)
    else:
        z = h.double() @ w.double().t()
        top = ids.gather(1, tl.argmax(1, keepdim=True))
        want = temperature * (z.amax(1) - z.gather(1, top)[:, 0])
    # A logit is off by less than 2^-14; the sums of 4000 equal terms by 2^-16.
    assert ((loss - want).abs() <= 2.0 ** -13 * want + temperature * 2.0 ** -13 * (temperature < 1)).all()
