"""Distillation of no tokens, with any number of entries and any temperature: 0 and gradients of 0."""

import ctypes

import pytest
import torch

import mamba_cpu
from test_linear_loss import DEV


@pytest.mark.parametrize("k,temperature", [(5, 1.0), (1, 2.0), (64, 0.5)])
def test_a_block_without_tokens_is_not_refused(k, temperature):
    """Empty tensors have no address, a teacher's logits among them. Nothing is written: no row, no place for a list of
    rows."""
    from mamba_cpu import _C

    a = _C.LinearLossArgs()
    a.tokens, a.vocab, a.dim, a.k, a.hidden_stride, a.weight_stride = 0, 500, 64, k, 64, 64
    a.temperature, a.dtype, a.ids64, a.reduction = temperature, _C.MCPU_BF16, 1, 0
    for name in ("fwd", "bwd"):
        assert getattr(_C.lib, f"mcpu_linear_loss_{name}_workspace_size")(ctypes.byref(a)) == 0
        rc = getattr(_C.lib, f"mcpu_linear_loss_{name}")(ctypes.byref(a), None, 0, None)
        assert rc != _C.MCPU_ERR_INVALID, (name, _C.lib.mcpu_last_error())


@pytest.mark.gpu
@pytest.mark.parametrize("k,temperature", [(5, 1.0), (1, 2.0), (64, 0.5), (0, 2.0)])
@pytest.mark.parametrize("lead", [(0,), (2, 0)])
def test_no_tokens(k, temperature, lead):
    for reduction in ("mean", "sum", "none"):
        h = torch.zeros(*lead, 64, device=DEV, requires_grad=True)
        w = torch.randn(500, 64, device=DEV, requires_grad=True)
        loss = mamba_cpu.linear_distillation_fn(h, w, torch.zeros(*lead, k, dtype=torch.long, device=DEV),
                                                torch.zeros(*lead, k, device=DEV), temperature=temperature,
                                                reduction=reduction)
        assert loss.shape == (lead if reduction == "none" else ())
        dh, dw = torch.autograd.grad(loss.sum(), [h, w])
        assert dh.shape == h.shape and dw.shape == w.shape
        assert torch.count_nonzero(loss) == 0 and torch.count_nonzero(dw) == 0
