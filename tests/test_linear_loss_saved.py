"""Hooks on the tensors that the head's losses save for their backward: operands come back contiguous and aligned,
whatever they were in the forward."""

import pytest
import torch

import mamba_cpu
from test_linear_loss import DEV, DTYPES, inputs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first,stride", [(0, 64), (1, 131), (1, 72)])
@pytest.mark.parametrize("t,v", [(40, 260), (1100, 4000)])
def test_saved_tensors_in_host_memory(dtype, first, stride, t, v):
    h, w, ids, _ = inputs(dtype, t, v, 64)
    room = torch.zeros(v * stride + first, device=DEV, dtype=w.dtype)[first:].view(v, stride)
    room[:, :64] = w.to(DEV)
    grads = []
    for save in (False, True):
        hg, wg = h.to(DEV).requires_grad_(), room[:, :64].detach().requires_grad_()
        if save:
            with torch.autograd.graph.save_on_cpu():
                loss = mamba_cpu.linear_cross_entropy_fn(hg, wg, ids.to(DEV))
        else:
            loss = mamba_cpu.linear_cross_entropy_fn(hg, wg, ids.to(DEV))
        grads.append(torch.autograd.grad(loss, [hg, wg]))
    for a, b in zip(*grads):
        if t > 64:  # tiles: the same terms in the same order
            assert torch.equal(a, b)
        else:  # another order of the terms: roundings of float32 sums, then one of ds and of the result
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=2.0 ** -9 * float(a.abs().max()))
