"""gated_linear_update with int64 indices past 31 bits: out of range, so skipped,
and no other row's."""

import pytest
import torch

DEV = "cuda"


@pytest.mark.gpu
def test_indices_past_31_bits_are_skipped():
    import mamba_cpu

    print("gated update, indices past 31 bits", flush=True)
    x = torch.randn(6, 40, device=DEV)
    decay = torch.randn(40, device=DEV)
    state = torch.randn(5, 40, device=DEV)
    before = state.clone()
    idx = torch.tensor([2 ** 32, -2 ** 63, 3, 2 ** 63 - 1, 2 ** 33 + 1, 2 ** 31], device=DEV)
    y = mamba_cpu.gated_linear_update(state, x, x, x, decay, state_batch_indices=idx)
    want = mamba_cpu.gated_linear_update(before[3:4].clone(), x[2:3], x[2:3], x[2:3], decay)
    assert torch.equal(y[2:3], want) and torch.equal(state[3:4], want)
    out = [0, 1, 3, 4, 5]
    assert torch.count_nonzero(y[out]) == 0
    rest = [0, 1, 2, 4]
    assert torch.equal(state[rest], before[rest])
