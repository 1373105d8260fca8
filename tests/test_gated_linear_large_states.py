"""The gated recurrence with states near the largest float32: they decay through
the edges of segments (16 steps) and chunks (64 and 128) as the formula says,
forward and backward.

Tolerances: s is formed in about 7 roundings, and the exponential's argument and
result in 3 more, so a step's decay exp(-s) is exact to (7 s + 3) 2**-24 and a
state after t steps to t times that of itself. The product of a segment's or
chunk's decays is a float32 number, whose smallest is 2**-149: a state h may come
out of an edge too large by 2**-149 h, at most 5e-7.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
gpu = pytest.mark.gpu


def gates(l, d, keep):
    """Inputs of zero whose decay is `keep` a step."""
    x = torch.zeros(1, l, d, device=DEV)
    a_gate = torch.full((1, l, d), 1.0, device=DEV)
    rho = 1 / (1 + np.exp(-1.0))
    decay = torch.full((d,), float(np.log(np.expm1(-np.log(keep) / 8.0 / rho))), device=DEV)
    return x, a_gate, torch.zeros_like(x), decay


@gpu
@pytest.mark.parametrize("start", [1e36, -3e38, 1e30])
@pytest.mark.parametrize("keep", [0.5, 0.01, 0.9, 0.1])
def test_large_states_decay_as_the_formula_says(keep, start):
    import mamba_cpu

    print(f"gated scan of a state of {start} kept by {keep}", flush=True)
    l, d = 700, 3
    x, a_gate, x_gate, decay = gates(l, d, keep)
    init = torch.full((1, d), start, device=DEV, requires_grad=True)
    y, last = mamba_cpu.gated_linear_scan_fn(x.requires_grad_(), a_gate, x_gate, decay, initial_state=init,
                                             return_last_state=True)
    want, want_last = O.gated_scan_fwd(x, a_gate, x_gate, decay, init)
    steps = np.arange(1, l + 1)[None, :, None]

    def close(got, want, t, name):
        err = np.abs(got.detach().double().cpu().numpy() - want)
        bound = (3 - 7 * np.log(keep)) * 2.0 ** -24 * t * np.abs(want) + 2.0 ** -149 * abs(start)
        assert np.all(err <= bound), f"{name}: {err.max()}, first at {np.argwhere(err > bound)[0]}"

    close(y, want, steps, "y")
    close(last, want_last, l, "last")
    dlast = torch.full((1, d), start, device=DEV)
    dx, dinit = torch.autograd.grad(last, [x, init], dlast)
    wx, _, _, _, winit = O.gated_scan_bwd(x, a_gate, x_gate, decay, torch.zeros_like(x), init, dlast=dlast)
    close(dx, wx, steps[:, ::-1], "dx")
    close(dinit, winit, l, "dinit")


@gpu
@pytest.mark.parametrize("keep", [0.5, 0.01])
def test_an_infinite_state_stays_one(keep):
    import mamba_cpu

    print(f"gated scan of an infinite state kept by {keep}", flush=True)
    l, d = 700, 3
    x, a_gate, x_gate, decay = gates(l, d, keep)
    init = torch.tensor([[float("inf"), -float("inf"), float("nan")]], device=DEV)
    y = mamba_cpu.gated_linear_scan_fn(x, a_gate, x_gate, decay, initial_state=init)
    assert torch.equal(y[..., :2], init[:, None, :2].expand(-1, l, -1)) and torch.isnan(y[..., 2]).all()
