"""layer_norm_fn on rows longer than a workgroup's registers hold (8192): a
value common to a whole row leaves it exactly, as it does shorter rows.

Tolerance, for a constant row of c: a thread adds n = dim / 256 values, so the
mean is off by at most n 2**-24 of c (and 8 more of the tree); what is left of
that once the mean of the rest has been taken out is the same fraction of it,
times rstd, 1 / sqrt(eps): c ((n + 8) 2**-24)**2 / sqrt(eps).
"""

import numpy as np
import pytest
import torch

DEV = "cuda"
gpu = pytest.mark.gpu
EPS = 1e-5


def bound(c, dim):
    return c * ((dim / 256 + 8) * 2.0 ** -24) ** 2 / np.sqrt(EPS) + 1e-6


@gpu
@pytest.mark.parametrize("c", [5.1, 1000.1, -77.7])
@pytest.mark.parametrize("dim", [300, 8192, 8193, 20_000, 100_000])
def test_a_constant_row_is_the_bias(dim, c):
    import mamba_cpu

    print(f"norm of constant rows, {dim} of {c}", flush=True)
    g = torch.Generator().manual_seed(dim)
    x = torch.full((3, dim), c, device=DEV)
    w, b = (torch.randn(dim, generator=g).to(DEV) for _ in range(2))
    x.requires_grad_()
    y = mamba_cpu.layer_norm_fn(x, w, b, eps=EPS)
    assert (y - b).abs().max().item() <= bound(abs(c), dim) * w.abs().max().item()
    # zhat = 0: dz = rstd (t - mean(t)), rstd = 1 / sqrt(eps).
    dy = torch.randn(3, dim, generator=g).to(DEV)
    (dx,) = torch.autograd.grad(y, x, dy)
    t = (dy * w).double()
    want = (t - t.mean(-1, keepdim=True)) / np.sqrt(EPS)
    assert (dx.double() - want).abs().max().item() <= 1e-5 * want.abs().max().item()


@gpu
@pytest.mark.parametrize("dim", [8192, 8193, 20_000])
def test_a_far_mean_keeps_the_spread(dim):
    """Around 1e4 with a spread of 1: the values themselves are rounded to 1e4 x 2**-24."""
    import mamba_cpu

    print(f"norm of rows around 1e4, {dim}", flush=True)
    g = torch.Generator().manual_seed(dim)
    x = (1e4 + torch.randn(4, dim, generator=g)).to(DEV)
    z = x.double()
    want = (z - z.mean(-1, keepdim=True)) / (z.var(-1, unbiased=False, keepdim=True) + EPS).sqrt()
    y = mamba_cpu.layer_norm_fn(x, torch.ones(dim, device=DEV), eps=EPS)
    assert (y.double() - want).abs().max().item() <= 1e-5 * want.abs().max().item()
