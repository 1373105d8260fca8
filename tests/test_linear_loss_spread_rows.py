"""Rows whose gradients are of very different sizes: confident tokens beside one that is not, and weights of tokens
over many powers of ten. Each row of the gradients is held to its own size.

Tolerances, beside those of test_linear_loss.py (u, KEPT, OUT, lse_tol). A row's unit is its ds's largest (cross
entropy) or its coefficient; r is the unit over the largest of all, of which 2^-16 goes to hidden's rows in dweight's
product and what is left, y = min(1, 2^16 r), to ds:

- ds in f16 pieces has steps of 2^-24 where its unit is 2^13: half of one is 2^-38 of the unit over y; a unit that is
  a power of two doubles it;
- hidden, with its largest magnitude at 2^13 or above, likewise 2^-38 of that over r / y, which is at least 2^-17.
"""

import math

import numpy as np
import pytest
import torch

import mamba_cpu
from oracle import loss as O
from test_linear_loss import DEV, DTYPES, KEPT, OUT, U, WAYS, check, inputs, lse_tol, run_ce, teacher


def held_to_its_size(dtype, h, w, ds, unit, ltol, dh, dw, shares=0.0):
    """shares: what ds has of its row's target distribution, taken from the probabilities, whose error is of their own
    size."""
    hd, wd = np.abs(h.double().numpy()), np.abs(w.double().numpy())
    e = KEPT[dtype] + 2 * float(np.max(ltol))
    r = (unit / unit.max())[:, None]
    low = 2.0 ** -37 * unit[:, None] / np.minimum(1, 2.0 ** 16 * r) if dtype != "bf16" else np.zeros_like(r)
    floor = 2.0 ** -24 if dtype == "f16" else 0.0
    mag = np.abs(ds) + shares
    want_h, want_w = O.grads(h, w, ds)
    assert dtype != "f16" or max(np.abs(want_h).max(), np.abs(want_w).max()) < 60000  # no overflow of the results
    check("dhidden", dh, want_h,
          (e + ds.shape[1] * U) * (mag @ wd) + low * wd.sum(0) + OUT[dtype] * np.abs(want_h) + floor)
    step = 2.0 ** -38 * hd.max() / np.maximum(r, 2.0 ** -17) if dtype != "bf16" else np.zeros_like(r)
    check("dweight", dw, want_w,
          (e + KEPT[dtype] + len(ds) * U) * (mag.T @ hd) + mag.T @ np.broadcast_to(step, hd.shape) + low.T @ hd
          + OUT[dtype] * np.abs(want_w) + floor)


def confident(t, v, beyond):
    """Token 0's target is 60 below word 41. The others' targets are words 0 to 31, above all others by as much as
    leaves those about exp(-beyond[word]) together; the words behind its own have next to nothing of a token, so that
    each word's gradient is of its own tokens' size. No row of weight has anything in columns 48 to 63: there hidden is
    0.5 to 2, to no word's favour."""
    g = torch.Generator().manual_seed(1)
    w = torch.zeros(v, 64)
    w[:32, :32] = torch.eye(32)
    w[41, 32:48] = 1.9375
    ids = torch.arange(t) % 32
    h = torch.zeros(t, 64)
    h[:, :32] = torch.where(torch.arange(32) > ids[:, None], -30.0, 0.0)
    h[torch.arange(t), ids] = math.log(v) + beyond[ids]
    h[:, 48:] = (0.5 + 1.5 * torch.rand(t, 16, generator=g)) * (1 - 2 * torch.randint(2, (t, 16), generator=g))
    h[0, :32], h[0, 32:48] = 0, 1.9375
    ids[0] = 40
    return h, w, ids


def verify(dtype, h, w, ids, dloss):
    h, w = h.to(DTYPES[dtype]), w.to(DTYPES[dtype])
    _, _, dh, dw = run_ce(dtype, h, w, ids, "none", dloss)
    _, lse, _ = O.rows(h, w, ids)
    ds = O.logits_grad(h, w, ids, dloss.double().numpy())
    unit = np.abs(ds).max(1)
    held_to_its_size(dtype, h, w, ds, unit, lse_tol(dtype, h, w, lse) + 2 * U * np.abs(lse), dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_confident_tokens_beside_one_that_is_not(dtype, t, v):
    """Under a loss scale of 2^13; ds of the confident tokens is 4e-3 to 5e-7 of the other's."""
    h, w, ids = confident(t, v, 5.5 + 9 * torch.linspace(0, 1, 32))
    verify(dtype, h, w, ids, torch.full((t,), 2.0 ** 13))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_weights_of_tokens_over_six_powers_of_ten(dtype, t, v):
    """One weight for all tokens of a word, so that each word's row of the gradient has a size of its own."""
    h, w, ids = confident(t, v, torch.full((32,), 3.0))
    dloss = 2.0 ** 10 * 10.0 ** (-6 * (torch.arange(t) % 32) / 31)
    dloss[0] = 2.0 ** 14
    verify(dtype, h, w, ids, dloss)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_distilled_tokens_of_weights_over_eight_powers_of_ten(dtype, t, v):
    h, w, _, g = inputs(dtype, t, v, 64)
    ids, tl = teacher(t, v, 8, g)
    dloss = 2.0 ** 11 * 10.0 ** (-8 * torch.linspace(0, 1, t)) * (1 - 2 * (torch.arange(t) % 2))
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = mamba_cpu.linear_distillation_fn(hg, wg, ids.to(DEV), tl.to(DEV), temperature=1.5, reduction="none")
    dh, dw = torch.autograd.grad(loss, [hg, wg], dloss.to(DEV))
    _, lse, _ = O.rows(h, w, ids, tl, 1.5)
    ds = O.logits_grad(h, w, ids, dloss.double().numpy(), teacher=tl, temperature=1.5)
    unit = 1.5 * np.abs(dloss.double().numpy())
    q, _ = O.shares(ids, v, tl, 1.5)
    shares = np.zeros_like(ds)
    np.put_along_axis(shares, ids.numpy(), q * unit[:, None], 1)
    ltol = lse_tol(dtype, h, w, lse, 1.5) + 2 * U * np.abs(lse) + 8 * U
    held_to_its_size(dtype, h, w, ds, unit, ltol, dh, dw, shares)
