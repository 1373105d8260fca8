"""Logits over a temperature of 2^16 and more: the softmax is of their differences, however large they are.

Operands are small integers and powers of two, so that every logit is exact in float32 in any order of its sum, and so
are the differences of two of a row. What is left: arguments of exp2 up to 2^7 rounded by 2^-18, sums of up to 200
positive terms in a row, 2^-24 each, together below 2^-16 of a probability; ds's rounding (KEPT) and the
result's (OUT), a sum of float32 terms (U each), float16's smallest step.
"""

import numpy as np
import pytest
import torch

import mamba_cpu
from oracle import loss as O
from test_linear_loss import DEV, DTYPES, KEPT, OUT, U, WAYS, check, inputs, logit_err, run_ce, teacher


def check_ds(dtype, h, w, ds, shares, dh, dw):
    mag, hd, wd = np.abs(ds) + shares, np.abs(h.double().numpy()), np.abs(w.double().numpy())
    e, floor = KEPT[dtype] + 2.0 ** -15, 2.0 ** -24 if dtype == "f16" else 0.0
    low = 2.0 ** -36 * mag.max() if dtype != "bf16" else 0.0  # steps of ds, whose largest coefficient is below 4
    want_h, want_w = O.grads(h, w, ds)
    check("dhidden", dh, want_h,
          (e + ds.shape[1] * U) * (mag @ wd) + low * wd.sum(0) + OUT[dtype] * np.abs(want_h) + floor)
    check("dweight", dw, want_w,
          (e + KEPT[dtype] + len(ds) * U) * (mag.T @ hd) + low * hd.sum(0) + OUT[dtype] * np.abs(want_w) + floor)


def whole(t, v, base, unit):
    """logits = base^2 + an integer times unit^2."""
    g = torch.Generator().manual_seed(t)
    h, w = torch.randint(-2, 3, (t, 64), generator=g) * unit, torch.randint(-1, 2, (v, 64), generator=g) * unit
    h[:, 0] = w[:, 0] = base
    return h, w, g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("base", [2.0 ** 8, 2.0 ** 11])
@pytest.mark.parametrize("t,v", WAYS)
def test_cross_entropy(dtype, base, t, v):
    h, w, g = whole(t, v, base, 1.0)
    best = (h.double() @ w.double().t()).argmax(1)
    ids = torch.where(torch.arange(t) % 3 == 0, best, torch.randint(v, (t,), generator=g))
    dloss = torch.randn(t, generator=g) / 8
    h, w = h.to(DTYPES[dtype]), w.to(DTYPES[dtype])
    loss, lse, dh, dw = run_ce(dtype, h, w, ids, "none", dloss)
    want, want_lse, _ = O.rows(h, w, ids)
    check("loss", loss, want, 2.0 ** -16 * (1 + want))
    check("lse", lse, want_lse, 2.0 ** -22 * want_lse + 2.0 ** -16)
    check_ds(dtype, h, w, O.logits_grad(h, w, ids, dloss.double().numpy()), 0.0, dh, dw)


def run_kd(h, w, ids, tl, temperature, dloss):
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = mamba_cpu.linear_distillation_fn(hg, wg, ids.to(DEV), tl.to(DEV), temperature=temperature, reduction="none")
    dh, dw = torch.autograd.grad(loss, [hg, wg], dloss.to(DEV))
    return loss, dh, dw


def shares_of(ids, tl, v, temperature, dloss):
    q, _ = O.shares(ids, v, tl, temperature)
    shares = np.zeros((len(ids), v))
    np.put_along_axis(shares, ids.numpy(), q * temperature * np.abs(dloss.double().numpy())[:, None], 1)
    return shares


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [16, 22])
@pytest.mark.parametrize("t,v", WAYS)
def test_distillation_at_a_small_temperature(dtype, power, t, v):
    """temperature = 2^-power and logits of 1 + an integer times it."""
    temperature = 2.0 ** -power
    h, w, g = whole(t, v, 1.0, 2.0 ** (-power / 2))
    ids, tl = teacher(t, v, 9, g)
    tl = tl * temperature
    dloss = (1 - 2.0 * (torch.arange(t) % 2)) / temperature / 4
    h, w = h.to(DTYPES[dtype]), w.to(DTYPES[dtype])
    loss, dh, dw = run_kd(h, w, ids, tl, temperature, dloss)
    want, _, _ = O.rows(h, w, ids, tl, temperature)
    # lse and the entries' logits, both near 1 / temperature, are rounded by half a step of float32 there.
    check("loss", loss, want, 8 * U / temperature * temperature ** 2 + 2.0 ** -16 * want)
    ds = O.logits_grad(h, w, ids, dloss.double().numpy(), teacher=tl, temperature=temperature)
    check_ds(dtype, h, w, ds, shares_of(ids, tl, v, temperature, dloss), dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [20, 40])
@pytest.mark.parametrize("t,v", WAYS)
def test_distillation_next_to_temperature_0(dtype, power, t, v):
    """Ordinary logits: the student's distribution is its best word alone, in whatever order the logits' sums were
    formed."""
    h, w, _, g = inputs(dtype, t, v, 64, seed=5)
    z = h.double() @ w.double().t()
    best = z.topk(2, 1)
    near = (best.values[:, 0] - best.values[:, 1]) * 2.0 ** power < 40  # rows whose best two are not apart
    near |= best.values[:, 0] - best.values[:, 1] < 4 * logit_err(dtype, h, w)
    ids, tl = teacher(t, v, 9, g)
    ids[:, 3] = torch.where((ids == best.indices[:, :1]).any(1), ids[:, 3], best.indices[:, 0])
    ids[near] = -1
    assert int(near.sum()) < t // 8
    temperature = 2.0 ** -power
    tl = tl * temperature
    dloss = (1 - 2.0 * (torch.arange(t) % 2)) / temperature / 4
    loss, dh, dw = run_kd(h, w, ids, tl, temperature, dloss)
    assert torch.isfinite(loss).all()
    ds = O.logits_grad(h, w, ids, dloss.double().numpy(), teacher=tl, temperature=temperature)
    check_ds(dtype, h, w, ds, shares_of(ids, tl, v, temperature, dloss), dh, dw)
