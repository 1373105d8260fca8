"""linear_cross_entropy_fn and linear_distillation_fn against the float64 oracle
(oracle/loss.py), both directions, and their refusals.

Tolerances, with u = eps / 2 of float32 (2^-24) and S = max_tv sum_d |h_td w_vd|:

- a logit: products of 16-bit operands are exact, their sum over dim terms is
  off by at most dim u S; float32 operands lose 2^-22 of each factor (three
  products instead of four, two pieces of 11 bits), 4 * 2^-22 S in all;
- lse: the largest logit error, and for exp2, the sum and the logarithm's
  terms 2^-20 (1 + |lse|): arguments up to 2^5 in base 2 are rounded at 2^-20,
  sums of V terms in tiles of 128, at most 200 additions in a row, 200 u < 2^-16
  relative in the worst case and so absolute in the logarithm;
- the loss: both of the above and the rounding of its own sum;
- ds: its rounding to the kept type (bf16 2^-8, f16 2^-11, float32 2^-21), and
  the relative error of p, which is that of its exponent, twice lse's;
- gradients: |ds| |operand| summed, times ds' error and n u for a sum of n
  float32 terms, and the result's own rounding; dweight takes hidden's rows times
  their unit, rounded to the kept type once more; f16 adds its smallest step.
"""

import numpy as np
import pytest
import torch

import mamba_cpu
from oracle import loss as O

DEV = "cuda"
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
KEPT = {"f32": 2.0 ** -21, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
OUT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def inputs(dtype, t, v, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, d, generator=g) / d ** 0.5
    ids = torch.randint(v, (t,), generator=g)
    h = torch.randn(t, d, generator=g) + 6 * torch.rand(t, 1, generator=g) * w[ids]
    return h.to(DTYPES[dtype]), w.to(DTYPES[dtype]), ids, g


def teacher(t, v, k, g):
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(t)])
    return ids, torch.randn(t, k, generator=g) * 3


def finite(h):
    """h without what rows left out may hold."""
    return h.double().nan_to_num(0.0, 0.0, 0.0)


def logit_err(dtype, h, w):
    s = float((finite(h).abs() @ w.double().abs().t()).max())
    return (h.shape[1] * U + (4 * 2.0 ** -22 if dtype == "f32" else 0)) * s


def lse_tol(dtype, h, w, lse, temperature=1.0):
    return logit_err(dtype, h, w) / temperature + 2.0 ** -16 + 2.0 ** -20 * (1 + np.abs(lse))


def check(name, got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = np.abs(got - want)
    ratio = np.where(err == 0, 0.0, err / np.where(tol > 0, tol, 1e-300))
    print(f"  {name}: max|want| {np.abs(want).max(initial=0):.3g} max err {err.max(initial=0):.3g} "
          f"worst err/tol {ratio.max(initial=0):.3g}", flush=True)
    good = bool(np.isfinite(got).all() and (err <= tol).all())
    assert good, f"{name}: {ratio.max()}"


def check_grads(dtype, h, w, ds, ltol, dh, dw):
    """dh, dw against ds's products; ltol: lse's tolerance (per row)."""
    hd, wd = np.abs(finite(h).numpy()), np.abs(w.double().numpy())
    e = KEPT[dtype] + 2 * float(np.max(ltol, initial=0))
    mag = np.abs(ds)
    # A row's ds near 0 is the difference of its coefficient times p and its share.
    top = mag.max(1, keepdims=True) if mag.size else mag
    mag = mag + 2 * float(np.max(ltol, initial=0)) / e * top * (mag > 0)
    floor = 2.0 ** -24 if dtype == "f16" else 0.0
    low = 2.0 ** -36 * np.abs(ds).max(initial=0) if dtype != "bf16" else 0.0
    low += 2.0 ** -100  # ds below that is kept beside the largest, which leaves float32's and f16's range
    want_h, want_w = O.grads(finite(h), w, ds)
    if dh is not None:
        check("dhidden", dh, want_h,
              (e + ds.shape[1] * U) * (mag @ wd) + low * wd.sum(0) + OUT[dtype] * np.abs(want_h) + floor)
    if dw is not None:
        live = (ds != 0).any(1)[:, None]
        check("dweight", dw, want_w,
              (e + KEPT[dtype] + ds.shape[0] * U) * (mag.T @ (hd * live)) + low * (hd * live).sum(0)
              + OUT[dtype] * np.abs(want_w) + floor)


def run_ce(dtype, h, w, ids, reduction, dloss, dlse=None, ignore_index=-100):
    """The op's outputs and gradients; dloss per row ("none") or a number."""
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss, lse = mamba_cpu.linear_cross_entropy_fn(hg, wg, ids.to(DEV), ignore_index=ignore_index,
                                                  reduction=reduction, return_lse=True)
    heads, gs = [loss], [torch.as_tensor(dloss, dtype=torch.float32, device=DEV).expand_as(loss)]
    if dlse is not None:
        heads.append(lse)
        gs.append(dlse.to(DEV))
    dh, dw = torch.autograd.grad(heads, [hg, wg], gs)
    torch.cuda.synchronize()
    return loss, lse, dh, dw


def verify_ce(dtype, h, w, ids, reduction="none", g=None, dlse=None, ignore_index=-100):
    print(f"ce {dtype} {tuple(h.shape)} x {tuple(w.shape)} {reduction}", flush=True)
    t = h.shape[0]
    dloss = torch.randn(t, generator=g) if reduction == "none" else 1.5
    loss, lse, dh, dw = run_ce(dtype, h, w, ids, reduction, dloss, dlse, ignore_index)
    want, want_lse, keep = O.rows(h, w, ids, ignore_index=ignore_index)
    ltol = lse_tol(dtype, h, w, want_lse) * keep
    check("lse", lse, want_lse, ltol)
    ptol = ltol + logit_err(dtype, h, w) * keep + 4 * U * np.abs(want_lse)
    if reduction == "none":
        check("loss", loss, want, ptol)
        per = dloss.double().numpy()
    else:
        n = max(1, keep.sum()) if reduction == "mean" else 1
        check("loss", loss, np.asarray(want.sum() / n), ptol.sum() / n + 32 * U * np.abs(want).sum() / n)
        per = np.full(t, 1.5 / n)
    ds = O.logits_grad(h, w, ids, per, dlse, ignore_index=ignore_index)
    check_grads(dtype, h, w, ds, ltol + 2 * U * np.abs(want_lse), dh, dw)
    return dh, dw


# The ways through the kernels, by tokens and vocabulary: up to 64 tokens; blocks of 64 tokens and 128 rows up to 512 of
# them; tiles of 256 x 256. WAYS has one of each.
WAYS = [(40, 260), (100, 260), (1100, 4000)]
SIZES = [(1, 1, 8), (66, 1, 70), (1, 2, 1), (1, 300, 8), (2, 128, 64), (5, 129, 65), (64, 257, 200), (255, 200, 77),
         (256, 256, 64), (257, 513, 128), (300, 1000, 192), (513, 70, 320), (40, 3001, 33), (700, 6600, 72),
         (129, 33000, 64), (1030, 4200, 33), (520, 8192, 256), (16, 260, 129), (17, 31, 1000), (32, 511, 512),
         (33, 1000, 264), (48, 300, 130), (65, 130, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v,d", SIZES)
def test_cross_entropy(dtype, t, v, d):
    h, w, ids, g = inputs(dtype, t, v, d, seed=t + v)
    verify_ce(dtype, h, w, ids, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("t,v", WAYS)
def test_cross_entropy_reduced(dtype, reduction, t, v):
    h, w, ids, g = inputs(dtype, t, v, 96)
    ids[::3] = -100
    ids[4] = v  # outside the vocabulary
    ids[5] = -1
    verify_ce(dtype, h, w, ids, reduction, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_gradient_of_lse(dtype, t, v):
    h, w, ids, g = inputs(dtype, t, v, 100)
    ids[7:20] = -100
    dlse = torch.randn(t, generator=g)
    verify_ce(dtype, h, w, ids, "none", g, dlse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", [(60, 270), (300, 270), (1100, 4000)])
def test_rows_left_out_reach_nothing(dtype, t, v):
    """NaN and infinities in rows left out: zero there, and the other rows as without them."""
    h, w, ids, g = inputs(dtype, t, v, 128)
    ids[torch.rand(t, generator=g) < 0.7] = -100
    out = ids == -100
    bad = h.clone()
    bad[out] = torch.tensor([float("nan"), float("inf"), -float("inf")]).repeat(43)[:128].to(h.dtype)
    g1, g2 = torch.Generator().manual_seed(1), torch.Generator().manual_seed(1)
    dh, dw = verify_ce(dtype, h, w, ids, "none", g1)
    dh2, dw2 = verify_ce(dtype, bad, w, ids, "none", g2)
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)
    assert torch.count_nonzero(dh2[out.to(DEV)]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", [(1, 270), (300, 270), (1100, 4000)])
def test_no_row_counts(dtype, t, v):
    h, w, ids, _ = inputs(dtype, t, v, 64)
    for reduction in ("mean", "sum", "none"):
        loss, lse, dh, dw = run_ce(dtype, h, w, torch.full_like(ids, -100), reduction, 1.0)
        for x in (loss, lse, dh, dw):
            assert torch.count_nonzero(x) == 0 and torch.isfinite(x).all()


def verify_kd(dtype, h, w, ids, tl, temperature, reduction, g):
    print(f"kd {dtype} {tuple(h.shape)} x {tuple(w.shape)} k {ids.shape[1]} T {temperature} {reduction}", flush=True)
    t = h.shape[0]
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    loss = mamba_cpu.linear_distillation_fn(hg, wg, ids.to(DEV), tl.to(DEV), temperature=temperature,
                                            reduction=reduction)
    dloss = torch.randn(t, generator=g) if reduction == "none" else torch.tensor(1.5)
    dh, dw = torch.autograd.grad(loss, [hg, wg], dloss.to(DEV))
    torch.cuda.synchronize()
    want, lse, keep = O.rows(h, w, ids, tl, temperature)
    ltol = lse_tol(dtype, h, w, lse, temperature) * keep
    # Terms of up to |lse| + |s| + |log q| <= 64 in sums of k entries.
    ptol = temperature ** 2 * (ltol + (logit_err(dtype, h, w) / temperature + 64 * (ids.shape[1] + 8) * U) * keep)
    if reduction == "none":
        check("loss", loss, want, ptol)
        per = dloss.double().numpy()
    else:
        n = max(1, keep.sum()) if reduction == "mean" else 1
        check("loss", loss, np.asarray(want.sum() / n), ptol.sum() / n + 32 * U * np.abs(want).sum() / n)
        per = np.full(t, 1.5 / n)
    ds = O.logits_grad(h, w, ids, per, teacher=tl, temperature=temperature)
    check_grads(dtype, h, w, ds, ltol + 2 * U * np.abs(lse) + 8 * U, dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v,d,k,temperature", [
    (1, 5, 3, 1, 1.0), (3, 300, 64, 8, 2.0), (65, 257, 100, 64, 1.0), (258, 200, 128, 65, 0.5),
    (30, 1500, 77, 200, 1.5), (9, 1100, 64, 1024, 1.0),
    (1100, 4000, 72, 20, 1.5), (600, 7700, 64, 70, 1.0)])
def test_distillation(dtype, t, v, d, k, temperature):
    h, w, _, g = inputs(dtype, t, v, d, seed=t)
    ids, tl = teacher(t, v, k, g)
    verify_kd(dtype, h, w, ids, tl, temperature, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("t,v", [(50, 310), (70, 310), (1100, 4000)])
def test_distillation_entries_left_out(dtype, reduction, t, v):
    """Rows that end early, rows without entries, ids outside the vocabulary with NaN beside them, an id twice."""
    h, w, _, g = inputs(dtype, t, v, 96)
    ids, tl = teacher(t, v, 9, g)
    for i in range(t):
        ids[i, i % 10:] = -1
        tl[i, i % 10:] = float("nan") if i % 2 else -float("inf")
    ids[5, 2] = v
    ids[8, 3] = ids[8, 1]
    ids[9, 0:9] = ids[9, 0]
    tl[13, 1] = -float("inf")
    ids[20], tl[20] = torch.arange(9), -float("inf")
    verify_kd(dtype, h, w, ids, tl, 1.5, reduction, g)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_one_entry_is_cross_entropy(t, v):
    h, w, ids, g = inputs("bf16", t, v, 128)
    ids[3:9] = -1
    ce = mamba_cpu.linear_cross_entropy_fn(h.to(DEV), w.to(DEV), ids.to(DEV), reduction="none")
    kd = mamba_cpu.linear_distillation_fn(h.to(DEV), w.to(DEV), ids[:, None].to(DEV), torch.randn(t, 1, device=DEV),
                                          reduction="none")
    assert (ce - kd).abs().max() <= 8 * U * ce.abs().max()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the float64 oracle's loss along a direction, at the op's own gradient."""
    h, w, ids, g = inputs("f32", 20, 150, 40)
    loss, lse, dh, dw = run_ce("f32", h, w, ids, "sum", 1.0)
    for x, dx, name in ((h, dh, "hidden"), (w, dw, "weight")):
        way = torch.randn(x.shape, generator=g).double()
        step = 1e-5
        ends = []
        for sign in (1, -1):
            moved = x.double() + sign * step * way
            args = (moved, w) if name == "hidden" else (h, moved)
            ends.append(O.rows(*args, ids)[0].sum())
        want = (ends[0] - ends[1]) / (2 * step)
        got = float((dx.double().cpu() * way).sum())
        # Differences: step^2 times a third derivative of order |way|^3; gradient: as in check_grads, 2^-14 overall.
        assert abs(got - want) <= 1e-4 * float((dx.double().cpu() * way).abs().sum()), (name, got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_same_result_every_time(dtype, t, v):
    h, w, ids, g = inputs(dtype, t, v, 192)
    first = run_ce(dtype, h, w, ids, "mean", 1.0)
    for _ in range(3):
        for a, b in zip(first, run_ce(dtype, h, w, ids, "mean", 1.0)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", [(60, 300), (100, 260), (1100, 4000)])
def test_strides_and_offsets(dtype, t, v):
    """Rows a distance apart, an unaligned first element, hidden of more dimensions, int32 targets. Blocks read
    unaligned rows in another order of the terms, so these are held to the oracle, tiles to the bit."""
    h, w, ids, g = inputs(dtype, t, v, 128)
    want = run_ce(dtype, h, w, ids, "none", 1.0)
    hs = torch.zeros(t, 150, dtype=h.dtype, device=DEV)
    ws = torch.full((v, 131), float("nan"), dtype=w.dtype, device=DEV)
    hs[:, 5:133], ws[:, 1:129] = h.to(DEV), w.to(DEV)
    hv, wv = hs[:, 5:133].detach().requires_grad_(), ws[:, 1:129].detach().requires_grad_()
    loss, lse = mamba_cpu.linear_cross_entropy_fn(hv.unflatten(0, (t // 20, 20)), wv,
                                                  ids.to(DEV, torch.int32).view(t // 20, 20), reduction="none",
                                                  return_lse=True)
    assert loss.shape == (t // 20, 20) and lse.shape == (t // 20, 20)
    dh, dw = torch.autograd.grad(loss.sum(), [hv, wv])
    if t > 1000:
        for a, b in zip((loss.view(-1), lse.view(-1), dh, dw), want):
            assert torch.equal(a, b)
    want_loss, want_lse, _ = O.rows(h, w, ids)
    ltol = lse_tol(dtype, h, w, want_lse)
    check("lse", lse.view(-1), want_lse, ltol)
    check("loss", loss.view(-1), want_loss, ltol + logit_err(dtype, h, w) + 4 * U * np.abs(want_lse))
    check_grads(dtype, h, w, O.logits_grad(h, w, ids, np.ones(t)), ltol + 2 * U * np.abs(want_lse), dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("t,v", WAYS)
def test_gradients_of_one_operand_alone(dtype, t, v):
    h, w, ids, _ = inputs(dtype, t, v, 128)
    _, _, dh, dw = run_ce(dtype, h, w, ids, "mean", 1.0)
    for which in (0, 1):
        ops = [h.to(DEV), w.to(DEV)]
        ops[which].requires_grad_()
        mamba_cpu.linear_cross_entropy_fn(*ops, ids.to(DEV)).backward()
        assert torch.equal(ops[which].grad, (dh, dw)[which])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 10, 8), (4, 0, 8), (0, 0, 8)])
def test_empty(shape):
    t, v, d = shape
    h, w = torch.randn(t, d, device=DEV, requires_grad=True), torch.randn(v, d, device=DEV, requires_grad=True)
    ids = torch.zeros(t, dtype=torch.long, device=DEV)
    for reduction in ("mean", "none"):
        loss, lse = mamba_cpu.linear_cross_entropy_fn(h, w, ids, reduction=reduction, return_lse=True)
        kd = mamba_cpu.linear_distillation_fn(h, w, ids[:, None], torch.zeros(t, 1, device=DEV), reduction=reduction)
        none = mamba_cpu.linear_distillation_fn(h, w, ids[:, None][:, :0], torch.zeros(t, 0, device=DEV),
                                                reduction=reduction)
        assert lse.shape == (t,)
        dh, dw = torch.autograd.grad(loss.sum() + kd.sum() + none.sum(), [h, w])
        for x in (loss, kd, none, dh, dw):
            assert torch.count_nonzero(x) == 0
        assert dh.shape == h.shape and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_nan_logits_stay_in_their_row(t, v):
    """A NaN in a row that counts makes that row's loss and gradient NaN, and no other row's."""
    h, w, ids, _ = inputs("bf16", t, v, 64)
    h[7, 3] = float("nan")
    loss, lse, dh, _ = run_ce("bf16", h, w, ids, "none", 1.0)
    bad = torch.arange(t, device=DEV) == 7
    assert torch.isnan(loss[bad]).all() and torch.isnan(lse[bad]).all() and torch.isnan(dh[bad]).all()
    assert torch.isfinite(loss[~bad]).all() and torch.isfinite(dh[~bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,wd", [(torch.bfloat16, torch.float32), (torch.float64, torch.float64)])
def test_other_types_go_by_float32(hd, wd):
    h, w, ids, _ = inputs("f32", 30, 200, 64)
    h, w = h.to(hd), w.to(wd)
    want = run_ce("f32", h.float(), w.float(), ids, "mean", 1.0)
    loss, lse, dh, dw = run_ce("f32", h, w, ids, "mean", 1.0)
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    assert dh.dtype == hd and dw.dtype == wd and torch.equal(dh, want[2].to(hd)) and torch.equal(dw, want[3].to(wd))


# ---- refusals ----


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.linear_cross_entropy_fn(torch.randn(2, 8), torch.randn(5, 8), torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.linear_distillation_fn(torch.randn(2, 8), torch.randn(5, 8), torch.zeros(2, 3, dtype=torch.long),
                                         torch.randn(2, 3))


@pytest.mark.gpu
def test_refusals():
    h, w = torch.randn(4, 8, device=DEV), torch.randn(10, 8, device=DEV)
    ids = torch.zeros(4, dtype=torch.long, device=DEV)
    ce, kd = mamba_cpu.linear_cross_entropy_fn, mamba_cpu.linear_distillation_fn
    top, tl = ids[:, None].expand(4, 3), torch.randn(4, 3, device=DEV)
    for call in (
        lambda: ce(h, w, ids, reduction="max"),
        lambda: ce(h, w[:, :7], ids),
        lambda: ce(h, w[0], ids),
        lambda: ce(h, w, ids[:3]),
        lambda: ce(h, w, ids.float()),
        lambda: ce(h, w, top),
        lambda: ce(h, w, ids.cpu()),
        lambda: ce(h, w.cpu(), ids),
        lambda: ce(h[:, :0], w[:, :0], ids),
        lambda: kd(h, w, top, tl, temperature=0.0),
        lambda: kd(h, w, top, tl, temperature=float("inf")),
        lambda: kd(h, w, top, tl, temperature=float("nan")),
        lambda: kd(h, w, top, tl[:, :2]),
        lambda: kd(h, w, ids, tl),
        lambda: kd(h, w, top, tl.cpu()),
        lambda: kd(h, w, top, tl.clone().requires_grad_()),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        kd(h, w, torch.zeros(4, 1025, dtype=torch.long, device=DEV), torch.zeros(4, 1025, device=DEV))
