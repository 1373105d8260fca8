"""The head's losses as a program calls them: argument blocks and refusals of the
C ABI, shape functions, streams, HIP graphs, operands past 4 GiB, a vocabulary in
pieces, extreme logits, and RecurrentLM's losses against its own logits.

Graph and stream checks ask for equal bits: sums are in a fixed order. Tolerances
elsewhere are those of test_linear_loss.py.
"""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

import mamba_cpu
from conftest import ROOT
from oracle import loss as O
from test_linear_loss import (KEPT, OUT, U, WAYS, check, inputs, logit_err, lse_tol, run_ce, teacher, verify_ce,
                              verify_kd)

DEV = "cuda"


# ---- without a device ----


def test_argument_block_follows_the_header_and_the_library():
    from mamba_cpu import _C

    cls = _C.LinearLossArgs
    assert _C.lib.mcpu_args_size(b"linear_loss") == ctypes.sizeof(cls)
    header = open(os.path.join(ROOT, "include", "mamba_hip.h")).read()
    body = re.search(r"typedef struct mcpu_linear_loss_args \{(.*?)\} mcpu_linear_loss_args;", header, re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"))):
        first, *more = decl.split(",")
        fields += [first.split()[-1].lstrip("*")] + [m.strip().lstrip("*") for m in more]
    assert [f[0] for f in cls._fields_] == fields


def _block(**kw):
    """A block of addresses that nothing follows, valid but for kw."""
    from mamba_cpu import _C

    a = _C.LinearLossArgs()
    for name in ("hidden", "weight", "ids", "loss", "lse", "picked", "stat", "rows", "dloss", "dhidden", "dweight"):
        setattr(a, name, 4096)
    a.tokens, a.vocab, a.dim, a.k, a.hidden_stride, a.weight_stride = 300, 500, 64, 1, 64, 64
    a.temperature, a.dtype, a.ids64, a.reduction = 1.0, _C.MCPU_BF16, 1, 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,unsupported", [
    (dict(tokens=-1), False), (dict(vocab=-1), False), (dict(dim=-1), False), (dict(dim=0), False),
    (dict(k=-1), False), (dict(hidden_stride=-1), False), (dict(weight_stride=-1), False), (dict(dtype=3), False),
    (dict(ids64=2), False), (dict(reduction=3), False), (dict(reduction=-1), False), (dict(temperature=0.0), False),
    (dict(temperature=-1.0), False), (dict(temperature=float("nan")), False), (dict(temperature=float("inf")), False),
    (dict(temperature=2.0), False), (dict(k=2), False), (dict(share=4096, dlse=4096), False),
    (dict(tokens=2 ** 26 + 1), True), (dict(vocab=2 ** 24 + 1), True), (dict(dim=2 ** 20 + 1), True),
    (dict(share=4096, teacher=4096, k=1025), True), (dict(hidden=0), False), (dict(weight=0), False),
    (dict(ids=0), False), (dict(stat=0), False), (dict(rows=0), False),
    (dict(share=4096, teacher=4096, picked=0), False)])
def test_bad_blocks_are_refused_before_a_device_is_touched(kw, unsupported):
    from mamba_cpu import _C

    want = _C.MCPU_ERR_UNSUPPORTED if unsupported else _C.MCPU_ERR_INVALID
    a = _block(**kw)
    for name in ("fwd", "bwd"):
        assert getattr(_C.lib, f"mcpu_linear_loss_{name}_workspace_size")(ctypes.byref(a)) == 0
        assert getattr(_C.lib, f"mcpu_linear_loss_{name}")(ctypes.byref(a), 4096, 2 ** 60, None) == want, name
        assert _C.lib.mcpu_last_error()


def test_missing_results_and_workspaces_are_refused():
    from mamba_cpu import _C

    L = _C.lib
    assert L.mcpu_linear_loss_fwd(None, None, 0, None) == _C.MCPU_ERR_INVALID
    for kw in (dict(loss=0), dict(lse=0), dict(teacher=4096)):
        assert L.mcpu_linear_loss_fwd(ctypes.byref(_block(**kw)), 4096, 2 ** 60, None) == _C.MCPU_ERR_INVALID
    assert L.mcpu_linear_loss_bwd(ctypes.byref(_block(dloss=0)), 4096, 2 ** 60, None) == _C.MCPU_ERR_INVALID
    for tokens in (8, 300):
        a = _block(tokens=tokens)
        for name in ("fwd", "bwd"):
            need = getattr(L, f"mcpu_linear_loss_{name}_workspace_size")(ctypes.byref(a))
            assert need > 0
            f = getattr(L, f"mcpu_linear_loss_{name}")
            assert f(ctypes.byref(a), 4096, need - 1, None) == _C.MCPU_ERR_INVALID
            assert f(ctypes.byref(a), None, need, None) == _C.MCPU_ERR_INVALID


def test_workspaces_stay_bounded():
    """ds of a piece is at most 1 GiB where 256 vocabulary rows of all tokens are, whatever the vocabulary."""
    from mamba_cpu import _C

    for tokens, vocab, dim in ((65536, 2 ** 24, 256), (2 ** 20, 131072, 256), (64, 2 ** 24, 64)):
        a = _block(tokens=tokens, vocab=vocab, dim=dim, hidden_stride=dim, weight_stride=dim)
        need = _C.lib.mcpu_linear_loss_bwd_workspace_size(ctypes.byref(a))
        rows = 2 * tokens * dim * 4 + 5 * 4 * tokens  # hidden twice, dhidden in float32, the rows' numbers
        parts = 1536 * 2 ** 18  # split results
        assert need <= 2 ** 30 + rows + parts + 2 ** 20, (tokens, vocab, need)


def test_shape_functions_follow_the_operators():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        h = torch.empty(3, 5, 8, device=DEV, dtype=torch.bfloat16)
        w = torch.empty(11, 8, device=DEV, dtype=torch.bfloat16)
        ids = torch.zeros(3, 5, dtype=torch.long, device=DEV)
        loss, lse = mamba_cpu.linear_cross_entropy_fn(h, w, ids, return_lse=True)
        assert loss.shape == () and lse.shape == (3, 5) and loss.dtype == lse.dtype == torch.float32
        assert mamba_cpu.linear_cross_entropy_fn(h, w, ids, reduction="none").shape == (3, 5)
        kd = mamba_cpu.linear_distillation_fn(h, w, ids[..., None].expand(3, 5, 4),
                                              torch.empty(3, 5, 4, device=DEV), reduction="none")
        assert kd.shape == (3, 5)
        dh, dw = torch.ops.mamba_cpu.linear_loss_bwd(
            None, None, h.view(15, 8), w, ids.view(15, 1), kd.new_empty(0, 1), kd.new_empty(4, 15),
            kd.new_empty(0, 1), ids.new_empty(16, dtype=torch.int32), kd.new_empty(0, dtype=torch.uint8), -100, 1.0, 0,
            False, True, True)
        assert dh.shape == (15, 8) and dw.shape == (11, 8) and dh.dtype == dw.dtype == torch.bfloat16


@pytest.mark.parametrize("which", ["hidden", "weight", "teacher"])
def test_forward_mode_raises(which):
    import torch.autograd.forward_ad as fwAD
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True), fwAD.dual_level():
        t = {"hidden": torch.empty(5, 8, device=DEV), "weight": torch.empty(7, 8, device=DEV),
             "teacher": torch.empty(5, 2, device=DEV)}
        t[which] = fwAD.make_dual(t[which], torch.empty_like(t[which]))
        ids = torch.zeros(5, 2, dtype=torch.long, device=DEV)
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            mamba_cpu.linear_distillation_fn(t["hidden"], t["weight"], ids, t["teacher"])
        if which != "teacher":
            with pytest.raises((RuntimeError, NotImplementedError)):
                mamba_cpu.linear_cross_entropy_fn(t["hidden"], t["weight"], ids[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["ce", "kd"])
def test_a_second_gradient_is_refused(op):
    h, w, ids, g = inputs("f32", 20, 50, 32)
    hh, ww = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    if op == "ce":
        loss = mamba_cpu.linear_cross_entropy_fn(hh, ww, ids.to(DEV))
    else:
        loss = mamba_cpu.linear_distillation_fn(hh, ww, *(x.to(DEV) for x in teacher(20, 50, 4, g)))
    dh, dw = torch.autograd.grad(loss, [hh, ww], create_graph=True)
    for d in (dh, dw):
        with pytest.raises(RuntimeError, match="not implemented"):
            torch.autograd.grad(d.sum(), [hh], retain_graph=True)


# ---- streams and graphs ----


def _draw(seed, t=300, dtype=torch.bfloat16, v=14000):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(t, 192, device=DEV, generator=g).to(dtype)
    w = (torch.randn(v, 192, device=DEV, generator=g) / 14).to(dtype)
    ids = torch.randint(v, (t,), device=DEV, generator=g)
    ids[torch.rand(t, device=DEV, generator=g) < 0.1 * (seed % 7)] = -100  # another number of rows each time
    top = torch.randint(-1, v, (t, 6), device=DEV, generator=g)
    return {"h": h, "w": w, "ids": ids, "top": top, "tl": torch.randn(t, 6, device=DEV, generator=g)}


def _step(d):
    """Both losses, forward and backward, through leaves of this call's own."""
    h, w = d["h"].detach().requires_grad_(), d["w"].detach().requires_grad_()
    ce, lse = mamba_cpu.linear_cross_entropy_fn(h, w, d["ids"], return_lse=True)
    kd = mamba_cpu.linear_distillation_fn(h, w, d["top"], d["tl"], temperature=2.0, reduction="sum")
    dh, dw = torch.autograd.grad([ce, kd, lse], [h, w], [torch.full_like(ce, 3.0), torch.ones_like(kd),
                                                         torch.full_like(lse, 1e-3)])
    return ce.detach(), kd.detach(), lse.detach(), dh, dw


@pytest.mark.gpu
@pytest.mark.parametrize("t,v,dtype", [(300, 14000, torch.bfloat16), (300, 14000, torch.float32),
                                       (20, 700, torch.bfloat16), (100, 700, torch.float32)])
def test_calls_replay_from_a_graph(t, v, dtype):
    static = _draw(0, t, dtype, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(static)
    torch.cuda.synchronize()
    for seed in (1, 2, 3, 4, 8):
        for k, x in _draw(seed, t, dtype, v).items():
            static[k].copy_(x)
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        want = _step(_draw(seed, t, dtype, v))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), seed


@pytest.mark.gpu
def test_two_streams_at_once():
    """Inputs made on each stream behind a queue of work, both calls on their way together."""
    want = [_step(_draw(s)) for s in (1, 2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for round_ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                a = torch.full((2048, 2048), 1.0 / 2048, device=DEV)
                for _ in range(20):
                    a = a @ a
                d = {k: v * 1 for k, v in _draw(i + 1).items()}
                got[i] = _step(d)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b), round_


# ---- sizes ----


def _gpu_rows(h, w, ids, per=1024):
    """loss and lse per row in float64 on the GPU, rows in parts."""
    loss, lse = [], []
    for i in range(0, h.shape[0], per):
        z = torch.matmul(h[i:i + per].double(), w.double().t())
        l = torch.logsumexp(z, 1)
        lse.append(l)
        loss.append(l - z.gather(1, ids[i:i + per, None])[:, 0])
    return torch.cat(loss), torch.cat(lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_vocabulary_in_pieces(dtype):
    """More than 1 GiB of ds: three pieces and two in float32; more rows than one turn of the rows' order."""
    t, v, d = 20000, 40000 if dtype == torch.bfloat16 else 20000, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(t, d, device=DEV, generator=g).to(dtype).requires_grad_()
    w = (torch.randn(v, d, device=DEV, generator=g) / 8).to(dtype).requires_grad_()
    ids = torch.randint(v, (t,), device=DEV, generator=g)
    ids[::5] = -100
    loss = mamba_cpu.linear_cross_entropy_fn(h, w, ids, reduction="sum")
    dh, dw = torch.autograd.grad(loss, [h, w])
    hd, wd = h.detach().double(), w.detach().double()
    want_h, want_w, total = torch.zeros_like(hd), torch.zeros_like(wd), 0.0
    mag_h, mag_w = torch.zeros_like(hd), torch.zeros_like(wd)
    for i in range(0, t, 2000):
        rows = (torch.arange(i, i + 2000, device=DEV))[ids[i:i + 2000] >= 0]
        z = torch.matmul(hd[rows], wd.t())
        lp = torch.log_softmax(z, 1)
        total -= float(lp.gather(1, ids[rows, None]).sum())
        ds = lp.exp_()
        ds.scatter_add_(1, ids[rows, None], -torch.ones(len(rows), 1, device=DEV, dtype=torch.double))
        want_h[rows] = ds @ wd
        want_w += ds.t() @ hd[rows]
        mag_h[rows] = ds.abs() @ wd.abs()
        mag_w += ds.abs().t() @ hd[rows].abs()
    key = "bf16" if dtype == torch.bfloat16 else "f32"
    # Logits up to 2^3 in sum: their error and lse's below 2^-15; dweight's operand is rounded too.
    e = 2 * KEPT[key] + 2.0 ** -14 + v * U
    assert abs(float(loss.detach()) - total) <= total * 2.0 ** -16
    assert bool(((dh.double() - want_h).abs() <= e * mag_h + OUT[key] * want_h.abs()).all())
    assert bool(((dw.double() - want_w).abs() <= e * mag_w + OUT[key] * want_w.abs() + 1e-9).all())
    assert torch.count_nonzero(dh[::5]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [9, 80])  # blocks, tiles
def test_weight_past_4_gib(t):
    """2^31 elements and more of weight: the last rows' logits and gradients are as those of the rows by themselves."""
    d = 2048
    v = 2 ** 20 + 2 ** 17 + 77
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.zeros(v, d, device=DEV, dtype=torch.bfloat16)
    tail = (torch.randn(1000, d, device=DEV, generator=g) / 45).to(torch.bfloat16)
    w[-1000:] = tail
    h = torch.randn(t, d, device=DEV, generator=g).to(torch.bfloat16)
    ids = v - 1 - torch.randint(1000, (t,), device=DEV, generator=g)
    hg, wg = h.requires_grad_(), w.requires_grad_()
    loss, lse = mamba_cpu.linear_cross_entropy_fn(hg, wg, ids, reduction="none", return_lse=True)
    dh, dw = torch.autograd.grad(loss.sum(), [hg, wg])
    z = torch.matmul(h.detach().double(), tail.double().t())
    want = torch.logsumexp(torch.cat([z, torch.full((t, 1), float(np.log(v - 1000)), device=DEV)], 1).double(), 1)
    assert (lse - want).abs().max() <= 2.0 ** -15 * 16
    p = torch.exp(z - want[:, None])
    p.scatter_add_(1, (ids - (v - 1000))[:, None], -torch.ones(t, 1, device=DEV, dtype=torch.double))
    mag_h, mag_w = p.abs() @ tail.double().abs(), p.abs().t() @ h.detach().double().abs()
    e = 2 * KEPT["bf16"] + 2.0 ** -12
    assert bool(((dh.double() - p @ tail.double()).abs() <= 2 * e * mag_h).all())
    assert bool(((dw[-1000:].double() - p.t() @ h.detach().double()).abs() <= 2 * e * mag_w).all())
    # The rows of zeros: one probability for all, so one gradient.
    one = (torch.exp(-want)[:, None] * h.detach().double()).sum(0)
    mag = (torch.exp(-want)[:, None] * h.detach().double().abs()).sum(0)
    for row in (0, 2 ** 20 - 1, 2 ** 20, v - 1001):
        assert bool(((dw[row].double() - one).abs() <= 2 * e * mag + 1e-12).all()), row


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", [(20, 300), (70, 300), (300, 14000)])
def test_rows_far_apart(t, v):
    """hidden's rows 2^26 (2^24) elements apart, weight's 2^21 (2^18): offsets past 32 bits, and rows the products
    cannot step over."""
    h, w, ids, _ = inputs("bf16", t, v, 64)
    want = run_ce("bf16", h, w, ids, "none", 1.0)
    far_h, far_w = (2 ** 26, 2 ** 21) if t < 100 else (2 ** 24, 2 ** 18)
    hs = torch.empty(t * far_h, device=DEV, dtype=torch.bfloat16).view(t, far_h)[:, :64]
    ws = torch.empty(v * far_w, device=DEV, dtype=torch.bfloat16).view(v, far_w)[:, :64]
    hs.copy_(h), ws.copy_(w)
    hs, ws = hs.detach().requires_grad_(), ws.detach().requires_grad_()
    loss, lse = mamba_cpu.linear_cross_entropy_fn(hs, ws, ids.to(DEV), reduction="none", return_lse=True)
    dh, dw = torch.autograd.grad(loss.sum(), [hs, ws])
    for a, b in zip((loss, lse, dh, dw), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_broadcast_hidden(t, v):
    """One row for all tokens, expanded: its gradient is the sum of theirs."""
    h, w, ids, _ = inputs("f32", t, v, 64)
    one = h[:1].to(DEV).requires_grad_()
    wg = w.to(DEV)
    mamba_cpu.linear_cross_entropy_fn(one.expand(t, 64), wg, ids.to(DEV), reduction="sum").backward()
    _, _, dh, _ = run_ce("f32", h[:1].expand(t, 64).contiguous(), w, ids, "sum", 1.0)
    assert torch.allclose(one.grad, dh.sum(0, keepdim=True), rtol=0, atol=t * U * float(dh.abs().sum(0).max()))


# ---- values ----


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v", WAYS)
def test_extreme_logits(dtype, t, v):
    """Logits of hundreds, targets far above all others (a loss of 0) and far below (a loss as large as the gap)."""
    h, w, ids, g = inputs(dtype, t, v, 64)
    h = h * 64
    best = (h.double() @ w.double().t()).argmax(1)
    ids = torch.where(torch.arange(t) % 2 == 0, best, ids)
    verify_ce(dtype, h, w, ids, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_a_small_loss_keeps_its_digits(t, v):
    """Targets 12 above the others: a loss of about 2e-3 or less, to the relative error of its own exponent."""
    h, w, ids, _ = inputs("f32", t, v, 64, seed=3)
    w = w / w.norm(dim=1, keepdim=True)
    h = 18 * w[ids] + 0.05 * h
    loss, _, _, _ = run_ce("f32", h, w, ids, "none", 1.0)
    want, _, _ = O.rows(h, w, ids)
    # The gap's error, twice a logit's, is the loss's relative one; log1p and the sums some 2^-20 more.
    check("loss", loss, want, (2 * logit_err("f32", h, w) + 2.0 ** -16) * want)
    assert want.max() < 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_float32_rows_of_unequal_size(t, v):
    """Rows of hidden and weight over six powers of ten: float32 operands are scaled by their largest value."""
    h, w, ids, g = inputs("f32", t, v, 64)
    h = h * 10.0 ** (-6 * torch.rand(t, 1, generator=g))
    w = w * 10.0 ** (-6 * torch.rand(v, 1, generator=g))
    verify_ce("f32", h, w, ids, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v", WAYS)
def test_constant_and_zero_operands(dtype, t, v):
    h, w, ids, g = inputs(dtype, t, v, 64)
    verify_ce(dtype, torch.zeros_like(h), w, ids, "none", g)
    verify_ce(dtype, h, torch.zeros_like(w), ids, "none", g)
    verify_kd(dtype, torch.zeros_like(h), w, *teacher(t, v, 5, g), 1.0, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_infinite_gradients_come_through(t, v):
    """A loss scale that overflowed: inf or NaN out, for the scaler to see."""
    h, w, ids, _ = inputs("f16", t, v, 64)
    _, _, dh, dw = run_ce("f16", h, w, ids, "mean", float("inf"))
    assert not torch.isfinite(dh).all(1).any() and not torch.isfinite(dw).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,v", WAYS)
@pytest.mark.parametrize("some", [True, False])
def test_targets_far_above_under_a_loss_scale(dtype, t, v, some):
    """Targets 60 to 100 above all others, under a loss scale of 2^16: ds down to the end of float32's range, with and
    without a row of ordinary size beside."""
    w = torch.eye(v, 64, dtype=torch.float64)
    ids = torch.arange(t) % 64
    h = torch.zeros(t, 64, dtype=torch.float64)
    h[torch.arange(t), ids] = torch.linspace(60, 100, t, dtype=torch.float64)
    if some:
        h[5] = 0
    h, w = h.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]), w.to(
        {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype])
    loss, lse, dh, dw = run_ce(dtype, h, w, ids, "none", 2.0 ** 16)
    want, want_lse, _ = O.rows(h, w, ids)
    check("loss", loss, want, 2.0 ** -16 * (1 + want))
    ds = O.logits_grad(h, w, ids, np.full(t, 2.0 ** 16))
    want_h, want_w = O.grads(h, w, ds)
    # One rounding of ds and one of the result, and f16's smallest steps: of ds beside the largest, of the result.
    u, low = 3 * OUT[dtype] + 2.0 ** -14, 2.0 ** -36 * 2.0 ** 16 + 2.0 ** -24 if some or dtype == "f16" else 2.0 ** -70
    check("dhidden", dh, want_h, u * np.abs(ds) @ np.abs(w.double().numpy()) + low)
    check("dweight", dw, want_w, u * np.abs(ds).T @ np.abs(h.double().numpy()) + 100 * low)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_ids_past_32_bits_are_no_other_ids(t, v):
    """An id of 2^32 + v is outside the vocabulary, and is not v, whichever comes first."""
    h, w, _, g = inputs("bf16", t, v, 64)
    ids, tl = teacher(t, v, 6, g)
    wild = torch.cat([ids[:, :2] + 2 ** 32, ids, ids[:, 3:4] - 2 ** 32, torch.full_like(ids[:, :1], 2 ** 62)], 1)
    wide = torch.cat([torch.zeros(t, 2), tl, torch.full((t, 2), 9.0)], 1)
    outs = []
    for i, l in ((ids, tl), (wild, wide)):
        hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        loss = mamba_cpu.linear_distillation_fn(hg, wg, i.to(DEV), l.to(DEV), reduction="none")
        outs.append((loss, *torch.autograd.grad(loss.sum(), [hg, wg])))
    for a, b in zip(*outs):
        assert torch.allclose(a, b, rtol=2.0 ** -7, atol=1e-6)
    ce = [mamba_cpu.linear_cross_entropy_fn(h.to(DEV), w.to(DEV), i.to(DEV), reduction="none")
          for i in (ids[:, 0], ids[:, 0] + 2 ** 32)]
    assert (ce[0] > 0).all() and torch.count_nonzero(ce[1]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,v", WAYS)
def test_what_lies_around_the_operands(dtype, t, v):
    """Operands in the middle of memory that holds NaN, where weight is read in place: nothing of it is read into a
    result."""
    key = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}[dtype]
    h, w, ids, _ = inputs(key, t, v, 64)
    want = run_ce(key, h, w, ids, "none", 1.0)
    hs = torch.full((t + 40, 192), float("nan"), dtype=dtype, device=DEV)
    ws = torch.full((v + 700, 192), float("nan"), dtype=dtype, device=DEV)
    hs[8:t + 8, 64:128], ws[200:v + 200, 64:128] = h.to(DEV), w.to(DEV)
    hv, wv = hs[8:t + 8, 64:128].detach().requires_grad_(), ws[200:v + 200, 64:128].detach().requires_grad_()
    loss, lse = mamba_cpu.linear_cross_entropy_fn(hv, wv, ids.to(DEV), reduction="none", return_lse=True)
    dh, dw = torch.autograd.grad(loss.sum(), [hv, wv])
    for a, b in zip((loss, lse, dh, dw), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_loss_scaled_float16(t, v):
    """Gradients of 2^-14 a token under a scale of 2^14 and without: the same but for float16's smallest step."""
    h, w, ids, _ = inputs("f16", t, v, 64)
    _, _, dh, dw = run_ce("f16", h, w, ids, "sum", 1.0)
    _, _, sh, sw = run_ce("f16", h, w, ids, "sum", 2.0 ** -10)
    for a, b in ((dh, sh), (dw, sw)):
        assert ((a.double() * 2.0 ** -10 - b.double()).abs() <= 2.0 ** -24).all()


# ---- RecurrentLM ----


@pytest.mark.gpu
@pytest.mark.parametrize("batch,seqlen", [(2, 17), (3, 50)])
def test_recurrent_lm_losses(batch, seqlen):
    """model.loss and distillation_loss against the same losses of the model's own logits, values and every gradient;
    packed rows; then two training steps."""
    from mamba_cpu.recurrent_lm import RecurrentLM

    torch.manual_seed(0)
    m = RecurrentLM(301, 64, 2, d_inner=96).cuda()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(301, (batch, seqlen + 1), generator=g).cuda()
    seq = (torch.arange(seqlen)[None].expand(batch, -1) >= 9).int().cuda()
    targets = ids[:, 1:].clone()
    targets[:, 3] = -100
    top = torch.randint(301, (batch, seqlen, 5), generator=g).cuda()
    tl = torch.randn(batch, seqlen, 5, generator=g).cuda()

    def own():
        return (m.loss(ids[:, :-1], targets, seq_idx=seq)
                + m.distillation_loss(ids[:, :-1], top, tl, temperature=1.5, seq_idx=seq))

    def plain():
        logits = m(ids[:, :-1], seq_idx=seq)
        ce = torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=-100)
        q = torch.softmax(tl / 1.5, -1)
        logp = torch.log_softmax(logits / 1.5, -1).gather(-1, top)
        return ce + 1.5 ** 2 * (q * (q.log() - logp)).sum(-1).mean()

    params = list(m.parameters())
    a, b = own(), plain()
    ga, gb = torch.autograd.grad(a, params), torch.autograd.grad(b, params)
    assert abs(float(a.detach()) - float(b.detach())) <= 1e-5 * float(b.detach())
    for x, y, (name, _) in zip(ga, gb, m.named_parameters()):
        # As test_recurrent_lm holds the model's gradients, from either loss.
        assert (x - y).abs().max() <= 2e-4 * y.abs().max(), name
    with torch.no_grad():
        lp = -m.loss(ids[:, :-1], targets, reduction="none")
        want = torch.log_softmax(m(ids[:, :-1]), -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    assert (lp - torch.where(targets >= 0, want, torch.zeros_like(want))).abs().max() <= 1e-4
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    for _ in range(2):
        opt.zero_grad()
        own().backward()
        opt.step()
    assert all(torch.isfinite(p).all() for p in m.parameters())
