"""More of the calls that the head's losses allow: distillation over strided and unaligned operands, hidden of one
token without a leading dimension, a gradient through lse alone, an ignored id of the vocabulary, one column, many
entries of many tokens, a traced training step, and rows' gradients from a captured graph.

Tolerances are those of test_linear_loss.py.
"""

import numpy as np
import pytest
import torch

import mamba_cpu
from oracle import loss as O
from test_linear_loss import (DEV, DTYPES, U, WAYS, check, check_grads, inputs, logit_err, lse_tol, teacher,
                              verify_ce, verify_kd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", [(60, 300), (100, 260), (1100, 4000)])
def test_distillation_over_strides_and_offsets(dtype, t, v):
    h, w, _, g = inputs(dtype, t, v, 130)
    ids, tl = teacher(t, v, 9, g)
    room_h = torch.full((t, 151), float("nan"), dtype=h.dtype, device=DEV)
    room_w = torch.full((v, 133), float("nan"), dtype=w.dtype, device=DEV)
    room_h[:, 5:135], room_w[:, 1:131] = h.to(DEV), w.to(DEV)
    hv, wv = room_h[:, 5:135].detach().requires_grad_(), room_w[:, 1:131].detach().requires_grad_()
    wide = torch.zeros(t, 20, dtype=torch.int32, device=DEV)
    wide[:, 1:19:2] = ids.to(DEV, torch.int32)
    loss = mamba_cpu.linear_distillation_fn(hv.unflatten(0, (t // 20, 20)), wv, wide[:, 1:19:2].view(t // 20, 20, 9),
                                            tl.to(DEV).t().contiguous().t().view(t // 20, 20, 9), temperature=1.5,
                                            reduction="none")
    assert loss.shape == (t // 20, 20)
    dloss = torch.randn(t, generator=g)
    dh, dw = torch.autograd.grad(loss, [hv, wv], dloss.to(DEV).view(t // 20, 20))
    want, lse, _ = O.rows(h, w, ids, tl, 1.5)
    ltol = lse_tol(dtype, h, w, lse, 1.5)
    check("loss", loss.view(-1), want, 1.5 ** 2 * (ltol + logit_err(dtype, h, w) / 1.5 + 64 * 17 * U))
    ds = O.logits_grad(h, w, ids, dloss.double().numpy(), teacher=tl, temperature=1.5)
    check_grads(dtype, h, w, ds, ltol + 2 * U * np.abs(lse) + 8 * U, dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_without_a_leading_dimension(dtype):
    h, w, ids, g = inputs(dtype, 1, 300, 64)
    want = mamba_cpu.linear_cross_entropy_fn(h.to(DEV), w.to(DEV), ids.to(DEV), reduction="none", return_lse=True)
    got = mamba_cpu.linear_cross_entropy_fn(h[0].to(DEV), w.to(DEV), ids[0].to(DEV), reduction="none", return_lse=True)
    for a, b in zip(got, want):
        assert a.shape == () and torch.equal(a, b[0])
    top, tl = teacher(1, 300, 5, g)
    kd = [mamba_cpu.linear_distillation_fn(x.to(DEV), w.to(DEV), i.to(DEV), l.to(DEV), reduction="none")
          for x, i, l in ((h, top, tl), (h[0], top[0], tl[0]))]
    assert kd[1].shape == () and torch.equal(kd[1], kd[0][0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t,v", WAYS)
def test_gradient_through_lse_alone(dtype, reduction, t, v):
    h, w, ids, g = inputs(dtype, t, v, 96)
    ids[3:9] = -100
    dlse = torch.randn(t, generator=g)
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    _, lse = mamba_cpu.linear_cross_entropy_fn(hg, wg, ids.to(DEV), reduction=reduction, return_lse=True)
    dh, dw = torch.autograd.grad(lse, [hg, wg], dlse.to(DEV))
    _, want_lse, keep = O.rows(h, w, ids)
    ltol = lse_tol(dtype, h, w, want_lse) * keep
    check_grads(dtype, h, w, O.logits_grad(h, w, ids, np.zeros(t), dlse), ltol + 2 * U * np.abs(want_lse), dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("t,v", WAYS)
def test_an_id_of_the_vocabulary_is_ignored(t, v):
    h, w, ids, g = inputs("bf16", t, v, 64)
    ids[::4] = 3
    verify_ce("bf16", h, w, ids, "none", g, ignore_index=3)
    verify_ce("bf16", h, w, ids, "mean", g, ignore_index=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v,d", [(40, 260, 1), (100, 260, 1), (1100, 4000, 1), (1100, 4000, 63)])
def test_few_columns(dtype, t, v, d):
    h, w, ids, g = inputs(dtype, t, v, d)
    verify_ce(dtype, h, w, ids, "none", g)
    verify_kd(dtype, h, w, *teacher(t, v, 3, g), 1.0, "mean", g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", [(100, 1100), (600, 14000)])
def test_most_entries_of_many_tokens(dtype, t, v):
    h, w, _, g = inputs(dtype, t, v, 64)
    ids, tl = teacher(t, v, 1024, g)
    ids[:, 1000] = ids[:, 5]
    verify_kd(dtype, h, w, ids, tl, 1.0, "none", g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_a_traced_training_step(dtype, t, v):
    h, w, ids, g = inputs(dtype, t, v, 72)
    torch._dynamo.reset()
    top, tl = (x.to(DEV) for x in teacher(t, v, 4, g))
    ids = ids.to(DEV)

    def step(hidden, weight):
        return (mamba_cpu.linear_cross_entropy_fn(hidden, weight, ids)
                + mamba_cpu.linear_distillation_fn(hidden, weight, top, tl, temperature=2.0, reduction="sum"))

    outs = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        loss = f(hg, wg)
        outs.append((loss.detach(), *torch.autograd.grad(loss, [hg, wg])))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("t,v", WAYS)
def test_rows_gradients_replay_from_a_graph(dtype, t, v):
    """Units of rows that other replays' inputs set, hidden's largest magnitude among them."""
    def draw(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        h = (torch.randn(t, 72, device=DEV, generator=g) * 4.0 ** (seed % 5 - 2)).to(dtype)
        w = (torch.randn(v, 72, device=DEV, generator=g) / 9).to(dtype)
        ids = torch.randint(-2, v, (t,), device=DEV, generator=g)
        top = torch.randint(-1, v, (t, 6), device=DEV, generator=g)
        return {"h": h, "w": w, "ids": ids, "top": top, "tl": torch.randn(t, 6, device=DEV, generator=g),
                "g": 10.0 ** (-8 * torch.rand(t, device=DEV, generator=g)) * (1 + seed)}

    def step(d):
        h, w = d["h"].detach().requires_grad_(), d["w"].detach().requires_grad_()
        ce = mamba_cpu.linear_cross_entropy_fn(h, w, d["ids"], reduction="none")
        kd = mamba_cpu.linear_distillation_fn(h, w, d["top"], d["tl"], temperature=2.0, reduction="none")
        return (*torch.autograd.grad(ce, [h, w], d["g"]), *torch.autograd.grad(kd, [h, w], d["g"]))

    static = draw(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    torch.cuda.synchronize()
    for seed in (1, 2, 3, 4, 8):
        for k, x in draw(seed).items():
            static[k].copy_(x)
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        for a, b in zip(got, step(draw(seed))):
            assert torch.equal(a, b), seed
