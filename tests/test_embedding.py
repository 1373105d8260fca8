"""embedding_fn: the scaled lookup and its gradient by sorted tokens.

Tolerances, from the formats: a row is one product, so float32 rows are within
one rounding (2**-24) of the oracle's and 16-bit rows within half a unit
(2**-8, 2**-11 relative). A gradient sums up to n tokens in float32: within
n x 2**-24 of the sum of their magnitudes, plus the format's rounding.
"""

import ctypes

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def test_oracle_gradient_is_the_transpose_of_the_lookup():
    g = torch.Generator().manual_seed(0)
    ids = torch.tensor([3, 0, 3, -1, 7, 9, 3])
    w, dout = torch.randn(8, 5, generator=g).double(), torch.randn(7, 5, generator=g).double()
    onehot = torch.zeros(7, 8, dtype=torch.float64)
    for t, v in enumerate(ids.tolist()):
        if 0 <= v < 8:
            onehot[t, v] = 1.0
    np.testing.assert_allclose(O.embedding_bwd(ids, dout, 8, 3.0), 3.0 * (onehot.T @ dout).numpy(), rtol=1e-14)
    assert w.shape == (8, 5)


def test_refusals_on_the_cpu():
    import mamba_cpu
    from mamba_cpu import _C

    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.embedding_fn(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 2))
    L = _C.lib

    def block(**kw):
        a = _C.EmbeddingArgs()
        a.ids = a.weight = a.out = a.dout = a.dweight = 16
        a.tokens, a.vocab, a.dim, a.weight_stride, a.dout_stride, a.scale = 5, 7, 8, 8, 8, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    need = L.mcpu_embedding_bwd_workspace_size(block())
    assert need >= 4 * (5 + 8)
    bad = _C.MCPU_ERR_INVALID
    for kw in ({"ids": None}, {"tokens": -1}, {"dtype": 4}, {"ids64": 2}, {"weight_stride": -1}):
        assert L.mcpu_embedding_fwd(block(**kw), None) == bad, kw
        assert L.mcpu_embedding_bwd(block(**kw), 16, need, None) == bad, kw
    assert L.mcpu_embedding_fwd(block(out=None), None) == bad
    assert L.mcpu_embedding_bwd(block(dweight=None), 16, need, None) == bad
    assert L.mcpu_embedding_bwd(block(), 16, need - 1, None) == bad
    assert L.mcpu_embedding_fwd(block(vocab=1 << 40), None) == _C.MCPU_ERR_UNSUPPORTED
    assert L.mcpu_embedding_fwd(None, None) == bad and L.mcpu_embedding_bwd(None, None, 0, None) == bad
    assert L.mcpu_embedding_bwd_workspace_size(None) == 0


gpu = pytest.mark.gpu


def draw(tokens, vocab, dim, dtype, seed=0, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(vocab, (tokens,), generator=g)
    ids = torch.where(torch.rand(tokens, generator=g) < skew, torch.full_like(ids, vocab // 2), ids)
    return (ids.to(DEV), torch.randn(vocab, dim, generator=g).to(dtype).to(DEV),
            torch.randn(tokens, dim, generator=g).to(dtype).to(DEV))


def check(ids, w, dout, scale, layout=lambda v: v):
    import mamba_cpu

    dtype, vocab = w.dtype, w.shape[0]
    scale = float(np.float32(scale))  # as the operator takes it
    leaf = layout(w).detach().requires_grad_()
    out = mamba_cpu.embedding_fn(ids, leaf, scale=scale)
    assert out.shape == (*ids.shape, w.shape[1]) and out.dtype == dtype
    flat = ids.reshape(-1)
    inside = (flat >= 0) & (flat < vocab)
    want = torch.where(inside[:, None], w[flat.clamp(0, vocab - 1).long()].double() * scale, 0.0)
    tiny = 6e-8 if dtype == torch.float16 else 0.0
    err = (out.reshape(-1, w.shape[1]).double() - want).abs()
    assert (err <= 1.01 * HALF[dtype] * want.abs() + tiny).all()
    (dw,) = torch.autograd.grad([out], [leaf], [dout.reshape(out.shape)])
    assert dw.dtype == dtype and dw.shape == w.shape
    want = O.embedding_bwd(ids, dout.reshape(-1, w.shape[1]), vocab, scale)
    size = O.embedding_bwd(ids, dout.reshape(-1, w.shape[1]).abs(), vocab, abs(scale))
    counts = np.bincount(flat[inside].cpu().numpy(), minlength=vocab)[:, None]
    bound = (counts + 2) * 2.0 ** -24 * size + HALF[dtype] * np.abs(want) * 1.01 + tiny
    err = np.abs(dw.double().cpu().numpy() - want)
    assert np.all(err <= bound), f"dweight worst err/bound {np.nanmax(err / np.maximum(bound, 1e-300)):.3g}"


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (7, 5, 3), (64, 300, 64), (1000, 257, 130), (65, 50280, 33),
                                              (4097, 1000, 768), (3000, 7, 20)])
def test_matches_oracle(tokens, vocab, dim, dtype):
    print(f"embedding {tokens} of {vocab} x {dim} {dtype}", flush=True)
    check(*draw(tokens, vocab, dim, dtype, seed=tokens), scale=dim ** 0.5)


@gpu
@pytest.mark.parametrize("skew", [0.3, 0.97, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_id_with_most_of_the_tokens(skew, dtype):
    print(f"embedding skew {skew} {dtype}", flush=True)
    check(*draw(5003, 999, 70, dtype, seed=3, skew=skew), scale=1.0)


@gpu
def test_few_ids_with_all_the_tokens():
    print("embedding of a tiny vocabulary, runs of equal ids", flush=True)
    ids, w, dout = draw(2100, 3, 96, torch.float32, seed=4)
    check(torch.sort(ids).values, w, dout, scale=0.5)
    check(ids, w, dout, scale=0.5)


@gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_ids_outside_the_vocabulary_and_their_shape(kind):
    print(f"embedding ids outside, {kind}", flush=True)
    ids, w, dout = draw(60, 40, 24, torch.float32, seed=5)
    ids[::5] = torch.tensor([-1, 40, 1000, -7, 39, 40, -40, 41, 0, 2 ** 31 - 1, -2 ** 31, 5], device=DEV)
    check(ids.to(kind).view(3, 20), w, dout, scale=2.0)
    if kind == torch.int64:
        ids[0], ids[1] = 2 ** 40, -2 ** 62
        check(ids, w, dout, scale=2.0)
    every = torch.full((9,), -1, dtype=kind, device=DEV)
    check(every, w, dout[:9], scale=1.0)


@gpu
@pytest.mark.parametrize("kind", ["wide rows", "offset by one", "transposed", "expanded gradient"])
def test_any_strides(kind):
    print(f"embedding strides: {kind}", flush=True)
    ids, w, dout = draw(90, 50, 66, torch.bfloat16, seed=6)
    make = {"wide rows": lambda v: torch.cat([v, v], -1)[:, :66], "transposed": lambda v: v.t().contiguous().t(),
            "offset by one": lambda v: torch.cat([v[:, :1], v], -1)[:, 1:]}.get(kind, lambda v: v)
    dout = dout[:1, :1].expand(90, 66) if kind == "expanded gradient" else make(dout)
    check(ids, w, dout, 1.0, layout=make)
    check(torch.stack([ids, ids], 1)[:, 0], w, dout, 1.0)  # ids every other element


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", [(0, 5, 4), (0, 0, 4), (3, 5, 0), (3, 0, 4)])
def test_empty(tokens, vocab, dim):
    import mamba_cpu

    print(f"embedding empty {tokens, vocab, dim}", flush=True)
    w = torch.ones(vocab, dim, device=DEV, requires_grad=True)
    out = mamba_cpu.embedding_fn(torch.zeros(tokens, dtype=torch.int64, device=DEV), w)
    assert out.shape == (tokens, dim)
    out.sum().backward()
    assert w.grad.shape == w.shape and torch.count_nonzero(w.grad) == 0


@gpu
def test_results_do_not_change_from_call_to_call():
    import mamba_cpu

    print("embedding twice", flush=True)
    ids, w, dout = draw(20000, 700, 256, torch.float32, seed=7, skew=0.4)
    grads = []
    for _ in range(2):
        leaf = w.detach().requires_grad_()
        grads.append(torch.autograd.grad([mamba_cpu.embedding_fn(ids, leaf)], [leaf], [dout])[0])
    assert torch.equal(*grads)


@gpu
def test_gpu_refusals_and_operator_checks():
    import mamba_cpu

    print("embedding refusals, opcheck", flush=True)
    ids, w, _ = draw(6, 9, 4, torch.float32)
    for args in ((ids.float(), w), (ids, w[0]), (ids.cpu(), w), (ids.to(torch.int16), w)):
        with pytest.raises(ValueError):
            mamba_cpu.embedding_fn(*args)
    torch.library.opcheck(torch.ops.mamba_cpu.embedding_fwd.default, (ids, w.requires_grad_(), 2.0),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
