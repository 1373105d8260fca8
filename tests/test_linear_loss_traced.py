"""The head's losses as traced programs see them: the shape function's sizes are the operator's."""

import ctypes
import itertools

import pytest
import torch

import mamba_cpu  # noqa: F401  (loads the operators)
from test_linear_loss import DEV, DTYPES, inputs, teacher


def traced_sizes(tokens, vocab, dim, k, stride, dtype, distil):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        h = torch.empty(tokens, dim, device=DEV, dtype=dtype)
        w = torch.empty(vocab, stride, device=DEV, dtype=dtype)[:, :dim]
        ids = torch.zeros(tokens, k, device=DEV, dtype=torch.long)
        tl = torch.zeros(tokens, k, device=DEV) if distil else None
        outs = torch.ops.mamba_cpu.linear_loss_fwd(h, w, ids, tl, -100, 1.0, 0, True)
        return [tuple(x.shape) for x in outs]


def test_the_kept_weight_has_the_size_that_is_traced():
    from mamba_cpu import _C

    kinds = ((torch.float32, _C.MCPU_F32), (torch.bfloat16, _C.MCPU_BF16), (torch.float16, _C.MCPU_F16))
    some = 0
    for tokens, vocab, dim, more, k, (dtype, tag) in itertools.product(
            (0, 1, 64, 65, 300, 1100), (0, 1, 128, 4000, 13200), (1, 64, 96, 128), (0, 3, 8), (0, 1, 5), kinds):
        a = _C.LinearLossArgs()
        for name in ("hidden", "weight", "ids", "stat", "rows", "picked", "share", "teacher"):
            setattr(a, name, 4096)
        a.tokens, a.vocab, a.dim, a.k, a.hidden_stride, a.weight_stride = tokens, vocab, dim, k, dim, dim + more
        a.temperature, a.dtype, a.ids64 = 1.0, tag, 1
        want = _C.lib.mcpu_linear_loss_laid_size(ctypes.byref(a))
        got = traced_sizes(tokens, vocab, dim, k, dim + more, dtype, True)
        assert got[6] == (want,), (tokens, vocab, dim, more, k, dtype)
        some += want > 0
    assert some > 100


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first,stride", [(0, 64), (1, 72), (8, 72), (0, 67)])
def test_operator_returns_what_is_traced(dtype, first, stride):
    t, v = 1100, 4000
    h, _, ids, _ = inputs(dtype, t, v, 64)
    w = torch.zeros(v * stride + first, device=DEV, dtype=DTYPES[dtype])[first:].view(v, stride)[:, :64]
    outs = torch.ops.mamba_cpu.linear_loss_fwd(h.to(DEV), w, ids[:, None].to(DEV), None, -100, 1.0, 0, True)
    assert [tuple(x.shape) for x in outs] == traced_sizes(t, v, 64, 1, stride, DTYPES[dtype], False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", ["ce", "kd"])
@pytest.mark.parametrize("t,v,d", [(20, 60, 64), (1100, 4000, 72)])
def test_operator_checks(dtype, op, t, v, d):
    h, w, ids, g = inputs(dtype, t, v, d)
    h, w = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    ids, tl = (ids[:, None], None) if op == "ce" else teacher(t, v, 4, g)
    if tl is not None:
        tl = tl.to(DEV)
    torch.library.opcheck(torch.ops.mamba_cpu.linear_loss_fwd.default, (h, w, ids.to(DEV), tl, -100, 1.0, 2, True),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
