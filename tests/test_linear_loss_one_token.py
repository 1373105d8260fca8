"""A single confident token, scored: a loss of about 0.01 has float32's digits, though lse - s_target in float32, with
lse near 16, has none behind the fourth.

Operands are multiples of 2^-3 and 2^-5, so that every logit is a multiple of 2^-8 below 2^8 and exact in float32 in any
order of its sum. What is left: arguments of exp2 up to 2^5, each rounded by at most 2^-20 (a logit's difference, its
part's maximum, the target's), 2^-20 log 2 of the value each; 30 additions of positive terms in a row, 2^-24 each; exp2
and the logarithm, 2^-22. Together below 2^-18; the tolerance is twice that.
"""

import pytest
import torch

import mamba_cpu
from test_linear_loss import DEV, DTYPES


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,dim", [(50280, 768), (1000, 128)])
def test_a_confident_token_scored(dtype, vocab, dim):
    worst = 0.0
    for seed in range(8):
        g = torch.Generator(device=DEV).manual_seed(seed)
        w = (torch.randint(4, (vocab, dim), device=DEV, generator=g) - 1).clamp_(-1, 1) / 32
        w = torch.where(w > 0, w * (1 - 2 * torch.randint(2, w.shape, device=DEV, generator=g)), w * 0)
        y = torch.randint(vocab, (1,), device=DEV, generator=g)
        h = torch.randint(-8, 9, (1, dim), device=DEV, generator=g) / 8
        # So many of the target's columns point its way that its logit is 12 to 16.
        pull = torch.round((12 + 4 * torch.rand(1, device=DEV, generator=g)) * 8 / w[y].abs().sum()) / 8
        h = h + pull * w[y].sign()
        assert float((h.abs() @ w.abs().t()).max()) < 2 ** 7
        loss, lse = mamba_cpu.linear_cross_entropy_fn(h.to(DTYPES[dtype]), w.to(DTYPES[dtype]), y, reduction="none",
                                                      return_lse=True)
        z = torch.matmul(h.double(), w.double().t())[0]
        others = torch.cat([z[:y], z[y + 1:]])
        want = torch.log1p(torch.exp(others - z[y]).sum())
        rel = float((loss.double() - want).abs() / want)
        print(f"{dtype} {vocab} x {dim} loss {float(loss):.6g} off by {rel:.3g}", flush=True)
        worst = max(worst, rel)
        assert abs(float(lse) - float(torch.logsumexp(z, 0))) <= 2.0 ** -19 * float(lse)
    assert worst <= 2.0 ** -17
