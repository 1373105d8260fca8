"""sample_fn with top-p close to 1, where the cut lies in a tail of very
unlikely tokens: there is always a token, it lies in the vocabulary, its
logprob is written, and the cut is where the definition has it.

The oracle is float64 (oracle/lm.py). Where the cut itself is measured, the
noise rises towards smaller indices so that the last token kept wins, and the
mass before that token is compared with top_p times the total: within 1.2e-7
of the total, two spacings of a float32 top_p next to 1.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
gpu = pytest.mark.gpu
BELOW_ONE = float(np.nextafter(np.float32(1), np.float32(0)))


def check(logits, noise, **kw):
    """Every row as the oracle has it; rows it calls too near to tell (1e-5) have
    a token of the vocabulary. The seeds here leave most rows to be compared."""
    import mamba_cpu

    token, logprob = mamba_cpu.sample_fn(logits, noise, return_logprobs=True, **kw)
    token, logprob = token.cpu().numpy(), logprob.cpu().numpy()
    logits, noise, compared = logits.cpu(), noise.cpu(), 0
    for r in range(len(token)):
        assert 0 <= token[r] < logits.shape[1], f"row {r}: token {token[r]}"
        lp = torch.log_softmax(logits[r].double(), -1)[token[r]].item()
        assert abs(logprob[r] - lp) <= 5e-6 + 2.0 ** -23 * abs(lp), f"row {r}: logprob {logprob[r]} for {lp}"
        want, _, kept, near = O.sample(logits[r], noise[r], **kw)
        if near < 1e-5:
            continue
        compared += 1
        assert token[r] == want, f"row {r}: {token[r]} instead of {want}, {kept} kept, near {near:.2g}"
    assert compared >= len(token) * 3 // 4


@gpu
@pytest.mark.parametrize("top_p", [0.9999, 0.99999, 0.999999, BELOW_ONE])
@pytest.mark.parametrize("top_k", [0, 700])
@pytest.mark.parametrize("v,dtype", [(1500, torch.float32), (50280, torch.float32), (50280, torch.bfloat16)])
def test_random_rows(v, dtype, top_k, top_p):
    print(f"sample top_p {top_p} of {v} {dtype} top_k {top_k}", flush=True)
    g = torch.Generator().manual_seed(v + top_k)
    logits = (torch.randn(40, v, generator=g) * 2.5).to(dtype)
    noise = torch.empty(40, v).exponential_(generator=g).clamp_(min=1e-30)
    check(logits.to(DEV), noise.to(DEV), top_k=top_k, top_p=top_p)


@gpu
@pytest.mark.parametrize("top_p", [0.99999, 0.999999, BELOW_ONE])
@pytest.mark.parametrize("top_k", [0, 100_000])
def test_one_likely_token_and_a_long_equal_tail(top_k, top_p):
    """131071 tokens of e**-23 each: none is 2**-32 of the mass, together they are 1.3e-5 of it."""
    print(f"sample peaked row top_p {top_p} top_k {top_k}", flush=True)
    g = torch.Generator().manual_seed(1)
    logits = torch.full((4, 131_072), -23.0)
    logits[:, 0] = 0.0
    noise = torch.empty(4, 131_072).exponential_(generator=g).clamp_(min=1e-6)
    check(logits.to(DEV), noise.to(DEV), top_k=top_k, top_p=top_p)


@gpu
@pytest.mark.parametrize("top_p", [0.99999, 0.999995, 0.9999])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_cut_lies_where_the_definition_has_it(dtype, top_p):
    import mamba_cpu

    print(f"sample cut of a long tail, top_p {top_p} {dtype}", flush=True)
    v = 131_072
    for far in (23.0, 20.5):
        logits = torch.full((1, v), -far)
        logits[0, 0] = 0.0
        logits = logits.to(dtype)
        w = np.exp(logits[0].double().numpy())
        score = 1 + 1e-4 * np.arange(v)  # rises with the index: the last kept token wins
        noise = torch.from_numpy((w / score)[None]).float()
        token = mamba_cpu.sample_fn(logits.to(DEV), noise.to(DEV), top_p=top_p).item()
        p, total = float(np.float32(top_p)), w.sum()
        assert 0 <= token < v
        before = w[:token].sum()
        # The last kept: the mass before it is below p, the mass with it no longer.
        assert before < p * total + 1.2e-7 * total, f"{token}: {before / total}"
        assert token == v - 1 or before + w[token] >= p * total - 1.2e-7 * total, f"{token}: {before / total}"


@gpu
def test_a_row_always_has_a_token():
    """Also where the one logit's score is infinity over infinity."""
    import mamba_cpu

    print("sample one infinite logit", flush=True)
    inf = torch.full((1, 1), float("inf"), device=DEV)
    for kw in ({}, {"top_p": 0.5}, {"min_p": 0.1}, {"top_k": 1}):
        token, logprob = mamba_cpu.sample_fn(inf, inf, return_logprobs=True, **kw)
        assert token.tolist() == [0] and logprob.tolist() == [0.0], kw
