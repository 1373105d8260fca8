"""sample_fn gives the same token for the same noise, call after call, also where
top-p lies at the mass that its short list holds: one row of logits with 4096
values of top_p, and every token compared with the oracle's.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("lo,hi", [(0.05, 0.999), (0.5, 0.6)])
def test_the_same_noise_gives_the_same_token(lo, hi):
    import mamba_cpu

    print(f"sample top_p {lo} to {hi}, repeated", flush=True)
    b, v = 4096, 3000
    g = torch.Generator().manual_seed(0)
    logits = (torch.randn(1, v, generator=g) * 2.5).to(DEV).expand(b, v)
    noise = torch.empty(1, v).exponential_(generator=g).clamp_(min=1e-30).to(DEV).expand(b, v)
    top_p = torch.linspace(lo, hi, b).to(DEV)
    first = mamba_cpu.sample_fn(logits, noise, top_p=top_p, return_logprobs=True)
    for _ in range(10):
        again = mamba_cpu.sample_fn(logits, noise, top_p=top_p, return_logprobs=True)
        assert all(torch.equal(x, y) for x, y in zip(again, first))
    compared = 0
    for r in range(0, b, 16):
        want, _, kept, near = O.sample(logits[r], noise[r], top_p=top_p[r].item())
        if near < 1e-5:
            continue
        compared += 1
        assert first[0][r].item() == want, f"top_p {top_p[r].item()}: {first[0][r].item()} for {want}, {kept} kept"
    assert compared >= 250
    assert np.isfinite(first[1].cpu().numpy()).all()
