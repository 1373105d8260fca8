"""sample_fn on one and two rows, every row compared: the seed of each case is the
first whose rows the oracle (oracle/lm.py) calls clear, by 1e-5 of what is compared.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O
from test_sampling import SETTINGS

DEV = "cuda"


def clear(b, v, dtype, kw):
    """Logits and noise, and the oracle's (token, logprob) of each row."""
    for seed in range(50):
        g = torch.Generator().manual_seed(seed)
        logits = (torch.randn(b, v, generator=g) * 2.5).to(dtype)
        noise = torch.empty(b, v).exponential_(generator=g).clamp_(min=1e-30)
        rows = [O.sample(logits[r], noise[r], **kw) for r in range(b)]
        if all(near >= 1e-5 for *_, near in rows):
            return logits, noise, rows
    raise AssertionError("no seed with clear rows")


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("b,v,dtype", [(1, 1, torch.float32), (1, 1025, torch.float32), (2, 7, torch.bfloat16),
                                       (1, 16385, torch.bfloat16), (2, 50280, torch.float32),
                                       (1, 131072, torch.float16)])
def test_every_row_is_the_oracle_s(b, v, dtype, kw):
    import mamba_cpu

    print(f"sample {b} x {v} {dtype} {kw}", flush=True)
    logits, noise, rows = clear(b, v, dtype, kw)
    token, logprob = mamba_cpu.sample_fn(logits.to(DEV), noise.to(DEV), return_logprobs=True, **kw)
    assert token.tolist() == [r[0] for r in rows]
    for got, (_, lp, *_) in zip(logprob.tolist(), rows):
        assert np.isfinite(lp) and abs(got - lp) <= 5e-6 + 2.0 ** -23 * abs(lp)
