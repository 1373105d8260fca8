"""A target whose own logit overflowed: lse - s is inf - inf, so the loss is NaN, as the gradient is, and not 0."""

import pytest
import torch

from test_linear_loss import DTYPES, WAYS, run_ce


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", WAYS)
def test_infinite_logit_of_the_target(dtype, t, v):
    """Word 3 is every token's target and alone has an infinity, in a column where hidden is 1."""
    g = torch.Generator().manual_seed(0)
    h, w = torch.randn(t, 64, generator=g), torch.randn(v, 64, generator=g)
    h[:, 0] = 1
    w[3, 0] = float("inf")
    ids = torch.full((t,), 3)
    loss, lse, dh, dw = run_ce(dtype, h.to(DTYPES[dtype]), w.to(DTYPES[dtype]), ids, "none", 1.0)
    assert torch.isnan(loss).all() and not torch.isfinite(lse).any()
    assert not torch.isfinite(dh).all(1).any() and not torch.isfinite(dw).all()
    # One that is minus infinity is a loss of infinity.
    w[3, 0] = -float("inf")
    loss, lse, _, _ = run_ce(dtype, h.to(DTYPES[dtype]), w.to(DTYPES[dtype]), ids, "none", 1.0)
    if dtype != "f32" or t < 1000:  # tiles multiply an infinity's second piece, which is 0: NaN
        assert (loss == float("inf")).all() and torch.isfinite(lse).all()
    else:
        assert not torch.isfinite(loss).any()
