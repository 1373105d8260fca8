"""Forward-mode derivatives: an operator with a backward but no forward-mode
rule raises, as the scans do; none hands back a result without its tangent.
On fake tensors: what raises does so before any kernel runs."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

DEV = "cuda"


def _dual(*shape):
    return fwAD.make_dual(torch.empty(*shape, device=DEV), torch.empty(*shape, device=DEV))


def _calls():
    import mamba_cpu as m

    plain = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    ids = lambda: torch.zeros(5, dtype=torch.long, device=DEV)  # noqa: E731
    scan = lambda u: m.selective_scan_fn(u, plain(2, 4, 9), plain(4, 8), plain(2, 8, 9), plain(2, 8, 9))  # noqa: E731
    return {
        "gated scan, x": lambda: m.gated_linear_scan_fn(_dual(2, 9, 4), plain(2, 9, 4), plain(2, 9, 4), plain(4)),
        "gated scan, decay": lambda: m.gated_linear_scan_fn(plain(2, 9, 4), plain(2, 9, 4), plain(2, 9, 4), _dual(4)),
        "gated scan, state": lambda: m.gated_linear_scan_fn(plain(2, 9, 4), plain(2, 9, 4), plain(2, 9, 4), plain(4),
                                                            initial_state=_dual(2, 4)),
        "norm, x": lambda: m.layer_norm_fn(_dual(3, 8), plain(8)),
        "norm, weight": lambda: m.layer_norm_fn(plain(3, 8), _dual(8)),
        "norm, bias": lambda: m.layer_norm_fn(plain(3, 8), plain(8), _dual(8)),
        "norm, residual": lambda: m.layer_norm_fn(plain(3, 8), plain(8), residual=_dual(3, 8), prenorm=True),
        "embedding": lambda: m.embedding_fn(ids(), _dual(7, 8)),
        # The older operators, which these follow.
        "selective scan": lambda: scan(_dual(2, 4, 9)),
        "conv": lambda: m.causal_conv1d_fn(_dual(2, 4, 9), plain(4, 3)),
    }


@pytest.mark.parametrize("name", sorted(_calls()))
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_not_dropped(name, grad):
    with FakeTensorMode(), fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises((RuntimeError, NotImplementedError), match="(?i)jvp|forward"):
            _calls()[name]()


@pytest.mark.parametrize("name", ["gated scan, x", "norm, x", "embedding"])
def test_calls_without_a_tangent_run_inside_a_dual_level(name):
    import mamba_cpu as m

    with FakeTensorMode(), fwAD.dual_level(), torch.no_grad():
        plain = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
        out = {"gated scan, x": lambda: m.gated_linear_scan_fn(plain(2, 9, 4), plain(2, 9, 4), plain(2, 9, 4), plain(4)),
               "norm, x": lambda: m.layer_norm_fn(plain(3, 8), plain(8)),
               "embedding": lambda: m.embedding_fn(torch.zeros(5, dtype=torch.long, device=DEV), plain(7, 8))}[name]()
        assert fwAD.unpack_dual(out).tangent is None
