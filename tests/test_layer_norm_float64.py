"""layer_norm_fn of a float64 stream: computed in float32, but the residual it
hands back without a new one is the caller's own tensor."""

import pytest
import torch

DEV = "cuda"


def _fake(f):
    """On fake tensors: types and identities, without a device."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        f()


def test_prenorm_without_a_residual_hands_x_back():
    import mamba_cpu

    def run():
        w = torch.empty(16, device=DEV)
        for dtype in (torch.float64, torch.float32, torch.bfloat16):
            x = torch.empty(3, 16, device=DEV, dtype=dtype)
            y, z = mamba_cpu.layer_norm_fn(x, w, prenorm=True)
            assert z is x and y.dtype == dtype, dtype
            _, z = mamba_cpu.layer_norm_fn(x, w, prenorm=True, residual_in_fp32=True)
            assert z.dtype == torch.float32 and z.shape == x.shape, dtype
        x = torch.empty(3, 16, device=DEV, dtype=torch.float64)
        y, z = mamba_cpu.layer_norm_fn(x, w, residual=x, prenorm=True)
        assert y.dtype == z.dtype == torch.float64

    _fake(run)


@pytest.mark.gpu
def test_the_stream_keeps_its_bits():
    import mamba_cpu

    print("norm of a float64 stream", flush=True)
    x = torch.randn(5, 40, device=DEV, dtype=torch.float64, requires_grad=True)
    w = torch.ones(40, device=DEV)
    y, z = mamba_cpu.layer_norm_fn(x, w, prenorm=True)
    assert z is x and y.dtype == torch.float64
    dy = torch.randn_like(y)
    (grad,) = torch.autograd.grad([y, z], x, [dy, dy])
    want = torch.autograd.grad(torch.nn.functional.layer_norm(x, (40,)), x, dy)[0] + dy
    assert grad.dtype == torch.float64
    torch.testing.assert_close(grad, want, rtol=1e-5, atol=1e-5)
