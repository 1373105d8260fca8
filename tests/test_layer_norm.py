"""layer_norm_fn: layer norm and RMS norm of a residual stream.

The oracle is float64 numpy (oracle/lm.py); on the CPU its gradients are
pinned against central differences. The kernels are checked on the GPU.

Tolerances, from the formats: a row's sums have dim terms and a parameter's
gradient has one per row; summed in blocks, their rounding stays below
sqrt(terms) x 2**-24 of the sum of magnitudes, under 1e-5 of the result's
scale for the sizes here (sums of random signs cancel to 1 / sqrt(terms) of
their magnitudes, so 2**-24 x terms / sqrt(terms) at most 64 x 6e-8 = 4e-6).
16-bit outputs add half a unit in the last place, 2**-8 or 2**-11 relative.
dx is a difference of terms of size rstd t, which cancel in rows of one
element: its scale is theirs where that is larger.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
STORE = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 1e-5


def close(got, want, name="", terms=0.0):
    """`terms`: the size of what a difference was formed from, where that cancels."""
    dtype = got.dtype
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, name
    scale = max(np.abs(want).max(), terms, 1e-30) if want.size else 1.0
    bound = F32 * scale + STORE[dtype] * np.abs(want) * (1 + 1e-3) + (6e-8 if dtype == torch.float16 else 0.0)
    err = np.abs(got - want)
    assert np.all(err <= bound), f"{name}: worst err/bound {np.nanmax(err / bound):.3g}"


def draw(shape, dtype, res, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = shape[-1]
    t = {"x": (r(*shape) + 0.3).to(dtype), "w": 1 + 0.2 * r(d), "b": 0.2 * r(d), "dy": r(*shape).to(dtype)}
    t["res"] = None if res is None else (2 * r(*shape)).to(res)
    t["dz"] = r(*shape).to(res or dtype)
    return {k: None if v is None else v.to(device) for k, v in t.items()}


@pytest.mark.parametrize("rms", [False, True])
def test_oracle_gradients_match_differences(rms):
    t = {k: v.double() for k, v in draw((3, 5), torch.float64, torch.float64, seed=1).items()}

    def loss():
        y, z = O.norm_fwd(t["x"], t["w"], t["b"], t["res"], rms=rms)
        return (y * t["dy"].numpy()).sum() + (z * t["dz"].numpy()).sum()

    dz, dw, db = O.norm_bwd(t["x"], t["w"], t["dy"], t["b"], t["res"], t["dz"], rms=rms)
    for name, grad in (("x", dz), ("res", dz), ("w", dw), ("b", db)):
        flat, num = t[name].reshape(-1), np.empty(t[name].numel())
        for i in range(flat.numel()):
            old = flat[i].item()
            flat[i] = old + 1e-5
            up = loss()
            flat[i] = old - 1e-5
            num[i] = (up - loss()) / 2e-5
            flat[i] = old
        np.testing.assert_allclose(grad.reshape(-1), num, rtol=1e-6, atol=1e-8, err_msg=name)


def test_refuses_cpu_tensors():
    import mamba_cpu

    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.layer_norm_fn(torch.zeros(2, 4), torch.ones(4))


def _block(**kw):
    from mamba_cpu import _C

    a = _C.NormArgs()
    a.x = a.weight = a.y = a.rstd = a.mean = a.dy = a.dx = a.dweight = 16
    a.rows, a.dim, a.eps = 4, 8, 1e-5
    a.x_stride = a.res_stride = a.y_stride = a.dy_stride = 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_abi_refuses_bad_blocks():
    import ctypes

    from mamba_cpu import _C

    L, bad = _C.lib, _C.MCPU_ERR_INVALID
    for kw in ({"x": None}, {"weight": None}, {"rows": -1}, {"dtype": 5}, {"dtype": 1, "res_dtype": 2},
               {"rms": 2}, {"eps": -1.0}, {"eps": float("nan")}, {"x_stride": -8}, {"y": None}):
        assert L.mcpu_norm_fwd(ctypes.byref(_block(**kw)), None) == bad, kw
    assert L.mcpu_norm_fwd(ctypes.byref(_block(rows=1 << 40)), None) == _C.MCPU_ERR_UNSUPPORTED
    assert L.mcpu_norm_fwd(None, None) == bad and L.mcpu_norm_bwd(None, None, 0, None) == bad
    a = _block()
    need = L.mcpu_norm_bwd_workspace_size(ctypes.byref(a))
    assert need >= 2 * 4 * 8
    assert L.mcpu_norm_bwd(ctypes.byref(a), 16, need - 1, None) == bad
    assert "workspace" in L.mcpu_last_error().decode()
    for kw in ({"dy": None}, {"rstd": None}, {"mean": None}, {"dweight": None}, {"bias": 16}):
        assert L.mcpu_norm_bwd(ctypes.byref(_block(**kw)), 16, need, None) == bad, kw
    assert L.mcpu_norm_bwd_workspace_size(None) == 0


gpu = pytest.mark.gpu
# One element, odd widths, one row, widths of a wave and of many waves, the widest in a few rows.
SHAPES = [(1, 1), (3, 7), (5, 64), (1, 768), (70, 129), (33, 1000), (9, 2560), (4, 8191), (2, 20000), (300, 16)]


def _check(t, rms, prenorm, bias=True, layout=lambda v: v, wide=False):
    import mamba_cpu

    names = [k for k in ("x", "res", "w", "b") if t[k] is not None and (bias or k != "b")]
    leaves = {k: (layout(t[k]) if k in ("x", "res") else t[k]).detach().requires_grad_() for k in names}
    out = mamba_cpu.layer_norm_fn(leaves["x"], leaves["w"], leaves.get("b"), residual=leaves.get("res"),
                                  prenorm=prenorm, residual_in_fp32=wide, is_rms_norm=rms)
    y, z = out if prenorm else (out, None)
    wy, wz = O.norm_fwd(t["x"], t["w"], t["b"] if bias else None, t["res"], rms=rms)
    assert y.dtype == t["x"].dtype
    close(y, wy, "y")
    dz_out = None
    if prenorm:
        close(z, wz, "residual")
        dz_out = t["dz"].to(z.dtype)
    grads = torch.autograd.grad([y, z] if prenorm else [y], list(leaves.values()),
                                [t["dy"], dz_out] if prenorm else [t["dy"]])
    dz, dw, db = O.norm_bwd(t["x"], t["w"], t["dy"], None, t["res"], dz_out, rms=rms)
    centred = wz if rms else wz - wz.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt((centred ** 2).mean(-1) + 1e-5)
    terms = rstd.max() * (t["dy"] * t["w"]).abs().max().item()
    for k, got in zip(names, grads):
        close(got, {"x": dz, "res": dz, "w": dw, "b": db}[k], "d" + k, terms if k in ("x", "res") else 0.0)


@gpu
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype,res", [(torch.float32, None), (torch.float32, torch.float32),
                                       (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                       (torch.float16, torch.float32), (torch.float16, None)])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_oracle(shape, dtype, res, rms):
    print(f"norm {shape} {dtype} residual {res} rms {rms}", flush=True)
    _check(draw(shape, dtype, res, seed=shape[0], device=DEV), rms, prenorm=res is not None)


@gpu
@pytest.mark.parametrize("prenorm,wide", [(False, False), (True, False), (True, True)])
def test_forms_of_the_residual(prenorm, wide):
    print(f"norm prenorm {prenorm} residual_in_fp32 {wide}", flush=True)
    for res in (None, torch.float32, torch.bfloat16):
        t = draw((3, 5, 96), torch.bfloat16, res, seed=4, device=DEV)
        if prenorm and res is None and not wide:
            import mamba_cpu

            y, z = mamba_cpu.layer_norm_fn(t["x"], t["w"], prenorm=True)
            assert z is t["x"]
            continue
        _check(t, False, prenorm, bias=False, wide=wide)


@gpu
@pytest.mark.parametrize("kind", ["wide rows", "offset by one", "transposed", "expanded"])
def test_any_strides(kind):
    print(f"norm strides: {kind}", flush=True)
    t = draw((6, 130), torch.bfloat16, torch.float32, seed=5, device=DEV)
    make = {
        "wide rows": lambda v: torch.cat([v, v], -1)[:, :130],
        "offset by one": lambda v: torch.cat([v[:, :1], v], -1)[:, 1:],
        "transposed": lambda v: v.t().contiguous().t(),
        "expanded": lambda v: v,
    }[kind]
    t["dy"] = t["dy"][:1, :1].expand(6, 130) if kind == "expanded" else make(t["dy"])
    if kind == "expanded":
        t["res"] = t["res"][:1].expand(6, 130)
    _check(t, True, True, layout=make)


@gpu
def test_constant_and_extreme_rows():
    """A constant row has zero variance: y = bias. A row holding NaN or an
    infinity leaves the others alone. A mean far from zero keeps its variance:
    the row's own rounding is 1e4 x 2**-24 against a spread of 1."""
    import mamba_cpu

    print("norm extremes", flush=True)
    t = draw((8, 300), torch.float32, None, seed=6, device=DEV)
    t["x"][0] = 5.0
    t["x"][2, 7], t["x"][5, 0] = float("nan"), float("inf")
    y = mamba_cpu.layer_norm_fn(t["x"], t["w"], t["b"])
    torch.testing.assert_close(y[0], t["b"], rtol=0, atol=1e-6)
    want, _ = O.norm_fwd(t["x"], t["w"], t["b"])
    good = [0, 1, 3, 4, 6, 7]
    close(y[good], want[good], "rows beside NaN")
    assert torch.isnan(y[2]).all() and torch.isnan(y[5]).any()
    far = t["x"][[1, 3]] + 1e4
    want, _ = O.norm_fwd(far, t["w"], t["b"])
    np.testing.assert_allclose(mamba_cpu.layer_norm_fn(far, t["w"], t["b"]).cpu().numpy(), want, atol=2e-3)


@gpu
@pytest.mark.parametrize("shape", [(0, 8), (2, 0, 8), (3, 0)])
def test_empty(shape):
    import mamba_cpu

    print(f"norm empty {shape}", flush=True)
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
    res = torch.zeros(shape, device=DEV, requires_grad=True)
    y, z = mamba_cpu.layer_norm_fn(x, w, b, residual=res, prenorm=True)
    assert y.shape == shape and z.shape == shape
    grads = torch.autograd.grad([y, z], [x, w, b, res], [torch.zeros_like(y), torch.zeros_like(z)])
    assert all(torch.count_nonzero(g) == 0 for g in grads)


@gpu
def test_results_do_not_change_from_call_to_call():
    import mamba_cpu

    print("norm twice", flush=True)
    t = draw((1000, 520), torch.bfloat16, torch.float32, seed=7, device=DEV)
    runs = []
    for _ in range(2):
        leaves = [t[k].detach().requires_grad_() for k in ("x", "w", "b", "res")]
        y, z = mamba_cpu.layer_norm_fn(*leaves[:3], residual=leaves[3], prenorm=True)
        runs.append([y, z, *torch.autograd.grad([y, z], leaves, [t["dy"], t["dz"]])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
def test_gpu_refusals():
    import mamba_cpu

    t = draw((4, 10), torch.float32, torch.float32, device=DEV)
    f = mamba_cpu.layer_norm_fn
    for args, kw in (((t["x"], t["w"][:9]), {}), ((t["x"], t["w"], t["b"][:9]), {}), ((t["x"], t["w"]), {"eps": -1.0}),
                     ((t["x"], t["w"]), {"residual": t["res"][:2]}), ((t["x"], t["w"].cpu()), {}),
                     ((t["x"], t["w"][None]), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)


@gpu
def test_operator_checks():
    print("norm opcheck", flush=True)
    t = draw((6, 40), torch.float32, torch.float32, device=DEV)
    x, w, b, res = (t[k].requires_grad_() for k in ("x", "w", "b", "res"))
    torch.library.opcheck(torch.ops.mamba_cpu.norm_fwd.default, (x, w, b, res, 1e-5, False, True, False),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
