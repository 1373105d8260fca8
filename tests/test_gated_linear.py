"""Gated linear recurrence: gated_linear_scan_fn and gated_linear_update.

The oracle is a float64 loop over the steps (oracle/lm.py); on the CPU it is
pinned against central differences and against each packed sequence run alone.
The kernels are checked on the GPU against it.

Tolerances, fixed from the formats: a float32 result is a chain of products
and sums whose rounding errors decay with the state itself; with decays up to
0.999 a state remembers about 1000 steps, whose 2**-24 errors add up as a
random walk to about 30 x 2**-24 = 2e-6 of the state's size: 2e-5 leaves ten
times that for sums of gradients. 16-bit outputs add half a unit in the last
place: 2**-8 for bfloat16 (8 significant bits), 2**-11 for float16 (11 bits, whose smallest steps near zero
are 6e-8), relative to the value.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
STORE = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2e-5


def draw(b, l, d, dtype=torch.float32, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": r(b, l, d), "a_gate": 1.5 * r(b, l, d), "x_gate": r(b, l, d), "dy": r(b, l, d)}
    t = {k: v.to(dtype).to(device) for k, v in t.items()}
    keep = 0.9 + 0.099 * torch.rand(d, generator=g)
    t["decay"] = torch.log(torch.expm1(-torch.log(keep) / 8.0)).to(device)
    t["init"], t["dlast"] = r(b, d).to(device), r(b, d).to(device)
    return t


def packed(b, l, count, seed=1):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.sort((torch.rand(b, count - 1, generator=g) * l).long(), dim=1).values
    return (torch.arange(l)[None, :, None] >= cuts[:, None, :]).sum(-1)


def close(got, want, dtype=torch.float32, name=""):
    """Within the format's half unit of each value, and F32 of the tensor's largest."""
    got = got.detach().double().cpu().numpy() if hasattr(got, "detach") else np.asarray(got)
    assert got.shape == want.shape, name
    scale = max(np.abs(want).max(), 1e-30) if want.size else 1.0
    tiny = 6e-8 if dtype == torch.float16 else 0.0
    err = np.abs(got - want)
    bound = F32 * scale + STORE[dtype] * np.abs(want) * (1 + 1e-3) + tiny
    assert np.all(err <= bound), f"{name}: worst err/bound {np.nanmax(err / bound):.3g}, finite {np.isfinite(got).all()}"


# ---- the oracle, on the CPU ----


def test_oracle_gradients_match_differences():
    t = draw(2, 5, 3, seed=3)
    t = {k: v.double() for k, v in t.items()}
    ids = torch.tensor([[0, 0, 1, 1, 1], [0, 0, 0, 0, 2]])
    names = ("x", "a_gate", "x_gate", "decay", "init")

    def loss(v):
        y, last = O.gated_scan_fwd(v["x"], v["a_gate"], v["x_gate"], v["decay"], v["init"], ids)
        return (y * v["dy"].numpy()).sum() + (last * v["dlast"].numpy()).sum()

    grads = O.gated_scan_bwd(t["x"], t["a_gate"], t["x_gate"], t["decay"], t["dy"], t["init"], ids, dlast=t["dlast"])
    for name, grad in zip(names, grads):
        flat, num = t[name].reshape(-1), np.empty(t[name].numel())
        for i in range(flat.numel()):
            old = flat[i].item()
            hi, lo = old + 1e-5, old - 1e-5
            flat[i] = hi
            up = loss(t)
            flat[i] = lo
            num[i] = (up - loss(t)) / (hi - lo)
            flat[i] = old
        # Central differences: truncation about 1e-10, rounding about 1e-16 / 1e-5.
        np.testing.assert_allclose(grad.reshape(-1), num, rtol=1e-6, atol=1e-8, err_msg=name)


def test_oracle_packed_equals_separate_sequences():
    t = draw(1, 9, 4, seed=4)
    ids = torch.tensor([[3, 3, 3, 3, 7, 7, 8, 8, 8]])
    y, last = O.gated_scan_fwd(t["x"], t["a_gate"], t["x_gate"], t["decay"], t["init"], ids)
    for lo, hi, init in ((0, 4, t["init"]), (4, 6, None), (6, 9, None)):
        sl = [t[k][:, lo:hi] for k in ("x", "a_gate", "x_gate")]
        part, end = O.gated_scan_fwd(*sl, t["decay"], init)
        np.testing.assert_allclose(y[:, lo:hi], part, rtol=1e-14)
    np.testing.assert_allclose(last, end, rtol=1e-14)


def test_oracle_step_is_the_scan():
    t = draw(2, 4, 3, seed=5)
    y, _ = O.gated_scan_fwd(t["x"], t["a_gate"], t["x_gate"], t["decay"], t["init"])
    h = t["init"]
    for i in range(4):
        h = O.gated_step(h, t["x"][:, i], t["a_gate"][:, i], t["x_gate"][:, i], t["decay"])
        np.testing.assert_allclose(h, y[:, i], rtol=1e-14)


# ---- refusals, on the CPU ----


def test_refuses_cpu_tensors_and_bad_arguments():
    import mamba_cpu

    t = draw(1, 4, 3)
    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.gated_linear_scan_fn(t["x"], t["a_gate"], t["x_gate"], t["decay"])
    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.gated_linear_update(t["init"], t["x"][:, 0], t["a_gate"][:, 0], t["x_gate"][:, 0], t["decay"])


def _block(**kw):
    from mamba_cpu import _C

    a = _C.GatedScanArgs()
    a.x = a.a_gate = a.x_gate = a.decay = a.y = a.dy = a.dx = a.da_gate = a.dx_gate = a.ddecay = a.ckpt = 16
    a.batch, a.seqlen, a.dim, a.c, a.dtype = 2, 33, 8, 8.0, _C.MCPU_F32
    for s in (a.x_stride, a.a_stride, a.i_stride, a.y_stride, a.dy_stride, a.dx_stride, a.da_stride, a.di_stride):
        s[:] = (33 * 8, 8, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code,word", [
    ({"x": None}, "INVALID", "required"), ({"decay": None}, "INVALID", "required"),
    ({"batch": -1}, "INVALID", "negative size"), ({"dtype": 9}, "INVALID", "dtype"),
    ({"c": -1.0}, "INVALID", "c must"), ({"c": float("nan")}, "INVALID", "c must"),
    ({"batch": 1 << 40}, "UNSUPPORTED", "too large"), ({"y": None}, "INVALID", "y is required"),
])
def test_abi_refuses_bad_scan_blocks(change, code, word):
    import ctypes

    from mamba_cpu import _C

    rc = _C.lib.mcpu_gated_scan_fwd(ctypes.byref(_block(**change)), None, 0, None)
    assert rc == getattr(_C, "MCPU_ERR_" + code) and word in _C.lib.mcpu_last_error().decode()


def test_abi_sizes_and_backward_refusals():
    import ctypes

    from mamba_cpu import _C

    L, a = _C.lib, _block()
    assert L.mcpu_gated_scan_ckpt_size(ctypes.byref(a)) == 4 * 2 * 3 * 8  # a state per 16 of 33 steps
    need = L.mcpu_gated_scan_bwd_workspace_size(ctypes.byref(a))
    assert need >= 4 * 2 * 8
    for change in ({"ckpt": None}, {"ddecay": None}, {"dy": None}):
        assert L.mcpu_gated_scan_bwd(ctypes.byref(_block(**change)), 16, need, None) == _C.MCPU_ERR_INVALID
    rc = L.mcpu_gated_scan_bwd(ctypes.byref(a), 16, need - 1, None)
    assert rc == _C.MCPU_ERR_INVALID and "workspace" in L.mcpu_last_error().decode()
    a.a_stride[1] = -8
    assert L.mcpu_gated_scan_bwd(ctypes.byref(a), 16, need, None) == _C.MCPU_ERR_INVALID
    assert L.mcpu_gated_scan_ckpt_size(None) == 0
    assert L.mcpu_gated_scan_bwd(None, None, 0, None) == _C.MCPU_ERR_INVALID
    assert L.mcpu_gated_step(None, None) == _C.MCPU_ERR_INVALID


def test_abi_refuses_bad_step_blocks():
    import ctypes

    from mamba_cpu import _C

    def rc(**kw):
        a = _C.GatedStepArgs()
        a.state = a.x = a.a_gate = a.x_gate = a.decay = a.y = 16
        a.batch, a.dim, a.state_batch, a.c = 2, 8, 2, 8.0
        for s in (a.state_stride, a.x_stride, a.a_stride, a.i_stride):
            s[:] = (8, 1)
        for k, v in kw.items():
            setattr(a, k, v)
        return _C.lib.mcpu_gated_step(ctypes.byref(a), None)

    for kw in ({"y": None}, {"state": None}, {"state_batch": 1}, {"dim": -1}, {"c": -2.0}, {"dtype": 3}):
        assert rc(**kw) == _C.MCPU_ERR_INVALID, kw


# ---- the kernels ----

gpu = pytest.mark.gpu
# One token, odd lengths and widths, segment and chunk edges (8 and 32 steps), long rows.
SHAPES = [(1, 1, 1), (2, 7, 3), (1, 8, 64), (3, 33, 65), (2, 32, 130), (1, 257, 128), (2, 1021, 40), (1, 3001, 96)]


def _gpu(t):
    return {k: v.to(DEV) for k, v in t.items()}


def _check(t, dtype, ids=None, init=True, dlast=True, c=8.0, layout=lambda v: v):
    import mamba_cpu

    names = ["x", "a_gate", "x_gate", "decay"] + (["init"] if init else [])
    leaves = {k: layout(t[k]).detach().requires_grad_() if k in ("x", "a_gate", "x_gate")
              else t[k].detach().requires_grad_() for k in names}
    y, last = mamba_cpu.gated_linear_scan_fn(
        leaves["x"], leaves["a_gate"], leaves["x_gate"], leaves["decay"], initial_state=leaves.get("init"),
        seq_idx=ids, c=c, return_last_state=True)
    assert y.dtype == dtype and last.dtype == torch.float32
    args = (t["x"], t["a_gate"], t["x_gate"], t["decay"])
    wy, wlast = O.gated_scan_fwd(*args, t["init"] if init else None, ids, c)
    close(y, wy, dtype, "y")
    close(last, wlast, name="last")
    grads = torch.autograd.grad([y, last] if dlast else [y], list(leaves.values()),
                                [t["dy"], t["dlast"]] if dlast else [t["dy"]])
    want = O.gated_scan_bwd(*args, t["dy"], t["init"] if init else None, ids, c, t["dlast"] if dlast else None)
    for k, got, w in zip(names, grads, want):
        close(got, w, dtype if k in ("x", "a_gate", "x_gate") else torch.float32, "d" + k)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_matches_oracle(shape, dtype):
    print(f"gated scan {shape} {dtype}", flush=True)
    _check(_gpu(draw(*shape, dtype=dtype, seed=sum(shape))), dtype)


@gpu
@pytest.mark.parametrize("shape", [(2, 65, 70), (1, 1500, 33)])
@pytest.mark.parametrize("count", [2, 6])
def test_packed_sequences_match_oracle(shape, count):
    print(f"gated scan packed {shape} x{count}", flush=True)
    t = _gpu(draw(*shape, dtype=torch.bfloat16, seed=7))
    ids = packed(shape[0], shape[1], count).to(DEV)
    _check(t, torch.bfloat16, ids)
    _check(t, torch.bfloat16, torch.arange(shape[1], device=DEV).expand(shape[0], -1))  # every step its own


@gpu
def test_without_states_and_with_another_c():
    print("gated scan without initial or last state's gradient, c 2 and 0", flush=True)
    t = _gpu(draw(2, 100, 20, seed=8))
    _check(t, torch.float32, init=False, dlast=False)
    _check(t, torch.float32, init=False, dlast=False, c=2.0)
    _check(t, torch.float32, c=0.0)  # no decay and no input: the state stays


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["time-contiguous", "every other channel", "wide rows", "offset by one", "expanded"])
def test_any_strides(kind, dtype):
    print(f"gated scan strides: {kind} {dtype}", flush=True)
    t = _gpu(draw(2, 77, 66, dtype=dtype, seed=9))
    make = {
        "time-contiguous": lambda v: v.transpose(1, 2).contiguous().transpose(1, 2),
        "every other channel": lambda v: torch.stack([v, v + 1], -1).flatten(2)[..., ::2],
        "wide rows": lambda v: torch.cat([v, v], -1)[..., :v.shape[-1]],
        "offset by one": lambda v: torch.cat([v[..., :1], v], -1)[..., 1:],
        "expanded": lambda v: v,
    }[kind]
    if kind == "expanded":
        t["dy"] = t["dy"][:1, :1, :1].expand_as(t["dy"])
        t["a_gate"] = t["a_gate"][:, :, :1].expand_as(t["x"])
    else:
        t["dy"] = make(t["dy"])
    _check(t, dtype, layout=make)


@gpu
def test_extreme_gates():
    """Gates and decays at both ends: closed (a = 1, m = 0), wide open (a = 0), infinite."""
    print("gated scan extreme gates", flush=True)
    t = _gpu(draw(1, 24, 8, seed=10))
    t["a_gate"][0, :, 0], t["a_gate"][0, :, 1], t["a_gate"][0, :, 2] = -200.0, 200.0, float("inf")
    t["a_gate"][0, :, 3], t["x_gate"][0, :, 4], t["x_gate"][0, :, 5] = -30.0, -200.0, float("inf")
    t["x_gate"][0, :, 3] = -float("inf")
    t["decay"][6], t["decay"][7] = -60.0, 30.0
    _check(t, torch.float32)


@gpu
def test_nan_stays_in_its_channel():
    import mamba_cpu

    print("gated scan NaN", flush=True)
    t = _gpu(draw(1, 40, 70, seed=11))
    clean = mamba_cpu.gated_linear_scan_fn(t["x"], t["a_gate"], t["x_gate"], t["decay"])
    t["x"][0, 20, 5] = float("nan")
    t["a_gate"][0, 3, 66] = float("nan")
    y = mamba_cpu.gated_linear_scan_fn(t["x"], t["a_gate"], t["x_gate"], t["decay"])
    nan = torch.isnan(y[0])
    assert nan[20:, 5].all() and nan[3:, 66].all()
    nan[20:, 5] = False
    nan[3:, 66] = False
    assert not nan.any()
    other = torch.ones(70, dtype=torch.bool, device=DEV)
    other[[5, 66]] = False
    assert torch.equal(y[..., other], clean[..., other])


@gpu
@pytest.mark.parametrize("b,l,d", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
def test_without_steps_rows_or_channels(b, l, d):
    import mamba_cpu

    print(f"gated scan empty {b, l, d}", flush=True)
    t = _gpu(draw(b, l, d)) if d else {k: torch.zeros(s, device=DEV) for k, s in
                                       (("x", (b, l, d)), ("a_gate", (b, l, d)), ("x_gate", (b, l, d)),
                                        ("dy", (b, l, d)), ("decay", (d,)), ("init", (b, d)), ("dlast", (b, d)))}
    leaves = [t[k].requires_grad_() for k in ("x", "a_gate", "x_gate", "decay", "init")]
    y, last = mamba_cpu.gated_linear_scan_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
    assert y.shape == (b, l, d) and torch.equal(last, t["init"].detach())
    grads = torch.autograd.grad([y, last], leaves, [t["dy"], t["dlast"]])
    assert [g.shape for g in grads] == [v.shape for v in leaves]
    assert torch.count_nonzero(grads[3]) == 0 and torch.equal(grads[4], t["dlast"])


@gpu
def test_results_do_not_change_from_call_to_call():
    import mamba_cpu

    t = _gpu(draw(2, 500, 200, dtype=torch.bfloat16, seed=12))
    print("gated scan twice", flush=True)
    runs = []
    for _ in range(2):
        leaves = [t[k].detach().requires_grad_() for k in ("x", "a_gate", "x_gate", "decay")]
        y = mamba_cpu.gated_linear_scan_fn(*leaves)
        runs.append([y, *torch.autograd.grad([y], leaves, [t["dy"]])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
def test_mixed_and_wide_dtypes_are_computed_in_float32():
    import mamba_cpu

    t = _gpu(draw(1, 20, 6, seed=13))
    want, _ = O.gated_scan_fwd(t["x"].bfloat16(), t["a_gate"], t["x_gate"], t["decay"])
    y = mamba_cpu.gated_linear_scan_fn(t["x"].bfloat16(), t["a_gate"], t["x_gate"], t["decay"])
    assert y.dtype == torch.bfloat16
    close(y, want, torch.bfloat16, "bf16 x, float32 gates")
    y = mamba_cpu.gated_linear_scan_fn(t["x"].double(), t["a_gate"].double(), t["x_gate"].double(), t["decay"])
    assert y.dtype == torch.float64


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,d", [(1, 1), (3, 70), (64, 129)])
def test_update_matches_oracle(b, d, dtype):
    import mamba_cpu

    print(f"gated update {b, d} {dtype}", flush=True)
    t = _gpu(draw(b, 2, d, dtype=dtype, seed=14))
    state = t["init"].clone()
    for i in range(2):
        step = [t[k][:, i] for k in ("x", "a_gate", "x_gate")]
        want = O.gated_step(state, *step, t["decay"])
        y = mamba_cpu.gated_linear_update(state, *step, t["decay"])
        close(state, want, name="state")
        close(y, want, dtype, "y")


@gpu
def test_update_indices_and_strides():
    import mamba_cpu

    print("gated update indexed", flush=True)
    t = _gpu(draw(4, 1, 10, seed=15))
    pool = torch.randn(7, 20, device=DEV)[:, ::2]
    before = pool.clone()
    step = [t[k][:, 0] for k in ("x", "a_gate", "x_gate")]
    y = mamba_cpu.gated_linear_update(pool, *step, t["decay"], state_batch_indices=torch.tensor([5, -1, 0, 7]))
    assert torch.count_nonzero(y[1]) == 0 and torch.count_nonzero(y[3]) == 0
    for row, b in ((5, 0), (0, 2)):
        want = O.gated_step(before[row], *(v[b] for v in step), t["decay"])
        close(pool[row], want, name="state")
    for row in (1, 2, 3, 4, 6):
        assert torch.equal(pool[row], before[row])


@gpu
def test_gpu_refusals():
    import mamba_cpu

    t = _gpu(draw(2, 6, 4))
    ok = [t[k] for k in ("x", "a_gate", "x_gate", "decay")]
    call = mamba_cpu.gated_linear_scan_fn
    for args, kw in (
        ([t["x"][0], *ok[1:]], {}), ([ok[0], t["a_gate"][:, :5], *ok[2:]], {}), ([*ok[:3], t["decay"][:3]], {}),
        (ok, {"c": -1.0}), (ok, {"seq_idx": torch.zeros(2, 5, dtype=torch.int32, device=DEV)}),
        (ok, {"seq_idx": torch.zeros(2, 6, device=DEV)}), (ok, {"initial_state": t["init"][:1]}),
        ([*ok[:3], t["decay"].cpu()], {}),
    ):
        with pytest.raises(ValueError):
            call(*args, **kw)
    step = [v[:, 0] for v in ok[:3]]
    for state, args, kw in (
        (t["init"].bfloat16(), step, {}), (t["init"][:1], step, {}), (t["init"], [step[0], step[1][:1], step[2]], {}),
        (t["init"], step, {"state_batch_indices": torch.zeros(3, dtype=torch.int32, device=DEV)}),
        (t["init"], step, {"c": float("nan")}),
    ):
        with pytest.raises(ValueError):
            mamba_cpu.gated_linear_update(state, *args, t["decay"], **kw)


@gpu
def test_operator_checks():
    """torch.library.opcheck: schema, autograd registration and shape functions."""
    print("gated scan opcheck", flush=True)
    t = _gpu(draw(2, 9, 5, seed=16))
    leaves = [t[k].requires_grad_() for k in ("x", "a_gate", "x_gate", "decay")]
    ids = packed(2, 9, 2).to(DEV, torch.int32)
    torch.library.opcheck(torch.ops.mamba_cpu.gated_scan_fwd.default, (*leaves, t["init"], ids, 8.0, True),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    torch.library.opcheck(torch.ops.mamba_cpu.gated_step.default,
                          (t["init"].clone(), *(t[k].detach()[:, 0] for k in ("x", "a_gate", "x_gate")),
                           t["decay"].detach(), 8.0), test_utils=("test_schema", "test_faketensor"))
