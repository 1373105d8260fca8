"""sample_fn: temperature, top-k, top-p, min-p and the race of exponentials.

The oracle is float64 numpy (oracle/lm.py), one row at a time; on the CPU it is
pinned by what the definitions say (what is kept, the frequencies of a race).
On the GPU tokens have to be the oracle's. The oracle also says how near its
choice was (the relative distance of the closest things it compared); a row
nearer than 1e-5, a hundred float32 roundings, is left out, and at most one row in a
hundred may be. Log-probabilities: each is a difference of numbers up to 40, so
within 40 x 2**-23 = 5e-6, plus 2**-23 of itself.
"""

import ctypes

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"


# ---- the oracle, on the CPU ----


def test_oracle_keeps_what_the_cuts_say():
    l = torch.tensor([[1.0, 3.0, 3.0, 0.0, -float("inf"), float("nan"), 2.0]])
    w = np.exp([3.0, 3.0, 2.0, 1.0, 0.0])
    p = w / w.sum()
    noise = torch.ones(1, 7)
    assert O.sample(l, noise, 1.0)[0] == 1  # ties by index
    assert O.sample(l, noise, 0.0)[:1] == (1,)
    for k, n in ((1, 1), (2, 2), (3, 3), (100, 7)):
        assert O.sample(l, noise, top_k=k)[2] == n
    assert O.sample(l, noise, top_p=p[0] + 1e-3)[2] == 2
    assert O.sample(l, noise, top_p=p[:3].sum() - 1e-3)[2] == 3
    assert O.sample(l, noise, top_p=0.0)[2] == 1
    assert O.sample(l, noise, top_k=2, top_p=0.4)[2] == 1  # of the two kept
    assert O.sample(l, noise, min_p=np.exp(-1.5))[2] == 3
    assert O.sample(l, noise, min_p=1.0)[2] == 2
    assert O.sample(torch.full((1, 3), -float("inf")), noise)[:2] == (-1, -np.inf)
    assert abs(O.sample(l, noise)[1] - np.log(p[0])) < 1e-12


def test_oracle_race_draws_by_weight():
    """Frequencies of 20000 draws against the kept weights: each within five
    standard deviations."""
    rng = np.random.default_rng(0)
    l = torch.tensor([[0.3, 1.0, -0.5, 2.0, 0.9]])
    n = 20000
    got = np.bincount([O.sample(l, torch.from_numpy(rng.exponential(size=(1, 5))), 0.8, top_k=3)[0]
                       for _ in range(n)], minlength=5) / n
    w = np.exp(l[0].double().numpy() / 0.8) * [0, 1, 0, 1, 1]
    want = w / w.sum()
    assert np.all(np.abs(got - want) <= 5 * np.sqrt(want * (1 - want) / n))


# ---- refusals, on the CPU ----


def test_refusals_on_the_cpu():
    import mamba_cpu
    from mamba_cpu import _C

    with pytest.raises(ValueError, match="ROCm GPU"):
        mamba_cpu.sample_fn(torch.zeros(2, 4), torch.ones(2, 4))
    L, bad = _C.lib, _C.MCPU_ERR_INVALID

    def rc(**kw):
        a = _C.SampleArgs()
        a.logits = a.noise = a.token = 16
        a.rows, a.vocab, a.logits_stride, a.noise_stride = 2, 50, 50, 50
        a.temperature, a.top_p = 1.0, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return L.mcpu_sample(ctypes.byref(a), None, 0, None)

    for kw in ({"logits": None}, {"noise": None}, {"token": None}, {"rows": -1}, {"vocab": 0}, {"dtype": 7},
               {"logits_stride": -1}, {"temperature": float("nan")}, {"top_p": 1.5}, {"top_p": -0.1},
               {"top_p": float("nan")}, {"min_p": 2.0}, {"top_k": -1}):
        assert rc(**kw) == bad, kw
    assert rc(vocab=(1 << 23) + 1) == _C.MCPU_ERR_UNSUPPORTED
    assert L.mcpu_sample(None, None, 0, None) == bad and L.mcpu_sample_workspace_size(None) == 0


gpu = pytest.mark.gpu


def draw(b, v, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, v, generator=g) * spread).to(dtype)
    return logits.to(DEV), torch.empty(b, v).exponential_(generator=g).clamp_(min=1e-30).to(DEV)


def check(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    import mamba_cpu

    token, logprob = mamba_cpu.sample_fn(logits, noise, temperature, top_k, top_p, min_p, return_logprobs=True)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    only = mamba_cpu.sample_fn(logits, noise, temperature, top_k, top_p, min_p)
    assert torch.equal(only, token)
    token, logprob = token.cpu().numpy(), logprob.cpu().numpy()
    at = lambda s, r: s[r].item() if isinstance(s, torch.Tensor) else s  # noqa: E731
    b, left_out = logits.shape[0], 0
    for r in range(b):
        want, lp, kept, near = O.sample(logits[r], noise[r], at(temperature, r), at(top_k, r), at(top_p, r),
                                        at(min_p, r))
        if near < 1e-5:
            left_out += 1
            continue
        assert token[r] == want, f"row {r}: {token[r]} instead of {want}, {kept} kept, near {near:.2g}"
        if np.isinf(lp):
            assert logprob[r] == lp
        else:
            assert abs(logprob[r] - lp) <= 5e-6 + 2.0 ** -23 * abs(lp), f"row {r}: logprob {logprob[r]} for {lp}"
    assert left_out <= max(1, b // 100), f"{left_out} of {b} rows too near to tell"


SETTINGS = [{}, {"temperature": 0.0}, {"temperature": 0.7, "top_k": 50}, {"top_k": 1}, {"top_p": 0.9},
            {"top_p": 0.0}, {"top_p": 0.999, "temperature": 1.5}, {"min_p": 0.05}, {"min_p": 1.0},
            {"temperature": 0.8, "top_k": 40, "top_p": 0.95}, {"top_k": 700, "top_p": 0.6, "min_p": 0.01},
            {"top_k": 10 ** 9}, {"top_k": 3000, "top_p": 0.99, "temperature": 3.0}]


@gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("b,v,dtype", [(1, 1, torch.float32), (5, 7, torch.float32), (3, 1024, torch.bfloat16),
                                       (2, 50280, torch.float32), (2, 50280, torch.bfloat16),
                                       (2, 33333, torch.float16), (1, 131072, torch.float32)])
def test_matches_oracle(b, v, dtype, kw):
    print(f"sample {b} x {v} {dtype} {kw}", flush=True)
    check(*draw(b, v, dtype, seed=v + b), **kw)


@gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_flat_and_tied_logits(kw):
    """All equal, two levels, and 16-bit logits of a narrow range: large classes
    of equal logits on both sides of every cut."""
    print(f"sample ties {kw}", flush=True)
    logits, noise = draw(4, 9001, torch.bfloat16, seed=2, spread=0.05)
    logits[0] = 1.5
    logits[1] = (torch.arange(9001, device=DEV) % 3 == 1).to(torch.bfloat16)
    logits[2] = torch.where(logits[2] > 0, 0.0, -0.0)
    if kw.get("top_p", 1.0) not in (0.0, 1.0):  # j < p n is decided by p's rounding for equal logits
        logits, noise = logits[1:].clone(), noise[1:]
        logits[1, ::2] = 0.25
    check(logits, noise, **kw)


@gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_masked_and_infinite_logits(kw):
    print(f"sample masks {kw}", flush=True)
    inf = float("inf")
    logits, noise = draw(9, 2000, seed=3)
    logits[0] = -inf
    logits[1] = float("nan")
    logits[2, 1:] = -inf
    logits[3, ::2] = -inf
    logits[4, 5:] = torch.finfo(torch.float32).min
    logits[5, 100] = inf
    logits[6, 100], logits[6, 7], logits[6, 3] = inf, inf, float("nan")
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 17] = float("nan")
    if 0 < kw.get("top_p", 1.0) < 1:  # the equal logits of row 7 again
        logits[7, 0] = 0.0
    check(logits, noise, **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_settings_per_row(dtype):
    print(f"sample settings per row {dtype}", flush=True)
    b = 64
    logits, noise = draw(b, 5000, dtype, seed=4)
    g = torch.Generator().manual_seed(5)
    pick = lambda vals, dt: torch.tensor(vals, dtype=dt)[torch.randint(len(vals), (b,), generator=g)].to(DEV)  # noqa: E731
    check(logits, noise, temperature=pick([0.0, 0.6, 1.0, 1.7], torch.float32),
          top_k=pick([0, 1, 50, 2000, 9000], torch.int64), top_p=pick([1.0, 0.9, 0.3, 0.0], torch.float32),
          min_p=pick([0.0, 0.02, 1.0], torch.float32))


@gpu
@pytest.mark.parametrize("kind", ["wide rows", "offset by one", "transposed", "one row for all"])
def test_any_strides(kind):
    print(f"sample strides: {kind}", flush=True)
    logits, noise = draw(5, 3001, torch.bfloat16, seed=6)
    make = {"wide rows": lambda v: torch.cat([v, v], -1)[:, :3001],
            "offset by one": lambda v: torch.cat([v[:, :1], v], -1)[:, 1:],
            "transposed": lambda v: v.t().contiguous().t(), "one row for all": lambda v: v[:1].expand(5, -1)}[kind]
    check(make(logits), make(noise), temperature=0.9, top_k=60, top_p=0.9)


@gpu
def test_odd_noise():
    """Noise at its ends: the smallest float32 wins, infinity loses; equal
    scores go to the lowest index."""
    import mamba_cpu

    print("sample odd noise", flush=True)
    logits, noise = torch.zeros(3, 500, device=DEV), torch.ones(3, 500, device=DEV)
    noise[0, 77] = 1e-37
    noise[1, :400] = float("inf")
    got = mamba_cpu.sample_fn(logits, noise)
    assert got.tolist() == [77, 400, 0]


@gpu
def test_greedy_without_noise_and_no_rows():
    import mamba_cpu

    print("sample greedy, no rows", flush=True)
    logits, _ = draw(3, 50280, torch.bfloat16, seed=8)
    want = [int((row == row.max()).nonzero()[0]) for row in logits.cpu()]
    assert mamba_cpu.sample_fn(logits, temperature=0.0).tolist() == want
    token, logprob = mamba_cpu.sample_fn(logits[:0], torch.ones(0, 50280, device=DEV), return_logprobs=True)
    assert token.shape == (0,) and logprob.shape == (0,)


@gpu
def test_draws_by_weight():
    """20000 rows of one distribution: frequencies within five standard deviations."""
    import mamba_cpu

    print("sample frequencies", flush=True)
    l = torch.tensor([0.3, 1.0, -0.5, 2.0, 0.9], device=DEV)
    n = 20000
    noise = torch.empty(n, 5, device=DEV).exponential_(generator=torch.Generator(DEV).manual_seed(9))
    got = torch.bincount(mamba_cpu.sample_fn(l.expand(n, 5), noise, 0.8, top_k=3), minlength=5).cpu().numpy() / n
    w = np.exp(l.double().cpu().numpy() / 0.8) * [0, 1, 0, 1, 1]
    want = w / w.sum()
    assert np.all(np.abs(got - want) <= 5 * np.sqrt(want * (1 - want) / n))


@gpu
def test_gpu_refusals_and_operator_checks():
    import mamba_cpu

    print("sample refusals, opcheck", flush=True)
    logits, noise = draw(3, 100)
    f = mamba_cpu.sample_fn
    for args, kw in (((logits[0], noise[0]), {}), ((logits, noise[:2]), {}), ((logits, noise.half()), {}),
                     ((logits, None), {}), ((logits, noise.cpu()), {}), ((logits, noise), {"top_k": -1}),
                     ((logits, noise), {"top_p": 1.1}), ((logits, noise), {"min_p": -0.1}),
                     ((logits, noise), {"temperature": float("nan")}),
                     ((logits, noise), {"top_k": torch.zeros(2, dtype=torch.int32, device=DEV)}),
                     ((logits[:, :0], noise[:, :0]), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    torch.library.opcheck(torch.ops.mamba_cpu.sample.default,
                          (logits, noise, 1.0, 5, 0.9, 0.0, None, None, None, None, True),
                          test_utils=("test_schema", "test_faketensor"))
