"""sample_fn with settings that mean "off" given per row: a top_k of 0 or below
keeps every token, as the oracle (oracle/lm.py) has it, whatever else cuts; and
a top_k past 31 bits is not another top_k.
"""

import pytest
import torch

from oracle import lm as O

DEV = "cuda"
gpu = pytest.mark.gpu


def draw(b, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, v, generator=g) * 2.5).to(dtype)
    return logits.to(DEV), torch.empty(b, v).exponential_(generator=g).clamp_(min=1e-30).to(DEV)


def check(logits, noise, top_k, top_p, min_p=0.0):
    import mamba_cpu

    token, logprob = mamba_cpu.sample_fn(logits, noise, top_k=top_k, top_p=top_p, min_p=min_p, return_logprobs=True)
    for r in range(len(token)):
        want, lp, kept, near = O.sample(logits[r], noise[r], top_k=int(top_k[r]), top_p=float(top_p[r]), min_p=min_p)
        if near < 1e-5:
            continue
        assert token[r].item() == want, f"row {r}: {token[r].item()} instead of {want}, {kept} kept"
        assert abs(logprob[r].item() - lp) <= 5e-6 + 2.0 ** -23 * abs(lp), f"row {r}"


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [7, 1000, 5000, 50280])
@pytest.mark.parametrize("min_p", [0.0, 0.02])
def test_top_k_below_0_is_off(v, dtype, min_p):
    print(f"sample top_k below 0, {v} {dtype} min_p {min_p}", flush=True)
    b = 24
    logits, noise = draw(b, v, dtype, seed=v)
    top_k = torch.tensor([-1, 0, -1, -2 ** 31, 20, -5], dtype=torch.int32).repeat(4).to(DEV)
    top_p = torch.tensor([0.9, 0.5, 0.99, 1.0]).repeat_interleave(6).to(DEV)
    check(logits, noise, top_k, top_p, min_p)


@gpu
def test_top_k_past_31_bits_keeps_every_token():
    import mamba_cpu

    print("sample top_k past 31 bits", flush=True)
    logits, noise = draw(6, 3000, torch.float32, seed=1)
    top_k = torch.tensor([2 ** 31, 2 ** 32 + 1, 2 ** 63 - 1, -2 ** 63, -2 ** 32 + 3, 2 ** 31 - 1], device=DEV)
    check(logits, noise, top_k, torch.full((6,), 0.9, device=DEV))
    want = mamba_cpu.sample_fn(logits, noise, top_p=0.9)
    assert torch.equal(mamba_cpu.sample_fn(logits, noise, top_k=2 ** 40, top_p=0.9), want)
    for k in (-1, -2 ** 32, -2 ** 63):
        with pytest.raises(ValueError, match="top_k"):
            mamba_cpu.sample_fn(logits, noise, top_k=k)


@gpu
def test_generate_takes_such_settings():
    from mamba_cpu.recurrent_lm import RecurrentLM, generate

    print("generate with top_k below 0 and past 31 bits", flush=True)
    torch.manual_seed(0)
    model = RecurrentLM(vocab_size=300, d_model=32, n_layer=1).to(DEV)
    prompt = torch.randint(300, (3, 5), device=DEV)

    def run(top_k):
        return generate(model, prompt, 6, top_k=torch.tensor(top_k, device=DEV), top_p=0.9,
                        generator=torch.Generator(DEV).manual_seed(2))

    want = run([0, 0, 4])
    assert torch.equal(run([-1, 2 ** 32 + 1, 4]), want)
