"""RecurrentLM and generate: the operators together, against a float64 model
written out in plain torch on the CPU.

Tolerances, from the arithmetic: two blocks are a chain of some 20 operators
whose float32 roundings (2**-24) grow with the square root of the at most 100
terms of a product: 20 x 10 x 6e-8 = 1.2e-5 of a tensor's largest value.
Logits are held to 5e-5 of it and gradients, a chain twice as long, to 1e-4.
"""

import math

import pytest
import torch
import torch.nn.functional as F

from mamba_cpu.recurrent_lm import RecurrentLM, generate

DEV = "cuda"
VOCAB, DMODEL, LAYERS, INNER, CONV = 101, 32, 2, 48, 4


def model(dtype=torch.float32, seed=0, device=DEV):
    torch.manual_seed(seed)
    m = RecurrentLM(VOCAB, DMODEL, LAYERS, d_inner=INNER, d_conv=CONV)
    return m.to(device=device, dtype=dtype)


def draw(b, l, seed=1):
    return torch.randint(0, VOCAB, (b, l), generator=torch.Generator().manual_seed(seed))


def plain_logits(p, ids, eps=1e-6, c=8.0):
    """The model as its formulas read, from float64 parameters."""
    def rms(x, w):
        return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w

    h = F.embedding(ids, p["embedding"]) * math.sqrt(DMODEL)
    l = ids.shape[1]
    for i in range(LAYERS):
        q = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"blocks.{i}.")}
        u, z = (rms(h, q["norm_weight"]) @ q["in_proj.weight"].t()).chunk(2, -1)
        padded = F.pad(u, (0, 0, CONV - 1, 0))
        u = F.silu(sum(padded[:, k:k + l] * q["conv_weight"][:, k] for k in range(CONV)) + q["conv_bias"])
        ga, gx = (u @ q["gates.weight"].t() + q["gates.bias"]).chunk(2, -1)
        s = c * F.softplus(q["decay"]) * torch.sigmoid(ga)
        add = torch.sqrt(1 - torch.exp(-2 * s)) * torch.sigmoid(gx) * u
        state, y = torch.zeros_like(u[:, 0]), []
        for t in range(l):
            state = torch.exp(-s[:, t]) * state + add[:, t]
            y.append(state)
        h = h + (torch.stack(y, 1) * F.silu(z)) @ q["out_proj.weight"].t()
    return rms(h, p["norm_weight"]) @ p["embedding"].t()


def near(got, want, tol, name=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, name
    err = (got - want).abs().max() / want.abs().max()
    assert err <= tol, f"{name}: {err:.3g} of the largest"


def test_refuses_the_cpu():
    m = model(device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        m(draw(1, 4))
    with pytest.raises(ValueError, match="GPU"):
        generate(m, draw(1, 4), 2)


def test_the_plain_model_is_causal_and_differentiable():
    p = {k: v.detach().double().requires_grad_() for k, v in model(device="cpu").named_parameters()}
    ids = draw(1, 9)
    other = ids.clone()
    other[:, 6:] = (other[:, 6:] + 1) % VOCAB
    a, b = plain_logits(p, ids), plain_logits(p, other)
    assert torch.equal(a[:, :6], b[:, :6]) and not torch.equal(a[:, 6:], b[:, 6:])
    w = torch.randn(a.shape, generator=torch.Generator().manual_seed(2)).double()
    grad = torch.autograd.grad((a * w).sum(), p["blocks.0.decay"])[0]
    step = torch.zeros(INNER).double()
    step[5] = 1e-6
    up = plain_logits({**p, "blocks.0.decay": p["blocks.0.decay"] + step}, ids)
    down = plain_logits({**p, "blocks.0.decay": p["blocks.0.decay"] - step}, ids)
    diff = (((up - down) * w).sum() / 2e-6).item()
    assert abs(diff - grad[5].item()) <= 1e-6 * max(1.0, grad.abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("b,l", [(2, 37), (1, 1), (3, 130)])
def test_logits_and_gradients(b, l):
    m, ids = model(), draw(b, l)
    logits = m(ids.to(DEV))
    w = torch.randn(logits.shape, generator=torch.Generator().manual_seed(2))
    (logits * w.to(DEV)).sum().backward()
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in m.named_parameters()}
    want = plain_logits(p, ids)
    (want * w.double()).sum().backward()
    near(logits, want, 5e-5, "logits")
    for k, v in m.named_parameters():
        near(v.grad, p[k].grad, 1e-4, k)


@pytest.mark.gpu
@pytest.mark.parametrize("first", [1, 2, 20, 36])
def test_prompt_in_pieces_and_steps_continue_it(first):
    m, ids = model(), draw(2, 40).to(DEV)
    with torch.no_grad():
        want = m(ids)
    cache = m.new_cache(2)
    near(m.prefill(ids[:, :first], cache), want[:, first - 1], 1e-4, "first piece")
    near(m.prefill(ids[:, first:37], cache), want[:, 36], 1e-4, "second piece")
    for t in range(37, 40):
        near(m.step(ids[:, t], cache), want[:, t], 1e-4, f"token {t}")


@pytest.mark.gpu
def test_packed_rows_equal_separate_sequences():
    m, ids = model(), draw(1, 90).to(DEV)
    cuts = [0, 1, 30, 33, 90]
    seq = torch.zeros(1, 90, dtype=torch.long, device=DEV)
    for c in cuts[1:-1]:
        seq[:, c:] += 1
    with torch.no_grad():
        got = m(ids, seq_idx=seq)
        for lo, hi in zip(cuts, cuts[1:]):
            near(got[:, lo:hi], m(ids[:, lo:hi]), 1e-4, f"{lo}:{hi}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [False, True])
def test_generate_replays_what_single_steps_give(dtype, rows):
    m, prompt, n = model(dtype), draw(3, 7).to(DEV), 12
    settings = {"temperature": 0.8, "top_k": 20, "top_p": 0.95}
    if rows:
        settings = {"temperature": torch.tensor([0.0, 0.7, 1.3]), "top_k": torch.tensor([0, 5, 50]),
                    "top_p": torch.tensor([1.0, 0.9, 1.0]), "min_p": torch.tensor([0.0, 0.0, 0.05])}
    got = generate(m, prompt, n, generator=torch.Generator(DEV).manual_seed(3), **settings)
    again = generate(m, prompt, n, generator=torch.Generator(DEV).manual_seed(3), **settings)
    assert torch.equal(got, again)
    assert torch.equal(got[:, :7], prompt) and got.shape == (3, 7 + n)
    from mamba_cpu import sample_fn

    gen, cache, noise = torch.Generator(DEV).manual_seed(3), m.new_cache(3), torch.empty(3, VOCAB, device=DEV)
    logits = m.prefill(prompt, cache)
    for t in range(n):
        token = sample_fn(logits, noise.exponential_(generator=gen), **settings)
        assert torch.equal(token, got[:, 7 + t]), f"token {t}"
        logits = m.step(token, cache)


@pytest.mark.gpu
def test_greedy_generation_takes_the_largest_logit_of_the_whole_forward():
    m, prompt = model(), draw(2, 5).to(DEV)
    out = generate(m, prompt, 20, temperature=0)
    assert torch.equal(generate(m, prompt, 0), prompt)
    assert torch.equal(generate(m, prompt, 1, temperature=0), out[:, :6])
    with torch.no_grad():
        logits = m(out[:, :-1])[:, 4:]
    chosen = logits.gather(-1, out[:, 5:, None])[..., 0]
    assert (chosen >= logits.amax(-1) - 2e-4 * logits.abs().amax()).all()  # both within 1e-4 of the exact ones


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_learns_a_batch(dtype):
    m = model(dtype)
    opt = torch.optim.AdamW(m.parameters(), lr=3e-3, weight_decay=0.0)
    ids = draw(4, 65).to(DEV)
    losses = []
    for _ in range(30):
        loss = F.cross_entropy(m(ids[:, :-1]).float().flatten(0, 1), ids[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0] - 0.5


@pytest.mark.gpu
def test_generate_refusals():
    m = model()
    with pytest.raises(ValueError, match="prompt"):
        generate(m, torch.zeros(2, 0, dtype=torch.long, device=DEV), 3)
    with pytest.raises(ValueError, match="prompt"):
        generate(m, torch.zeros(4, dtype=torch.long, device=DEV), 3)
