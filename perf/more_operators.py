"""The losses of a language model's head as measurable cases: cross entropy and
distillation from a teacher's top logits, both of hidden @ weight.T without the
logits kept, each through its public entry point and in its plain form.

    own                 False: run() computes the plain form; True: it calls the framework
    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU
    run(state)          one pass and its outputs
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   run()'s outputs in 64 bits from the definitions

The plain forms are elementary torch operations in float32, rounded once to the
output's type. Definitions, with s = hidden @ weight.T over (tokens, vocab):

ce    L = log sum_v exp(s_v), loss = L - s_target. A token whose target is the
      ignore index or outside the vocabulary has loss 0 and no gradient, and
      the mean is over the others.
kd    q = softmax(teacher_logits / T) over the token's entries whose id is in
      the vocabulary, L = log sum_v exp(s_v / T),
      loss = T^2 (sum_k q_k log q_k + L - sum_k q_k s_id_k / T). A token
      without entries is left out as above.

Scoring returns the loss of each token (ce: and L); training the mean loss and
the gradients of hidden and weight, or, with "each", the loss of each token and
the gradients for a given gradient of each.

Sizes come from the models this repository runs (d_model 768 and 2560, vocabulary
50280, batches of 8 x 2048 tokens) and from generic odd ones.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100


def _ce(name, dtype, t, v, d, mode, masked=0.0):
    return {"name": name, "op": "ce", "dtype": dtype, "t": t, "v": v, "d": d, "mode": mode, "masked": masked}


def _kd(name, dtype, t, v, d, mode, k, tau, masked=0.0):
    return {**_ce(name, dtype, t, v, d, mode, masked), "op": "kd", "k": k, "tau": tau}


def listed():
    return [
        # The head of a training step on 8 x 2048 tokens.
        _ce("ce_train_bf16_16384_v50280_d768", "bf16", 16384, 50280, 768, "mean"),
        # The same of a wider model, half the tokens: the largest call.
        _ce("ce_train_bf16_8192_v50280_d2560", "bf16", 8192, 50280, 2560, "mean"),
        # Fine-tuning on answers: a ragged batch whose prompts (two thirds of the tokens) are masked.
        _ce("ce_train_bf16_6007_v50280_d768_masked", "bf16", 6007, 50280, 768, "mean", 0.66),
        # A float32 training step on a ragged batch.
        _ce("ce_train_f32_2039_v50280_d768", "f32", 2039, 50280, 768, "mean"),
        # Odd sizes throughout, each token's loss with a weight of its own, as policy gradients have it.
        _ce("ce_train_f16_1021_v32003_d1001_each", "f16", 1021, 32003, 1001, "each"),
        # Scoring of a document: the log-probability of each of its tokens.
        _ce("ce_score_bf16_4096_v50280_d2560", "bf16", 4096, 50280, 2560, "score"),
        # One token of one sequence, as a step of constrained decoding or speculation scores it.
        _ce("ce_score_bf16_1_v50280_d768", "bf16", 1, 50280, 768, "score"),
        # One token for each of a serving batch.
        _ce("ce_score_bf16_33_v50280_d2560", "bf16", 33, 50280, 2560, "score"),
        # Distillation of a small model from stored top logits of a large one.
        _kd("kd_train_bf16_8192_v50280_d768_k64", "bf16", 8192, 50280, 768, "mean", 64, 1.0),
        # Over a large vocabulary, softened, rows with fewer entries and rows without any.
        _kd("kd_train_bf16_2048_v131072_d2560_k32_t2", "bf16", 2048, 131072, 2560, "mean", 32, 2.0, 0.1),
        # A small ragged batch in float32.
        _kd("kd_train_f32_509_v50280_d768_k8", "f32", 509, 50280, 768, "mean", 8, 1.5),
        # The divergence from the teacher over a few validation tokens.
        _kd("kd_score_bf16_16_v50280_d768_k64", "bf16", 16, 50280, 768, "score", 64, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    d = rng.choice([768, 2560, _log(rng, 40, 2560), _log(rng, 40, 2560)])
    v = rng.choice([50280, _log(rng, 200, 131072), _log(rng, 200, 131072)])
    mode = rng.choice(["mean", "mean", "each", "score"])
    # At most a fifth of the largest listed case's products.
    t = max(1, min(_log(rng, 1, 16384), 8192 * 50280 * 2560 // (5 * v * d)))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    masked = rng.choice([0.0, 0.0, 0.3, 0.9])
    if rng.random() < 0.55:
        return {k: x for k, x in _ce("", dtype, t, v, d, mode, masked).items() if k != "name"}
    k = min(_log(rng, 1, 128), v // 2)
    case = _kd("", dtype, t, v, d, mode, k, rng.choice([1.0, 1.0, 2.0, 0.7]), masked)
    return {key: x for key, x in case.items() if key != "name"}


# ---- inputs ----

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    dt, t, v, d = DTYPES[case["dtype"]], case["t"], case["v"], case["d"]
    train = case["mode"] != "score"
    s = {"op": case["op"], "mode": case["mode"]}
    # Rows of about unit length, as embeddings are initialised and as tied heads keep them.
    w = (n(v, d) / math.sqrt(d)).to(dt)
    # Frequencies of tokens about 1 / rank.
    ids = ((torch.exp(u(t) * math.log(v)).long() - 1).clamp_(0, v - 1) * 7919 + 13) % v
    drop = u(t) < case["masked"]
    if case["op"] == "ce":
        s["targets"] = torch.where(drop, torch.full_like(ids, IGNORE), ids)
    else:
        k = case["k"]
        # Distinct ids of falling logits; some rows end early, padded with -1.
        step = (u(t) * (v // k)).long().clamp_(1, max(1, v // k - 1))
        rank = torch.arange(k, device=DEV)
        top = (ids[:, None] + rank[None] * step[:, None]) % v
        s["tl"] = 14 - torch.empty(t, k, device=DEV).exponential_(generator=g).cumsum(1) * min(1.0, 12.0 / k)
        length = torch.where(u(t) < 0.2, (u(t) * k).long() + 1, torch.full_like(ids, k))
        length = torch.where(drop, torch.zeros_like(length), length)
        none = rank[None] >= length[:, None]
        s["top"] = torch.where(none, torch.full_like(top, -1), top)
        s["tl"] = torch.where(none, torch.full_like(s["tl"], -math.inf), s["tl"])
        s["tau"] = case["tau"]
    # What a normalised last layer gives: unit elements, and a pull of any strength towards the right token.
    h = n(t, d) + (16 * u(t))[:, None] * w[ids].float()
    s["h"], s["w"] = h.to(dt), w
    # Loss scale of float16 training.
    s["scale"] = torch.full((), 4096.0 if case["dtype"] == "f16" else 1.0, device=DEV)
    s["g"] = n(t) / math.sqrt(t) * s["scale"] if case["mode"] == "each" else None
    if train:
        s["h"].requires_grad_()
        s["w"].requires_grad_()
    return s


# ---- the plain forms ----

def _teacher(s, real):
    """q and sum q log q per token, and which tokens have entries."""
    have = (s["top"] >= 0) & (s["top"] < s["w"].shape[0])
    x = torch.where(have, s["tl"].to(real), torch.full_like(s["tl"], -math.inf, dtype=real)) / s["tau"]
    mx = x.amax(1, keepdim=True)
    keep = mx[:, 0] > -math.inf
    e = torch.where(have & keep[:, None], torch.exp(x - torch.where(keep[:, None], mx, torch.zeros_like(mx))),
                    torch.zeros_like(x))
    q = e / torch.where(keep, e.sum(1), torch.ones_like(mx[:, 0]))[:, None]
    neg = torch.where(q > 0, q * torch.log(torch.where(q > 0, q, torch.ones_like(q))), torch.zeros_like(q)).sum(1)
    return q, neg, keep


def _plain(s):
    h, w = s["h"].float(), s["w"].float()
    t, dt = h.shape[0], s["h"].dtype
    logits = h @ w.t()
    if s["op"] == "ce":
        tau = 1.0
        keep = (s["targets"] != IGNORE) & (s["targets"] >= 0) & (s["targets"] < w.shape[0])
        at = torch.where(keep, s["targets"], torch.zeros_like(s["targets"]))[:, None]
        q, neg = keep.float()[:, None], torch.zeros(t, device=DEV)
    else:
        tau = s["tau"]
        q, neg, keep = _teacher(s, torch.float32)
        at = torch.where(s["top"] >= 0, s["top"], torch.zeros_like(s["top"]))
        logits /= tau
    mx = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    p = torch.exp(logits.sub_(mx))
    mass = p.sum(1, keepdim=True)
    lse = (mx + torch.log(mass))[:, 0]
    zero = torch.zeros_like(lse)
    each = torch.where(keep, tau * tau * (neg + lse - (q * picked).sum(1)), zero)
    if s["mode"] == "score":
        return {"loss": each, "lse": torch.where(keep, lse, zero)} if s["op"] == "ce" else {"loss": each}
    count = keep.sum().clamp(min=1)
    g = s["g"] if s["g"] is not None else (s["scale"] / count).expand(t)
    g = torch.where(keep, tau * g, zero)
    dl = p.mul_((g / mass[:, 0])[:, None])
    dl.scatter_add_(1, at, -q * g[:, None])
    loss = each if s["mode"] == "each" else each.sum() / count
    return {"loss": loss, "dhidden": (dl @ w).to(dt), "dweight": (dl.t() @ h).to(dt)}


# ---- the framework's calls ----

def _own(s):
    pkg = os.path.join(os.getcwd(), "mamba-cpu_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mamba_cpu

    reduction = "mean" if s["mode"] == "mean" else "none"
    if s["op"] == "ce":
        out = mamba_cpu.linear_cross_entropy_fn(s["h"], s["w"], s["targets"], ignore_index=IGNORE,
                                                reduction=reduction, return_lse=s["mode"] == "score")
        if s["mode"] == "score":
            return {"loss": out[0], "lse": out[1]}
    else:
        out = mamba_cpu.linear_distillation_fn(s["h"], s["w"], s["top"], s["tl"], temperature=s["tau"],
                                               reduction=reduction)
        if s["mode"] == "score":
            return {"loss": out}
    dh, dw = torch.autograd.grad(out, [s["h"], s["w"]], s["scale"] if s["g"] is None else s["g"])
    return {"loss": out.detach(), "dhidden": dh, "dweight": dw}


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _plain(s)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    t, v, d = case["t"], case["v"], case["d"]
    kept = max(1, round(t * (1 - case["masked"])))
    labels = 12 * t * case["k"] if case["op"] == "kd" else 8 * t
    b = (kept + v) * d * e + labels + 4 * t
    if case["mode"] == "score":
        return {"bytes": b, "flops": 2 * kept * v * d}
    return {"bytes": b + (t + v) * d * e, "flops": 6 * kept * v * d}


# ---- 64 bits, from the definitions ----

def exact(case, seed):
    s = prepare(case, seed)
    w = s["w"].detach().double()
    t, (v, d) = case["t"], w.shape
    tau = case.get("tau", 1.0)
    train = case["mode"] != "score"
    # One target distribution per token over the vocabulary, a block of tokens at a time.
    if case["op"] == "ce":
        rows = s["targets"].clamp(0, v - 1)[:, None]
        share = ((s["targets"] != IGNORE) & (s["targets"] >= 0) & (s["targets"] < v)).double()[:, None]
    else:
        rows = s["top"].clamp(0, v - 1)
        score = (s["tl"].double() / tau).masked_fill((s["top"] < 0) | (s["top"] >= v), -math.inf)
        share = torch.softmax(score, 1).nan_to_num(0.0)
    kept = share.sum(1) > 0.5
    count = max(1, int(kept.sum()))
    weight = s["g"].double() if s["g"] is not None else (s["scale"].double() / count).expand(t)
    each = torch.zeros(t, dtype=torch.float64, device=DEV)
    lse = torch.zeros_like(each)
    dh = torch.zeros(t, d, dtype=torch.float64, device=DEV) if train else None
    dw = torch.zeros_like(w) if train else None
    block = max(1, 100_000_000 // v)
    for i in range(0, t, block):
        j = slice(i, min(i + block, t))
        x = s["h"].detach()[j].double()
        z = torch.matmul(x, w.T).div_(tau)
        lse[j] = torch.logsumexp(z, 1).masked_fill(~kept[j], 0.0)
        logp = torch.log_softmax(z, 1)
        cross = torch.special.xlogy(share[j], share[j]) - share[j] * logp.gather(1, rows[j])
        each[j] = cross.sum(1).mul_(tau * tau).masked_fill(~kept[j], 0.0)
        if train:
            dz = logp.exp_()
            dz.scatter_add_(1, rows[j], -share[j])
            dz.mul_((tau * weight[j] * kept[j])[:, None])
            dh[j] = torch.matmul(dz, w)
            dw += torch.matmul(dz.T, x)
    if not train:
        return {"loss": each, "lse": lse} if case["op"] == "ce" else {"loss": each}
    loss = each if case["mode"] == "each" else each.sum() / count
    return {"loss": loss, "dhidden": dh, "dweight": dw}
