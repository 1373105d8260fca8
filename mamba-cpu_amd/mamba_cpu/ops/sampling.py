"""sample_fn on MI355X: one token per row of logits, with temperature, top-k,
top-p and min-p, from given random numbers, over the gfx950 kernels of
csrc/sampling.hip. The reference has no such op.
"""

import torch

from mamba_cpu import _C  # noqa: F401  (loads the operator library)

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


# mamba_cpu::sample is defined in C++ (csrc/torch_lm_ops.cpp, loaded by
# mamba_cpu._C); this is its shape function for FakeTensor tracing.


@torch.library.register_fake("mamba_cpu::sample")
def _(logits, noise, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows,
      logprobs):
    rows = logits.shape[0]
    return (logits.new_empty(rows, dtype=torch.int64),
            logits.new_empty(rows if logprobs else 0, dtype=torch.float32))


# Each setting's type where it is given per row, and what it is where it is off.
SETTINGS = {"temperature": (torch.float32, 1.0), "top_k": (torch.int32, 0), "top_p": (torch.float32, 1.0),
            "min_p": (torch.float32, 0.0)}


def setting_rows(name, value, device):
    """A setting given per row, as the kernel reads it."""
    dtype = SETTINGS[name][0]
    if dtype == torch.int32 and value.dtype == torch.int64:
        value = value.clamp(0, 2 ** 31 - 1)  # below 0 is off, as 0 is
    return value.to(device=device, dtype=dtype).contiguous()


def _setting(name, value, rows, device):
    """(number, per-row tensor or None) of a setting given either way."""
    if not isinstance(value, torch.Tensor):
        return value, None
    if value.shape != (rows,):
        raise ValueError(f"{name} must be a number or a tensor of shape ({rows},), got {tuple(value.shape)}")
    return SETTINGS[name][1], setting_rows(name, value, device)


def sample_fn(logits, noise=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprobs=False):
    """
    logits: (batch, vocab); noise: (batch, vocab) float32 from Exp(1), e.g.
        torch.empty(batch, vocab, device=...).exponential_(); above 0. May be
        None where temperature is the number 0.
    temperature, top_k, top_p, min_p: numbers, or tensors of shape (batch,)
        with one setting for each row. top_k 0 (per row also below 0), top_p 1
        and min_p 0 are off; temperature 0 takes the largest logit.
    Returns tokens: (batch,) int64 [, logprobs: (batch,) float32, the
    log-softmax of the logits (before temperature and cuts) at the token].

    In the order of the logits (descending, equal ones by index), with
    w = exp((l - max) / temperature): top-k keeps the first k; then top-p keeps
    a token while the mass before it is below top_p of what top-k kept; then
    min-p keeps w >= min_p. The first token is always kept. The token is the
    kept one with the largest w / noise, which draws from the kept in
    proportion to w; the same noise gives the same token. A row whose logits
    are all -inf or NaN gives token -1 and logprob -inf; NaN counts as -inf.
    No gradient: the log-probability is cut from the logits' graph.
    """
    if logits.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {logits.device}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be (batch, vocab), got {tuple(logits.shape)}")
    rows, dev = logits.shape[0], logits.device
    t, t_rows = _setting("temperature", temperature, rows, dev)
    k, k_rows = _setting("top_k", top_k, rows, dev)
    p, p_rows = _setting("top_p", top_p, rows, dev)
    m, m_rows = _setting("min_p", min_p, rows, dev)
    if logits.dtype not in _DTYPES:
        logits = logits.float()
    token, logprob = torch.ops.mamba_cpu.sample(logits, noise, float(t), int(k), float(p), float(m), t_rows, k_rows,
                                                p_rows, m_rows, bool(return_logprobs))
    return (token, logprob) if return_logprobs else token
