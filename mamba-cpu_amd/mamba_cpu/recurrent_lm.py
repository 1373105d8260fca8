"""A language model of gated linear recurrences over this package's ops:
training, prompts (whole or in pieces), packed sequences, and sampled decoding
with each token's step replayed from a HIP graph.

    model = RecurrentLM(vocab_size=50280, d_model=768, n_layer=24).cuda()
    loss = model.loss(ids[:, :-1], ids[:, 1:])
    tokens = generate(model, prompt, max_new_tokens=128, temperature=0.8, top_p=0.95)

A block is RMS norm -> in_proj (to u and a gate z) -> causal conv1d with silu
-> the recurrence, its two gates a linear function of the conv's output ->
times silu(z) -> out_proj, on a residual stream kept in float32. The blocks are
those of Griffin ("Griffin: Mixing Gated Linear Recurrences with Local
Attention for Efficient Language Models", 2024) without its attention and MLP
layers and with one dense matrix for the gates. The reference has no such model.

Per call the token embedding is embedding_fn, the norms (with the residual
sum) layer_norm_fn, the recurrence gated_linear_scan_fn or, for one token,
gated_linear_update, and the choice of a token sample_fn; the losses are
linear_cross_entropy_fn and linear_distillation_fn over the embedding's weight, so
that training keeps no logits; the blocks' products are the library's.
"""

import math

import torch
from torch import nn

from mamba_cpu.ops import (
    causal_conv1d_fn,
    causal_conv1d_update,
    embedding_fn,
    gated_linear_scan_fn,
    gated_linear_update,
    layer_norm_fn,
    linear_cross_entropy_fn,
    linear_distillation_fn,
    sample_fn,
)
from mamba_cpu.ops.sampling import setting_rows


class RecurrentBlock(nn.Module):
    def __init__(self, d_model, d_inner, d_conv, c):
        super().__init__()
        self.c = c
        self.norm_weight = nn.Parameter(torch.ones(d_model))
        self.in_proj = nn.Linear(d_model, 2 * d_inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(d_inner, d_conv).uniform_(-1, 1) / math.sqrt(d_conv))
        self.conv_bias = nn.Parameter(torch.zeros(d_inner))
        self.gates = nn.Linear(d_inner, 2 * d_inner)
        # A fully open gate decays by 0.9 to 0.999 a step.
        open_decay = torch.empty(d_inner).uniform_(0.9, 0.999)
        self.decay = nn.Parameter(torch.log(torch.expm1(-torch.log(open_decay) / c)))
        self.out_proj = nn.Linear(d_inner, d_model, bias=False)

    def forward(self, normed, seq_idx=None, conv_state=None, state=None):
        """normed: (batch, seqlen, d_model). conv_state (batch, d_inner, d_conv - 1) and state
        (batch, d_inner) are what the tokens before left, and are overwritten with what these leave."""
        u, z = self.in_proj(normed).chunk(2, dim=-1)
        keep = conv_state is not None
        u = causal_conv1d_fn(u.transpose(1, 2), self.conv_weight, self.conv_bias, seq_idx=seq_idx,
                             initial_states=conv_state, return_final_states=keep, activation="silu")
        if keep:
            u, final = u
            conv_state.copy_(final)
        u = u.transpose(1, 2)
        a_gate, x_gate = self.gates(u).chunk(2, dim=-1)
        y, last = gated_linear_scan_fn(u, a_gate, x_gate, self.decay, initial_state=state, seq_idx=seq_idx, c=self.c,
                                       return_last_state=True)
        if state is not None:
            state.copy_(last)
        return self.out_proj(y * nn.functional.silu(z))

    def step(self, normed, conv_state, state):
        """normed: (batch, d_model), one token per row."""
        u, z = self.in_proj(normed).chunk(2, dim=-1)
        u = causal_conv1d_update(u, conv_state, self.conv_weight, self.conv_bias, activation="silu")
        a_gate, x_gate = self.gates(u).chunk(2, dim=-1)
        y = gated_linear_update(state, u, a_gate, x_gate, self.decay, c=self.c)
        return self.out_proj(y * nn.functional.silu(z))


class RecurrentLM(nn.Module):
    """forward(ids (batch, seqlen)[, seq_idx]) -> logits (batch, seqlen, vocab_size). The head shares the
    embedding's weight, which embedding_fn scales by sqrt(d_model)."""

    def __init__(self, vocab_size, d_model, n_layer, d_inner=None, d_conv=4, c=8.0, eps=1e-6):
        super().__init__()
        self.d_inner, self.d_conv, self.eps = d_inner or 2 * d_model, d_conv, eps
        self.scale = math.sqrt(d_model)
        self.embedding = nn.Parameter(torch.randn(vocab_size, d_model) / self.scale)
        self.blocks = nn.ModuleList(RecurrentBlock(d_model, self.d_inner, d_conv, c) for _ in range(n_layer))
        self.norm_weight = nn.Parameter(torch.ones(d_model))

    def _run(self, ids, block_call):
        hidden, residual = embedding_fn(ids, self.embedding, self.scale), None
        for i, block in enumerate(self.blocks):
            normed, residual = layer_norm_fn(hidden, block.norm_weight, residual=residual, eps=self.eps, prenorm=True,
                                             residual_in_fp32=True, is_rms_norm=True)
            hidden = block_call(i, block, normed)
        return layer_norm_fn(hidden, self.norm_weight, residual=residual, eps=self.eps, is_rms_norm=True)

    def forward(self, ids, seq_idx=None):
        return self._hidden(ids, seq_idx) @ self.embedding.t()

    def _hidden(self, ids, seq_idx=None):
        return self._run(ids, lambda i, block, x: block(x, seq_idx=seq_idx))

    def loss(self, ids, targets, seq_idx=None, ignore_index=-100, reduction="mean"):
        """Cross entropy of targets (batch, seqlen) against forward(ids)'s logits, which are not formed as a whole
        (linear_cross_entropy_fn). With "none" and no gradient: minus the targets' log-probabilities."""
        return linear_cross_entropy_fn(self._hidden(ids, seq_idx), self.embedding, targets, ignore_index=ignore_index,
                                       reduction=reduction)

    def distillation_loss(self, ids, teacher_ids, teacher_logits, temperature=1.0, seq_idx=None, reduction="mean"):
        """Divergence of forward(ids)'s logits from a teacher's top ones, (batch, seqlen, k) each
        (linear_distillation_fn)."""
        return linear_distillation_fn(self._hidden(ids, seq_idx), self.embedding, teacher_ids, teacher_logits,
                                      temperature=temperature, reduction=reduction)

    def new_cache(self, batch):
        """Per block the conv window and the state, as before the first token."""
        w = self.embedding
        return [(w.new_zeros(batch, self.d_inner, self.d_conv - 1),
                 w.new_zeros(batch, self.d_inner, dtype=torch.float32)) for _ in self.blocks]

    @torch.no_grad()
    def prefill(self, ids, cache):
        """ids (batch, seqlen >= 1), the next tokens of each row -> logits (batch, vocab_size) after the last;
        advances the cache in place."""
        hidden = self._run(ids, lambda i, block, x: block(x, None, *cache[i]))
        return hidden[:, -1] @ self.embedding.t()

    @torch.no_grad()
    def step(self, token, cache):
        """token (batch,) -> logits (batch, vocab_size); advances the cache in place."""
        return self._run(token, lambda i, block, x: block.step(x, *cache[i])) @ self.embedding.t()


@torch.no_grad()
def generate(model, prompt, max_new_tokens, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator=None):
    """The prompt (batch, seqlen) in one forward, then one HIP graph replay a token: the embedding through the
    logits and the choice of the token (sample_fn's settings, numbers or one for each row). `generator` (of the
    model's device) gives the noise, drawn between replays, one (batch, vocab) draw a token.
    Returns (batch, seqlen + max_new_tokens) int64 ids."""
    dev = model.embedding.device
    if dev.type != "cuda":
        raise ValueError(f"graph-captured decoding runs on ROCm GPU models, got device {dev}")
    if prompt.dim() != 2 or prompt.shape[1] == 0:
        raise ValueError(f"generate expects a prompt (batch, seqlen >= 1), got {tuple(prompt.shape)}")
    if max_new_tokens < 1:
        return prompt.long()
    batch, vocab = prompt.shape[0], model.embedding.shape[0]
    # Settings given per row are put where the kernel reads them before the capture.
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    settings = {k: setting_rows(k, v, dev) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    cache = model.new_cache(batch)
    new = torch.empty(batch, max_new_tokens, dtype=torch.long, device=dev)
    noise = torch.empty(batch, vocab, device=dev).exponential_(generator=generator)
    token = sample_fn(model.prefill(prompt, cache), noise, **settings)
    new[:, 0] = token
    if max_new_tokens > 1:
        saved = [tuple(t.clone() for t in layer) for layer in cache]
        # One step on a side stream first (first-call work stays out of the
        # graph), then the cache as the prompt left it.
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            sample_fn(model.step(token, cache), noise, **settings)
        torch.cuda.current_stream(dev).wait_stream(side)
        for layer, kept in zip(cache, saved):
            for t, s in zip(layer, kept):
                t.copy_(s)
        torch.cuda.synchronize(dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            token.copy_(sample_fn(model.step(token, cache), noise, **settings))
        for i in range(1, max_new_tokens):
            noise.exponential_(generator=generator)
            graph.replay()
            new[:, i] = token
    return torch.cat([prompt.long(), new], dim=1)
