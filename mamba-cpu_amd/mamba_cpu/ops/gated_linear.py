"""Gated linear recurrence on MI355X: sequences (forward and backward) and one
token at a time, over the gfx950 kernels of csrc/gated_scan.hip.

The recurrent block beside Mamba's: each channel keeps one number, decayed by
a gate of the input. Per batch row, step t and channel d:

    rho = sigmoid(a_gate)    iota = sigmoid(x_gate)    s = c softplus(decay_d) rho
    a = exp(-s)              m = sqrt(1 - exp(-2 s))
    h_t = a h_{t-1} + m iota x_t,    y_t = h_t         (h_{-1} = initial_state or 0)

The reference has no such op. Arithmetic and states are float32 for every
storage type; y and the gradients of x and the gates are rounded once to x's.
"""

import torch

from mamba_cpu import _C  # noqa: F401  (loads the operator library)

_X_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_SEG = 16  # steps between the states the forward keeps


# mamba_cpu::gated_scan_fwd (autograd through mamba_cpu::gated_scan_bwd) and
# the in-place mamba_cpu::gated_step are defined in C++ (csrc/torch_lm_ops.cpp,
# loaded by mamba_cpu._C); these are their shape functions for FakeTensor
# tracing.


@torch.library.register_fake("mamba_cpu::gated_scan_fwd")
def _(x, a_gate, x_gate, decay, initial_state, seq_idx, c, save):
    b, l, d = x.shape
    kept = b * ((l + _SEG - 1) // _SEG) * d if save else 0
    return x.new_empty(x.shape), decay.new_empty(b, d), decay.new_empty(kept)


@torch.library.register_fake("mamba_cpu::gated_scan_bwd")
def _(dy, dlast_state, x, a_gate, x_gate, decay, initial_state, seq_idx, c, ckpt):
    return (x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape), decay.new_empty(decay.shape),
            decay.new_empty(initial_state.shape if initial_state is not None else (0,)))


@torch.library.register_fake("mamba_cpu::gated_step")
def _(state, x, a_gate, x_gate, decay, c, state_batch_indices=None):
    return x.new_empty(x.shape)


def _one_dtype(*tensors):
    """The storage type of x and the gates: x's if all share it and the
    kernels take it, float32 otherwise."""
    dt = tensors[0].dtype
    return dt if dt in _X_DTYPES and all(t.dtype == dt for t in tensors) else torch.float32


def gated_linear_scan_fn(x, a_gate, x_gate, decay, initial_state=None, seq_idx=None, c=8.0,
                         return_last_state=False):
    """
    x: (batch, seqlen, dim); a_gate, x_gate: like x, before their sigmoids
    decay: (dim,), before its softplus
    initial_state: optional (batch, dim), the state before the first step
    seq_idx: optional (batch, seqlen) int32 or int64 (compared in their low 32
        bits) ids of packed sequences: the state does not cross a change of id;
        the initial state belongs to the first id of each row
    c: the decay's factor, not negative
    Returns y like x, in x's dtype [, last_state: (batch, dim) float32].

    Any strides; differentiable in x, a_gate, x_gate, decay and initial_state
    (through y and last_state).
    """
    if x.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {x.device}")
    if x.dim() != 3:
        raise ValueError(f"gated_linear_scan_fn expects x (batch, seqlen, dim), got {tuple(x.shape)}")
    if not c >= 0:
        raise ValueError(f"c must not be negative, got {c}")
    in_dtype = x.dtype
    dt = _one_dtype(x, a_gate, x_gate)
    if seq_idx is not None:
        if seq_idx.dtype not in (torch.int32, torch.int64) or seq_idx.shape != x.shape[:2]:
            raise ValueError(f"seq_idx must be an integer tensor of shape {tuple(x.shape[:2])}")
        seq_idx = seq_idx.to(device=x.device, dtype=torch.int32).contiguous()
    init = None if initial_state is None else initial_state.float().contiguous()
    save = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, a_gate, x_gate, decay, initial_state))
    y, last, _ = torch.ops.mamba_cpu.gated_scan_fwd(
        x.to(dt), a_gate.to(dt), x_gate.to(dt), decay.float().contiguous(), init, seq_idx, float(c), save)
    y = y.to(in_dtype)
    return (y, last) if return_last_state else y


def gated_linear_update(state, x, a_gate, x_gate, decay, c=8.0, state_batch_indices=None):
    """One token per batch row. Updates state in place.

    state: (batch, dim) float32; x, a_gate, x_gate: (batch, dim); decay: (dim,)
    state_batch_indices: optional (batch,) int; batch row b then updates
        state[state_batch_indices[b]] (state may have more rows than the batch;
        rows whose index is out of range are skipped and get a zero output).
        Indices must be distinct.
    Returns y like x, in x's dtype: the new state, rounded. No gradient.
    """
    if x.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {x.device}")
    if state.dtype != torch.float32:
        raise ValueError(f"gated_linear_update keeps its state in float32, got {state.dtype}")
    if not c >= 0:
        raise ValueError(f"c must not be negative, got {c}")
    idx = None
    if state_batch_indices is not None:
        if (state_batch_indices.dtype not in (torch.int32, torch.int64)
                or state_batch_indices.shape != (x.shape[0],)):
            raise ValueError(f"state_batch_indices must be an integer tensor of shape ({x.shape[0]},)")
        if state_batch_indices.dtype == torch.int64:  # out of range stays out of range
            state_batch_indices = state_batch_indices.clamp(-1, 2 ** 31 - 1)
        idx = state_batch_indices.to(device=x.device, dtype=torch.int32).contiguous()
    dt = _one_dtype(x, a_gate, x_gate)
    if dt == x.dtype:
        return torch.ops.mamba_cpu.gated_step(state, x, a_gate, x_gate, decay, float(c), idx)
    return torch.ops.mamba_cpu.gated_step(
        state, x.to(dt), a_gate.to(dt), x_gate.to(dt), decay, float(c), idx).to(x.dtype)
