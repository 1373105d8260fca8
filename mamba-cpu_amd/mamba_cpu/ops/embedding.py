"""embedding_fn on MI355X: the scaled lookup of token embeddings and its
gradient, over the gfx950 kernels of csrc/embedding.hip. The reference has no
such op.
"""

import torch

from mamba_cpu import _C  # noqa: F401  (loads the operator library)

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


# mamba_cpu::embedding_fwd (autograd through mamba_cpu::embedding_bwd) is
# defined in C++ (csrc/torch_lm_ops.cpp, loaded by mamba_cpu._C); these are its
# shape functions for FakeTensor tracing.


@torch.library.register_fake("mamba_cpu::embedding_fwd")
def _(ids, weight, scale):
    return weight.new_empty(ids.shape[0], weight.shape[1])


@torch.library.register_fake("mamba_cpu::embedding_bwd")
def _(dout, ids, vocab, scale):
    return dout.new_empty(vocab, dout.shape[1])


def embedding_fn(ids, weight, scale=1.0):
    """
    ids: integer tensor of any shape; weight: (vocab, dim); scale: a number,
        taken as float32
    Returns scale * weight[ids], (*ids.shape, dim) in weight's dtype, formed in
    float32. An id outside [0, vocab) has a zero row and no gradient, so a rank
    that holds a slice of the vocabulary looks up ids minus its first one, and
    the ranks' results add up.

    Differentiable in weight: the gradient of a row is the float32 sum over its
    tokens in a fixed order, rounded once, and does not change from call to call.
    """
    if weight.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {weight.device}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    if weight.dim() != 2:
        raise ValueError(f"weight must be (vocab, dim), got {tuple(weight.shape)}")
    w = weight if weight.dtype in _DTYPES else weight.float()
    out = torch.ops.mamba_cpu.embedding_fwd(ids.reshape(-1), w, float(scale))
    return out.view(*ids.shape, weight.shape[1]).to(weight.dtype)
