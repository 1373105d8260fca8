"""The losses of a language model's head on MI355X: cross entropy, and
distillation from a teacher's top logits, of logits = hidden @ weight.T that are
never kept, forward and backward, over the gfx950 kernels of
csrc/linear_loss.hip. The reference has no such op.

Per token, with s = hidden @ weight.T formed in float32:

    cross entropy   loss = log sum_v exp(s_v) - s_target
    distillation    q = softmax(teacher / T) over the teacher's entries,
                    loss = T^2 sum_k q_k (log q_k - log softmax(s / T)_id_k)

Logits are of hidden and weight as given, summed in float32 (many tokens of
float32: as two float16 pieces each, which keep 22 bits of a value and 2^-38 of
the tensor's largest). hidden and weight of different types, or of others than
float32, bfloat16 and float16, go as float32.

The gradients are products over the logits' gradients ds, rounded once to the
operands' type (float32: to 22 bits, two float16 pieces). A row of ds is kept in a
unit of its own: its target's ds, or with a distillation loss for each row that
row's gradient (bfloat16, and reduced distillation losses, one for all). dweight
takes unit / largest unit from hidden's rows, which cross entropy then rounds once
more to that type. In float16 pieces this holds for rows far below the largest:
down to 2^-16 of it their ds has steps of 2^-37 of its unit, and hidden's elements all
their bits down to 2^-11 of hidden's largest (float32: next to the largest); below,
ds's steps grow as the row gets smaller. The results' sums are float32, rounded
once, in an order that does not change from call to call.

Between forward and backward a call keeps a few numbers a token and, where the
kernels do not read weight as it lies (float32, or 16 bits with a number of columns
that is no multiple of 64 or rows that are no multiple of 16 bytes apart), a copy of it.
"""

import torch

from mamba_cpu import _C  # noqa: F401  (loads the operator library)

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


# mamba_cpu::linear_loss_fwd (autograd through mamba_cpu::linear_loss_bwd) is
# defined in C++ (csrc/torch_loss_ops.cpp, loaded by mamba_cpu._C); these are
# its shape functions for FakeTensor tracing.


def _laid_size(hidden, weight, k, save):
    """Bytes of weight in the products' layout, where it is kept for the backward and would not be read in place from
    an aligned first element on."""
    (tokens, dim), vocab = hidden.shape, weight.shape[0]
    wide = hidden.dtype == torch.float32
    stride = weight.stride(0) if weight.stride(1) == 1 or dim <= 1 else dim
    blocks = tokens <= 64 or -(-vocab // 128) * -(-tokens // 64) <= 512  # read in place too
    if not save or blocks or k == 0 or (
            not wide and dim % 64 == 0 and stride % 8 == 0 and stride <= 2 ** 20):
        return 0
    return 256 + (vocab * -(-dim // 64) * 64 * (4 if wide else 2) + 255) // 256 * 256


@torch.library.register_fake("mamba_cpu::linear_loss_fwd")
def _(hidden, weight, ids, teacher, ignore_index, temperature, reduction, save):
    tokens, k = ids.shape
    f32 = dict(dtype=torch.float32)
    return (hidden.new_empty(() if reduction else (tokens,), **f32), hidden.new_empty(tokens, **f32),
            hidden.new_empty(tokens if teacher is not None else 0, k, **f32), hidden.new_empty(4, tokens, **f32),
            hidden.new_empty(tokens if teacher is not None else 0, k, **f32),
            hidden.new_empty(tokens + 1, dtype=torch.int32),
            hidden.new_empty(_laid_size(hidden, weight, k, save), dtype=torch.uint8))


@torch.library.register_fake("mamba_cpu::linear_loss_bwd")
def _(dloss, dlse, hidden, weight, ids, picked, stat, share, rows, laid, ignore_index, temperature, reduction, distil,
      want_hidden, want_weight):
    return (hidden.new_empty(hidden.shape[0] if want_hidden else 0, hidden.shape[1]),
            weight.new_empty(weight.shape[0] if want_weight else 0, weight.shape[1]))


def _operands(hidden, weight, reduction):
    """hidden as (tokens, dim) and weight, of one type that the kernels take."""
    if hidden.device.type != "cuda":
        raise ValueError(f"mamba_cpu (MI355X build) runs on ROCm GPU tensors, got device {hidden.device}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden must be (..., dim) and weight (vocab, dim), got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if weight.shape[1] == 0:
        raise ValueError("hidden and weight have no columns")
    dt = hidden.dtype if hidden.dtype in _DTYPES and weight.dtype == hidden.dtype else torch.float32
    tokens = hidden.numel() // hidden.shape[-1]
    return hidden.to(dt).reshape(tokens, hidden.shape[-1]), weight.to(dt)


def _saved(hidden, weight):
    """Whether a backward may follow, for which the forward then keeps the weight as it laid it out."""
    return torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)


def _ids(name, ids, shape, device):
    if ids.dtype not in (torch.int32, torch.int64) or ids.shape[:len(shape)] != shape:
        raise ValueError(f"{name} must be an integer tensor of shape {tuple(shape)}, got {tuple(ids.shape)} "
                         f"{ids.dtype}")
    if ids.device != device:
        raise ValueError(f"{name} must be on {device}, got {ids.device}")
    return ids


def linear_cross_entropy_fn(hidden, weight, targets, ignore_index=-100, reduction="mean", return_lse=False):
    """
    hidden: (..., dim); weight: (vocab, dim); targets: integer, hidden's shape
        without its last
    ignore_index: a target that leaves its token out, as any target outside
        [0, vocab) does
    reduction: "mean" over the tokens not left out (0 when there is none), "sum",
        or "none"
    Returns loss: () or, for "none", targets' shape, float32 [, lse: targets' shape,
    float32, log sum_v exp(s_v)]. Tokens left out have loss and lse 0 and no
    gradient, and nothing in them, NaN included, reaches another. Without a
    gradient wanted, -loss of "none" is the targets' log-probability.

    Differentiable in hidden and weight, through loss and lse (once: the gradient
    has no gradient of its own); the backward forms the logits again.
    """
    h, w = _operands(hidden, weight, reduction)
    ids = _ids("targets", targets, hidden.shape[:-1], hidden.device).reshape(-1, 1)
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must be {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}")
    loss, lse, *_ = torch.ops.mamba_cpu.linear_loss_fwd(h, w, ids.contiguous(), None, int(ignore_index), 1.0,
                                                       _REDUCTIONS[reduction], _saved(h, w))
    if reduction == "none":
        loss = loss.view(targets.shape)
    return (loss, lse.view(targets.shape)) if return_lse else loss


def linear_distillation_fn(hidden, weight, teacher_ids, teacher_logits, temperature=1.0, reduction="mean"):
    """
    hidden: (..., dim); weight: (vocab, dim)
    teacher_ids: integer (..., k), the tokens a teacher rated highest, and
        teacher_logits: (..., k), their logits or log-probabilities; k at most 1024.
        An id outside [0, vocab) or a logit of -inf leaves its entry out; an id
        given twice has both entries' shares.
    temperature: divides both sides' logits, 2^-60 to 2^60
    reduction: as linear_cross_entropy_fn's; tokens without entries are left out
    Returns loss: () or, for "none", hidden's shape without its last, float32:
    temperature^2 times the divergence of softmax(s / temperature) over the whole
    vocabulary from the teacher's softmax over its entries.

    Differentiable in hidden and weight (once); teacher_logits must not require
    a gradient.
    """
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
        raise ValueError(f"temperature must lie in 2^-60 to 2^60, got {temperature}")
    h, w = _operands(hidden, weight, reduction)
    lead = hidden.shape[:-1]
    ids = _ids("teacher_ids", teacher_ids, lead, hidden.device)
    if ids.dim() != len(lead) + 1 or teacher_logits.shape != ids.shape:
        raise ValueError(f"teacher_ids and teacher_logits must be {tuple(lead)} + (k,), got {tuple(ids.shape)} and "
                         f"{tuple(teacher_logits.shape)}")
    if teacher_logits.device != hidden.device:
        raise ValueError(f"teacher_logits must be on {hidden.device}, got {teacher_logits.device}")
    shape = (h.shape[0], ids.shape[-1])
    loss, *_ = torch.ops.mamba_cpu.linear_loss_fwd(
        h, w, ids.reshape(shape).contiguous(), teacher_logits.float().reshape(shape).contiguous(), -1,
        float(temperature), _REDUCTIONS[reduction], _saved(h, w))
    return loss.view(lead) if reduction == "none" else loss
