"""Calls whose workgroups have 2**32 threads together or more, which is more than
one launch takes: short rows, many of them. The rows are independent, so the
last ones have to be those of the same call on them alone, bit for bit; equal
rows have equal results.
"""

import pytest
import torch

DEV = "cuda"
gpu = pytest.mark.gpu
TAIL = 1000


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _rows(n, d, tail, dtype=torch.float32):
    """n rows: the first one's values repeated, then `tail`."""
    v = tail[:1].to(dtype).expand(n, d).contiguous()
    v[n - len(tail):] = tail.to(dtype)
    return v


def _same(got, want, name):
    """got's last rows are want's, its others equal to want's first."""
    assert torch.equal(got[-len(want):], want), name
    head = got[:len(got) - len(want)]
    assert bool((head == want[:1]).all()), name


@pytest.mark.parametrize("kw", [{"top_k": 3, "top_p": 0.9}, {}, {"temperature": 0.0}], ids=str)
@gpu
def test_sampled_rows(kw):
    import mamba_cpu

    n = 2 ** 22 + 5000  # workgroups of 1024
    print(f"sample {n} rows {kw}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    logits, noise = torch.randn(TAIL, 5, device=DEV, generator=g), torch.rand(TAIL, 5, device=DEV, generator=g) + 0.1
    want = mamba_cpu.sample_fn(logits, noise, return_logprobs=True, **kw)
    got = mamba_cpu.sample_fn(_rows(n, 5, logits), _rows(n, 5, noise), return_logprobs=True, **kw)
    for a, b, name in zip(got, want, ("token", "logprob")):
        _same(a, b, name)


@gpu
def test_sampled_rows_in_slices():
    """Two slices a row, workgroups of 512; one row's logits for all."""
    import mamba_cpu

    n, v = 2 ** 22 + 5000, 8200
    print(f"sample {n} rows of {v}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    logits = torch.randn(1, v, device=DEV, generator=g)
    noise = torch.rand(1, v, device=DEV, generator=g) + 0.1
    want = mamba_cpu.sample_fn(logits, noise, return_logprobs=True)
    got = mamba_cpu.sample_fn(logits.expand(n, v), noise.expand(n, v), return_logprobs=True)
    for a, b in zip(got, want):
        assert bool((a == b).all())


@pytest.mark.parametrize("rms", [True, False])
@gpu
def test_norm_rows(rms):
    import mamba_cpu

    n = 2 ** 26 + 5000  # four rows a workgroup of 256
    print(f"norm {n} rows, rms {rms}", flush=True)
    x = torch.randn(TAIL, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    w = torch.tensor([1.0, -2.0, 0.5], device=DEV)
    _same(mamba_cpu.layer_norm_fn(_rows(n, 3, x), w, is_rms_norm=rms),
          mamba_cpu.layer_norm_fn(x, w, is_rms_norm=rms), "y")


@gpu
def test_embedding_tokens():
    import mamba_cpu

    n = 2 ** 26 + 5000  # four tokens a workgroup of 256
    print(f"embedding of {n} tokens", flush=True)
    table = torch.randn(7, 2, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    ids = torch.arange(n, device=DEV, dtype=torch.int32) % 9 - 1  # -1 and 7 have zero rows
    out = mamba_cpu.embedding_fn(ids, table)
    rows = torch.cat([torch.zeros(1, 2, device=DEV), table, torch.zeros(1, 2, device=DEV)])
    assert torch.equal(out[:9 * (n // 9)].view(-1, 9, 2), rows.expand(n // 9, 9, 2))
    assert torch.equal(out[9 * (n // 9):], rows[:n % 9])


@gpu
def test_embedding_gradient_of_many_tokens():
    """Ids over every chunk of 32 tokens, ids over many: sums of ones are exact to 2**24."""
    import mamba_cpu

    n = 2 ** 27 + 5000  # a workgroup of 1024 per chunk
    print(f"embedding gradient of {n} tokens", flush=True)
    ids = torch.arange(n, device=DEV, dtype=torch.int32) % 1000
    ids[-40:] = 1000
    table = torch.zeros(1001, 1, device=DEV, requires_grad=True)
    out = mamba_cpu.embedding_fn(ids, table)
    (grad,) = torch.autograd.grad(out, table, torch.ones(1, device=DEV).expand_as(out))
    assert torch.equal(grad[:, 0].long(), torch.bincount(ids, minlength=1001))


@gpu
def test_gated_scan_rows():
    """One channel and step a row: workgroups of 512 forward and 256 backward."""
    import mamba_cpu

    n = 2 ** 24 + 5000
    print(f"gated scan of {n} rows", flush=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    parts = [torch.randn(TAIL, 1, device=DEV, generator=g) for _ in range(4)]
    decay = torch.tensor([0.3], device=DEV)

    def run(x, a, i, init):
        leaves = [v.unsqueeze(1).requires_grad_() for v in (x, a, i)] + [init.requires_grad_()]
        y, last = mamba_cpu.gated_linear_scan_fn(*leaves[:3], decay, initial_state=leaves[3], return_last_state=True)
        return [v.detach().view(-1, 1) for v in (y, last, *torch.autograd.grad(y, leaves, torch.ones_like(y)))]

    want = run(*(p.clone() for p in parts))
    for got, ref, name in zip(run(*(_rows(n, 1, p) for p in parts)), want, ("y", "last", "dx", "da", "di", "dinit")):
        _same(got, ref, name)


@gpu
def test_gated_scan_chunks_of_many_rows():
    """Two chunks a row, handed on from workgroup to workgroup, over more than one launch."""
    import mamba_cpu

    n, l = 2 ** 22 + 3000, 130
    print(f"gated scan of {n} rows of {l} steps", flush=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    x, a, i = (torch.randn(1, l, 1, device=DEV, generator=g).bfloat16() for _ in range(3))
    decay = torch.tensor([-1.0], device=DEV)
    want, want_last = mamba_cpu.gated_linear_scan_fn(x, a, i, decay, return_last_state=True)
    y, last = mamba_cpu.gated_linear_scan_fn(*(v.expand(n, l, 1) for v in (x, a, i)), decay, return_last_state=True)
    assert bool((y == want).all()) and bool((last == want_last).all())


@gpu
def test_gated_update_rows():
    """2**32 channels and more; their inputs are one number."""
    import mamba_cpu

    b, d = 2 ** 16 + 3, 2 ** 16
    print(f"gated update of {b} x {d}", flush=True)
    one = torch.full((1, 1), 0.5, device=DEV, dtype=torch.bfloat16)
    decay = torch.full((d,), -1.0, device=DEV)
    small = torch.full((1, 1), 0.25, device=DEV)
    want = mamba_cpu.gated_linear_update(small, one, one, one, decay[:1])
    state = torch.full((b, d), 0.25, device=DEV)
    y = mamba_cpu.gated_linear_update(state, *(one.expand(b, d) for _ in range(3)), decay)
    assert all(bool((y[r:r + 4096] == want).all()) and bool((state[r:r + 4096] == small).all())
               for r in range(0, b, 4096))


def test_abi_refuses_columns_past_the_grid():
    """The embedding's gradient joins 256 columns a workgroup of the grid's second dimension."""
    import ctypes

    from mamba_cpu import _C

    a = _C.EmbeddingArgs()
    a.ids = a.dout = a.dweight = 16  # placeholders: never dereferenced
    a.tokens, a.vocab, a.dim, a.scale = 1, 1, 65535 * 256 + 1, 1.0
    rc = _C.lib.mcpu_embedding_bwd(ctypes.byref(a), 16, 1 << 40, None)
    assert rc == _C.MCPU_ERR_UNSUPPORTED and "columns" in _C.lib.mcpu_last_error().decode()


@pytest.mark.parametrize("batch,dim", [(2 ** 38 + 1, 1), (2 ** 40, 2 ** 40), (2 ** 62, 4), (3, 2 ** 62)])
def test_abi_refuses_more_channels_than_it_counts(batch, dim):
    """Also where batch x dim itself passes 63 bits."""
    import ctypes

    from mamba_cpu import _C

    a = _C.GatedStepArgs()
    a.state = a.x = a.a_gate = a.x_gate = a.decay = a.y = 16  # placeholders: never dereferenced
    a.batch, a.dim, a.state_batch, a.c = batch, dim, batch, 8.0
    rc = _C.lib.mcpu_gated_step(ctypes.byref(a), None)
    assert rc == _C.MCPU_ERR_UNSUPPORTED and "too large" in _C.lib.mcpu_last_error().decode()
