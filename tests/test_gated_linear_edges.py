"""The gated recurrence at the lengths where its work is split: segments of 16
steps, chunks of 128 forward and 64 backward, windows of 8 and 4 chunks of the
look back (4 windows are kept, those further back are read again).

Against the float64 loop of oracle/lm.py. A state remembers its past over
hundreds of steps, so an error of the split would show in every step behind it;
its rounding, a random walk of 2**-24 a step over 1000 steps, stays within 2e-6
of the largest value: 2e-5 leaves ten times that. bfloat16 adds half a unit,
2**-8 of the value.
"""

import numpy as np
import pytest
import torch

from oracle import lm as O

DEV = "cuda"
gpu = pytest.mark.gpu
FWD, BWD = 128, 64  # steps of a chunk
EDGES = sorted({n + e for n in (16, 48, BWD, FWD, 2 * FWD, 4 * BWD, 5 * BWD) for e in (-1, 0, 1)})
# A window of the forward and of the backward (8 chunks, and 4), two, and those kept (32 and 16), with the first behind.
WINDOWS = [8 * FWD, 9 * FWD + 1, 16 * BWD + 1, 17 * BWD, 32 * FWD + 1, 33 * FWD, 33 * FWD + 1, 41 * FWD + 17]


def run(l, d, dtype, seq_idx=None):
    import mamba_cpu

    g = torch.Generator().manual_seed(l)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, a, i, dy = (r(2, l, d).to(dtype).to(DEV) for _ in range(4))
    init, dlast = r(2, d).to(DEV), r(2, d).to(DEV)
    keep = 0.99 + 0.0095 * torch.rand(d, generator=g)
    decay = torch.log(torch.expm1(-torch.log(keep) / 8.0)).to(DEV)
    leaves = [t.requires_grad_() for t in (x, a, i, decay, init)]
    y, last = mamba_cpu.gated_linear_scan_fn(*leaves[:4], initial_state=init, seq_idx=seq_idx, return_last_state=True)
    grads = torch.autograd.grad([y, last], leaves, [dy, dlast])
    wy, wlast = O.gated_scan_fwd(x, a, i, decay, init, seq_idx)
    want = O.gated_scan_bwd(x, a, i, decay, dy, init, seq_idx, dlast=dlast)
    for name, got, ref in zip(("y", "last", "dx", "da", "di", "ddecay", "dinit"), (y, last, *grads), (wy, wlast, *want)):
        got = got.detach()
        half = 2.0 ** -8 * 1.001 if got.dtype == torch.bfloat16 else 0.0
        err = np.abs(got.double().cpu().numpy() - ref)
        bound = 2e-5 * np.abs(ref).max() + half * np.abs(ref)
        assert np.all(err <= bound), f"{name}, {l} steps: worst err/bound {np.nanmax(err / bound):.3g}"


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("l", EDGES)
def test_segment_and_chunk_edges(l, dtype):
    print(f"gated scan of {l} steps, {dtype}", flush=True)
    run(l, 5, dtype)


@gpu
@pytest.mark.parametrize("l", WINDOWS)
def test_window_edges(l):
    print(f"gated scan of {l} steps", flush=True)
    run(l, 3, torch.float32)


@gpu
@pytest.mark.parametrize("at", [1, 16, 17, 63, 64, 65, 127, 128, 129, 256])
def test_a_sequence_starts_at_an_edge(at):
    print(f"gated scan, another sequence from step {at}", flush=True)
    seq_idx = (torch.arange(300, device=DEV) >= at).int().expand(2, -1)
    run(300, 5, torch.float32, seq_idx)
