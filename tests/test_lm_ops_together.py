"""What the recurrence, norm, embedding and sampling operators share: their
argument blocks, the stream they run on, HIP graphs, tensors past 4 GiB, and
what a NaN or infinity may reach.

The graph and stream checks ask for equal bits: the kernels sum in a fixed
order. Tensors past 4 GiB are checked against the same operator on a copied
part, bit for bit where its rows are independent; the recurrence's part starts
elsewhere, so it is held to the recurrence's own tolerance (2e-5 of the largest
value, and half a unit of the 16-bit type).
"""

import ctypes
import os
import re
import time

import pytest
import torch

from conftest import ROOT

DEV = "cuda"
HEADER = os.path.join(ROOT, "include", "mamba_hip.h")
BLOCKS = [("gated_scan", "GatedScanArgs"), ("gated_step", "GatedStepArgs"), ("norm", "NormArgs"),
          ("embedding", "EmbeddingArgs"), ("sample", "SampleArgs")]


# ---- the argument blocks, on the CPU ----


@pytest.mark.parametrize("name,cls_name", BLOCKS)
def test_argument_blocks_follow_the_header_and_the_library(name, cls_name):
    from mamba_cpu import _C

    cls = getattr(_C, cls_name)
    assert _C.lib.mcpu_args_size(name.encode()) == ctypes.sizeof(cls)
    body = re.search(r"typedef struct mcpu_%s_args \{(.*?)\} mcpu_%s_args;" % (name, name), open(HEADER).read(), re.S)
    text = re.sub(r"/\*.*?\*/", "", body.group(1), flags=re.S)
    fields = []
    for decl in filter(None, (d.strip() for d in text.split(";"))):
        first, *more = re.sub(r"\[\d+\]", "", decl).split(",")
        fields += [first.split()[-1].lstrip("*")] + [m.strip().lstrip("*") for m in more]
    assert [f[0] for f in cls._fields_] == fields


def test_shape_functions_follow_the_operators():
    """The outputs that tracing expects, without a device."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import mamba_cpu

    with FakeTensorMode():
        x = torch.empty(2, 9, 16, device=DEV, dtype=torch.bfloat16)
        y, last = mamba_cpu.gated_linear_scan_fn(x, x, x, torch.empty(16, device=DEV), return_last_state=True)
        assert y.shape == x.shape and y.dtype == x.dtype and last.shape == (2, 16) and last.dtype == torch.float32
        y, z = mamba_cpu.layer_norm_fn(x, torch.empty(16, device=DEV), prenorm=True, residual_in_fp32=True)
        assert y.dtype == x.dtype and z.shape == x.shape and z.dtype == torch.float32
        e = mamba_cpu.embedding_fn(torch.zeros(3, 5, dtype=torch.long, device=DEV), torch.empty(7, 16, device=DEV))
        assert e.shape == (3, 5, 16)
        token, logprob = mamba_cpu.sample_fn(torch.empty(4, 50, device=DEV), torch.empty(4, 50, device=DEV),
                                             return_logprobs=True)
        assert token.shape == (4,) and token.dtype == torch.int64 and logprob.shape == (4,)


# ---- streams and graphs ----


def _draw(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    b, l, d, v = 2, 300, 64, 9000
    return {
        "ids": torch.randint(0, 500, (b, l), device=DEV, generator=g), "table": r(500, d), "w": 1 + 0.1 * r(d),
        "a": r(b, l, d), "i": r(b, l, d), "decay": r(d), "init": r(b, d),
        "dy": r(b, l, d), "dlast": r(b, d), "logits": 3 * r(4, v), "noise": r(4, v).abs() + 1e-3,
        "state": r(b, d),
    }


LEAVES = ("table", "w", "a", "i", "decay", "init")


def _step(t):
    """Embedding -> norm -> recurrence with their gradients, one token's update, a token."""
    from mamba_cpu import embedding_fn, gated_linear_scan_fn, gated_linear_update, layer_norm_fn, sample_fn

    x, z = layer_norm_fn(embedding_fn(t["ids"], t["table"], 2.0), t["w"], residual=t["a"], prenorm=True,
                         is_rms_norm=True)
    y, last = gated_linear_scan_fn(x, t["a"], t["i"], t["decay"], initial_state=t["init"], return_last_state=True)
    torch.autograd.backward([y, last, z], [t["dy"], t["dlast"], t["dy"]])
    with torch.no_grad():
        state = t["state"].clone()
        step = gated_linear_update(state, y[:, 0], t["a"][:, 0], t["i"][:, 0], t["decay"])
        cut, logprob = sample_fn(t["logits"], t["noise"], temperature=0.9, top_k=40, top_p=0.9, return_logprobs=True)
        free = sample_fn(t["logits"][:1], t["noise"][:1])
    return {"y": y, "last": last, "z": z, "state": state, "step": step, "cut": cut, "logprob": logprob, "free": free}


def _results(t, outs):
    r = {k: v.detach().clone() for k, v in outs.items()}
    r.update({"d" + k: t[k].grad.clone() for k in LEAVES})
    return r


def _eager(seed):
    t = _draw(seed)
    for k in LEAVES:
        t[k].requires_grad_()
    return _results(t, _step(t))


def _equal(got, want, name):
    for k, v in want.items():
        torch.testing.assert_close(got[k], v, rtol=0, atol=0, msg=lambda m, k=k: f"{name}, {k}: {m}")


@pytest.mark.gpu
def test_calls_replay_from_a_graph():
    static = _draw(0)
    for k in LEAVES:
        static[k].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            for k in LEAVES:
                static[k].grad = None
            _step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in LEAVES:
        static[k].grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(static)
    torch.cuda.synchronize()
    for seed in (1, 2, 3, 4):
        with torch.no_grad():
            for k, v in _draw(seed).items():
                static[k].copy_(v)
        graph.replay()
        got = _results(static, outs)
        torch.cuda.synchronize()
        want = _eager(seed)  # eager work between replays
        torch.cuda.synchronize()
        _equal(got, want, f"replay of seed {seed}")


@pytest.mark.gpu
def test_calls_run_on_the_current_stream_without_waiting():
    want = _eager(5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        source = _draw(5)
        torch.cuda.synchronize()
        t = {k: torch.zeros_like(v) for k, v in source.items()}
        t["noise"].fill_(1.0)
        for k in LEAVES:
            t[k].requires_grad_()
        torch.cuda.synchronize()
        torch.cuda._sleep(400_000_000)  # the inputs arrive behind this
        with torch.no_grad():
            for k in t:
                t[k].copy_(source[k])
        start = time.perf_counter()
        outs = _step(t)
        issued = time.perf_counter() - start
        drained = side.query()
        got = _results(t, outs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert not drained, f"the calls returned after {issued:.3f} s, with the queue drained"
    _equal(got, want, "side stream")


# ---- what a NaN or an infinity may reach ----


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_sequence_does_not_see_what_another_of_its_row_holds(bad, dtype):
    """Also where the chunks of 64 steps are bridged, and backward through the cut."""
    from mamba_cpu import gated_linear_scan_fn

    g = torch.Generator(device=DEV).manual_seed(0)
    b, l, d = 2, 700, 66
    x, a, i, dy = (torch.randn(b, l, d, device=DEV, generator=g).to(dtype) for _ in range(4))
    decay = torch.randn(d, device=DEV, generator=g)
    seq = torch.zeros(b, l, dtype=torch.long, device=DEV)
    seq[:, 150:] += 1
    seq[:, 391:] += 1

    def run(x, dy):
        leaves = [v.clone().requires_grad_() for v in (x, a, i)]
        y = gated_linear_scan_fn(*leaves, decay, seq_idx=seq)
        y.backward(dy)
        return [y.detach()] + [v.grad for v in leaves]

    want = run(x, dy)
    x2, dy2 = x.clone(), dy.clone()
    x2[:, 200], dy2[:, 230] = bad, bad
    for name, got, clean in zip(("y", "dx", "da", "di"), run(x2, dy2), want):
        assert torch.equal(got[:, :150], clean[:, :150]) and torch.equal(got[:, 391:], clean[:, 391:]), name
        assert torch.isfinite(clean).all(), name
    assert not torch.isfinite(run(x2, dy2)[0][:, 200:391]).any()


@pytest.mark.gpu
def test_a_bad_row_stays_a_row():
    from mamba_cpu import layer_norm_fn, sample_fn

    g = torch.Generator(device=DEV).manual_seed(0)
    x, dy = (torch.randn(9, 100, device=DEV, generator=g) for _ in range(2))
    w = torch.ones(100, device=DEV)

    def run(x):
        leaf = x.clone().requires_grad_()
        y = layer_norm_fn(leaf, w, eps=1e-5)
        y.backward(dy)
        return y.detach(), leaf.grad

    bad = x.clone()
    bad[3, 7], bad[5, 0] = float("nan"), float("inf")
    keep = [r for r in range(9) if r not in (3, 5)]
    for got, clean in zip(run(bad), run(x)):
        assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[3]).all()
    noise = torch.rand(9, 100, device=DEV, generator=g) + 0.1
    assert torch.equal(sample_fn(bad, noise, top_k=5)[keep], sample_fn(x, noise, top_k=5)[keep])


# ---- many windows of look back ----


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_row_of_few_channels_equals_its_pieces(dtype):
    """400 chunks of one tile, whose states reach far; the pieces hand the state on in float32."""
    from mamba_cpu import gated_linear_scan_fn

    g = torch.Generator(device=DEV).manual_seed(0)
    b, l, d = 1, 25_637, 10
    x, a, i = (torch.randn(b, l, d, device=DEV, generator=g).to(dtype) for _ in range(3))
    decay = torch.full((d,), -9.0, device=DEV)  # a near 0.9995
    whole, last = gated_linear_scan_fn(x, a, i, decay, return_last_state=True)
    state, parts = None, []
    for lo in range(0, l, 4000):
        y, state = gated_linear_scan_fn(x[:, lo:lo + 4000], a[:, lo:lo + 4000], i[:, lo:lo + 4000], decay,
                                        initial_state=state, return_last_state=True)
        parts.append(y)
    want = torch.cat(parts, 1).float()
    bound = 2e-5 * want.abs().max() + (2.0 ** -7 * want.abs() if dtype == torch.bfloat16 else 0)  # both are rounded
    assert ((whole.float() - want).abs() <= bound).all()
    assert ((last - state).abs() <= 2e-5 * state.abs().max()).all()


# ---- tensors past 4 GiB ----


@pytest.fixture
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_norm_rows_past_4_gib(room):
    from mamba_cpu import layer_norm_fn

    rows, dim, tail = 1_100_000, 2048, 100
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.zeros(rows, dim, device=DEV, dtype=torch.bfloat16)
    x[-tail:] = torch.randn(tail, dim, device=DEV, generator=g).bfloat16()
    w = torch.randn(dim, device=DEV, generator=g)
    big, small = x.requires_grad_(), x.detach()[-tail:].clone().requires_grad_()
    y, want = layer_norm_fn(big, w, is_rms_norm=True), layer_norm_fn(small, w, is_rms_norm=True)
    assert torch.equal(y[-tail:], want)
    dy = torch.zeros_like(y)
    dy[-tail:] = torch.randn(tail, dim, device=DEV, generator=g).bfloat16()
    y.backward(dy)
    want.backward(dy[-tail:].clone())
    assert torch.equal(big.grad[-tail:], small.grad)


@pytest.mark.gpu
def test_embedding_table_past_4_gib(room):
    from mamba_cpu import embedding_fn

    vocab, dim = 1_100_000, 2048
    g = torch.Generator(device=DEV).manual_seed(0)
    table = torch.zeros(vocab, dim, device=DEV, dtype=torch.bfloat16)
    table[-500:] = torch.randn(500, dim, device=DEV, generator=g).bfloat16()
    ids = torch.randint(vocab - 500, vocab, (300,), device=DEV, generator=g)
    small = table[-500:].clone().requires_grad_()
    table.requires_grad_()
    y, want = embedding_fn(ids, table), embedding_fn(ids - (vocab - 500), small)
    assert torch.equal(y, want)
    dy = torch.randn(y.shape, device=DEV, generator=g).bfloat16()
    y.backward(dy)
    want.backward(dy)
    assert torch.equal(table.grad[-500:], small.grad)
    assert not table.grad[:100_000].any() and not table.grad[-1000:-500].any()


@pytest.mark.gpu
def test_logits_past_4_gib(room):
    from mamba_cpu import sample_fn

    rows, vocab = 17_000, 131_072
    g = torch.Generator(device=DEV).manual_seed(0)
    logits = torch.zeros(rows, vocab, device=DEV, dtype=torch.bfloat16)
    noise = torch.ones(rows, vocab, device=DEV)
    logits[-20:] = torch.randn(20, vocab, device=DEV, generator=g).bfloat16()
    noise[-20:].exponential_(generator=g)
    cut, logprob = sample_fn(logits, noise, top_k=50, top_p=0.9, return_logprobs=True)
    want, want_logprob = sample_fn(logits[-20:].clone(), noise[-20:].clone(), top_k=50, top_p=0.9,
                                   return_logprobs=True)
    assert torch.equal(cut[-20:], want) and torch.equal(logprob[-20:], want_logprob)
    assert not cut[:100].any()  # equal logits and noise: the first
    free = sample_fn(logits, noise)
    assert torch.equal(free[-20:], sample_fn(logits[-20:].clone(), noise[-20:].clone()))


@pytest.mark.gpu
def test_recurrence_past_4_gib(room):
    from mamba_cpu import gated_linear_scan_fn

    l, d, tail, skip = 1_100_000, 2048, 1500, 800
    g = torch.Generator(device=DEV).manual_seed(0)
    x, a, i, dy = (torch.empty(1, l, d, device=DEV, dtype=torch.bfloat16) for _ in range(4))
    for t in (x, a, i, dy):
        t.fill_(0.5)
        t[:, -tail:] = torch.randn(1, tail, d, device=DEV, generator=g).bfloat16()
    decay = torch.full((d,), 0.0, device=DEV)  # forgets within 100 steps
    small = [t[:, -tail:].clone().requires_grad_() for t in (x, a, i)]
    big = [t.requires_grad_() for t in (x, a, i)]
    y = gated_linear_scan_fn(*big, decay)
    want = gated_linear_scan_fn(*small, decay)
    y.backward(dy)
    want.backward(dy[:, -tail:].clone())
    for name, got, ref in [("y", y, want)] + [(n, p.grad, q.grad) for n, p, q in zip("xai", big, small)]:
        got, ref = got[:, -tail + skip:].detach().float(), ref[:, skip:].detach().float()
        assert ((got - ref).abs() <= 2e-5 * ref.abs().max() + 2.0 ** -7 * ref.abs()).all(), name
    assert torch.equal(y[:, 5000], y[:, 500_000]) and y[0, 5000, 0] > 0  # settled


@pytest.mark.gpu
@pytest.mark.parametrize("step", [130_000_000, 140_000_000, 270_000_000])
def test_recurrence_steps_far_apart(room, step):
    """16 steps of 2-byte elements on both sides of 4 GiB, and 8 steps beyond it."""
    from mamba_cpu import gated_linear_scan_fn

    l, d = 20, 70
    g = torch.Generator(device=DEV).manual_seed(0)
    x, a, i, dy = (torch.randn(1, l, d, device=DEV, generator=g).bfloat16() for _ in range(4))
    decay = torch.randn(d, device=DEV, generator=g)
    store = torch.empty((l - 1) * step + d, device=DEV, dtype=torch.bfloat16)

    def run(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, a, i)]
        y = gated_linear_scan_fn(*leaves, decay)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = run(x, dy)
    far = store.as_strided((1, l, d), (0, step, 1))
    far.copy_(x)
    got = run(far, dy)
    far.copy_(dy)
    got += run(x, far)
    for have, ref in zip(got, want + want):
        assert torch.equal(have, ref)


def test_abi_refuses_steps_too_far_apart():
    from mamba_cpu import _C

    a = _C.GatedScanArgs()
    a.x = a.a_gate = a.x_gate = a.decay = a.y = 16  # placeholders: never dereferenced
    a.batch, a.seqlen, a.dim, a.c, a.dtype = 1, 20, 70, 8.0, _C.MCPU_BF16
    for s in (a.x_stride, a.a_stride, a.i_stride, a.y_stride):
        s[:] = (1400, 70, 1)
    assert _C.lib.mcpu_gated_scan_ckpt_size(ctypes.byref(a)) == 4 * 2 * 70
    for far in ((0, 2 ** 27, 1), (0, 1, 2 ** 31 // 70 + 1), (0, 2 ** 26, 2 ** 30 // 70 + 1), (0, 2 ** 62, 2 ** 62)):
        a.x_stride[:] = far
        rc = _C.lib.mcpu_gated_scan_fwd(ctypes.byref(a), None, 0, None)
        assert rc == _C.MCPU_ERR_UNSUPPORTED and "far apart" in _C.lib.mcpu_last_error().decode(), far
