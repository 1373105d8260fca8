"""Float64 numpy restatements of the operators beside the scans, as their
definitions read: the gated linear recurrence step by step, the residual norm,
the embedding's gradient, token sampling. Test infrastructure only.
"""

import numpy as np


def _f64(t):
    return np.asarray(t.detach().double().cpu().numpy() if hasattr(t, "detach") else t, dtype=np.float64)


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def _gates(x, a_gate, x_gate, decay, c):
    rho, iota = sigmoid(a_gate), sigmoid(x_gate)
    s = c * softplus(decay) * rho
    return rho, iota, s, np.exp(-s), np.sqrt(-np.expm1(-2 * s))


def _resets(seq_idx, b, l):
    k = np.ones((b, l, 1))
    if seq_idx is not None:
        ids = np.asarray(seq_idx.cpu() if hasattr(seq_idx, "cpu") else seq_idx)
        k[:, 1:, 0] = ids[:, 1:] == ids[:, :-1]
    return k


def gated_scan_fwd(x, a_gate, x_gate, decay, init=None, seq_idx=None, c=8.0):
    """y (batch, seqlen, dim) and the last state (batch, dim)."""
    x, a_gate, x_gate, decay = (_f64(t) for t in (x, a_gate, x_gate, decay))
    b, l, d = x.shape
    _, iota, _, a, m = _gates(x, a_gate, x_gate, decay, c)
    k = _resets(seq_idx, b, l)
    h = np.zeros((b, d)) if init is None else _f64(init).copy()
    y = np.empty_like(x)
    for t in range(l):
        h = k[:, t] * a[:, t] * h + m[:, t] * iota[:, t] * x[:, t]
        y[:, t] = h
    return y, h


def gated_scan_bwd(x, a_gate, x_gate, decay, dy, init=None, seq_idx=None, c=8.0, dlast=None):
    """Gradients of x, a_gate, x_gate, decay and the initial state."""
    y, _ = gated_scan_fwd(x, a_gate, x_gate, decay, init, seq_idx, c)
    x, a_gate, x_gate, decay, dy = (_f64(t) for t in (x, a_gate, x_gate, decay, dy))
    b, l, d = x.shape
    rho, iota, s, a, m = _gates(x, a_gate, x_gate, decay, c)
    k = _resets(seq_idx, b, l)
    h0 = np.zeros((b, d)) if init is None else _f64(init)
    carry = np.zeros((b, d)) if dlast is None else _f64(dlast).copy()
    dx, da, di, ddecay = np.empty_like(x), np.empty_like(x), np.empty_like(x), np.zeros(d)
    for t in range(l - 1, -1, -1):
        g = dy[:, t] + carry
        prev = k[:, t] * (h0 if t == 0 else y[:, t - 1])
        mt = m[:, t]
        with np.errstate(divide="ignore", invalid="ignore"):
            dm_ds = np.where(mt > 0, a[:, t] ** 2 / mt, 0.0)
        ds = g * (iota[:, t] * x[:, t] * dm_ds - a[:, t] * prev)
        dx[:, t] = g * mt * iota[:, t]
        di[:, t] = g * mt * x[:, t] * iota[:, t] * sigmoid(-x_gate[:, t])
        da[:, t] = ds * s[:, t] * sigmoid(-a_gate[:, t])
        ddecay += (ds * c * rho[:, t] * sigmoid(decay)).sum(0)
        carry = k[:, t] * a[:, t] * g
    return dx, da, di, ddecay, carry


def gated_step(state, x, a_gate, x_gate, decay, c=8.0):
    """The state after one token."""
    state, x, a_gate, x_gate, decay = (_f64(t) for t in (state, x, a_gate, x_gate, decay))
    _, iota, _, a, m = _gates(x, a_gate, x_gate, decay, c)
    return a * state + m * iota * x


def norm_fwd(x, weight, bias=None, residual=None, eps=1e-5, rms=False):
    """y and z = x + residual, rows along the last axis."""
    z = _f64(x) if residual is None else _f64(x) + _f64(residual)
    mean = 0.0 if rms else z.mean(-1, keepdims=True)
    var = ((z - mean) ** 2).mean(-1, keepdims=True)
    y = (z - mean) / np.sqrt(var + eps) * _f64(weight)
    return (y if bias is None else y + _f64(bias)), z


def norm_bwd(x, weight, dy, bias=None, residual=None, dz_out=None, eps=1e-5, rms=False):
    """Gradients of z (x's and the residual's), weight and bias. Through the
    row's Jacobian: d zhat_i / d z_j = (delta_ij - [layer] 1 / n - zhat_i zhat_j / n) / std."""
    z = _f64(x) if residual is None else _f64(x) + _f64(residual)
    n = z.shape[-1]
    centre = np.eye(n) if rms else np.eye(n) - 1.0 / n
    zc = z @ centre
    std = np.sqrt((zc ** 2).mean(-1, keepdims=True) + eps)
    zhat = zc / std
    t = _f64(dy) * _f64(weight)
    dz = (t / std - zhat * (t * zhat).sum(-1, keepdims=True) / (n * std)) @ centre
    if dz_out is not None:
        dz = dz + _f64(dz_out)
    flat = lambda v: v.reshape(-1, n)  # noqa: E731
    return dz, flat(_f64(dy) * zhat).sum(0), flat(_f64(dy)).sum(0)


def embedding_bwd(ids, dout, vocab, scale=1.0):
    """Gradient of the embedding's weight; ids outside [0, vocab) have none."""
    ids, dout = np.asarray(ids.cpu()).reshape(-1), _f64(dout)
    dw = np.zeros((vocab, dout.shape[-1]))
    for t, v in enumerate(ids):
        if 0 <= v < vocab:
            dw[v] += dout[t]
    return dw * scale


def sample(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: the token, its logprob, how many tokens were kept, and how near
    the choice was: the relative distance of the race's second and of a weight
    from min_p, 0 where the token changes if the top-p edge moves by 1e-5 of
    the mass."""
    l = _f64(logits).reshape(-1)
    l = np.where(np.isnan(l), -np.inf, l)
    m = l.max() if l.size else -np.inf
    if m == -np.inf:
        return -1, -np.inf, 0, np.inf
    with np.errstate(invalid="ignore"):
        flat = np.where(l == m, 0.0, l - m)
    logprob = lambda i: flat[i] - np.log(np.exp(flat).sum())  # noqa: E731
    order = np.lexsort((np.arange(l.size), -l))
    if not temperature > 0:
        return int(order[0]), logprob(order[0]), 1, np.inf
    w = np.exp(flat[order] / temperature)
    n = min(top_k, l.size) if top_k > 0 else l.size
    near, moved = np.inf, (n, n)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        mass = w[:n].sum()
        edge = float(np.float32(top_p)) * mass
        moved = [max(1, int((before < edge + by * mass).sum())) for by in (-1e-5, 1e-5)]
        n = max(1, int((before < edge).sum()))
    mp = min(float(np.float32(min_p)), 1.0)
    if mp > 0:
        near = min(near, np.abs(w[:n] / mp - 1)[w[:n] != 1].min(initial=np.inf))
    if moved[0] < moved[1]:
        race = (w / _f64(noise).reshape(-1)[order])[:moved[1]]
        race[1:][w[1:moved[1]] < mp] = -1
        if race[:moved[0]].max() <= race[moved[0]:].max():
            near = 0.0
    n = max(1, int((w[:n] >= mp).sum()))
    score = w[:n] / _f64(noise).reshape(-1)[order[:n]]
    best = score.max()
    ties = order[:n][score == best]
    rest = score[score < best]
    if rest.size and best > 0:
        near = min(near, 1 - rest.max() / best)
    return int(ties.min()), logprob(ties.min()), n, near
