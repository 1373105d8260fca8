"""Float64 numpy restatements of the operators beside the scans: the gated
linear recurrence, step by step as its definition reads. Test infrastructure
only.
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
