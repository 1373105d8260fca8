"""Float64 numpy restatement of the head's losses, as their definitions read:
cross entropy and distillation of logits = hidden @ weight.T, with gradients.
Test infrastructure only.
"""

import numpy as np

from oracle.lm import _f64


def _ints(t):
    return np.asarray(t.cpu() if hasattr(t, "cpu") else t).astype(np.int64)


def shares(ids, vocab, teacher=None, temperature=1.0, ignore_index=-100):
    """Per row the target distribution over its entries, (rows, k), 0 for entries left out, and which rows count."""
    ids = _ints(ids)
    if teacher is None:
        q = ((ids >= 0) & (ids < vocab) & (ids != ignore_index)).astype(np.float64)[:, None]
        return q, q[:, 0] > 0
    t = _f64(teacher) / temperature
    t = np.where((ids >= 0) & (ids < vocab), t, -np.inf)
    q, keep = np.zeros(t.shape), np.zeros(len(t), bool)
    for i, row in enumerate(t):
        if (row != -np.inf).any():
            with np.errstate(invalid="ignore"):
                e = np.exp(row - np.nanmax(row))
            q[i], keep[i] = e / e.sum(), True
    return q, keep


def rows(hidden, weight, ids, teacher=None, temperature=1.0, ignore_index=-100):
    """(loss, lse, counts) per row; rows left out have 0."""
    vocab = weight.shape[0]
    q, keep = shares(ids, vocab, teacher, temperature, ignore_index)
    at = _ints(ids).reshape(len(q), -1)
    loss, lse = np.zeros(len(q)), np.zeros(len(q))
    h, w = _f64(hidden), _f64(weight)
    for i in np.flatnonzero(keep):
        s = w @ h[i] / temperature
        m = s.max()
        lse[i] = m + np.log(np.exp(s - m).sum())
        if teacher is None:  # log(1 + sum over the others of exp(s - s_target)), whose digits lse - s_target loses
            with np.errstate(over="ignore"):
                others = np.delete(np.exp(s - s[at[i, 0]]), at[i, 0]).sum()
            loss[i] = np.log1p(others) if others < 1e300 else lse[i] - s[at[i, 0]]
            continue
        for k, share in enumerate(q[i]):
            if share != 0:
                loss[i] += share * (np.log(share) + lse[i] - s[at[i, k]])
    return loss * temperature ** 2, lse, keep


def logits_grad(hidden, weight, ids, dloss, dlse=None, teacher=None, temperature=1.0, ignore_index=-100):
    """(rows, vocab): the gradient of the logits for dloss and dlse given per row."""
    vocab = weight.shape[0]
    q, keep = shares(ids, vocab, teacher, temperature, ignore_index)
    at = _ints(ids).reshape(len(q), -1)
    _, lse, _ = rows(hidden, weight, ids, teacher, temperature, ignore_index)
    h, w = _f64(hidden), _f64(weight)
    ds = np.zeros((len(q), vocab))
    for i in np.flatnonzero(keep):
        p = np.exp(w @ h[i] / temperature - lse[i])
        g = temperature * float(dloss[i])
        e = 0.0 if dlse is None else float(dlse[i])
        ds[i] = (g + e) * p
        if teacher is None:  # p - 1 is minus the others' sum
            y = at[i, 0]
            ds[i, y] = e * p[y] - g * np.delete(p, y).sum()
            continue
        for k, share in enumerate(q[i]):
            if share != 0:
                ds[i, at[i, k]] -= g * share
    return ds


def grads(hidden, weight, ds):
    """Gradients of hidden and weight; rows of hidden whose ds is 0 take no part."""
    live = (ds != 0).any(1)
    h = np.where(live[:, None], _f64(hidden), 0.0)
    return ds @ _f64(weight), ds.T @ h
