"""Attention under a key mask and its gradients in float64, from their formulas."""

from __future__ import annotations

import numpy as np


def probabilities(q, k, keep=None):
    """(S, P, lse) of one head, q (Lq, D), k (Lk, D), ``keep`` (Lk,) bool; masked S are -inf, and a row that keeps
    nothing has P = 0 and lse = -inf."""
    s = np.where(True if keep is None else keep, q @ np.where(True if keep is None else keep[:, None], k, 0.0).T, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    base = np.where(np.isfinite(top), top, 0.0)
    e = np.exp(s - base)
    total = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, base + np.log(total), -np.inf)
    return s, e / np.where(total > 0, total, 1.0), lse[:, 0]


def attention(q, k, v, keep=None):
    """o of one head."""
    if keep is not None:
        v = np.where(keep[:, None], v, 0.0)
    return probabilities(q, k, keep)[1] @ v


def attention_grads(do, q, k, v, keep=None):
    """(dq, dk, dv) of one head."""
    if keep is not None:
        k, v = (np.where(keep[:, None], t, 0.0) for t in (k, v))
    p = probabilities(q, k, keep)[1]
    dp = do @ v.T
    ds = p * (dp - (do * (p @ v)).sum(-1, keepdims=True))
    return ds @ k, ds.T @ q, p.T @ do
