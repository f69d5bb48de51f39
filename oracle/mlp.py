"""Float64 restatement of the blocks' norm and gated MLP, and of their gradients (src/flicker/nn.py:17-21,
modules.py:38-40, 157-167), from the formulas; no rounding anywhere."""

from __future__ import annotations

import numpy as np


def _stats(x, eps):
    centred = x - x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt((centred * centred).mean(-1, keepdims=True) + eps)
    return centred * rstd, rstd


def layer_norm(x, factor=1.0, offset=0.0, eps=1e-6):
    """x (..., K); factor and offset broadcast against it (modulate: factor = 1 + scale)."""
    return _stats(np.asarray(x, np.float64), eps)[0] * factor + offset


def layer_norm_grads(dy, x, factor=1.0, eps=1e-6):
    """(dx, dy * n, dy): the last two summed over a parameter's rows are its gradient."""
    n, rstd = _stats(np.asarray(x, np.float64), eps)
    t = np.asarray(dy, np.float64) * factor
    dx = rstd * (t - t.mean(-1, keepdims=True) - n * (t * n).mean(-1, keepdims=True))
    return dx, dy * n, np.asarray(dy, np.float64) * np.ones_like(n)


def _sigmoid(g):
    e = np.exp(-np.abs(g))
    return np.where(g >= 0, 1.0, e) / (1.0 + e)


def swiglu(gu):
    g, u = np.split(np.asarray(gu, np.float64), 2, -1)
    return g * _sigmoid(g) * u


def swiglu_grads(dh, gu):
    g, u = np.split(np.asarray(gu, np.float64), 2, -1)
    s, rest = _sigmoid(g), _sigmoid(-g)
    return np.concatenate((dh * u * s * (1.0 + g * rest), dh * g * s), -1)


def gated_mlp(x, w_in, w_out):
    return swiglu(np.asarray(x, np.float64) @ w_in) @ w_out


def gated_mlp_grads(dy, x, w_in, w_out):
    """(dx, dw_in, dw_out) for 2-D x and dy."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    gu = x @ w_in
    dgu = swiglu_grads(dy @ np.asarray(w_out, np.float64).T, gu)
    return dgu @ np.asarray(w_in, np.float64).T, x.T @ dgu, swiglu(gu).T @ dy
