"""norm.residual_modulate and its gradients on the GPU against the float64 oracle.

Tolerances are test_gpu_norm's for the norm of r = x + gate * branch, which one more rounding (u |r|, inside the
norm's 300 u) computes; the sum's gradient d = dr + dx adds 4 u (|dr| + |dx|), dbranch = gate d 4 u of itself, and dgate,
over R rows, (R + 64) u sum|d branch| and d's own error times |branch|.
"""

import numpy as np
import pytest
import torch

from flicker_amd import norm
from tests.test_gpu_norm import TYPES, U, WIDTHS, _close, _f64, _norm_case, _stream

pytestmark = pytest.mark.gpu


def _operands(seed, batch, length, width, dtype, params, device, row_shape=True):
    x, g = _stream(seed, batch, length, width, TYPES[dtype], device)
    branch, dr, dy = (torch.randn(batch, length, width, generator=g).to(TYPES[dtype]).to(device) for _ in range(3))
    shape = (batch, 1, width) if row_shape else (batch, width)
    rows = [torch.randn(shape, generator=g).to(TYPES[params]).to(device) for _ in range(3)]
    return x, branch, dr, dy, rows


def _check(x, branch, dr, dy, rows, eps=norm.EPS):
    gate, shift, scale = rows
    r, y = norm.residual_modulate(x, branch, gate, shift, scale, eps=eps)
    grads = norm.residual_modulate_backward(dr, dy, x, branch, gate, shift, scale, eps=eps)
    batch, length, width = x.shape
    b64, g64 = _f64(branch), _f64(gate).reshape(batch, 1, width)
    s64 = _f64(x) + g64 * b64
    (yw, yt), (dxw, dxt), (daw, dat), (dcw, dct) = _norm_case(
        s64, 1 + _f64(scale).reshape(batch, 1, width), _f64(shift).reshape(batch, 1, width), _f64(dy), (1,), eps)
    _close("r", r, s64, 2 * U * (np.abs(s64) + np.abs(g64 * b64)))
    _close("y", y, yw, yt)
    d = _f64(dr) + dxw
    dt = dxt + 4 * U * (np.abs(_f64(dr)) + np.abs(dxw))
    _close("dx", grads[0], d, dt)
    _close("dbranch", grads[1], g64 * d, np.abs(g64) * dt + 4 * U * np.abs(g64 * d))
    dg, dg_tol = (d * b64).sum(1), (dt * np.abs(b64)).sum(1) + (length + 64) * U * np.abs(d * b64).sum(1)
    for name, got, p, want, tol in zip(("dgate", "dshift", "dscale"), grads[2:], rows, (dg, dcw, daw), (dg_tol, dct, dat)):
        _close(name, got, want.reshape(p.shape), tol.reshape(p.shape))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,params", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_widths(device, width, dtype, params):
    print(f"residual width={width} {dtype}/{params}", flush=True)
    _check(*_operands(width, 2, 11, width, dtype, params, device))


@pytest.mark.parametrize("batch,length", [(1, 1), (3, 1), (1, 2), (5, 37), (2, 700)])
@pytest.mark.parametrize("width", [40, 1000, 24 * 128])
def test_lengths(device, batch, length, width):
    print(f"residual batch={batch} length={length} width={width}", flush=True)
    _check(*_operands(length, batch, length, width, "bf16", "bf16", device, row_shape=False))


def test_many_entries(device):
    """More batch entries than one entry's rows, each with its own rows of parameters."""
    _check(*_operands(4, 300, 2, 96, "bf16", "fp32", device))


def test_strided_views(device):
    """Rows of a joint sequence and columns of wider buffers are read in place."""
    x, branch, dr, dy, rows = _operands(1, 2, 40, 520, "bf16", "bf16", device)
    wide = torch.full((2, 50, 1100), float("nan"), dtype=x.dtype, device=device)
    views = []
    for i, t in enumerate((x, branch, dr, dy)):
        buffer = wide.clone()
        view = buffer[:, 3 + i:43 + i, 7 * i:7 * i + 520]
        view.copy_(t)
        views.append(view)
    _check(*views, rows)


def test_zero_gate_is_the_norm(device):
    """gate = 0: r is x, y modulate's result, bit for bit."""
    x, branch, _, _, (gate, shift, scale) = _operands(2, 2, 33, 1000, "bf16", "bf16", device)
    r, y = norm.residual_modulate(x, branch, gate * 0, shift, scale)
    assert torch.equal(r, x) and torch.equal(y, norm.modulate(x, shift, scale))


def test_against_differences(device):
    """The gradients against central differences of the float32 forward pass along random directions."""
    x, branch, dr, dy, rows = _operands(3, 1, 8, 64, "fp32", "fp32", device)
    args = [x, branch, *rows]
    grads = norm.residual_modulate_backward(dr, dy, *args)
    g = torch.Generator().manual_seed(9)
    step = 2.0 ** -6
    for i, (a, grad) in enumerate(zip(args, grads)):
        way = torch.randn(a.shape, generator=g).to(device)
        way = way / way.norm() * a.norm() / a.numel() ** 0.5

        def loss(t):
            r, y = norm.residual_modulate(*args[:i], a + t * way, *args[i + 1:])
            return float((r.double() * dr.double()).sum() + (y.double() * dy.double()).sum())
        slope = (loss(step) - loss(-step)) / (2 * step)
        # rounding: each of 2 * 512 terms of the loss, off by 400 u of itself at each end; and the third derivative's step^2
        scale = float((x.abs() * dr.abs()).sum() + dy.abs().sum() * 4)
        want = float((grad.double() * way.double()).sum())
        assert abs(slope - want) <= 400 * U * scale / step + 4 * step ** 2 * float(way.abs().max()) * scale ** 0.5 + 1e-3 * abs(want), i


def test_empty(device):
    x = torch.empty(2, 0, 64, dtype=torch.bfloat16, device=device)
    row = torch.ones(2, 64, dtype=torch.bfloat16, device=device)
    r, y = norm.residual_modulate(x, x, row, row, row)
    assert r.shape == y.shape == x.shape
    grads = norm.residual_modulate_backward(x, x, x, x, row, row, row)
    assert grads[0].shape == x.shape and not any(t.any() for t in grads[2:])


def test_captured_and_replayed(device):
    x, branch, dr, dy, rows = _operands(5, 2, 65, 768, "bf16", "bf16", device)

    def step():
        return (*norm.residual_modulate(x, branch, *rows), *norm.residual_modulate_backward(dr, dy, x, branch, *rows))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.add_(0.25)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals(device):
    x, branch, dr, dy, (gate, shift, scale) = _operands(6, 2, 5, 64, "bf16", "bf16", device)
    with pytest.raises(ValueError, match="branch must be"):
        norm.residual_modulate(x, branch[:, :4], gate, shift, scale)
    with pytest.raises(ValueError, match="branch must be"):
        norm.residual_modulate(x, branch.float(), gate, shift, scale)
    with pytest.raises(TypeError, match="share one dtype"):
        norm.residual_modulate(x, branch, gate.float(), shift, scale)
    with pytest.raises(TypeError, match="needs a gate"):
        norm.residual_modulate(x, branch, None, shift, scale)
    with pytest.raises(ValueError, match="gate must be"):
        norm.residual_modulate(x, branch, gate[:1], shift, scale)
    with pytest.raises(ValueError, match="dr must be"):
        norm.residual_modulate_backward(dr[:, 1:], dy, x, branch, gate, shift, scale)
    with pytest.raises(ValueError, match="dy must be"):
        norm.residual_modulate_backward(dr, dy.half(), x, branch, gate, shift, scale)
