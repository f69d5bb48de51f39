"""Layer norm of the DiT blocks, forward and backward.

  layer_norm   (x - mean) / sqrt(var + eps) * weight + bias        (src/flicker/nn.py:17-21 is weight = bias = None)
  modulate     (1 + scale) * layer_norm(x) + shift, a row of each per image   (src/flicker/modules.py:38-40)
  residual_modulate   r = x + gate * branch and modulate of that sum: what ends one part of a block and begins
               the next                                              (src/flicker/modules.py:157-167, 185-200)

``*_backward`` take the incoming gradient and the forward call's arguments and return the gradients
in the order of those arguments; nothing is kept from the forward call.  All arithmetic is
float32 and every output is rounded once, where the reference rounds each step of ``modulate`` to
bf16 (``w8a8.quantize_act_modulated`` reproduces those roundings); the two differ by bf16 ulps.

x is bfloat16, float16 or float32, (..., width) with rows of any stride (a (B, L, width) view, such
as one stream of a joint sequence, is read in place) and any width up to 16384; parameters are
of x's type or float32.  Parameter gradients are sums over tokens in a fixed order.  For gradients through
torch's autograd see ``flicker_amd.autograd``.
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from .kernels import EPS, _native, _on_gpu, _vector

_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # FLK_BF16, FLK_F16, FLK_F32


def _dtype(name: str, t: torch.Tensor) -> int:
    _on_gpu(name, t)
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    return code


def _blocks(t: torch.Tensor) -> torch.Tensor:
    """``t`` (..., N) as (B, L, N) with a contiguous last axis, in place where its strides allow it."""
    if t.dim() != 3:
        t = t.reshape(1, -1, t.shape[-1]) if t.dim() else t
    return t if t.shape[-1] <= 1 or t.stride(2) == 1 else t.contiguous()


def _output(out: torch.Tensor | None, shape, like: torch.Tensor) -> torch.Tensor:
    """``out`` checked, or a new tensor of ``shape``: (..., N), rows contiguous and apart."""
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _on_gpu("out", out)
    if out.shape != shape or out.dtype != like.dtype:
        raise ValueError(f"out must be {like.dtype} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
    return out


def _out_blocks(out: torch.Tensor) -> torch.Tensor:
    """An output as (B, L, N) over the same memory; refused where that is not possible, or where rows
    overlap."""
    if out.numel() == 0:
        return out
    if out.dim() != 3:
        try:
            out = out.view(1, -1, out.shape[-1])
        except RuntimeError:
            raise ValueError(f"out {tuple(out.shape)} with strides {out.stride()} has no common row stride") from None
    if not _rows_apart(out):
        raise ValueError(f"out needs contiguous rows that do not overlap, got strides {out.stride()}")
    return out


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether (B, L, N) has contiguous rows that do not overlap."""
    batch, length, width = t.shape
    row = t.stride(1) if length > 1 else width
    entry = t.stride(0) if batch > 1 else width
    apart = entry >= (length - 1) * row + width or row >= (batch - 1) * entry + width
    return (width <= 1 or t.stride(2) == 1) and min(row, entry) >= width and (apart or min(batch, length) == 1)


def _elements(t: torch.Tensor) -> np.ndarray:
    """``t``'s addresses as an array that is never read."""
    class Memory:
        __array_interface__ = {"version": 3, "typestr": f"|V{t.element_size()}", "data": (t.data_ptr(), True),
                               "shape": tuple(t.shape), "strides": tuple(s * t.element_size() for s in t.stride())}
    return np.asarray(Memory())


def _end(t: torch.Tensor) -> int:
    return t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _refuse_overlap(name: str, out: torch.Tensor, t: torch.Tensor, columns=()) -> None:
    """Refuses an output over an input ``t`` that is still being read.  In place, row by row, is not refused: both are
    (B, L, N) blocks of the same strides, and out's rows begin one of ``columns`` after t's."""
    if out.data_ptr() >= _end(t) or t.data_ptr() >= _end(out):
        return
    if (out.data_ptr() - t.data_ptr()) in [c * t.element_size() for c in columns] and _rows_apart(t) and all(
            a == b or n == 1 for n, a, b in zip(t.shape[:2], out.stride(), t.stride())):
        return
    if np.shares_memory(_elements(out), _elements(t)):
        raise ValueError(f"out shares memory with {name}, and not in place")


def _param(name: str, t: torch.Tensor | None, shape, x: torch.Tensor) -> torch.Tensor | None:
    if t is None:
        return None
    _dtype(name, t)
    if t.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name} must be {x.dtype} like x, or float32, got {t.dtype}")
    if t.shape not in shape:
        raise ValueError(f"{name} must be one of {[tuple(s) for s in shape]}, got {tuple(t.shape)}")
    return t


def _params(named, x, shapes):
    """Two checked parameters of one dtype (or None) as dense tensors."""
    (n0, p0), (n1, p1) = named
    p0, p1 = _param(n0, p0, shapes, x), _param(n1, p1, shapes, x)
    if p0 is not None and p1 is not None and p0.dtype != p1.dtype:
        raise TypeError(f"{n0} and {n1} must share one dtype, got {p0.dtype} and {p1.dtype}")
    return tuple(None if p is None else _vector(p) for p in (p0, p1))


def _forward(x, factor, offset, per_entry: bool, add_one: bool, eps: float, out):
    code = _dtype("x", x)
    given, out = out is not None, _output(out, x.shape, x)
    yb = _out_blocks(out)
    if x.numel() == 0:
        return out
    xb = _blocks(x)
    batch, length, width = xb.shape
    if given:
        _refuse_overlap("x", yb, xb, (0,))
        for p in (factor, offset):
            if p is not None:
                _refuse_overlap("a parameter", yb, p)
    param = factor if factor is not None else offset
    _lib.run("flk_layer_norm", (x, factor, offset, out), xb.data_ptr(), *_strides(xb), code, _lib.ptr(factor),
             _lib.ptr(offset), code if param is None else _CODES[param.dtype], width if per_entry else 0,
             int(add_one), float(eps), batch, length, width, yb.data_ptr(), *_strides(yb), _lib.stream_of(x))
    return out


def _strides(t: torch.Tensor) -> tuple[int, int]:
    return t.stride(0), t.stride(1)


def _backward(dy, x, factor, wanted, param_dtype, per_entry: bool, add_one: bool, eps: float):
    """(dx, dfactor, doffset), the last two None where not ``wanted``."""
    code = _dtype("x", x)
    _on_gpu("dy", dy)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {x.dtype} {tuple(x.shape)} like x, got {dy.dtype} {tuple(dy.shape)}")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    width = x.shape[-1]
    shape = (x.shape[0], width) if per_entry else (width,)
    if x.numel() == 0:   # sums over no rows
        return dx, *(torch.zeros(shape, dtype=param_dtype, device=x.device) if w else None for w in wanted)
    dparams = tuple(torch.empty(shape, dtype=param_dtype, device=x.device) if w else None for w in wanted)
    xb, gb, ob = _blocks(x), _blocks(dy), _out_blocks(dx)
    batch, length, _ = xb.shape
    workspace, nbytes = None, 0
    if any(wanted):
        size = ctypes.c_int64(0)
        _lib.check(_lib.lib().flk_layer_norm_backward_plan(batch, length, width, int(not per_entry), ctypes.byref(size)),
                   "flk_layer_norm_backward_plan")
        nbytes = size.value
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.run("flk_layer_norm_backward", (dy, x, factor, dx, *dparams, workspace), gb.data_ptr(), *_strides(gb),
             xb.data_ptr(), *_strides(xb), code, _lib.ptr(factor), _CODES[param_dtype], width if per_entry else 0,
             int(add_one), float(eps), batch, length, width, ob.data_ptr(), *_strides(ob), *map(_lib.ptr, dparams),
             _lib.ptr(workspace), nbytes, _lib.stream_of(x))
    return dx, *dparams


def _check_x(x: torch.Tensor) -> None:
    _dtype("x", x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must be (..., width), got {tuple(x.shape)}")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = EPS, out: torch.Tensor | None = None) -> torch.Tensor:
    """Layer norm over the last axis of x (..., width); ``weight`` and ``bias`` (width,) or None.  ``out`` may be
    a view with strided rows, or x itself; any other overlap with an operand is refused."""
    if out is None:
        done = _native.layer_norm(x, weight, bias, eps)
        if done is not None:
            return done
    _check_x(x)
    weight, bias = _params((("weight", weight), ("bias", bias)), x, ((x.shape[-1],),))
    return _forward(x, weight, bias, False, False, eps, out)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, *, eps: float = EPS):
    """(dx, dweight, dbias) of ``layer_norm(x, weight, bias)`` for the incoming gradient dy; None for a
    parameter that is None."""
    done = _native.layer_norm_backward(dy, x, weight, bias, eps)
    if done is not None:
        return done
    _check_x(x)
    w, b = _params((("weight", weight), ("bias", bias)), x, ((x.shape[-1],),))
    dtype = next((p.dtype for p in (w, b) if p is not None), x.dtype)
    return _backward(dy, x, w, (w is not None, b is not None), dtype, False, False, eps)


def _modulation(x, shift, scale):
    _check_x(x)
    if x.dim() != 3:
        raise ValueError(f"x must be (B, L, width), got {tuple(x.shape)}")
    batch, _, width = x.shape
    if shift is None or scale is None:
        raise TypeError("modulate needs both shift and scale")
    return _params((("shift", shift), ("scale", scale)), x, ((batch, width), (batch, 1, width)))


def modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, eps: float = EPS,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """modules.py:38-40 -- (1 + scale) * layer_norm(x) + shift of x (B, L, width) with one row of shift and
    scale per batch entry, (B, width) or (B, 1, width).  ``out`` as for layer_norm."""
    if out is None:
        done = _native.modulate(x, shift, scale, eps)
        if done is not None:
            return done
    shift, scale = _modulation(x, shift, scale)
    return _forward(x, scale, shift, True, True, eps, out)


def modulate_backward(dy: torch.Tensor, x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *,
                      eps: float = EPS):
    """(dx, dshift, dscale) of ``modulate(x, shift, scale)`` for the incoming gradient dy, the last two shaped as
    shift and scale."""
    done = _native.modulate_backward(dy, x, shift, scale, eps)
    if done is not None:
        return done
    shift_row, scale_row = _modulation(x, shift, scale)
    dx, dscale, dshift = _backward(dy, x, scale_row, (True, True), scale_row.dtype, True, True, eps)
    return dx, dshift.view(shift.shape), dscale.view(scale.shape)


def _residual(x, branch, gate, shift, scale):
    """Checked (gate, shift, scale) rows."""
    if gate is None:
        raise TypeError("residual_modulate needs a gate")
    shift_row, scale_row = _modulation(x, shift, scale)
    _same("branch", branch, x)
    batch, _, width = x.shape
    gate = _param("gate", gate, ((batch, width), (batch, 1, width)), x)
    if gate.dtype != scale_row.dtype:
        raise TypeError(f"gate, shift and scale must share one dtype, got {gate.dtype} and {scale_row.dtype}")
    return _vector(gate), shift_row, scale_row


def _same(name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    _on_gpu(name, t)
    if t.shape != x.shape or t.dtype != x.dtype:
        raise ValueError(f"{name} must be {x.dtype} {tuple(x.shape)} like x, got {t.dtype} {tuple(t.shape)}")


def _rows(t: torch.Tensor) -> tuple[int, int, int]:
    return t.data_ptr(), t.stride(0), t.stride(1)


def residual_modulate(x: torch.Tensor, branch: torch.Tensor, gate: torch.Tensor, shift: torch.Tensor,
                      scale: torch.Tensor, *, eps: float = EPS) -> tuple[torch.Tensor, torch.Tensor]:
    """(r, y) with r = x + gate * branch and y = (1 + scale) * layer_norm(r) + shift: x and branch (B, L, width), one row
    of gate, shift and scale per batch entry, (B, width) or (B, 1, width).  y is of the unrounded sum."""
    done = _native.residual_modulate(x, branch, gate, shift, scale, eps)
    if done is not None:
        return done
    gate, shift, scale = _residual(x, branch, gate, shift, scale)
    r, y = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
    if x.numel() == 0:
        return r, y
    xb, bb = _blocks(x), _blocks(branch)
    batch, length, width = x.shape
    _lib.run("flk_residual_norm", (x, branch, gate, scale, shift, r, y), *_rows(xb), *_rows(bb), _CODES[x.dtype],
             gate.data_ptr(), scale.data_ptr(), shift.data_ptr(), _CODES[scale.dtype], width, 1, float(eps), batch, length,
             width, *_rows(r), *_rows(y), _lib.stream_of(x))
    return r, y


def residual_modulate_backward(dr: torch.Tensor, dy: torch.Tensor, x: torch.Tensor, branch: torch.Tensor,
                               gate: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, eps: float = EPS,
                               wanted: tuple[bool, bool, bool] = (True, True, True)):
    """(dx, dbranch, dgate, dshift, dscale) of ``residual_modulate`` for the incoming gradients dr of r and dy of y, the
    last three shaped as gate, shift and scale.  Where ``wanted`` is false (a frozen modulation) one of those is None; its
    sum is not stored, and without any of them none is formed."""
    if all(wanted):
        done = _native.residual_modulate_backward(dr, dy, x, branch, gate, shift, scale, eps)
        if done is not None:
            return done
    shapes = gate, shift, scale
    gate, shift, scale = _residual(x, branch, gate, shift, scale)
    _same("dr", dr, x)
    _same("dy", dy, x)
    batch, length, width = x.shape
    dx, dbranch = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
    make = torch.empty if x.numel() else torch.zeros   # sums over no rows
    dgate, dshift, dscale = (make(t.shape, dtype=t.dtype, device=x.device) if want else None
                             for t, want in zip(shapes, wanted, strict=True))
    if x.numel() == 0:
        return dx, dbranch, dgate, dshift, dscale
    size, ws = ctypes.c_int64(0), None
    if any(wanted):
        _lib.check(_lib.lib().flk_residual_norm_backward_plan(batch, length, width, 0, ctypes.byref(size)),
                   "flk_residual_norm_backward_plan")
        ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
    rb, yb, xb, bb = (_blocks(t) for t in (dr, dy, x, branch))
    _lib.run("flk_residual_norm_backward", (dr, dy, x, branch, gate, scale, dx, dbranch, dgate, dscale, dshift, ws),
             *_rows(rb), *_rows(yb), *_rows(xb), *_rows(bb), _CODES[x.dtype], gate.data_ptr(), scale.data_ptr(),
             _CODES[scale.dtype], width, 1, float(eps), batch, length, width, *_rows(dx), *_rows(dbranch),
             *(_lib.ptr(t) for t in (dgate, dscale, dshift, ws)), size.value, _lib.stream_of(x))
    return dx, dbranch, dgate, dshift, dscale
