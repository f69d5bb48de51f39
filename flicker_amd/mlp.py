"""The gated MLP of the DiT blocks, forward and backward.

  swiglu      silu(g) * u of gu = [g | u], silu(z) = z / (1 + exp(-z))
  gated_mlp   swiglu(x @ w_in) @ w_out, the projections, the gate and its gradient in one kernel each way

Double blocks run ``gated_mlp`` over each stream (src/flicker/modules.py:157-167).  Single blocks project QKV
and both MLP halves in one linear1, so there ``swiglu`` reads its halves in place from
``modules.single_attention``'s mlp columns and may write next to the attention's output in the
buffer that linear2 reads (modules.py:185-200).

``*_backward`` take the incoming gradient and the forward call's operands.  Sums are float32 and outputs are
rounded once; between the two projections h, and backwards [dg | du], are rounded to the operands' type,
which the matrix cores take, while g and u stay float32.  In float16 that rounding has the type's range: an h
past 65504 is infinite, and a dg or du below 2^-25 is zero (bfloat16 has float32's range).  For gradients
through torch's autograd see ``flicker_amd.autograd``.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from .kernels import _native, _on_gpu
from .norm import _blocks, _dtype, _out_blocks, _output, _refuse_overlap, _strides

_GATE, _GATE_BACKWARD, _MATMUL, _MATMUL_BT, _MATMUL_AT = range(5)   # FLK_MLP_*
_MAX_STRIDE = 1 << 22   # elements between two rows of an operand of the products


class Kept(NamedTuple):
    """What gated_mlp keeps for its backward pass: h (tokens, hidden) of x's type and gu = [g | u]
    (tokens, 2 * hidden) float32."""

    h: torch.Tensor
    gu: torch.Tensor


def swiglu(gu: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(g) * u of gu (..., 2 * hidden) = [g | u] -> (..., hidden); bfloat16, float16 or float32.  gu and
    ``out`` may be columns of wider buffers, and ``out`` one of gu's halves; any other overlap is refused."""
    if out is None:
        done = _native.swiglu(gu)
        if done is not None:
            return done
    code = _dtype("gu", gu)
    if gu.dim() == 0 or gu.shape[-1] == 0 or gu.shape[-1] % 2:
        raise ValueError(f"gu must be (..., 2 * hidden), got {tuple(gu.shape)}")
    hidden = gu.shape[-1] // 2
    given, out = out is not None, _output(out, (*gu.shape[:-1], hidden), gu)
    if gu.numel() == 0:
        return out
    gb, ob = _blocks(gu), _out_blocks(out)
    if given:
        _refuse_overlap("gu", ob, gb, (0, hidden))
    _lib.run("flk_swiglu", (gu, out), gb.data_ptr(), *_strides(gb), code, gb.shape[0], gb.shape[1], hidden,
             ob.data_ptr(), *_strides(ob), _lib.stream_of(gu))
    return out


def swiglu_backward(dh: torch.Tensor, gu: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """dgu = [dg | du] of ``swiglu(gu)`` for the incoming gradient dh; ``out`` may be gu itself, and dh one of its
    halves; any other overlap is refused."""
    if out is None:
        done = _native.swiglu_backward(dh, gu)
        if done is not None:
            return done
    code = _dtype("gu", gu)
    _on_gpu("dh", dh)
    if gu.dim() == 0 or gu.shape[-1] == 0 or gu.shape[-1] % 2:
        raise ValueError(f"gu must be (..., 2 * hidden), got {tuple(gu.shape)}")
    hidden = gu.shape[-1] // 2
    if dh.shape != (*gu.shape[:-1], hidden) or dh.dtype != gu.dtype:
        raise ValueError(f"dh must be {gu.dtype} {(*gu.shape[:-1], hidden)}, got {dh.dtype} {tuple(dh.shape)}")
    given, out = out is not None, _output(out, gu.shape, gu)
    if gu.numel() == 0:
        return out
    gb, db, ob = _blocks(gu), _blocks(dh), _out_blocks(out)
    if given:
        _refuse_overlap("gu", ob, gb, (0,))
        _refuse_overlap("dh", ob, db, (0, -hidden))
    _lib.run("flk_swiglu_backward", (dh, gu, out), db.data_ptr(), *_strides(db), gb.data_ptr(), *_strides(gb), code,
             gb.shape[0], gb.shape[1], hidden, ob.data_ptr(), *_strides(ob), _lib.stream_of(gu))
    return out


def _matrix(name: str, t: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """A 2-D view with a contiguous last axis and 16-byte aligned rows at most _MAX_STRIDE apart (a copy where t
    has none)."""
    _on_gpu(name, t)
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} like x, got {t.dtype}")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    row = t.stride(0)
    if t.stride(1) != 1 or row % 8 or not t.shape[1] <= row <= _MAX_STRIDE or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


@functools.lru_cache(maxsize=1024)
def _plan(product: int, rows: int, cols: int, inner: int) -> int:
    """Workspace bytes of one product (a pure function of the sizes)."""
    size = ctypes.c_int64(0)
    _lib.check(_lib.lib().flk_mlp_plan(product, rows, cols, inner, ctypes.byref(size)), "flk_mlp_plan")
    return size.value


def _workspace(product: int, rows: int, cols: int, inner: int, device):
    nbytes = _plan(product, rows, cols, inner)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


def _matmul(a, b, out, *, a_t: bool = False, b_t: bool = False) -> None:
    """out = a @ b, of a's transpose with ``a_t`` or b's with ``b_t``."""
    rows, cols = out.shape
    inner = a.shape[0] if a_t else a.shape[1]
    ws, nbytes = _workspace(_MATMUL_AT if a_t else _MATMUL_BT if b_t else _MATMUL, rows, cols, inner, a.device)
    _lib.run("flk_mlp_matmul", (a, b, out, ws), a.data_ptr(), a.stride(0), int(a_t), b.data_ptr(), b.stride(0),
             int(b_t), _dtype("a", a), rows, cols, inner, out.data_ptr(), out.stride(0), _lib.ptr(ws), nbytes,
             _lib.stream_of(a))


def _operands(x, w_in, w_out):
    """Checked (x rows, w_in, w_out, width, hidden)."""
    _on_gpu("x", x)
    if x.dim() == 0 or w_in.dim() != 2 or w_out.dim() != 2:
        raise ValueError(f"gated_mlp takes x (..., width), w_in (width, 2 * hidden), w_out (hidden, width), got "
                         f"{tuple(x.shape)}, {tuple(w_in.shape)}, {tuple(w_out.shape)}")
    width, hidden = x.shape[-1], w_out.shape[0]
    if w_in.shape != (width, 2 * hidden) or w_out.shape != (hidden, width):
        raise ValueError(f"w_in must be ({width}, 2 * hidden) and w_out (hidden, {width}) for x {tuple(x.shape)}, got "
                         f"{tuple(w_in.shape)} and {tuple(w_out.shape)}")
    if width % 8 or hidden % 8 or not width or not hidden:
        raise ValueError(f"gated_mlp needs a width and a hidden width that are multiples of 8, got {width} and {hidden}")
    xr = _matrix("x", x)
    return xr, _matrix("w_in", w_in, x.dtype), _matrix("w_out", w_out, x.dtype), width, hidden


def gated_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, *, keep: bool = False,
              out: torch.Tensor | None = None):
    """(silu(x @ w_g) * (x @ w_u)) @ w_out with w_in = [w_g | w_u]: x (..., width), w_in (width, 2 * hidden), w_out
    (hidden, width), all bfloat16 or all float16, widths multiples of 8 -> (..., width).  With ``keep`` also
    returns the ``Kept`` that gated_mlp_backward takes.  ``out`` must be contiguous; it may
    overlap x, but not w_out."""
    if out is None:
        done = _native.gated_mlp(x, w_in, w_out, keep)
        if done is not None:
            return (done[0], Kept(done[1], done[2])) if keep else done[0]
    xr, w_in, w_out, width, hidden = _operands(x, w_in, w_out)
    m = xr.shape[0]
    given, out = out is not None, _output(out, x.shape, x)
    if not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous and 16-byte aligned")
    if given and m:
        _refuse_overlap("w_out", out.view(m, width), w_out)
    h = torch.empty((m, hidden), dtype=x.dtype, device=x.device)
    gu = torch.empty((m, 2 * hidden), dtype=torch.float32, device=x.device) if keep else None
    if m:
        ws, nbytes = _workspace(_GATE, m, hidden, width, x.device)
        _lib.run("flk_mlp_gate", (xr, w_in, h, gu, ws), xr.data_ptr(), xr.stride(0), w_in.data_ptr(), w_in.stride(0),
                 _dtype("x", x), m, width, hidden, h.data_ptr(), hidden, _lib.ptr(gu), _lib.ptr(ws), nbytes,
                 _lib.stream_of(x))
        _matmul(h, w_out, out.view(m, width))
    return (out, Kept(h, gu)) if keep else out


def gated_mlp_backward(dy: torch.Tensor, x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, kept: Kept, *,
                       wanted: tuple[bool, bool, bool] = (True, True, True)):
    """(dx, dw_in, dw_out) of ``gated_mlp(x, w_in, w_out, keep=True)`` for the incoming gradient dy and the
    ``kept`` that call returned.  Where ``wanted`` is false (frozen weights) a gradient is None, and its product
    is not computed."""
    if all(wanted):
        done = _native.gated_mlp_backward(dy, x, w_in, w_out, *kept)
        if done is not None:
            return done
    xr, wi, wo, width, hidden = _operands(x, w_in, w_out)
    m = xr.shape[0]
    if dy.shape != x.shape:
        raise ValueError(f"dy must be {tuple(x.shape)} like x, got {tuple(dy.shape)}")
    gr = _matrix("dy", dy, x.dtype)
    h, gu = kept
    for name, t, shape, dtype in (("h", h, (m, hidden), x.dtype), ("gu", gu, (m, 2 * hidden), torch.float32)):
        _on_gpu(f"kept.{name}", t)
        if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"kept.{name} must be contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    dx, dw_in, dw_out = (torch.empty(t.shape, dtype=x.dtype, device=x.device) if want else None
                         for t, want in zip((x, w_in, w_out), wanted, strict=True))
    if m == 0:
        for dw in (dw_in, dw_out):
            if dw is not None:
                dw.zero_()
        return dx, dw_in, dw_out
    if dx is not None or dw_in is not None:
        dgu = torch.empty((m, 2 * hidden), dtype=x.dtype, device=x.device)
        ws, nbytes = _workspace(_GATE_BACKWARD, m, hidden, width, x.device)
        _lib.run("flk_mlp_gate_backward", (gr, wo, gu, dgu, ws), gr.data_ptr(), gr.stride(0), wo.data_ptr(),
                 wo.stride(0), gu.data_ptr(), _dtype("x", x), m, width, hidden, dgu.data_ptr(), 2 * hidden, _lib.ptr(ws),
                 nbytes, _lib.stream_of(x))
    if dw_out is not None:
        _matmul(h, gr, dw_out, a_t=True)
    if dw_in is not None:
        _matmul(xr, dgu, dw_in, a_t=True)
    if dx is not None:
        _matmul(dgu, wi, dx.view(m, width), b_t=True)
    return dx, dw_in, dw_out
