"""Attention of any lengths under a mask over the keys, forward and backward.

  attention   softmax(q k^T) v, merged heads: merge_heads(attend(q, k, v)) (src/flicker/kernels.py:105-145,
              modules.py:63-65) without its conditions

Next to ``kernels.attend``, which takes bf16 operands of one length and leaves out the running maximum because
QK-norm bounds its logits, these take logits of any size, bfloat16 or float16, queries and keys of different
lengths, several query heads to a key head, and a mask over each batch entry's keys (a prompt's padding).
``attention_backward`` returns the gradients of q, k and v; it takes what the forward call keeps with
``keep=True``.  As for ``attend``, q comes scaled by 1 / sqrt(D) (``Freqs.q_gain``).

Logits may have any size that float32 holds; backwards P = exp(S - lse) is off by lse's rounding, up to 2^-24 |lse| of
itself.  Statistics and sums are float32; P, and backwards dS, are rounded to the operands' type, which the matrix cores take,
and every output is rounded once.  In float16 the gradients' P and dS are held times powers of two, by do's and v's norms, so
that they neither overflow nor lose what small gradients leave of them; forwards P has all its bits down to 2^-22 of its row's
largest, and below 2^-33 is zero.
In bfloat16 a term P v below 2^-106 is.
For gradients through torch's autograd see ``flicker_amd.autograd``.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from .kernels import HEAD_DIM, _native, _on_gpu
from .norm import _CODES, _refuse_overlap, _rows_apart

_MAX_ROW = 1 << 25   # elements between two rows


class Kept(NamedTuple):
    """What attention keeps for its backward pass: the o that it returned, ``low``, what o's rounding left of it, in o's
    type and shape, and ``lse``, (B, H, Lq) float32, each row's log sum exp (-inf where the mask keeps nothing)."""

    o: torch.Tensor
    low: torch.Tensor
    lse: torch.Tensor


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` (B, H, L, D), or a copy where its last axis is not dense or its rows are not 16-byte aligned or too far apart."""
    if t.numel() and (t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride(), t.shape[:3]) if n > 1)
                      or (t.shape[2] > 1 and t.stride(2) > _MAX_ROW)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t: torch.Tensor):
    """Batch, head and row strides (0 along an axis of one)."""
    return (ctypes.c_int64 * 3)(*(s if n > 1 else 0 for s, n in zip(t.stride(), t.shape[:3])))


def _operands(q, k, v, key_mask):
    """Checked (q, k, v, mask bytes or None, sizes)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _on_gpu(name, t)
        if t.dim() != 4:
            raise ValueError(f"{name} must be (B, H, L, D), got {tuple(t.shape)}")
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if t.dtype != q.dtype:
            raise TypeError(f"{name} must be {q.dtype} like q, got {t.dtype}")
    batch, heads, queries, dim = q.shape
    if k.shape != v.shape or k.shape[0] != batch or k.shape[3] != dim:
        raise ValueError(f"k and v must be ({batch}, kv heads, keys, {dim}) of one shape, got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    kv_heads, keys = k.shape[1:3]
    if dim != HEAD_DIM:
        raise ValueError(f"attention: head_dim {dim} unsupported (kernels are built for {HEAD_DIM})")
    if not heads or not kv_heads or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key heads evenly")
    if key_mask is not None:
        _on_gpu("key_mask", key_mask)
        if key_mask.dtype != torch.bool:
            raise TypeError(f"key_mask must be bool, True where a key is kept, got {key_mask.dtype}")
        if key_mask.shape != (batch, keys):
            raise ValueError(f"key_mask must be ({batch}, {keys}), got {tuple(key_mask.shape)}")
        if keys > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    return _aligned(q), _aligned(k), _aligned(v), key_mask, (batch, heads, kv_heads, queries, keys)


@functools.lru_cache(maxsize=1024)
def _plan(sizes, masked: bool, backward: bool) -> int:
    """Workspace bytes of a call (a pure function of the sizes)."""
    size = ctypes.c_int64(0)
    _lib.check(_lib.lib().flk_attention_plan(*sizes, int(masked), int(backward), ctypes.byref(size)), "flk_attention_plan")
    return size.value


def _workspace(sizes, masked: bool, backward: bool, device):
    nbytes = _plan(sizes, masked, backward)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


def _mask_args(key_mask):
    return (None, 0) if key_mask is None else (key_mask.data_ptr(), key_mask.stride(0))


def _split(o: torch.Tensor, heads: int) -> torch.Tensor:
    """(B, L, H * D) as (B, H, L, D) over the same memory."""
    batch, length, width = o.shape
    return o.view(batch, length, heads, width // heads).transpose(1, 2)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, key_mask: torch.Tensor | None = None,
              keep: bool = False, out: torch.Tensor | None = None):
    """softmax(q k^T) v of q (B, H, Lq, D) and k, v (B, Hkv, Lk, D), bfloat16 or float16, Hkv dividing H, views of any
    strides -> (B, Lq, H * D).  ``key_mask`` (B, Lk) bool is True where a key is kept; a query that keeps none (or
    only such as its logits are -inf for) gets zeros, and what masked keys and values hold is never read into a result.  With ``keep`` also returns the ``Kept`` that
    attention_backward takes.  ``out`` may be a (B, Lq, H * D) view with strided rows that overlaps no operand."""
    if out is None:
        done = _native.attention(q, k, v, key_mask, keep)
        if done is not None:
            return (done[0], Kept(*done)) if keep else done[0]
    q, k, v, key_mask, sizes = _operands(q, k, v, key_mask)
    batch, heads, _, queries, keys = sizes
    dim = q.shape[3]
    if out is None:
        out = torch.empty((batch, queries, heads * dim), dtype=q.dtype, device=q.device)
    else:
        _on_gpu("out", out)
        if (out.shape != (batch, queries, heads * dim) or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(0) % 8
                or out.stride(1) % 8 or out.data_ptr() % 16):
            raise ValueError(f"out must be a {q.dtype} ({batch}, {queries}, {heads * dim}) view with contiguous, "
                             "16-byte aligned rows")
        if out.numel():
            if not _rows_apart(out):
                raise ValueError(f"out needs rows that do not overlap, got strides {out.stride()}")
            for name, t in (("q", q), ("k", k), ("v", v), ("key_mask", key_mask)):
                if t is not None and t.numel():
                    _refuse_overlap(name, out, t)
    low = torch.empty((batch, queries, heads * dim), dtype=q.dtype, device=q.device) if keep else None
    lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=q.device) if keep else None
    if out.numel():
        ws, nbytes = _workspace(sizes, key_mask is not None, False, q.device)
        _lib.run("flk_attention", (q, k, v, key_mask, out, low, lse, ws), q.data_ptr(), _strides(q), k.data_ptr(),
                 _strides(k), v.data_ptr(), _strides(v), _CODES[q.dtype], *_mask_args(key_mask), *sizes, dim, out.data_ptr(),
                 _strides(_split(out, heads)), _lib.ptr(low), _lib.ptr(lse), _lib.ptr(ws), nbytes, _lib.stream_of(q))
    return (out, Kept(out, low, lse)) if keep else out


def attention_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kept: Kept, *,
                       key_mask: torch.Tensor | None = None):
    """(dq, dk, dv) of ``attention(q, k, v, key_mask=key_mask, keep=True)`` for the incoming gradient do (B, Lq, H * D) and
    the ``kept`` that call returned; masked keys get zeros."""
    done = _native.attention_backward(do, q, k, v, *kept, key_mask)
    if done is not None:
        return done
    grads = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    q, k, v, key_mask, sizes = _operands(q, k, v, key_mask)
    batch, heads, _, queries, keys = sizes
    dim = q.shape[3]
    shape = (batch, queries, heads * dim)
    _on_gpu("do", do)
    if do.shape != shape or do.dtype != q.dtype:
        raise ValueError(f"do must be {q.dtype} {shape}, got {do.dtype} {tuple(do.shape)}")
    o, low, lse = kept
    for name, t, want, dtype in (("o", o, shape, q.dtype), ("low", low, shape, q.dtype),
                                 ("lse", lse, (batch, heads, queries), torch.float32)):
        _on_gpu(f"kept.{name}", t)
        if t.shape != want or t.dtype != dtype or (name != "o" and not t.is_contiguous()):
            raise ValueError(f"kept.{name} must be contiguous {dtype} {want}, got {t.dtype} {tuple(t.shape)}")
    if not q.numel() or not k.numel():
        return tuple(t.zero_() for t in grads)
    # splitting the merged axis needs a dense one
    do, o = (_aligned(_split(t if t.stride(2) == 1 else t.contiguous(), heads)) for t in (do, o))
    ws, nbytes = _workspace(sizes, key_mask is not None, True, q.device)
    _lib.run("flk_attention_backward", (do, q, k, v, o, low, lse, key_mask, *grads, ws),
             *(x for t in (do, q, k, v, o) for x in (t.data_ptr(), _strides(t))), low.data_ptr(), lse.data_ptr(),
             _CODES[q.dtype], *_mask_args(key_mask), *sizes, dim,
             *(x for t in grads for x in (t.data_ptr(), _strides(t))), ws.data_ptr(), nbytes, _lib.stream_of(q))
    return grads
