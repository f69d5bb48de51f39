"""``norm`` and ``mlp`` under torch's autograd: the same functions, differentiable.

Each call records the matching ``*_backward`` call; first derivatives only, and no forward mode (an operand
with a tangent raises NotImplementedError).  They are not captured into a HIP graph with gradients: autograd
accumulates into a leaf on the stream of whichever graph of that leaf is alive, which need not be the captured
one, so such a call is refused -- capture the explicit forward and backward calls of ``norm`` and ``mlp``
instead, which touch no leaves.
"""

from __future__ import annotations

import functools

import torch

from . import mlp as _mlp
from . import norm as _norm
from .kernels import EPS


def _not_captured() -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("flicker_amd.autograd is not captured into a graph with gradients: capture the explicit "
                           "forward and backward calls of flicker_amd.norm and flicker_amd.mlp")


def _recorded(*tensors) -> bool:
    """Whether autograd records a call on these operands."""
    recorded = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    if recorded:
        _not_captured()
    return recorded


def _first_only(backward):
    """A backward pass whose result is not differentiable again.  create_graph=True asks for that, and would get
    gradients that pass for constants."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("flicker_amd.autograd has first derivatives only: create_graph=True is not supported")
        _not_captured()
        return backward(ctx, *grads)
    return run


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return _norm.layer_norm(x, weight, bias, eps=eps)

    @staticmethod
    @_first_only
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        return *_norm.layer_norm_backward(dy, x, weight, bias, eps=ctx.eps), None


class _Modulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, shift, scale, eps):
        ctx.save_for_backward(x, shift, scale)
        ctx.eps = eps
        return _norm.modulate(x, shift, scale, eps=eps)

    @staticmethod
    @_first_only
    def backward(ctx, dy):
        return *_norm.modulate_backward(dy, *ctx.saved_tensors, eps=ctx.eps), None


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        ctx.save_for_backward(gu)
        return _mlp.swiglu(gu)

    @staticmethod
    @_first_only
    def backward(ctx, dh):
        return _mlp.swiglu_backward(dh, *ctx.saved_tensors)


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, keep):
        if not keep:
            return _mlp.gated_mlp(x, w_in, w_out)
        y, kept = _mlp.gated_mlp(x, w_in, w_out, keep=True)
        ctx.save_for_backward(x, w_in, w_out, *kept)
        return y

    @staticmethod
    @_first_only
    def backward(ctx, dy):
        x, w_in, w_out, h, gu = ctx.saved_tensors
        return *_mlp.gated_mlp_backward(dy, x, w_in, w_out, _mlp.Kept(h, gu), wanted=ctx.needs_input_grad[:3]), None


def layer_norm(x, weight=None, bias=None, *, eps: float = EPS) -> torch.Tensor:
    """norm.layer_norm, differentiable in x, weight and bias."""
    _recorded(x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, eps)


def modulate(x, shift, scale, *, eps: float = EPS) -> torch.Tensor:
    """norm.modulate, differentiable in x, shift and scale."""
    _recorded(x, shift, scale)
    return _Modulate.apply(x, shift, scale, eps)


def swiglu(gu) -> torch.Tensor:
    """mlp.swiglu, differentiable in gu."""
    _recorded(gu)
    return _Swiglu.apply(gu)


def gated_mlp(x, w_in, w_out) -> torch.Tensor:
    """mlp.gated_mlp, differentiable in x, w_in and w_out; keeps what the backward pass needs only where one
    of them requires a gradient."""
    return _GatedMLP.apply(x, w_in, w_out, _recorded(x, w_in, w_out))
