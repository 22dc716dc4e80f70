"""The training operators under torch's autograd.

`functional` holds each operator and its gradient as plain calls; here they are joined:

    layer_norm(x, weight, bias)            functional.layer_norm, layer_norm_backward
    gated_feed_forward(x, w_in, w_out)     functional.gated_feed_forward, gated_feed_forward_backward
    dropout(x, p, rng, ...)                functional.dropout, which is its own gradient

`modules.LayerNorm`, `modules.Transition` and `modules.Dropout` call them while autograd records.  Nothing but the operators' own inputs is
kept for the backward pass: row statistics and hidden channels are computed again, a dropout mask comes from its generator again.  Gradients
have a fixed order of summation; second derivatives are refused.  The calls are CUDA only, as everything here.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import functional as F

__all__ = ["layer_norm", "gated_feed_forward", "dropout"]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return F.layer_norm(x, weight, bias, eps, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        dx, dw, db = F.layer_norm_backward(dy, x, weight, ctx.eps, need_weight=ctx.needs_input_grad[1], need_bias=ctx.needs_input_grad[2])
        return dx if ctx.needs_input_grad[0] else None, _as(dw, weight), _as(db, bias), None, None


def _as(g: torch.Tensor | None, like: torch.Tensor | None) -> torch.Tensor | None:
    """The gradient of a parameter that the forward pass took in any shape of C elements."""
    if g is None or (g.dtype == like.dtype and g.shape == like.shape):
        return g
    return g.to(like.dtype).view(like.shape)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """LayerNorm over the last dim (model/primitives/normalization.py:61-91), x (..., C) bfloat16 or float32, C <= 1024."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype)


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out):
        ctx.save_for_backward(x, w_in, w_out)
        return F.gated_feed_forward(x, w_in, w_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return F.gated_feed_forward_backward(dy, *ctx.saved_tensors, *ctx.needs_input_grad)


def gated_feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor) -> torch.Tensor:
    """(silu(x Wa^T) * (x Wb^T)) Wo^T, [Wa; Wb] = w_in (2 hidden, C), Wo = w_out (C, hidden): SwiGLU and output projection of a Transition
    (model/layers/folding/transition.py:48-68).  x bfloat16 with bfloat16 or float32 parameters, or all float32."""
    return _GatedFeedForward.apply(x, w_in, w_out)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, shared_dim):
        if isinstance(rng, torch.Tensor) and p:      # the caller may move it on before the backward pass
            rng = rng.clone()
            ctx.save_for_backward(rng)
            ctx.rng = None
        else:
            ctx.rng = rng
        ctx.p, ctx.shared_dim, ctx.dtype = p, shared_dim, x.dtype
        return F.dropout(x, p, rng, shared_dim, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            if ctx.p:
                dy_kept = F.dropout(dy, ctx.p, ctx.saved_tensors[0] if ctx.rng is None else ctx.rng, ctx.shared_dim)
            else:
                dy_kept = dy
            dx = dy_kept.to(ctx.dtype)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, rng, shared_dim: int | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """(residual +) dropout(x) with the mask of `functional.dropout`: rng = (seed, offset) or an int64 CUDA tensor of the two."""
    return _Dropout.apply(x, residual, p, rng, shared_dim)
