"""The training operators under torch's autograd.

`functional` holds each operator and its gradient as plain calls; here they are joined:

    layer_norm(x, weight, bias)            functional.layer_norm, layer_norm_backward
    gated_feed_forward(x, w_in, w_out)     functional.gated_feed_forward, gated_feed_forward_backward
    dropout(x, p, rng, ...)                functional.dropout, which is its own gradient
    residual_norm(x, u, gate, ...)         functional.residual_norm, residual_norm_backward
    fused_linear(x, w, bias, ...)          functional.fused_linear, fused_linear_backward

`modules.LayerNorm`, `Transition`, `Dropout`, `Linear`, `AdaLN` and `ConditionedTransitionBlock` and `trunk.ParcaeRecurrence` call them while autograd records.
Nothing but the operators' own inputs is kept for the backward pass: row statistics and hidden channels are computed again, a dropout mask comes from its
generator again.  Under ``compressed()`` those inputs are kept in 8 bits.  Gradients have a fixed order of summation; second derivatives are
refused.  The calls are CUDA only, as everything here.
"""
from __future__ import annotations

import threading
from contextlib import ContextDecorator

import torch
from torch.autograd.function import once_differentiable

from . import functional as F

__all__ = ["layer_norm", "gated_feed_forward", "dropout", "residual_norm", "fused_linear", "compressed", "checkpoint_contexts"]

_this_thread = threading.local()


class compressed(ContextDecorator):
    """``with compressed():`` -- calls of this thread keep rows for the backward pass in 8 bits (``functional.compress``: 33 / 32 bytes a value, off by
    at most 2^-7 of the largest of 32 neighbours): the inputs of layer_norm, gated_feed_forward and fused_linear, the stream and the block's
    output of residual_norm.  Results of the forward pass stay what they are, but for the last bit of layer_norm, which residual_norm's kernel then
    computes; gradients are those at the kept values.

    A checkpoint repeats the forward pass on a thread of autograd's own, where this one's choice does not hold: the ``with`` stands inside the function that is
    checkpointed, or the checkpoint is given ``checkpoint_contexts``."""

    def __init__(self, enabled: bool = True):
        self.enabled = enabled

    def __enter__(self) -> None:
        if not hasattr(_this_thread, "before"):
            _this_thread.before = []
        _this_thread.before.append(_compressing())
        _this_thread.compressed = self.enabled

    def __exit__(self, *exc) -> None:
        _this_thread.compressed = _this_thread.before.pop()


def checkpoint_contexts() -> tuple:
    """``checkpoint(block, x, use_reentrant=False, context_fn=checkpoint_contexts)`` (torch.utils.checkpoint): the pass that is repeated keeps rows as the first
    one does, which is as this thread keeps them now (``compressed``)."""
    as_now = compressed(_compressing())
    return as_now, as_now


def _compressing() -> bool:
    return getattr(_this_thread, "compressed", False)


def _keep(ctx, kept: list, *others) -> None:
    """Save `kept`, rows as tensors, Compressed or None, and `others` for the backward pass."""
    ctx.kept_as = [t.dtype if type(t) is F.Compressed else None for t in kept]
    flat = []
    for t in kept:
        flat += [t.values, t.exponents] if type(t) is F.Compressed else [t]
    ctx.save_for_backward(*flat, *others)


def _kept(ctx) -> list:
    """What `_keep` was given."""
    saved, out = iter(ctx.saved_tensors), []
    for dtype in ctx.kept_as:
        out.append(next(saved) if dtype is None else F.Compressed(next(saved), next(saved), dtype))
    return out + list(saved)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        ctx.eps = eps
        if _compressing() and any(ctx.needs_input_grad) and (x.dtype, out_dtype or x.dtype) in F._STREAM_CODES and x.shape[-1] <= 1024:
            _, y, kept = F.residual_norm(x, weight=weight, bias=bias, eps=eps, out_dtype=out_dtype, compress=True)
            _keep(ctx, [kept], weight, bias)
            return y
        _keep(ctx, [x], weight, bias)
        return F.layer_norm(x, weight, bias, eps, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = _kept(ctx)
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
        _keep(ctx, [F.compress(x) if _compressing() and any(ctx.needs_input_grad) else x], w_in, w_out)
        return F.gated_feed_forward(x, w_in, w_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return F.gated_feed_forward_backward(dy, *_kept(ctx), *ctx.needs_input_grad)


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


class _ResidualNorm(torch.autograd.Function):
    """(r, y), of which r is missing where it is x itself and y without a norm."""

    @staticmethod
    def forward(ctx, x, u, gate, scale, weight, bias, gate_shift, samples, eps, norm, out_dtype):
        ctx.set_materialize_grads(False)
        ctx.samples, ctx.eps = samples, eps
        ctx.stream, ctx.norm = u is not None or scale is not None, norm
        need_u, need_x = gate is not None and ctx.needs_input_grad[2], scale is not None and ctx.needs_input_grad[3]
        small = _compressing() and any(ctx.needs_input_grad)
        r, y, *kept = F.residual_norm(x, u, gate, scale, weight, bias, gate_shift, samples, eps, norm, out_dtype, compress=small and norm)
        put = lambda t: F.compress(t) if small else t
        # (without a norm the backward pass reads nothing of r: dr has its shape and type)
        ctx.u_dtype, ctx.x_missing = None if u is None else u.dtype, x is None
        _keep(ctx, [(kept[0] if kept else r) if norm else None, put(u) if need_u else None, put(x) if need_x else None], gate, scale, weight, bias, gate_shift)
        return (r, y) if ctx.stream and norm else r if ctx.stream else y

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        dr, dy = grads if ctx.stream and ctx.norm else (grads[0], None) if ctx.stream else (None, grads[0])
        if dr is None and dy is None:
            return (None,) * 11
        r, u, x, gate, scale, weight, bias, gate_shift = _kept(ctx)
        need = ctx.needs_input_grad
        if r is None:
            r = dr                       # (of its shape and type)
        if u is None and ctx.u_dtype is not None:
            u = dr if dr is not None and dr.dtype == ctx.u_dtype else dy if dy is not None else dr.new_empty((), dtype=ctx.u_dtype).expand(dr.shape)
        g = F.residual_norm_backward(dr, dy, r, u, gate, x, scale, weight, gate_shift, ctx.samples, ctx.eps, need[0], need[1], need[2] and gate is not None,
                                     need[3] and scale is not None, need[4], need[5], need[6])
        return (None if ctx.x_missing else g.x, g.u, g.gate, _as(g.scale, scale), _as(g.weight, weight), _as(g.bias, bias), g.gate_shift, None, None, None, None)


def residual_norm(x, u=None, gate=None, scale=None, weight=None, bias=None, gate_shift=None, samples: int = 1, eps: float = 1e-5, norm: bool = True,
                  out_dtype: torch.dtype | None = None):
    """``functional.residual_norm``: (r, y), r being x itself without u and scale, y None without ``norm``."""
    out = _ResidualNorm.apply(x, u, gate, scale, weight, bias, gate_shift, samples, eps, norm, out_dtype)
    if u is None and scale is None:
        return x, out
    return out if norm else (out, None)


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        ctx.activation = activation
        wanted = activation is not None or ctx.needs_input_grad[1]         # (x is read by nothing else)
        _keep(ctx, [(F.compress(x) if _compressing() and any(ctx.needs_input_grad) else x) if wanted else None], w, bias)
        ctx.x_like = (x.shape, x.dtype)
        return F.fused_linear(x, w, bias, activation, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, bias = _kept(ctx)
        need = ctx.needs_input_grad
        if x is None:
            x = dy.new_empty((), dtype=ctx.x_like[1]).expand(ctx.x_like[0])          # (of its shape and type)
        dx, dw, db = F.fused_linear_backward(dy, x, w, bias, ctx.activation, need[0], need[1], need[2])
        return dx, dw, _as(db, bias), dy if need[3] else None, None


def fused_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """``functional.fused_linear``: f(x w^T + bias) (+ residual)."""
    return _FusedLinear.apply(x, w, bias, residual, activation)
