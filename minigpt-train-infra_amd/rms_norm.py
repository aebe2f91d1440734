"""RMS norm, with the addition that comes before it in a residual stream.

    h = round(x + residual)        y = h / sqrt(mean(h^2) + eps) * weight

h is rounded to the stream's type before it is normed, and is what the backward
pass reads; a program keeps it anyway, as the stream.  Without a residual, h is x.
rms_norm_int8 gives y in 8 bits, for int8_linear.
"""

from __future__ import annotations

import torch

from . import _native as N
from ._autograd import apart, recorded
from .int8_linear import Int8Rows


def rms_norm_backward(grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, *, grad_h: torch.Tensor | None = None,
                      eps: float = 1e-6, want_weight: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(d_x, d_weight) from the gradient of y, that of h (None: there is none) and
    h itself: d_x is the gradient of x and of the residual alike.  d_weight, of
    the weight's dtype, is a sum over all rows in a fixed order; None without
    want_weight.  The gradients have h's shape and dtype."""
    return N.ops().rms_norm_backward(grad_y, grad_h, h, weight, eps, want_weight, N.ops_stream(h))


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return N.ops().rms_norm(x, None, weight, eps, False, N.ops_stream(x))[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, weight = ctx.saved_tensors
        return (*rms_norm_backward(grad_y, x, weight, eps=ctx.eps, want_weight=ctx.needs_input_grad[1]), None)


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h = N.ops().rms_norm(x, residual, weight, eps, False, N.ops_stream(x))
        ctx.save_for_backward(h, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_h):
        h, weight = ctx.saved_tensors
        if grad_y is None:              # the stream alone was used: the sum's gradient, and none of the weight
            return grad_h, grad_h, None, None
        d_x, d_weight = rms_norm_backward(grad_y, h, weight, grad_h=grad_h, eps=ctx.eps, want_weight=ctx.needs_input_grad[2])
        return d_x, d_x, d_weight, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6) -> torch.Tensor:
    """The normed rows (the last dimension, of at most 32,768 elements) of x, of
    x's dtype, differentiable by x and weight.  weight: (width,), of x's dtype or
    another of the three."""
    if recorded(x, weight):
        return _RmsNorm.apply(x, weight, eps)
    return N.ops().rms_norm(x, None, weight, eps, False, N.ops_stream(x))[0]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): the normed rows of h = x + residual, and h, the stream that goes
    on.  x and residual have one shape and dtype.  Differentiable by all three."""
    if recorded(x, residual, weight):
        return _AddRmsNorm.apply(x, residual, weight, eps)
    return N.ops().rms_norm(x, residual, weight, eps, False, N.ops_stream(x))


def _normed_rows(x, residual, weight, eps) -> tuple[torch.Tensor, ...]:
    codes, scales, h = N.ops().rms_norm(x, residual, weight, eps, True, N.ops_stream(x))
    return (codes, scales) if residual is None else (codes, scales, h)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                  eps: float = 1e-6) -> tuple[Int8Rows, torch.Tensor]:
    """(rows, h): y in 8 bits with a scale for each row, rounded from 32 bits,
    and h (x itself without a residual).  Nothing is recorded for autograd: an x
    and a residual that ask for a gradient, which h would lose, are refused."""
    if torch.is_grad_enabled():
        for name, t in (("x", x), ("the residual", residual)):
            if t is not None and t.requires_grad:
                raise ValueError(f"rms_norm_int8 has no gradient by {name}: detach it")
    rows = apart(_normed_rows, x, residual, weight, eps)
    return Int8Rows(*rows[:2]), x if residual is None else rows[2]
