"""RMS norm of every query and key head, and the rotary rotation, in one pass.

    out = rotate(x / sqrt(mean(x^2) + eps) * weight)

for each head's vector x of q and k.  The rotation turns the pairs
(i, i + rotary/2) of the first `rotary` elements, or (2i, 2i + 1) when
interleaved, by the angles of the token's position; the others pass through.
"""

from __future__ import annotations

import torch

from . import _native as N
from ._autograd import recorded


def rope_tables(length: int, rotary: int, *, base: float = 10000.0,
                device: torch.device | str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) of the angles position * base^(-2i / rotary) for positions
    0..length-1 and i < rotary/2: float32, formed in 64 bits."""
    if rotary < 2 or rotary % 2:
        raise ValueError(f"rotary must be even and at least 2, got {rotary}")
    frequency = float(base) ** (-torch.arange(0, rotary, 2, device=device, dtype=torch.float64) / rotary)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * frequency
    return angle.cos().float(), angle.sin().float()


def qk_norm_rope_backward(grad_q: torch.Tensor, grad_k: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                          positions: torch.Tensor | None = None, *, eps: float = 1e-6, interleaved: bool = False,
                          heads_first: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(d_q, d_k, d_q_weight, d_k_weight) from the gradients of qk_norm_rope's
    outputs and its arguments; d_q and d_k are contiguous, the weights'
    gradients are sums over all tokens and heads in a fixed order."""
    return N.ops().qk_norm_rope_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved,
                                         heads_first, N.ops_stream(q))


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, *how):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = how
        return N.ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, *how, N.ops_stream(q))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        given = ctx.saved_tensors
        return (*N.ops().qk_norm_rope_backward(grad_q, grad_k, *given, *ctx.how, N.ops_stream(given[0])),) + (None,) * 6


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-6, interleaved: bool = False,
                 heads_first: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The normed and rotated (q, k), differentiable by q, k and the weights.

    q, k: (batch, length, heads, dim), of strides of their own (slices of one
    projection's output are read in place), dim at most 512.  q_weight,
    k_weight: (dim,), of q's dtype or another of the three.  cos, sin: float32
    (positions, rotary/2), as rope_tables makes them.  positions: int64 or int32
    of shape (length,) or (batch, length); None for 0, 1, ...; one outside the
    tables makes its token's rotated elements NaN.  heads_first: the outputs are
    (batch, heads, length, dim), as attention reads them.  cos and sin get no
    gradient; one that asks for it is refused."""
    if torch.is_grad_enabled():
        for name, t in (("cos", cos), ("sin", sin)):
            if t.requires_grad:
                raise ValueError(f"qk_norm_rope has no gradient by {name}: detach it")
    if recorded(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, heads_first)
    return N.ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, heads_first,
                                N.ops_stream(q))
