"""Which calls of an operator have to go through its autograd function."""

from __future__ import annotations

from collections.abc import Callable

import torch
from torch.autograd import forward_ad


def recorded(*tensors: torch.Tensor | None) -> bool:
    """Whether something watches a call on these tensors that sees autograd
    functions only: autograd, where one of them asks for a gradient; a level of
    forward-mode derivatives, which then raises for a dual tensor (it asks for no
    gradient, and its tangent would be dropped); torch.jit.trace, which would
    keep the result as a constant."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 or torch.jit.is_tracing()


class _Apart(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, *given):
        out = call(*given)
        ctx.mark_non_differentiable(*out)
        return out


def apart(call: Callable[..., tuple[torch.Tensor, ...]], *given) -> tuple[torch.Tensor, ...]:
    """call(*given), new tensors of which nothing is recorded for autograd.  Where
    something watches that would keep the results as constants, or drop a tangent,
    the call goes through an autograd function whose results ask for no gradient.
    A trace keeps what is given but tensors: `call` itself asks for the stream."""
    watched = forward_ad._current_level >= 0 or torch.jit.is_tracing()
    return _Apart.apply(call, *given) if watched else call(*given)
