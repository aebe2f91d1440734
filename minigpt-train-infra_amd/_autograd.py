"""Which calls of an operator have to go through its autograd function."""

from __future__ import annotations

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
