"""Token embedding: the lookup of scaled rows, and the weight's gradient.

    out[t] = scale * weight[ids[t]]
    grad[v] += scale * sum of grad_out[t] over the tokens t with ids[t] = v

The sums run in float32 over the tokens in their order, without atomics: the
same inputs give the same bits.
"""

from __future__ import annotations

import torch

from . import _native as N
from ._autograd import recorded


def embedding_grad_(grad: torch.Tensor, ids: torch.Tensor, grad_out: torch.Tensor, *, scale: float = 1.0,
                    padding_idx: int | None = None, accumulate: bool = True) -> torch.Tensor:
    """Adds the embedding's gradient into `grad` (rows, width), contiguous: only
    the rows that the ids name are read and written, so a weight that is tied to
    the output projection, or a later micro-batch, costs no pass over the whole
    gradient.  accumulate=False writes every row instead, zeros where no id
    names it.  grad_out: ids.shape + (width,), of grad's dtype or another of the
    three.  Ids outside the rows and equal to padding_idx add nothing.  Fewer than
    2^30 ids and 2^31 rows."""
    N.ops().embedding_grad(grad, ids, grad_out, scale, padding_idx, accumulate, N.ops_stream(grad))
    return grad


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, dtype):
        ctx.save_for_backward(ids)
        ctx.how = weight.shape, weight.dtype, scale, padding_idx
        return N.ops().embedding(ids, weight, scale, dtype, N.ops_stream(weight))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        shape, dtype, scale, padding_idx = ctx.how
        grad = torch.empty(shape, dtype=dtype, device=grad_out.device)
        embedding_grad_(grad, ids, grad_out, scale=scale, padding_idx=padding_idx, accumulate=False)
        return None, grad, None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None,
              dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale * weight[ids], of shape ids.shape + (width,) and of weight's dtype
    (or `dtype`), differentiable by weight.  ids: int64 or int32 of any shape;
    an id outside the rows gives a row of NaN and no gradient.  padding_idx: the
    row that gets no gradient."""
    if padding_idx is not None and not -weight.shape[0] <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is outside {weight.shape[0]} rows")
    if recorded(weight):
        return _Embedding.apply(ids, weight, scale, padding_idx, dtype)
    return N.ops().embedding(ids, weight, scale, dtype, N.ops_stream(weight))
