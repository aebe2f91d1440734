"""Attention of grouped heads: over a batch, over packed sequences, of new tokens
over a cache; and its backward pass.

    out_i = sum_j softmax_j(scale * q_i . k_j) v_j

over the keys that query i of a sequence of n queries and m keys sees: j <= i +
m - n if causal, so that the last query sees the last key, and else all.  A query
that sees none has out 0, lse -inf and no gradient; one whose largest score passes
32 bits is NaN.  Scores, softmax statistics and sums are held in 32 bits; probabilities and the scores' gradients are rounded
to the inputs' type for the products that follow them.
"""

from __future__ import annotations

import torch

from . import _native as N
from ._autograd import apart, recorded


def attention_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, *, offsets: torch.Tensor | None = None, key_offsets: torch.Tensor | None = None,
                       lengths: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None, causal: bool = True,
                       scale: float | None = None,
                       heads_first: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(d_q, d_k, d_v), contiguous and of the inputs' shapes, from the gradient of
    out, what attention_lse returned and its arguments.  The heads that share
    keys are summed in a fixed order."""
    return N.ops().attention_backward(grad_out, q, k, v, out, lse, offsets, key_offsets, lengths, key_lengths, causal, scale,
                                      heads_first, N.ops_stream(q))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, *how):
        out, lse = N.ops().attention(q, k, v, *how, True, N.ops_stream(q))
        ctx.save_for_backward(q, k, v, out, lse, *how[:4])
        ctx.how = how[4:]
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        given = ctx.saved_tensors
        return (*N.ops().attention_backward(grad_out, *given, *ctx.how, N.ops_stream(given[0])),) + (None,) * 7


def _with_lse(q, *given) -> tuple[torch.Tensor, ...]:
    return N.ops().attention(q, *given, True, N.ops_stream(q))


def attention_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, offsets: torch.Tensor | None = None,
                  key_offsets: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                  key_lengths: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
                  heads_first: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, lse): attention and, for attention_backward or to join parts of the
    keys, the logarithm of each row's sum of exp(scores), float32 (batch, heads,
    length).  Nothing is recorded for autograd."""
    return apart(_with_lse, q, k, v, offsets, key_offsets, lengths, key_lengths, causal, scale, heads_first)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, offsets: torch.Tensor | None = None,
              key_offsets: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
              key_lengths: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
              heads_first: bool = False) -> torch.Tensor:
    """out (batch, length, heads, dim), contiguous, differentiable by q, k and v.

    q: (batch, length, heads, dim); k, v: (batch, keys, k_heads, dim), heads a
    multiple of k_heads, dim at most 128; with heads_first (batch, heads, length,
    dim), as qk_norm_rope returns them, and out as the output projection reads it
    all the same.  Strides are free but for the last dimension's: slices of a
    fused projection and a cache's filled part are read in place.

    lengths, key_lengths: int64 or int32 (batch,) on the GPU, how many queries and
    keys of each row of the batch are real (a cache's filled part); the others are
    not read, and out is 0 there.  offsets: int64 or int32 (sequences + 1,), not
    decreasing: packed sequences in a batch of 1, sequence s the tokens from
    offsets[s] to offsets[s + 1]; key_offsets where the keys are packed otherwise.
    Tokens of no sequence are not read, and out is 0 there.

    scale: from 2^-100 to below 2^100, 1/sqrt(dim) by default.  A key or value that is not finite
    reaches queries of its own sequence only, but there also some before it."""
    if recorded(q, k, v):
        return _Attention.apply(q, k, v, offsets, key_offsets, lengths, key_lengths, causal, scale, heads_first)
    return N.ops().attention(q, k, v, offsets, key_offsets, lengths, key_lengths, causal, scale, heads_first, False,
                             N.ops_stream(q))[0]
