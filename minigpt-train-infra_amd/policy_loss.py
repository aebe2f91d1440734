"""The clipped policy loss with a KL term, over the logits of a batch's tokens.

With logp = log_softmax(logits / temperature)[target] of each row, ratio =
exp(logp - old_logp), r = ref_logp - logp and a temperature from 2^-120 to 2^120:

    policy = -min(ratio * A, clip(ratio, 1 - low, 1 + high) * A)
    kl     = exp(r) - r - 1
    loss   = mean(policy) + kl_coef * mean(kl)

the means weighted by the mask.  Rows the mask leaves out are not read, so
their targets and logits may hold anything; a batch of nothing else has loss 0
and gradient 0.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # 0-dim float32
    log_probs: torch.Tensor       # float32, one per row; 0 for rows the mask leaves out
    policy: torch.Tensor          # 0-dim: the mean of the policy term
    kl: torch.Tensor              # 0-dim: the mean of the KL term (0 without ref_logp)
    clip_fraction: torch.Tensor   # 0-dim: the share of rows whose gradient the clip holds at 0


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, *, mask: torch.Tensor | None = None,
                    temperature: float = 1.0) -> torch.Tensor:
    """The log-probability of each row's target, float32 of logits.shape[:-1]
    (what policy_loss takes as old_logp and ref_logp).  targets: int64 or int32; a
    target outside the vocabulary gives NaN.  mask: bool, or float32 weights; rows
    of weight 0 give 0.  Values per row have the shape logits.shape[:-1] or are a
    flat list of the rows.  Nothing is recorded for autograd."""
    return N.ops().token_log_probs(logits, targets, mask, temperature, N.ops_stream(logits))


def policy_loss_grad(logits: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                     ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                     clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0, temperature: float = 1.0,
                     grad_scale: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> tuple[PolicyLoss, torch.Tensor]:
    """The loss and its gradient by the logits in one pass over them, for
    `logits.backward(gradient)`.  grad_scale: a float32 GPU scalar the gradient
    is multiplied by (a GradScaler's scale).  out: where the gradient goes; the
    logits themselves may be given, where no other backward pass needs them (one
    that saved them raises).  Nothing is recorded for autograd."""
    *r, grad, _ = N.ops().policy_loss(logits, targets, old_logp, advantages, ref_logp, mask, clip[0], clip[1], kl_coef,
                                      temperature, grad_scale, True, out, N.ops_stream(logits))
    return PolicyLoss(*r), grad


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, old_logp, advantages, ref_logp, mask, *scalars):
        *r, _, work = N.ops().policy_loss(logits, targets, old_logp, advantages, ref_logp, mask, *scalars, None, False, None,
                                          N.ops_stream(logits))
        ctx.save_for_backward(logits, targets, old_logp, advantages, ref_logp, mask, r[1], work)
        ctx.scalars = scalars
        ctx.mark_non_differentiable(*r[1:])
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, *_):
        *given, log_probs, work = ctx.saved_tensors
        grad = N.ops().policy_loss_backward(*given, *ctx.scalars, grad_loss, log_probs, work, N.ops_stream(given[0]))
        return (grad,) + (None,) * 9


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0, temperature: float = 1.0) -> PolicyLoss:
    """The loss, differentiable by the logits: the backward pass reads them once
    more.  logits: (..., vocab) in float32, float16 or bfloat16; targets: int64
    or int32; the others float32, one value per row.  mask: bool, or float32
    weights.  A target outside the vocabulary in a row that counts makes the
    loss NaN.  old_logp, advantages, ref_logp and mask get no gradient; one that
    asks for it is refused."""
    for name, t in (("old_logp", old_logp), ("advantages", advantages), ("ref_logp", ref_logp), ("mask", mask)):
        if t is not None and t.requires_grad:
            raise ValueError(f"policy_loss has no gradient by {name}: detach it")
    return PolicyLoss(*_PolicyLoss.apply(logits, targets, old_logp, advantages, ref_logp, mask, float(clip[0]),
                                         float(clip[1]), float(kl_coef), float(temperature)))
