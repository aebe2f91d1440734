"""The MLP's activation, with its inputs kept for the backward pass in 8 bits.

    y = act(gate) * up            (SwiGLU with act="silu"), or act(gate) without up

A training pass keeps, instead of gate, up and y, an 8-bit checkpoint of gate
and up: int8 codes and one fp32 scale per 128 elements of a row, about half of
what bf16 gate and up take.  Its format is in include/mgopt_ops.h.  The
backward pass computes from it the gradients of gate and up and, for the weight
gradient of the projection that follows, y once more.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from ._autograd import recorded


class ActCheckpoint(NamedTuple):
    """What gated_act_backward needs of a forward pass."""

    codes: torch.Tensor      # int8 [inputs, rows, groups * 128]
    scales: torch.Tensor     # float32 [inputs, rows, groups]
    act: str
    shape: tuple[int, ...] | None = None     # the activation's; without it, gated_act_backward checks the count of rows only


def gated_act_pack(gate: torch.Tensor, up: torch.Tensor | None = None, *,
                   act: str = "silu") -> tuple[torch.Tensor, ActCheckpoint]:
    """(y, checkpoint) of gate and up, of any shape and any strides whose rows
    (the last dimension) are contiguous and evenly spaced; others are copied
    first.  act: "silu" or "gelu_tanh".  Nothing is recorded for autograd."""
    y, codes, scales = N.ops().gated_act(gate, up, act, True, N.ops_stream(gate))
    return y, ActCheckpoint(codes, scales, act, tuple(y.shape))


def gated_act_backward(grad_out: torch.Tensor, saved: ActCheckpoint, *,
                       want_y: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """(d_gate, d_up, y) from the gradient of y: d_up is None without a gate, y
    without want_y.  The outputs have grad_out's shape and dtype; its rows are
    those of y, in their order."""
    return N.ops().gated_act_backward(grad_out, saved.codes, saved.scales, saved.act, saved.shape, want_y, N.ops_stream(grad_out))


class _GatedAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, act):
        y, saved = gated_act_pack(gate, up, act=act)
        ctx.save_for_backward(saved.codes, saved.scales)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        d_gate, d_up, _ = gated_act_backward(grad_out, ActCheckpoint(*ctx.saved_tensors, ctx.act), want_y=False)
        return d_gate, d_up, None


def gated_act(gate: torch.Tensor, up: torch.Tensor | None = None, *, act: str = "silu") -> torch.Tensor:
    """act(gate) * up, or act(gate); where a gradient will be asked for, autograd
    keeps the 8-bit checkpoint and neither gate nor up."""
    if recorded(gate, up):
        return _GatedAct.apply(gate, up, act)
    return N.ops().gated_act(gate, up, act, False, N.ops_stream(gate))[0]
