"""Products of 8-bit integers with a scale for each token and each output
channel, for forward passes that need no gradient (a rollout's).

    y[t, n] = x.scales[t] * weight.scales[n] * sum of x.codes[t] * weight.codes[n]  (+ bias[n])
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from ._autograd import apart


class Int8Rows(NamedTuple):
    """Rows in 8 bits: row t stands for codes[t] * scales[t]."""

    codes: torch.Tensor      # int8 (..., width); rows may lie further apart than their width
    scales: torch.Tensor     # float32 (...)


def _rows(x) -> tuple[torch.Tensor, ...]:
    return N.ops().int8_rows(x, N.ops_stream(x))


def int8_rows(x: torch.Tensor) -> Int8Rows:
    """x (..., width) in 8 bits, a scale for each row: tokens of an activation, or
    the output channels of a weight (channels, width).  With m a row's largest
    magnitude, scale = m / 127 and the codes are the integers nearest to
    x * (127 / m); m below 2^-119 counts as 0, a row with an inf or a NaN has the
    scale NaN.  Nothing is recorded for autograd."""
    return Int8Rows(*apart(_rows, x))


def _linear(codes, *given) -> tuple[torch.Tensor]:
    return (N.ops().int8_linear(codes, *given, N.ops_stream(codes)),)


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y (..., channels) of `dtype` (float32, float16 or bfloat16) from x (...,
    width) and weight (channels, width), of at most 131,071 codes a row: their sums
    are exact in 32 bits.  bias: (channels,), of any of the three types.  Rows of
    codes may lie any distance apart, as int8_rows and rms_norm_int8 leave them.
    Nothing is recorded for autograd: scales and a bias that ask for a gradient are
    refused."""
    if torch.is_grad_enabled():
        for name, t in (("x's scales", x.scales), ("weight's scales", weight.scales), ("bias", bias)):
            if t is not None and t.requires_grad:
                raise ValueError(f"int8_linear has no gradient by {name}: detach it")
    return apart(_linear, x.codes, x.scales, weight.codes, weight.scales, bias, dtype)[0]
