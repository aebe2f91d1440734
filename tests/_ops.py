"""What the tests of the training-step operators share: types, unit roundoffs
and comparisons against results in 64 bits."""

from __future__ import annotations

import importlib

import torch

from tests._live import live

mg = importlib.import_module("minigpt-train-infra_amd")
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: the largest relative error of one rounding to the type, and its smallest positive value
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINIEST = {torch.float32: 2.0**-126, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-126}
EPS32 = 2.0**-23


def generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(gen, shape, dtype, sigma=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, sigma, generator=gen)


def case(*what):
    """Names the case on the terminal before it runs."""
    live("case: " + " ".join(str(w) for w in what))


def same_bits(got, want) -> bool:
    """Whether the tensors of both lists have the same bits (NaN among them)."""
    whole = {2: torch.int16, 4: torch.int32}
    return all(a.shape == b.shape and torch.equal(a.contiguous().view(whole[a.element_size()]),
                                                  b.contiguous().view(whole[b.element_size()]))
               for a, b in zip(got, want, strict=True))


def near(got: torch.Tensor, want: torch.Tensor, within: torch.Tensor, what: str) -> None:
    """got against want (64 bits): off by at most `within` (the error of the
    32-bit arithmetic) plus the rounding to got's type."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    g = got.double()
    bound = within + want.abs() * ROUND[got.dtype] * 1.001 + TINIEST[got.dtype]
    bad = ~((g - want).abs() <= bound)
    # equal infinities are no difference, and NaN has to meet NaN
    bad &= ~((g == want) | (g.isnan() & want.isnan()))
    if bool(bad.any()):
        at = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} values are off, the first at {at}: got "
                             f"{float(g.flatten()[at])!r}, want {float(want.flatten()[at])!r}, "
                             f"bound {float((bound + torch.zeros_like(want)).flatten()[at])!r}")
