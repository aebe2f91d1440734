"""What sends an operator's call through its autograd function (no GPU)."""

from __future__ import annotations

import importlib

import torch
from torch.autograd import forward_ad

recorded = importlib.import_module("minigpt-train-infra_amd._autograd").recorded


def test_gradients():
    plain, asks = torch.ones(3), torch.ones(3, requires_grad=True)
    assert not recorded(plain) and not recorded(plain, None)
    assert recorded(asks) and recorded(plain, None, asks)
    with torch.no_grad():
        assert not recorded(asks)
    with torch.inference_mode():
        assert not recorded(asks, torch.ones(3))


def test_forward_mode_levels():
    x = torch.ones(3)
    with forward_ad.dual_level():
        assert recorded(forward_ad.make_dual(x, x))
        with torch.no_grad():
            assert recorded(forward_ad.make_dual(x, x))
    assert not recorded(x)
    seen = []
    torch.func.jvp(lambda v: (seen.append(recorded(v)), v * 2)[1], (x,), (x,))
    assert seen == [True]


def test_traces():
    seen = []
    torch.jit.trace(lambda v: (seen.append(recorded(v)), v * 2)[1], (torch.ones(3),), check_trace=False)
    assert seen == [True] and not recorded(torch.ones(3))
