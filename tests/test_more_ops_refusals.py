"""CPU-only: calls of attention and the residual's norm that are refused."""

from __future__ import annotations

import pytest
import torch

from tests.test_more_ops_host import E_INVALID, _attention, _refused, lib, vp  # noqa: F401


@pytest.mark.parametrize("scale", [2.0**-101, 2.0**-151, 5e-324, 2.0**100])
def test_scales_beyond_fp32(lib, scale):  # noqa: F811
    for call in (lib.mgopt_attention, lib.mgopt_attention_backward):
        _refused(lib, call(_attention(scale=scale), vp(None)), E_INVALID, b"scale")
    for backward in (0, 1):
        assert lib.mgopt_attention_workspace(_attention(scale=scale), backward) == -1


def test_scales_at_the_ends(lib):  # noqa: F811
    for scale in (2.0**-100, 2.0**99):
        assert lib.mgopt_attention(_attention(scale=scale, batch=0), vp(None)) == 0
        assert lib.mgopt_attention_workspace(_attention(scale=scale), 1) > 0


def test_rms_norm_int8_cuts_no_stream(mg):
    """h goes on as the residual stream: one that asks for a gradient is not returned without it."""
    x, w = torch.ones(2, 4), torch.ones(4, requires_grad=True)
    asks = torch.ones(2, 4, requires_grad=True)
    for call, name in ((lambda: mg.rms_norm_int8(asks, w), "x"), (lambda: mg.rms_norm_int8(asks, w, residual=x), "x"),
                       (lambda: mg.rms_norm_int8(x, w, residual=asks), "the residual")):
        with pytest.raises(ValueError, match=f"no gradient by {name}: detach it"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU"):
            call()
    for call in (lambda: mg.rms_norm_int8(asks.detach(), w, residual=x), lambda: mg.rms_norm_int8(x, w)):
        with pytest.raises(RuntimeError, match="no CPU"):
            call()
