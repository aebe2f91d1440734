"""CPU-only: calls of attention and the residual's norm that are refused."""

from __future__ import annotations

import pytest

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
