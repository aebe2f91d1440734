"""attention at the ends of the scale's range, and of its scores' in 32 bits."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, DTYPES, mg
from tests.test_gpu_attention import compare, inputs, reference, run, whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_that_leave_nothing_of_the_scores(dtype):
    """At the smallest scale that is taken a row is the mean of what it sees; its
    gradient by q and k is below every type's smallest value, or near it."""
    q, k, v, g = inputs(2, 150, 150, 2, 1, 64, DTYPES[dtype], 30)
    got = run(q, k, v, g, scale=2.0**-100)
    compare(got, *reference(q, k, v, g, whole(2, 150, 150), scale=2.0**-100))


@pytest.mark.parametrize("scale", [2.0**-101, 2.0**-151, 1e-300])
def test_smaller_scales_are_refused(scale):
    """log2(e) * scale would lose bits in fp32, and then be 0, whose product with a masked score's -inf is a NaN."""
    q, k, v, g = inputs(1, 5, 5, 2, 1, 32, torch.float32, 31)
    out, lse = mg.attention_lse(q, k, v)
    for call in (lambda: mg.attention(q, k, v, scale=scale), lambda: mg.attention_lse(q, k, v, scale=scale),
                 lambda: mg.attention_backward(g, q, k, v, out, lse, scale=scale)):
        with pytest.raises(ValueError, match="scale must be at least 2\\^-100"):
            call()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N, M", [(3, 5), (70, 300), (1, 5000)])
def test_scores_beyond_32_bits_are_no_empty_rows(dtype, N, M):
    """q . k is finite and its product with the scale is not: NaN, as inf - inf is in
    elementary operations in 32 bits, and not the 0 and -inf of a row without keys."""
    t = DTYPES[dtype]
    for sign in (1.0, -1.0):
        q = torch.full((1, N, 2, 32), 2.0**60, dtype=t, device=DEV)
        k = torch.full((1, M, 1, 32), sign * 2.0**60, dtype=t, device=DEV)
        v, g = torch.ones_like(k), torch.ones_like(q)
        out, lse = mg.attention_lse(q, k, v, scale=2.0**10, causal=False)
        assert bool(out.isnan().all()) and bool(lse.isnan().all())
        for d in mg.attention_backward(g, q, k, v, out, lse, scale=2.0**10, causal=False):
            assert bool(d.isnan().all())
