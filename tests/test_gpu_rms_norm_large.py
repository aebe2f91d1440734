"""The norm's backward pass over rows near the type's largest values, under the
bounds of test_gpu_rms_norm.py: the gradient's product with the row passes 32 bits
where that with the normed row, whose values are near 1, does not."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, randn
from tests.test_gpu_rms_norm import check_backward, check_y

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [7, 200, 1000, 4096, 9001, 20_000, 32_768])
def test_rows_near_the_largest_values(dtype, width):
    case("rms_norm_backward, large rows", dtype, width)
    t = DTYPES[dtype]
    gen, big = generator(width), torch.finfo(t).max
    # rows of the largest value, of values up to it, and of 1e30 beside gradients of 1e10 (fp16: as large as it takes)
    h = randn(gen, (5, width), torch.float32, 0.2).clamp_(-1.0, 1.0)
    h[0] = 1.0
    h = (h.double() * torch.tensor([big, big, 1e30 if big > 1e30 else 6e4, 1.0, 1.0], dtype=torch.float64, device=DEV)[:, None]).to(t)
    gy = randn(gen, (5, width), torch.float32)
    gy[0] = 1.0                     # all of one sign: the sum is as large as it gets
    gy = (gy.double() * torch.tensor([1.0, 1.0, 1e10 if big > 1e30 else 1e4, 1.0, 1e-3], dtype=torch.float64, device=DEV)[:, None]).to(t)
    w = randn(gen, (width,), torch.float32, 0.2).add_(1.0)         # whose gradient has fp32's range
    assert bool(h.isfinite().all()) and bool(gy.isfinite().all())
    check_y(mg.rms_norm(h, w), h, w)
    for gh in (None, gy):
        dx, dw = mg.rms_norm_backward(gy, h, w, grad_h=gh)
        assert bool(dx.isfinite().all())
        check_backward(dx, dw, gy, gh, h, w)
