"""Gradients of a padded batch's keys behind their row's length: 0, whatever the
scores of the real ones are, under the bounds of test_gpu_attention.py.

A key that is not there has a score of 0 in the kernel, and exp(0 - lse) passes
fp16's range (kept times 2^15) with an lse under -0.69, the others' under -88."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, DTYPES, case, mg, randn, generator
from tests.test_gpu_attention import compare, reference, run

pytestmark = pytest.mark.gpu
#: the first two: work-groups whose waves share keys; the others: waves with keys of their own
SHAPES = [(6, 64, 40, 2, 2, 64, False), (4, 64, 40, 32, 1, 128, True), (80, 64, 140, 8, 8, 64, False),
          (150, 70, 40, 4, 4, 128, False), (128, 40, 40, 128, 4, 32, True)]


def inputs(B, N, M, H, Hk, D, dtype, score):
    """Scores near `score`, in units of a softmax without a scale."""
    gen = generator(B + D)
    q, k = randn(gen, (B, N, H, D), dtype, 0.02).add_(1.0), randn(gen, (B, M, Hk, D), dtype, 0.02).add_(1.0)
    return q, k.mul_(score / D), randn(gen, (B, M, Hk, D), dtype), randn(gen, (B, N, H, D), dtype, 0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", [-2.0, -12.0, -150.0])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_keys_behind_the_length_have_no_gradient(dtype, score, i):
    B, N, M, H, Hk, D, causal = SHAPES[i]
    case("attention, few real keys", dtype, score, SHAPES[i])
    q, k, v, g = inputs(B, N, M, H, Hk, D, DTYPES[dtype], score)
    real = [(1, 2, 3, 4, 33, 0)[b % 6] for b in range(B)]
    for b in range(B):
        k[b, real[b]:] = v[b, real[b]:] = float("nan")
    got = run(q, k, v, g, causal=causal, scale=1.0, key_lengths=torch.tensor(real, device=DEV))
    for b in range(B):
        assert not bool(got["dk"][b, real[b]:].any()) and not bool(got["dv"][b, real[b]:].any()), b
    some = min(B, 6)                # the reference goes head by head
    if H > 32:
        some = 2
    clean = [t[:some].nan_to_num(0.0) for t in (q, k, v, g)]
    parts = [(b, slice(0, N), slice(0, real[b])) for b in range(some)]
    compare({n: t[:some] for n, t in got.items()}, *reference(*clean, parts, causal, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_through_autograd(dtype):
    """The value projection's weight gets a gradient without a NaN."""
    t = DTYPES[dtype]
    q, k, x, g = inputs(3, 64, 8, 2, 2, 64, t, -100.0 if dtype != "f16" else -3.0)
    weight = randn(generator(3), (64, 64), t, 0.1).requires_grad_(True)
    lengths = torch.tensor([1, 3, 8], device=DEV)
    out = mg.attention(q, k, torch.matmul(x, weight), key_lengths=lengths, causal=False, scale=1.0)
    assert bool(torch.autograd.grad(out, weight, g)[0].isfinite().all())
