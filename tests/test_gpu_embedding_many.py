"""The embedding's gradient over many tokens: right, and in a time that grows as
the tokens do.  Sums of ones in float32 are exact up to 2^24."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, case, generator, mg, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [96 * 2048 - 1, 96 * 2048, 96 * 2048 + 1, 700_001, (1 << 21) + 5])
@pytest.mark.parametrize("V", [300, 40_000, 700_000])
def test_counts_and_orders(T, V):
    """Column 0 counts a row's tokens; the others are sums of whole numbers."""
    case("embedding_grad_", "tokens", T, "vocab", V)
    gen = generator(T % 97)
    ids = torch.randint(-2, V + 2, (T,), generator=gen, device=DEV)
    ids[: T // 3] = torch.randint(0, 40, (T // 3,), generator=gen, device=DEV)
    g = torch.randint(-8, 9, (T, 4), generator=gen, device=DEV).float()
    g[:, 0] = 1.0
    ok = (ids >= 0) & (ids < V) & (ids != 17)
    want = torch.zeros((V, 4), dtype=torch.float64, device=DEV)
    want.index_add_(0, ids[ok], g[ok].double())
    grad = mg.embedding_grad_(torch.full((V, 4), float("nan"), device=DEV), ids, g, padding_idx=17, accumulate=False)
    assert torch.equal(grad.double(), want)
    again = mg.embedding_grad_(torch.zeros((V, 4), device=DEV), ids.int(), g, padding_idx=17)
    assert torch.equal(again.double(), want)
    # sums that do round: the same bits in every run
    g = torch.randn((T, 4), generator=gen, device=DEV)
    a, b = (mg.embedding_grad_(torch.empty((V, 4), device=DEV), ids, g, accumulate=False) for _ in range(2))
    assert same_bits([a], [b])


def test_time_grows_with_the_tokens():
    """16 times the tokens take about 16 times as long; where each tile of the
    sort reads every tile's counts, it is up to 256 times."""
    V, H = 600_000, 1
    gen, grad = generator(7), torch.zeros((V, H), device=DEV)
    best = {}
    for T in (1 << 20, 1 << 24):
        case("embedding_grad_", "tokens", T, "vocab", V)
        ids = torch.randint(0, V, (T,), generator=gen, device=DEV)
        g = torch.randn((T, H), generator=gen, device=DEV)
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            mg.embedding_grad_(grad, ids, g)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        best[T] = min(times)
    assert best[1 << 24] < 32 * best[1 << 20], best
