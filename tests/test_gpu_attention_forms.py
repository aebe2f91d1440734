"""Forms of attention's kernels that only larger calls reach (work-groups whose
waves have rows and keys of their own, parts of a long cache), and forms that
alignment and head counts choose, under the bounds of test_gpu_attention.py."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, randn, same_bits
from tests.test_gpu_attention import compare, inputs, reference, run, whole

pytestmark = pytest.mark.gpu
#: 512 work-groups of 128 rows and of 128 keys at least
MANY = [(35, 200, 200, 8, 8, 64), (33, 130, 150, 32, 8, 128), (64, 129, 190, 8, 4, 96), (30, 150, 150, 24, 8, 32),
        (70, 257, 100, 12, 4, 80), (64, 1, 140, 4, 4, 128), (26, 300, 260, 10, 10, 127)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("i", range(len(MANY)))
def test_many_work_groups(dtype, i):
    B, N, M, H, Hk, D = MANY[i]
    q, k, v, g = inputs(B, N, M, H, Hk, D, DTYPES[dtype], i, fused=N == M)
    causal = i % 3 != 1
    case("attention", dtype, "causal" if causal else "full", MANY[i])
    compare(run(q, k, v, g, first=i % 2 == 0, causal=causal), *reference(q, k, v, g, whole(B, N, M), causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_padded_rows(dtype):
    """As above, rows and keys beyond their lengths NaN."""
    B, N, M, H, Hk, D = 40, 170, 200, 12, 4, 64
    case("attention, padded", dtype, (B, N, M, H, Hk, D))
    q, k, v, g = inputs(B, N, M, H, Hk, D, DTYPES[dtype], 21)
    lengths, keys = [(37 * b) % (N + 1) for b in range(B)], [(53 * b + 11) % (M + 1) for b in range(B)]
    for b in range(B):
        q[b, lengths[b]:] = g[b, lengths[b]:] = float("nan")
        k[b, keys[b]:] = v[b, keys[b]:] = float("nan")
    more = {"lengths": torch.tensor(lengths, device=DEV), "key_lengths": torch.tensor(keys, device=DEV)}
    clean = [t.nan_to_num(0.0) for t in (q, k, v, g)]
    parts = [(b, slice(0, lengths[b]), slice(0, keys[b])) for b in range(B)]
    compare(run(q, k, v, g, **more), *reference(*clean, parts))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_many_packed_sequences(dtype, D):
    """300 sequences of 0 to 60 tokens and two long ones, tokens of none before and behind (NaN)."""
    lengths = [(17 * i) % 61 for i in range(150)] + [400] + [(29 * i) % 61 for i in range(150)] + [333]
    at = torch.tensor([3] + lengths).cumsum(0).tolist()
    N, H, Hk = at[-1] + 70, 4, 2
    case("attention, packed", dtype, D, len(lengths), N)
    q, k, v, g = inputs(1, N, N, H, Hk, D, DTYPES[dtype], 22, fused=True)
    for t in (q, k, v, g):
        t[:, :3] = t[:, at[-1]:] = float("nan")
    clean = [t.nan_to_num(0.0) for t in (q, k, v, g)]
    parts = [(0, slice(a, b), slice(a, b)) for a, b in zip(at, at[1:])]
    got = run(q, k, v, g, offsets=torch.tensor(at, dtype=torch.int32, device=DEV))
    compare(got, *reference(*clean, parts))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, N, M, H, Hk, D", [(8, 1, 9000, 32, 32, 128), (3, 2, 40_001, 8, 1, 96), (2, 1, 9001, 4, 2, 50)])
def test_parts_of_long_caches(dtype, B, N, M, H, Hk, D):
    case("attention, cache", dtype, (B, N, M, H, Hk, D))
    q, k, v, _ = inputs(B, N, M, H, Hk, D, DTYPES[dtype], 23)
    filled = [M, 0, 70, M // 2, M - 1, 1, 2000, 129][:B]
    for b in range(B):
        k[b, filled[b]:] = v[b, filled[b]:] = float("nan")
    clean = [t.nan_to_num(0.0) for t in (q, k, v)]
    parts = [(b, slice(0, N), slice(0, filled[b])) for b in range(B)]
    compare(run(q, k, v, None, key_lengths=torch.tensor(filled, device=DEV)), *reference(*clean, None, parts))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [1, 40])
def test_rows_that_start_anywhere(dtype, B):
    """Heads that do not start on 16 bytes give the same bits as those that do."""
    q, k, v, g = inputs(B, 150, 150, 6, 2, 64, DTYPES[dtype], 24)
    want = run(q, k, v, g)
    moved = []
    for t in (q, k, v, g):
        x = torch.full((*t.shape[:2], t.shape[2], 67), float("nan"), dtype=t.dtype, device=DEV)[..., 3:]
        moved.append(x.copy_(t))
    got = run(*moved[:3], moved[3])
    assert all(same_bits([got[n]], [want[n]]) for n in want)


def test_a_cache_beyond_32_bits():
    """Keys and values 2^32 bytes and more behind the first."""
    gen, N = generator(25), 3
    k = torch.zeros((N, 12_000, 128, 1024), dtype=torch.bfloat16, device=DEV)[..., :64]     # 3.1 GB a row of the batch
    spots = torch.tensor([0, 5000, 11_998, 11_999], device=DEV)
    k[:, spots, 126:] = randn(gen, (N, 4, 2, 64), torch.bfloat16, 3.0)
    keys = k[:, :, 126:]
    q = randn(gen, (N, 2, 4, 64), torch.bfloat16, 3.0)
    assert keys[2, 11_999, 1].data_ptr() - k.data_ptr() > 2 * 2**32
    near = keys.contiguous()
    assert same_bits([mg.attention(q, keys, keys)], [mg.attention(q, near, near)])
