"""attention, attention_lse and attention_backward against the formulas in 64 bits.

Bounds, with u = 2^-24 and rho the rounding to the inputs' type (0 for float32,
which is not rounded between the products).  A score's sum over dim elements is
off by (dim + 2) u times the sum of the products' magnitudes, and the exponent
rounds a few times more; a probability is off by that, relatively, and by rho.
Each sum over n keys or rows adds n u of the sum of its terms' magnitudes.  The
gradient's delta is a sum over the rounded out.
"""

from __future__ import annotations

import math

import pytest
import torch
from torch.autograd import forward_ad

from tests._ops import DEV, DTYPES, ROUND, case, generator, mg, near, randn, same_bits

pytestmark = pytest.mark.gpu
U = 2.0**-24


def one_head(q, k, v, g, causal, scale, rho):
    """(results, bounds) of one head of one sequence: out, lse, dq, dk, dv in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, D = q.shape[0], k.shape[0], q.shape[1]
    x = scale * (q @ k.t())
    seen = torch.ones((n, m), dtype=torch.bool, device=DEV)
    if causal:
        seen = seen.tril(m - n)
    some = seen.any(-1, keepdim=True) if m else torch.zeros((n, 1), dtype=torch.bool, device=DEV)
    x = x.masked_fill(~seen, float("-inf"))
    lse = torch.logsumexp(x, -1, keepdim=True) if m else torch.full((n, 1), float("-inf"), dtype=torch.float64, device=DEV)
    p = torch.where(seen, torch.exp(x - torch.where(some, lse, 0.0)), 0.0)
    out = p @ v
    # a probability's relative error before its rounding
    ex = (D + 2) * U * scale * (q.abs() @ k.abs().t())
    size = torch.where(seen, x.abs(), 0.0)
    rel = torch.where(seen, ex + (4 * size + 16) * U, 0.0)
    rel = (rel.amax(-1, keepdim=True) if m else torch.zeros((n, 1), dtype=torch.float64, device=DEV)) * 2
    floor = 2.0**-38 if rho == 2.0**-11 else 0.0           # fp16's smallest values, as they are scaled
    e_out = (p @ v.abs()) * (2 * rel + rho + (m + 40) * U) + floor * m * (v.abs().amax() if m else 0.0)
    e_lse = rel + (m + 8) * U + torch.where(some, lse.abs() * 4 * U, 0.0)
    got, within = {"out": out, "lse": lse[:, 0]}, {"out": e_out, "lse": e_lse[:, 0]}
    if g is None:
        return got, within
    g = torch.where(some, g.double(), 0.0)
    r = rel + e_lse + 8 * U
    dp, delta = g @ v.t(), (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_p = (D + 2) * U * (g.abs() @ v.abs().t())
    e_delta = (g.abs() * (e_out + (rho or U) * out.abs())).sum(-1, keepdim=True) + (D + 2) * U * (g * out).abs().sum(-1, keepdim=True)
    e_ds = p * (e_p + e_delta + (dp.abs() + delta.abs()) * U) + ds.abs() * (r + rho + 4 * U)
    e_ds = e_ds + floor * (ds.abs().amax() if ds.numel() else 0.0)
    got |= {"dq": scale * (ds @ k), "dk": scale * (ds.t() @ q), "dv": p.t() @ g}
    within |= {"dq": scale * (e_ds @ k.abs() + (m + 8) * U * (ds.abs() @ k.abs())),
               "dk": scale * (e_ds.t() @ q.abs() + (n + 8) * U * (ds.abs().t() @ q.abs())),
               "dv": (p * (r + rho + (n + 8) * U)).t() @ g.abs() + floor * (g.abs().sum(0) if n else 0.0)}
    return got, within


def reference(q, k, v, g, parts, causal=True, scale=None):
    """q, k, v, g in (batch, length, heads, dim); parts: (row of the batch, queries, keys) of each sequence, as slices."""
    B, N, H, D = q.shape
    group, scale = H // k.shape[2], scale or D**-0.5
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=DEV)  # noqa: E731
    want = {"out": zeros(q), "lse": torch.full((B, H, N), float("-inf"), dtype=torch.float64, device=DEV)}
    if g is not None:
        want |= {"dq": zeros(q), "dk": zeros(k), "dv": zeros(v)}
    within = {n: torch.zeros_like(t) for n, t in want.items()}
    rho = 0.0 if q.dtype == torch.float32 else ROUND[q.dtype]
    for b, rows, keys in parts:
        for h in range(H):
            got, off = one_head(q[b, rows, h], k[b, keys, h // group], v[b, keys, h // group],
                                None if g is None else g[b, rows, h], causal, scale, rho)
            for a, b_ in ((want, got), (within, off)):
                a["out"][b, rows, h] = b_["out"]
                a["lse"][b, h, rows] = b_["lse"]
                if g is not None:
                    a["dq"][b, rows, h] = b_["dq"]
                    a["dk"][b, keys, h // group] += b_["dk"]
                    a["dv"][b, keys, h // group] += b_["dv"]
    return want, within


def compare(got, want, within):
    for name, t in got.items():
        near(t, want[name], within[name] + torch.zeros_like(want[name]), name)


def inputs(B, N, M, H, Hk, D, dtype, seed, fused=False):
    gen = generator(seed)
    if fused:
        x = randn(gen, (B, N, H + 2 * Hk, D), dtype)
        q, k, v = x.split((H, Hk, Hk), 2)
    else:
        q, k, v = randn(gen, (B, N, H, D), dtype), randn(gen, (B, M, Hk, D), dtype), randn(gen, (B, M, Hk, D), dtype)
    q.mul_(1.5)
    return q, k, v, randn(gen, (B, N, H, D), dtype, 0.1)


def run(q, k, v, g, first=False, **more):
    """All outputs, in (batch, length, heads, dim)."""
    turn = (lambda t: t.transpose(1, 2)) if first else (lambda t: t)
    q, k, v = turn(q), turn(k), turn(v)
    out, lse = mg.attention_lse(q, k, v, heads_first=first, **more)
    assert out.is_contiguous() and same_bits([mg.attention(q, k, v, heads_first=first, **more)], [out])
    got = {"out": out, "lse": lse}
    if g is not None:
        grads = mg.attention_backward(g, q, k, v, out, lse, heads_first=first, **more)
        assert same_bits(mg.attention_backward(g, q, k, v, out, lse, heads_first=first, **more), grads)
        got |= {n: turn(t) for n, t in zip(("dq", "dk", "dv"), grads)}
    return got


def whole(B, N, M):
    return [(b, slice(0, N), slice(0, M)) for b in range(B)]


SHAPES = [(1, 1, 1, 1, 1, 32), (2, 5, 5, 2, 1, 16), (1, 33, 33, 4, 2, 64), (2, 128, 128, 4, 4, 32), (1, 129, 129, 3, 1, 80),
          (1, 200, 200, 6, 2, 128), (1, 31, 97, 2, 2, 96), (1, 97, 31, 2, 1, 64), (1, 300, 300, 1, 1, 127), (2, 65, 64, 5, 5, 1),
          (1, 7, 260, 8, 1, 128), (1, 64, 1, 2, 2, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_batches(dtype, causal):
    for seed, (B, N, M, H, Hk, D) in enumerate(SHAPES):
        case("attention", dtype, "causal" if causal else "full", (B, N, M, H, Hk, D))
        q, k, v, g = inputs(B, N, M, H, Hk, D, DTYPES[dtype], seed, fused=N == M and seed % 2 == 1)
        got = run(q, k, v, g, first=seed % 3 == 0, causal=causal)
        compare(got, *reference(q, k, v, g, whole(B, N, M), causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_longer_sequences(dtype):
    for B, N, H, Hk, D in ((1, 1027, 4, 1, 128), (1, 1500, 2, 2, 64)):
        case("attention", dtype, (B, N, H, Hk, D))
        q, k, v, g = inputs(B, N, N, H, Hk, D, DTYPES[dtype], 40)
        compare(run(q, k, v, g), *reference(q, k, v, g, whole(B, N, N)))


PACKED = [[7], [1, 0, 5], [0, 0], [64, 1, 63, 128, 2], [130, 0, 0, 300, 17], [3] * 90, [1] * 5 + [127, 129, 128]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 3, 4])
def test_packed_sequences(dtype, group):
    """Sequences of any lengths, tokens before the first and behind the last (whose
    values are NaN), offsets of both integer types."""
    for seed, lengths in enumerate(PACKED):
        case("attention, packed", dtype, group, lengths[:8], len(lengths))
        before, after = (0, 0) if seed % 2 else (5, 40)
        at = torch.tensor([before] + lengths).cumsum(0).tolist()
        N, Hk, D = at[-1] + after, 2, 64 if seed % 3 else 48
        q, k, v, g = inputs(1, N, N, group * Hk, Hk, D, DTYPES[dtype], seed, fused=True)
        for t in (q, k, v, g):
            t[:, :before] = t[:, at[-1]:] = float("nan")
        offsets = torch.tensor(at, dtype=torch.int32 if seed % 2 else torch.int64, device=DEV)
        parts = [(0, slice(a, b), slice(a, b)) for a, b in zip(at, at[1:])]
        clean = [t.nan_to_num(0.0) for t in (q, k, v, g)]
        for causal in (True, False):
            got = run(q, k, v, g, first=seed % 2 == 0, offsets=offsets, causal=causal)
            compare(got, *reference(*clean, parts, causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_with_other_keys(dtype):
    """Queries and keys packed each their own way: no keys, no queries, fewer keys than queries."""
    n, m = [3, 0, 140, 20, 1, 6], [9, 4, 70, 0, 300, 6]
    qa, ka = ([0] + torch.tensor(x).cumsum(0).tolist() for x in (n, m))
    q, k, v, g = inputs(1, qa[-1], ka[-1], 4, 2, 64, DTYPES[dtype], 3)
    parts = [(0, slice(a, b), slice(c, d)) for a, b, c, d in zip(qa, qa[1:], ka, ka[1:])]
    more = {"offsets": torch.tensor(qa, device=DEV), "key_offsets": torch.tensor(ka, device=DEV)}
    for causal in (True, False):
        case("attention, packed, other keys", dtype, causal)
        compare(run(q, k, v, g, causal=causal, **more), *reference(q, k, v, g, parts, causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_batches(dtype):
    """Rows and keys beyond their lengths hold NaN and are not read; the result is 0 there."""
    B, N, M = 6, 150, 170
    lengths, keys = [150, 0, 1, 77, 150, 33], [170, 20, 0, 77, 40, 169]
    q, k, v, g = inputs(B, N, M, 4, 2, 64, DTYPES[dtype], 5)
    for b in range(B):
        q[b, lengths[b]:] = g[b, lengths[b]:] = float("nan")
        k[b, keys[b]:] = v[b, keys[b]:] = float("nan")
    more = {"lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV),
            "key_lengths": torch.tensor(keys, dtype=torch.int32, device=DEV)}
    clean = [t.nan_to_num(0.0) for t in (q, k, v, g)]
    parts = [(b, slice(0, lengths[b]), slice(0, keys[b])) for b in range(B)]
    for causal in (True, False):
        case("attention, padded", dtype, causal)
        got = run(q, k, v, g, causal=causal, **more)
        compare(got, *reference(*clean, parts, causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_over_a_cache(dtype):
    """One or a few new tokens over caches filled to different lengths, cut in
    parts where the rows are few; a cache's unfilled part holds NaN."""
    for B, N, M, H, Hk, D in ((1, 1, 3000, 8, 2, 128), (3, 1, 1100, 4, 4, 64), (2, 5, 2049, 6, 2, 96), (1, 2, 70_000, 4, 1, 32),
                              (70, 1, 515, 32, 8, 128), (4, 1, 700, 64, 1, 128)):
        case("attention, cache", dtype, (B, N, M, H, Hk, D))
        filled = [max(N, M - 97 * b) if b % 4 != 3 else (N if b % 8 == 3 else 0) for b in range(B)]
        q, k, v, _ = inputs(B, N, M, H, Hk, D, DTYPES[dtype], 6)
        for b in range(B):
            k[b, filled[b]:] = v[b, filled[b]:] = float("nan")
        lengths = torch.tensor(filled, device=DEV)
        clean = [t.nan_to_num(0.0) for t in (q, k, v)]
        got = run(q, k, v, None, key_lengths=lengths, first=B % 2 == 0)
        compare(got, *reference(*clean, None, [(b, slice(0, N), slice(0, filled[b])) for b in range(B)]))


def test_parts_of_the_keys_joined_by_lse():
    """What lse is for: attention over two parts of the keys, joined."""
    q, k, v, _ = inputs(1, 4, 900, 4, 2, 64, torch.float32, 7)
    whole_out, whole_lse = mg.attention_lse(q, k, v, causal=False)
    parts = [mg.attention_lse(q, k[:, a:b], v[:, a:b], causal=False) for a, b in ((0, 333), (333, 900))]
    lse = torch.stack([x for _, x in parts])
    w = torch.softmax(lse, 0).transpose(-1, -2)[..., None]
    assert torch.allclose(torch.logsumexp(lse, 0), whole_lse, atol=1e-5)
    assert torch.allclose((w * torch.stack([x for x, _ in parts])).sum(0), whole_out, atol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_values(dtype):
    """Scores of some hundreds, where one key has all the weight; gradients so
    small that products with probabilities lie below fp16's smallest value."""
    t = DTYPES[dtype]
    q, k, v, g = inputs(1, 150, 150, 2, 1, 64, t, 8)
    compare(run(q * 12, k * 4, v, g), *reference(q * 12, k * 4, v, g, whole(1, 150, 150)))
    flat = q * 0.01
    for size in (2.0**-12, 2.0**10):
        small = (g * size).to(t)
        got = run(flat, k, v, small, scale=0.25)
        want, within = reference(flat, k, v, small, whole(1, 150, 150), scale=0.25)
        compare(got, want, within)


def test_values_that_are_not_finite():
    """An inf or NaN in one sequence's rows stays in that sequence."""
    q, k, v, g = inputs(3, 70, 70, 2, 1, 64, torch.bfloat16, 9)
    want = run(q, k, v, g)
    for t, bad in ((q, float("inf")), (k, float("nan")), (v, float("inf")), (g, float("nan"))):
        x = {id(a): a.clone() for a in (q, k, v, g)}
        x[id(t)][1, 40, 0, 3] = bad
        got = run(*(x[id(a)] for a in (q, k, v, g)))
        # what the value does not go into: out and lse are not of g, lse and dv = p^T g not of v
        spared = {id(g): ("out", "lse"), id(v): ("lse", "dv")}.get(id(t), ())
        for name in want:
            assert same_bits([got[name][[0, 2]]], [want[name][[0, 2]]])
            finite = bool(got[name][1].isfinite().all())
            assert finite == (name in spared), name


def test_empty_calls():
    for B, N, M in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q, k, v, g = inputs(B, N, M, 4, 2, 32, torch.float32, 10)
        got = run(q, k, v, g)
        assert got["out"].shape == (B, N, 4, 32) and got["dk"].shape == (B, M, 2, 32)
        for name, t in got.items():
            assert not bool(t.any()) if name != "lse" else bool((t == float("-inf")).all())
    q, k, v, g = inputs(1, 9, 9, 2, 2, 32, torch.float32, 11)
    none = torch.tensor([4], device=DEV)                 # offsets of no sequence
    assert not any(bool(t.any()) for n, t in run(q, k, v, g, offsets=none).items() if n != "lse")


def test_offsets_out_of_range_touch_nothing_else():
    """Offsets and lengths beyond the tokens are clamped, decreasing ones give something."""
    gen = generator(12)
    room = randn(gen, (3, 64, 4, 32), torch.float32)
    q = k = v = room[1:2]
    kept = room.clone()
    for bad in ([0, 64, 1000], [-5, 64], [40, 10, 64], [64, 0], [2**31 - 1, -2**31]):
        x = torch.tensor(bad, dtype=torch.int32, device=DEV)
        out, lse = mg.attention_lse(q, k, v, offsets=x)
        mg.attention_backward(out, q, k, v, out, lse, offsets=x)
        torch.cuda.synchronize()
        assert torch.equal(room, kept)
    want = mg.attention(q, k, v)
    assert same_bits([mg.attention(q, k, v, offsets=torch.tensor([-7, 99], device=DEV))], [want])
    for bad in (-3, 10**9):
        mg.attention(q, k, v, key_lengths=torch.tensor([bad], device=DEV))
    assert same_bits([mg.attention(q, k, v, key_lengths=torch.tensor([999], device=DEV))], [want])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_against_differences(dtype):
    """By autograd, against central differences in 64 bits of the formula: steps of
    1e-4 leave 1e-8 of a third derivative and 1e-12 of rounding, beside the bounds
    of the gradients themselves."""
    q, k, v, g = inputs(1, 6, 9, 4, 2, 16, DTYPES[dtype], 13)
    want, within = reference(q, k, v, g, whole(1, 6, 9))
    given = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(mg.attention(*given), given, g)

    def loss(*x):
        x = [t.transpose(1, 2) for t in x]
        x[1:] = [t.repeat_interleave(2, 1) for t in x[1:]]
        s = x[0] @ x[1].transpose(-1, -2) / 4
        s = s.masked_fill(~torch.ones(6, 9, dtype=torch.bool, device=DEV).tril(3), float("-inf"))
        return float(((s.softmax(-1) @ x[2]).transpose(1, 2) * g.double()).sum())

    d = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [t.double() for t in (q, k, v)]
        flat = x[i].contiguous().view(-1)
        for at in range(0, flat.numel(), 29):
            x[i] = flat.index_add(0, torch.tensor([at], device=DEV), torch.tensor([d], dtype=torch.float64, device=DEV)).view_as(x[i])
            up = loss(*x)
            x[i] = flat.index_add(0, torch.tensor([at], device=DEV), torch.tensor([-d], dtype=torch.float64, device=DEV)).view_as(x[i])
            slope = (up - loss(*x)) / (2 * d)
            off = float(within[name].reshape(-1)[at]) + abs(slope) * ROUND[q.dtype] * 1.001 + 1e-7
            assert abs(float(grads[i].reshape(-1)[at]) - slope) <= off, (name, at)


def test_through_autograd():
    q, k, v, g = inputs(2, 40, 40, 4, 2, 64, torch.bfloat16, 14, fused=True)
    want = run(q, k, v, g)
    given = [t.clone().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(mg.attention(*given), given, g)
    assert same_bits(got, [want[n] for n in ("dq", "dk", "dv")])
    # one tensor as keys and values; a gradient that is a broadcast
    kv = k.clone().requires_grad_(True)
    grad, = torch.autograd.grad(mg.attention(q, kv, kv), kv, torch.ones((), dtype=q.dtype, device=DEV).expand(q.shape))
    one = run(q, k, k, torch.ones_like(g))
    assert same_bits([grad], [(one["dk"].float() + one["dv"].float()).to(k.dtype)])
    out = mg.attention(*given)
    given[0].data.view(-1)[0] += 0
    with torch.no_grad():
        given[1].mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(g)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
        mg.attention(forward_ad.make_dual(q, q), k, v)
    with pytest.warns(DeprecationWarning):
        traced = torch.jit.trace(lambda *t: mg.attention(*t), (q, k, v))
    assert same_bits([traced(q * 2, k, v)], [mg.attention(q * 2, k, v)])


def test_strides():
    """Heads and tokens in any order and spacing; a last dimension that is not
    contiguous is copied; broadcast keys."""
    q, k, v, g = inputs(2, 33, 33, 4, 2, 64, torch.float16, 15)
    want = run(q, k, v, g)
    wide = torch.empty((33, 3, 9, 67), dtype=q.dtype, device=DEV)
    spaced = []
    for t in (q, k, v):
        x = wide.clone()[:, 1:, 2:2 + t.shape[2], 1:65].transpose(0, 1)
        spaced.append(x.copy_(t))
    assert all(same_bits([a], [b]) for a, b in zip(run(*spaced, g).values(), want.values()))
    turned = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v, g)]
    assert all(same_bits([a], [b]) for a, b in zip(run(*turned).values(), want.values()))
    shared = [k[:1, :, :1].expand(2, 33, 2, 64), v[:1, :, :1].expand(2, 33, 2, 64)]
    got, plain = run(q, *shared, g), run(q, *(t.contiguous() for t in shared), g)
    assert all(same_bits([got[n]], [plain[n]]) for n in got)


def test_streams_and_graphs():
    """On another stream than the default one; a captured call and its backward
    pass, replayed with new inputs in the same memory."""
    q, k, v, g = inputs(1, 90, 90, 4, 2, 64, torch.bfloat16, 16)
    want = run(q, k, v, g)
    long = inputs(1, 1, 2000, 8, 2, 64, torch.bfloat16, 17)[:3]          # cut in parts
    want_long = mg.attention(*long)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, g)
        got_long = mg.attention(*long)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same_bits([got[n]], [want[n]]) for n in want) and same_bits([got_long], [want_long])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = mg.attention_lse(q, k, v)
        grads = mg.attention_backward(g, q, k, v, out, lse)
        out_long = mg.attention(*long)
    for seed in (18, 19, 20):
        new, new_long = inputs(1, 90, 90, 4, 2, 64, torch.bfloat16, seed), inputs(1, 1, 2000, 8, 2, 64, torch.bfloat16, seed)[:3]
        for a, b in zip((q, k, v, g, *long), (*new, *new_long)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = run(*new)
        assert same_bits([out, lse, *grads], list(want.values())) and same_bits([out_long], [mg.attention(*new_long)])


def test_refusals():
    q, k = torch.ones(2, 5, 4, 32, device=DEV), torch.ones(2, 6, 2, 32, device=DEV)
    ids = torch.tensor([0, 5], device=DEV)
    for bad, what in (((q[0], k, k), "need shapes"), ((q, k, k[:, :5]), "need shapes"), ((q[:1], k, k), "need shapes"),
                      ((q[..., :31], k, k), "need shapes"), ((q[:, :, :3], k, k), "multiple"), ((q[:, :, :0], k, k), "multiple"),
                      ((q[..., :0], k[..., :0], k[..., :0]), "at least one element"),
                      ((q.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5)), "more than 128")):
        with pytest.raises(ValueError, match=what):
            mg.attention(*bad)
    for more, what in (({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"),
                       ({"offsets": ids}, "batch of 1"), ({"key_offsets": ids}, "without offsets"),
                       ({"lengths": ids[:1]}, "2 values"), ({"key_lengths": ids[None]}, "2 values")):
        with pytest.raises(ValueError, match=what):
            mg.attention(q, k, k, **more)
    one, other = q[:1], k[:1]
    for more, what in (({"offsets": ids}, "key_offsets too"), ({"offsets": ids, "key_offsets": ids[:1]}, "2 values"),
                       ({"offsets": ids, "key_offsets": ids, "lengths": ids[:1]}, "not lengths"),
                       ({"offsets": ids[:0], "key_offsets": ids}, "one value")):
        with pytest.raises(ValueError, match=what):
            mg.attention(one, other, other, **more)
    for more in ({"lengths": ids.float()}, {"lengths": ids, "key_lengths": ids.int()}):
        with pytest.raises(TypeError, match="integer|int64"):
            mg.attention(q, k, k, **more)
    with pytest.raises(TypeError, match="dtype"):
        mg.attention(q, k.half(), k)
    with pytest.raises(RuntimeError, match="no CPU"):
        mg.attention(q, k, k, lengths=ids.cpu())
    out, lse = mg.attention_lse(q, k, k)
    for bad, what in (((out[:1], q, k, k, out, lse), "grad_out and out"), ((out, q, k, k, out.transpose(1, 2), lse), "grad_out and out"),
                      ((out, q, k, k, out, lse[0]), "lse"), ((out, q, k, k, out, lse.double()), "lse")):
        with pytest.raises(ValueError, match=what):
            mg.attention_backward(*bad)


def test_one_key_of_any_stride():
    """A single key has no next: its token stride says nothing."""
    q, k, v, g = inputs(2, 3, 1, 4, 2, 32, torch.bfloat16, 24)
    far = [t.as_strided(t.shape, (64, 2**25, 32, 1)) for t in (k, v)]
    got, want = run(q, *far, g), run(q, k, v, g)
    assert all(same_bits([got[n]], [want[n]]) for n in want)


def test_too_many_heads():
    """Heads beyond 32 bits are refused before they are counted in 32."""
    x = torch.ones(1, 1, 1, 8, device=DEV)
    with pytest.raises(ValueError, match="2\\^20 heads"):
        mg.attention(x.expand(1, 1, 2**32 + 1, 8), x, x)
