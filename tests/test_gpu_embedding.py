"""embedding and embedding_grad_ against the formulas in 64 bits.

Bounds, u = 2^-24.  A looked-up value is one product: u relative.  A gradient
of k tokens is a sum of at most k + 8 additions however it is split, one product
by the scale and one sum with the old value, fused: (k + 8) u of |scale| times
the sum of magnitudes, and u of the result."""

from __future__ import annotations

import math

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, near, randn, same_bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
#: tokens, vocabulary, width
SIZES = [(1, 1, 1), (1, 50, 8), (2, 3, 7), (63, 96, 128), (64, 2, 33), (65, 700, 16), (257, 96, 300), (1000, 50, 768),
         (1025, 5000, 40), (3000, 513, 130), (4097, 40_000, 24), (5000, 600, 1030), (9000, 200_000, 8), (20_000, 96, 64),
         (33_000, 1500, 36)]


def draw_ids(kind, T, V, gen):
    if kind == "uniform":
        return torch.randint(0, V, (T,), generator=gen, device=DEV)
    if kind == "same":
        return torch.full((T,), V // 2, device=DEV)
    if kind == "distinct":
        return torch.randperm(max(T, V), generator=gen, device=DEV)[:T] % V
    u = torch.rand(T, generator=gen, device=DEV, dtype=torch.float64)          # frequencies as one over the rank
    return (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)


def reference(ids, grad_out, V, scale, padding, old):
    """The gradient and its bound in 64 bits."""
    g, H = grad_out.double().reshape(-1, grad_out.shape[-1]), grad_out.shape[-1]
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < V)
    if padding is not None:
        ok &= ids != padding
    want, size = (torch.zeros((V, H), dtype=torch.float64, device=DEV) for _ in range(2))
    want.index_add_(0, ids[ok], g[ok] * scale)
    size.index_add_(0, ids[ok], g[ok].abs() * abs(scale))
    k = torch.bincount(ids[ok], minlength=V)[:, None]
    if old is not None:
        want += old.double()
    return want, size * (k + 8) * U + want.abs() * U, k[:, 0] > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "same", "zipf", "distinct"])
def test_lookup_and_gradient(dtype, kind):
    t = DTYPES[dtype]
    for seed, (T, V, H) in enumerate(SIZES):
        case("embedding", dtype, kind, "tokens", T, "vocab", V, "width", H)
        gen = generator(seed)
        ids, weight = draw_ids(kind, T, V, gen), randn(gen, (V, H), t)
        scale = (1.0, -3.5, math.sqrt(H))[seed % 3]
        padding = int(ids[T // 2]) if seed % 2 else None
        out = mg.embedding(ids, weight, scale=scale, padding_idx=padding)
        want = weight.double()[ids] * scale
        near(out, want, want.abs() * 2 * U, "out")
        grad_out = randn(gen, (T, H), t)
        want, within, named = reference(ids, grad_out, V, scale, padding, None)
        grad = torch.full((V, H), float("nan"), dtype=t, device=DEV)
        got = mg.embedding_grad_(grad, ids, grad_out, scale=scale, padding_idx=padding, accumulate=False)
        assert got is grad
        near(grad, want, within, "gradient")
        assert bool((grad[~named] == 0).all())
        again = torch.empty_like(grad)
        assert same_bits([mg.embedding_grad_(again, ids.int(), grad_out, scale=scale, padding_idx=padding, accumulate=False)],
                         [grad])
        old = randn(gen, (V, H), t)
        old[~named] = float("nan")           # rows that no id names are not touched
        grad = old.clone()
        mg.embedding_grad_(grad, ids, grad_out, scale=scale, padding_idx=padding)
        want, within, _ = reference(ids, grad_out, V, scale, padding, old)
        near(grad[named], want[named], within[named], "accumulated")
        assert same_bits([grad[~named]], [old[~named]])


@pytest.mark.parametrize("grad_dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_mixed_types(grad_dtype, out_dtype):
    """A gradient kept in another type than the outputs' (fp32 gradients of a
    bf16 pass, a bf16 gradient of an fp32 one), and lookups into another type."""
    gen = generator(3)
    for T, V, H in ((300, 50, 65), (6000, 2000, 136)):
        ids, weight = draw_ids("zipf", T, V, gen), randn(gen, (V, H), DTYPES[grad_dtype])
        out = mg.embedding(ids, weight, scale=2.5, dtype=DTYPES[out_dtype])
        assert out.dtype == DTYPES[out_dtype]
        want = weight.double()[ids] * 2.5
        near(out, want, want.abs() * 2 * U, "out")
        grad_out = randn(gen, (T, H), DTYPES[out_dtype])
        for accumulate in (False, True):
            old = randn(gen, (V, H), DTYPES[grad_dtype])
            grad = mg.embedding_grad_(old.clone(), ids, grad_out, scale=2.5, accumulate=accumulate)
            want, within, _ = reference(ids, grad_out, V, 2.5, None, old if accumulate else None)
            near(grad, want, within, "gradient")


@pytest.mark.parametrize("T", [70, 6000])
def test_ids_outside_the_rows(T):
    gen, V, H = generator(4), 60, 24
    ids = torch.randint(0, V, (T,), generator=gen, device=DEV)
    bad = torch.zeros(T, dtype=torch.bool, device=DEV)
    bad[::7] = True
    for value in (-1, -100, V, V + 3, 2**31 - 1, -(2**31), 2**40, -(2**62), 2**63 - 1):
        wrong = torch.where(bad, value, ids)
        weight, grad_out = randn(gen, (V, H), torch.float32), randn(gen, (T, H), torch.float32)
        out = mg.embedding(wrong, weight)
        assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], weight[ids[~bad]])
        for accumulate in (False, True):
            a, b = torch.ones((V, H), device=DEV), torch.ones((V, H), device=DEV)
            mg.embedding_grad_(a, wrong, grad_out, accumulate=accumulate)
            want, within, _ = reference(wrong, grad_out, V, 1.0, None, b if accumulate else None)
            near(a, want, within, "gradient")
    every = torch.full((T,), -1, device=DEV)
    grad = torch.ones((V, H), device=DEV)
    assert bool((mg.embedding_grad_(grad, every, grad_out) == 1).all())
    assert bool((mg.embedding_grad_(grad, every, grad_out, accumulate=False) == 0).all())
    zero = torch.zeros(T, dtype=torch.int64, device=DEV)
    assert bool((mg.embedding_grad_(grad.fill_(2), zero, grad_out, padding_idx=0) == 2).all())
    assert bool((mg.embedding_grad_(grad, zero, grad_out, padding_idx=-V, accumulate=False) == 0).all())


@pytest.mark.parametrize("T", [80, 7000])
def test_values_that_are_not_finite_stay_in_their_rows(T):
    gen, V, H = generator(5), 90, 40
    ids = torch.arange(T, device=DEV) % V
    grad_out = randn(gen, (T, H), torch.bfloat16)
    clean = mg.embedding_grad_(torch.empty((V, H), dtype=torch.bfloat16, device=DEV), ids, grad_out, accumulate=False)
    grad_out[3, 5], grad_out[11, 7] = float("nan"), float("inf")
    grad = mg.embedding_grad_(torch.empty_like(clean), ids, grad_out, accumulate=False)
    assert bool(grad[3, 5].isnan()) and bool(grad[11, 7].isposinf())
    grad[3, 5], grad[11, 7] = clean[3, 5], clean[11, 7]
    assert same_bits([grad], [clean])
    # a row of zero gradient that holds NaN is left out by the padding index
    grad_out[ids == 3] = float("nan")
    grad = mg.embedding_grad_(torch.empty_like(clean), ids, grad_out, padding_idx=3, accumulate=False)
    assert bool((grad[3] == 0).all())


def test_shapes_strides_and_autograd():
    gen, V, H = generator(6), 500, 72
    weight = randn(gen, (V, H), torch.float32).requires_grad_(True)
    ids = torch.randint(0, V, (4, 33), generator=gen, device=DEV)
    out = mg.embedding(ids, weight, scale=2.0, padding_idx=7)
    assert out.shape == (4, 33, H)
    grad_out = randn(gen, out.shape, torch.float32)
    out.backward(grad_out)
    want = mg.embedding_grad_(torch.empty((V, H), device=DEV), ids, grad_out, scale=2.0, padding_idx=7, accumulate=False)
    assert torch.equal(weight.grad, want)
    mg.embedding(ids.t(), weight, scale=2.0, padding_idx=7).backward(grad_out.transpose(0, 1))
    near(weight.grad, 2 * want.double(), 64 * U * want.double().abs() + 400 * U, "accumulated by autograd")
    weight.grad = None
    mg.embedding(ids, weight).sum().backward()             # a broadcast gradient
    count = torch.bincount(ids.flatten(), minlength=V).float()
    assert torch.equal(weight.grad, count[:, None].expand(V, H))
    with torch.no_grad():
        assert mg.embedding(ids, weight).grad_fn is None
        assert mg.embedding(ids[0, 0], weight).shape == (H,)
        assert torch.equal(mg.embedding(ids, weight.t().contiguous().t()), weight[ids])
        empty = mg.embedding(ids[:0], weight)
        assert empty.shape == (0, 33, H)
        grad = torch.ones((V, H), device=DEV)
        assert bool((mg.embedding_grad_(grad, ids[:0], empty) == 1).all())
        assert bool((mg.embedding_grad_(grad, ids[:0], empty, accumulate=False) == 0).all())
    # the rows of a gradient arena: a contiguous part of a larger buffer, not 16-byte aligned
    arena = torch.zeros(V * H + 3, device=DEV)
    view = arena[3:].view(V, H)
    mg.embedding_grad_(view, ids, grad_out, scale=2.0, padding_idx=7)
    assert torch.equal(view, want) and bool((arena[:3] == 0).all())


def test_gradient_against_differences():
    """The gradient of the sum of out * g, which is linear: differences of 1."""
    gen, V, H = generator(7), 5, 3
    weight, ids = randn(gen, (V, H), torch.float32), torch.randint(0, V, (20,), generator=gen, device=DEV)
    g = randn(gen, (20, H), torch.float32)
    grad = mg.embedding_grad_(torch.empty_like(weight), ids, g, scale=1.5, accumulate=False)
    want = torch.zeros((V, H), dtype=torch.float64, device=DEV)
    for i in range(V):
        for j in range(H):
            w = weight.double().clone()
            w[i, j] += 1.0
            want[i, j] = ((w[ids] - weight.double()[ids]) * 1.5 * g.double()).sum()
    near(grad, want, torch.full_like(want, 28 * U * 1.5 * float(g.abs().sum())), "gradient")


def test_offsets_beyond_32_bits():
    """A gradient and a weight of more than 2^31 elements, and as many outputs."""
    V, H = 530_000, 4100
    case("embedding", V, H)
    gen = generator(8)
    ids = torch.tensor([V - 1, 5, V - 1, 17, V - 2, 0], device=DEV)
    grad_out = randn(gen, (6, H), torch.bfloat16)
    grad = torch.ones((V, H), dtype=torch.bfloat16, device=DEV)
    mg.embedding_grad_(grad, ids, grad_out)
    rows = torch.tensor([V - 1, V - 2, 17, 5, 0], device=DEV)
    small = torch.tensor([0, 3, 0, 2, 1, 4], device=DEV)
    want, within, _ = reference(small, grad_out, 5, 1.0, None, torch.ones((5, H), device=DEV))
    near(grad[rows], want, within, "accumulated")
    assert bool((grad[::1001][1:] == 1).all())
    out = mg.embedding(ids, grad)
    assert torch.equal(out, grad[ids])
    mg.embedding_grad_(grad, ids, grad_out, accumulate=False)
    want, within, _ = reference(small, grad_out, 5, 1.0, None, None)
    near(grad[rows], want, within, "gradient")
    assert bool((grad[1:5] == 0).all()) and bool((grad[V - 1003:V - 2] == 0).all())
    del grad, out
    ids = torch.arange(530_000, device=DEV) % 64
    out = mg.embedding(ids, randn(gen, (64, H), torch.bfloat16))
    assert torch.equal(out[-64:], out[(530_000 - 64) % 64:][:64])
    out.fill_(1.0)
    grad = mg.embedding_grad_(torch.empty((64, H), device=DEV), ids, out, accumulate=False)
    assert torch.equal(grad[:, 0], torch.bincount(ids, minlength=64).float()) and bool((grad == grad[:, :1]).all())


@pytest.mark.parametrize("T, V", [(100, 50), (6000, 3000), (40_000, 30_000)])
def test_streams_and_graphs(T, V):
    gen, H = generator(9), 96
    ids, grad_out = draw_ids("zipf", T, V, gen), randn(gen, (T, H), torch.bfloat16)
    weight = randn(gen, (V, H), torch.bfloat16)
    total = torch.zeros((V, H), dtype=torch.bfloat16, device=DEV)

    def run(total):
        return (mg.embedding(ids, weight), mg.embedding_grad_(torch.empty_like(weight), ids, grad_out, accumulate=False),
                mg.embedding_grad_(total, ids, grad_out))

    want = run(total.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(total.clone())
    side.synchronize()
    assert same_bits(got, want)
    run(total.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(total)
    for k in range(3):
        ids.copy_((ids * 7 + 1) % V)
        grad_out.mul_(-0.5)
        before = total.clone()
        graph.replay()
        want = run(before)
        torch.cuda.synchronize()
        assert same_bits(got, want), k


def test_refusals():
    w, ids = torch.ones((9, 4), device=DEV), torch.zeros(5, dtype=torch.int64, device=DEV)
    g = torch.ones((5, 4), device=DEV)
    with pytest.raises(TypeError, match="int64 or int32"):
        mg.embedding(ids.float(), w)
    with pytest.raises(ValueError, match="shape"):
        mg.embedding(ids, w[0])
    with pytest.raises(TypeError, match="expected float32"):
        mg.embedding(ids, w.double())
    with pytest.raises(TypeError, match="expected float32"):
        mg.embedding(ids, w, dtype=torch.float64)
    for bad in (9, -10):
        with pytest.raises(ValueError, match="padding_idx"):
            mg.embedding(ids, w, padding_idx=bad)
        with pytest.raises(ValueError, match="padding_idx"):
            mg.embedding_grad_(w, ids, g, padding_idx=bad)
    with pytest.raises(ValueError, match="finite"):
        mg.embedding(ids, w, scale=float("inf"))
    with pytest.raises(ValueError, match="ids' shape"):
        mg.embedding_grad_(w, ids, g[:3])
    with pytest.raises(ValueError, match="contiguous"):
        mg.embedding_grad_(w.t(), ids, g)
    with pytest.raises(TypeError, match="int64 or int32"):
        mg.embedding_grad_(w, ids.float(), g)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mg.embedding(ids.cpu(), w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mg.embedding_grad_(w.cpu(), ids, g)
