"""rms_norm, add_rms_norm and their 8-bit form against the formulas in 64 bits.

Bounds, with u = 2^-24.  y = (h * r) * w: r is rounded once from 64 bits, and
two products follow, 3 u of |y|.  The backward pass's dot product adds at most 64
products a thread and then lanes and waves, under 90 roundings of partial sums of
at most sum |g w h|; the terms that it goes into round a few times each.  Codes are
defined in 32 bits and have to be equal.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from tests._ops import DEV, DTYPES, case, generator, mg, near, randn, same_bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
EPS = 1e-6
SHAPES = [(1, 1), (3, 7), (5, 64), (2, 129), (300, 128), (7, 520), (3, 1000), (4, 2731), (9, 4096), (3, 5003), (2, 9001),
          (2, 16389), (2, 32768)]


def inputs(shape, dtype, seed, fused=False, weight_dtype=None):
    gen, (n, w) = generator(seed), shape
    wide = randn(gen, (n, 2 * w + 3), dtype, 2.0)
    x, res = (wide[:, 1:w + 1], wide[:, w + 2:2 * w + 2]) if fused else (wide[:, :w].contiguous(), wide[:, w:2 * w].contiguous())
    return x, res, randn(gen, (w,), weight_dtype or dtype, 0.2).add_(1.0)


def r_of(h, eps=EPS):
    return 1.0 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + eps)


def check_y(y, h, w, eps=EPS):
    want = h.double() * r_of(h, eps) * w.double()
    near(y, want, want.abs() * 3.1 * U, "y")


def check_backward(dx, dw, gy, gh, h, w, eps=EPS):
    g, t, wt = gy.double(), h.double(), w.double()
    r = r_of(h, eps)
    gw, xhat = g * wt, t * r
    mean = (gw * xhat).mean(-1, keepdim=True)
    size = (gw * xhat).abs().mean(-1, keepdim=True)
    want, add = r * (gw - xhat * mean), 0.0 if gh is None else gh.double()
    within = r * (gw.abs() * 4 + (xhat * mean).abs() * 6 + xhat.abs() * size * 90) * U + (want.abs() + abs(add)) * U
    near(dx, want + add, within, "dx")
    if dw is not None:
        rows = g.shape[0]
        near(dw, (g * xhat).sum(0), (g * xhat).abs().sum(0) * (rows / 256 + 50) * U, "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fused", [False, True])
def test_forward_and_backward(dtype, fused):
    for seed, shape in enumerate(SHAPES):
        case("rms_norm", dtype, shape, "fused" if fused else "")
        t = DTYPES[dtype]
        x, res, w = inputs(shape, t, seed, fused)
        y, h = mg.add_rms_norm(x, res, w)
        assert same_bits([h], [(x.float() + res.float()).to(t)])
        check_y(y, h, w)
        assert same_bits([mg.rms_norm(h, w)], [y])
        gy, gh, _ = inputs(shape, t, seed + 100, fused)
        dx, dw = mg.rms_norm_backward(gy, h, w, grad_h=gh)
        check_backward(dx, dw, gy, gh, h, w)
        dx, none = mg.rms_norm_backward(gy, x, w, want_weight=False)
        check_backward(dx, None, gy, None, x, w)
        assert none is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight", DTYPES)
def test_weights_of_another_type(dtype, weight):
    case("rms_norm", dtype, "weight", weight)
    x, res, w = inputs((11, 333), DTYPES[dtype], 3, weight_dtype=DTYPES[weight])
    y, h = mg.add_rms_norm(x, res, w)
    check_y(y, h, w)
    dx, dw = mg.rms_norm_backward(res, h, w)
    assert dw.dtype == DTYPES[weight]
    check_backward(dx, dw, res, None, h, w)


@pytest.mark.parametrize("dtype, rows, width", [("bf16", 5000, 130), ("f32", 3001, 1028), ("f16", 1500, 8196), ("f32", 700, 12001)])
def test_more_rows_than_work_groups(dtype, rows, width):
    case("rms_norm", dtype, rows, width)
    x, res, w = inputs((rows, width), DTYPES[dtype], 5)
    dx, dw = mg.rms_norm_backward(res, x, w)
    check_backward(dx, dw, res, None, x, w)
    assert same_bits(mg.rms_norm_backward(res, x, w), [dx, dw])


def codes_of(y):
    """(codes, scales) of the format's definition, in numpy's fp32."""
    a = y.cpu().numpy()
    m = np.abs(a).max(-1, keepdims=True)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(m >= np.float32(2.0**-119), np.float32(127) / m, np.float32(0)).astype(np.float32)
    return np.rint(a * inv).astype(np.int8), np.where(m >= np.float32(2.0**-119), m * np.float32(1 / 127), np.float32(0))[:, 0]


def same_codes(rows, y):
    codes, scales = codes_of(y)
    assert np.array_equal(rows.codes.cpu().numpy(), codes) and np.array_equal(rows.scales.cpu().numpy(), scales)
    # the codes between the width and the next row are zeros
    n, w = codes.shape
    whole = rows.codes.as_strided((n, rows.codes.stride(0)), (rows.codes.stride(0), 1))
    assert rows.codes.stride(0) == (w + 15) // 16 * 16 and not bool(whole[:, w:].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes(dtype):
    for seed, shape in enumerate(SHAPES):
        case("rms_norm_int8, int8_rows", dtype, shape)
        x, res, w = inputs(shape, DTYPES[dtype], seed, seed % 2 == 1)
        rows, h = mg.rms_norm_int8(x, w, residual=res)
        assert same_bits([h], [(x.float() + res.float()).to(x.dtype)])
        same_codes(rows, h.float() * r_of(h).float() * w.float())
        rows, h = mg.rms_norm_int8(x, w)
        assert h.data_ptr() == x.data_ptr()
        same_codes(rows, x.float() * r_of(x).float() * w.float())
        same_codes(mg.int8_rows(x), x.float())
    wide = randn(generator(9), (3, 70_001), DTYPES[dtype])       # beyond what the norm takes
    same_codes(mg.int8_rows(wide), wide.float())
    lead = mg.int8_rows(randn(generator(9), (2, 3, 5, 40), DTYPES[dtype]))
    assert lead.codes.shape == (2, 3, 5, 40) and lead.scales.shape == (2, 3, 5)
    assert lead.codes.stride() == (15 * 48, 5 * 48, 48, 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
    """Rows of zeros, of the type's smallest and largest values, with an inf and
    with a NaN; the other rows are as they are alone."""
    t = DTYPES[dtype]
    x = randn(generator(1), (8, 200), t)
    x[1], x[2], x[3] = 0.0, torch.finfo(t).tiny / 4, torch.finfo(t).max
    x[4, 7], x[5, 9] = float("inf"), float("nan")
    w = torch.ones(200, dtype=t, device=DEV)
    y = mg.rms_norm(x, w)
    good = [0, 1, 2, 6, 7]
    check_y(y[good], x[good], w)
    assert bool(y[5].isnan().all()) and bool(y[4, 7].isnan()) and bool((y[4, :7] == 0).all())
    near(y[3], torch.ones(200, dtype=torch.float64, device=DEV), torch.full((200,), 1e-6, dtype=torch.float64, device=DEV), "largest")
    rows, _ = mg.rms_norm_int8(x, w)
    assert bool(rows.scales[[4, 5]].isnan().all()) and not bool(rows.codes[[4, 5]].any()) and float(rows.scales[1]) == 0
    assert not bool(rows.codes[1].any())
    rows = mg.int8_rows(x)
    assert bool(rows.scales[[4, 5]].isnan().all()) and bool(rows.scales[[0, 1, 2, 3, 6, 7]].isfinite().all())
    gy = randn(generator(2), (8, 200), t)
    dx, _ = mg.rms_norm_backward(gy, x, w)
    check_backward(dx[good], None, gy[good], None, x[good], w)
    assert bool(dx[5].isnan().all())
    # without eps a row of zeros has no direction
    assert bool(mg.rms_norm(x[1:2], w, eps=0.0).isnan().all())


def test_gradients_against_differences():
    """d_x and d_weight of sum(gy * y + gh * h) by autograd in 32 bits against
    central differences of the formula in 64: steps of 1e-5 leave 1e-10 of a third
    derivative of some hundreds at most and 1e-11 of rounding, beside 32-bit
    gradients that are 1e-5 near."""
    gen = generator(7)
    x, res, w = (randn(gen, s, torch.float32) for s in ((4, 37), (4, 37), (37,)))
    gy, gh = randn(gen, (4, 37), torch.float32), randn(gen, (4, 37), torch.float32)
    x, res, w = (t.requires_grad_(True) for t in (x, res, w))
    y, h = mg.add_rms_norm(x, res, w)
    got = torch.autograd.grad([y, h], [x, res, w], [gy, gh])
    assert same_bits([got[0]], [got[1]])

    # the differences move h itself, which the 32-bit sum has rounded
    def loss(h64, w64):
        return float((h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + EPS) * w64 * gy.double() + h64 * gh.double()).sum())

    h64, w64, d = h.detach().double(), w.detach().double(), 1e-5
    for i in range(0, 4 * 37, 11):
        e = torch.zeros_like(h64)
        e.view(-1)[i] = d
        want = (loss(h64 + e, w64) - loss(h64 - e, w64)) / (2 * d)
        assert abs(float(got[0].view(-1)[i]) - want) < 1e-5 * (1 + abs(want)), i
    for i in range(37):
        e = torch.zeros_like(w64)
        e[i] = d
        want = (loss(h64, w64 + e) - loss(h64, w64 - e)) / (2 * d)
        assert abs(float(got[2][i]) - want) < 1e-5 * (1 + abs(want)), i


def test_through_autograd():
    """The differentiable calls give the backward pass's bits; outputs that nothing
    uses, weights that ask for nothing, inputs that are one tensor."""
    x, res, w = inputs((6, 300), torch.bfloat16, 8)
    gy, gh, _ = inputs((6, 300), torch.bfloat16, 9)
    h = (x.float() + res.float()).to(x.dtype)
    a, b, c = (t.clone().requires_grad_(True) for t in (x, res, w))
    y, s = mg.add_rms_norm(a, b, c)
    want = mg.rms_norm_backward(gy, h, w, grad_h=gh)
    assert same_bits(torch.autograd.grad([y, s], [a, b, c], [gy, gh], retain_graph=True), [want[0], want[0], want[1]])
    assert same_bits(torch.autograd.grad(s, [a, b], gh, retain_graph=True), [gh, gh])
    assert torch.autograd.grad(s, c, gh, retain_graph=True, allow_unused=True)[0] is None
    want = mg.rms_norm_backward(gy, h, w)
    assert same_bits(torch.autograd.grad(y, [a, b, c], gy), [want[0], want[0], want[1]])
    y, s = mg.add_rms_norm(a, res, w)
    y.backward(gy)
    assert same_bits([a.grad], [want[0]])
    a.grad = None
    y, _ = mg.add_rms_norm(a, a, c)
    y.backward(gy)
    twice = mg.rms_norm_backward(gy, (2 * x.float()).to(x.dtype), w)
    assert same_bits([a.grad, c.grad], [(twice[0].float() * 2).to(x.dtype), twice[1]])
    d = x.clone().requires_grad_(True)
    mg.rms_norm(d, c).backward(gy)
    assert same_bits([d.grad], [mg.rms_norm_backward(gy, x, w)[0]])
    y, s = mg.add_rms_norm(d, res, w)
    s.add_(1)                                       # the stream that the backward pass reads
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(gy)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
        mg.rms_norm(forward_ad.make_dual(x, x), w)
    with pytest.warns(DeprecationWarning):
        traced = torch.jit.trace(lambda *t: mg.add_rms_norm(*t), (x, res, w))
    assert same_bits(traced(gy, gh, w), mg.add_rms_norm(gy, gh, w))


def test_shapes_and_strides():
    gen = generator(10)
    t, w = randn(gen, (3, 5, 4, 96), torch.float16), randn(gen, (96,), torch.float16)
    want = mg.rms_norm(t.reshape(-1, 96), w).view(t.shape)
    for x in (t, t.transpose(0, 1), t[:, ::2], t.expand(2, 3, 5, 4, 96), t[:, :0], t[0, 0, 0]):
        y = mg.rms_norm(x, w)
        assert y.shape == x.shape and y.is_contiguous()
    assert same_bits([mg.rms_norm(t.transpose(0, 1), w)], [want.transpose(0, 1)])
    assert same_bits([mg.rms_norm(t[:, ::2], w)], [want[:, ::2]])
    assert same_bits([mg.rms_norm(t, w[::1].expand(2, 96).t().contiguous().t()[1])], [want])
    dx, dw = mg.rms_norm_backward(t[:, :0], t[:, :0], w)
    assert dx.shape == (3, 0, 4, 96) and not bool(dw.any())
    assert mg.int8_rows(t[:0]).codes.shape == (0, 5, 4, 96)


def test_refusals():
    x, w = torch.ones(3, 8, device=DEV), torch.ones(8, device=DEV)
    for bad, what in (((x, w[:7]), "weight needs shape"), ((x, w[None]), "weight needs shape"),
                      ((torch.ones(2, 0, device=DEV), w), "last dimension"), ((torch.ones((), device=DEV), w), "last dimension"),
                      ((torch.ones(1, 32769, device=DEV), w), "32768")):
        with pytest.raises(ValueError, match=what):
            mg.rms_norm(*bad)
    for bad, what in ((x[:2], "differ in shape"), (x[0], "differ in shape")):
        with pytest.raises(ValueError, match=what):
            mg.add_rms_norm(x, bad, w)
        with pytest.raises(ValueError, match="needs h's shape"):
            mg.rms_norm_backward(bad, x, w)
        with pytest.raises(ValueError, match="needs h's shape"):
            mg.rms_norm_backward(x, x, w, grad_h=bad)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            mg.rms_norm(x, w, eps=eps)
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError, match="dtype"):
            mg.rms_norm(bad, w)
        with pytest.raises(TypeError, match="dtype"):
            mg.add_rms_norm(x, bad, w)
        with pytest.raises(TypeError, match="dtype"):
            mg.int8_rows(bad)
    for f in (lambda: mg.rms_norm(x, w.cpu()), lambda: mg.add_rms_norm(x, x.cpu(), w), lambda: mg.rms_norm_backward(x.cpu(), x, w)):
        with pytest.raises(RuntimeError, match="no CPU"):
            f()
