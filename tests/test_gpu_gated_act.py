"""gated_act: the MLP's activation, its 8-bit checkpoint and its backward pass
against the formulas in 64 bits.

Bounds, per element, from the 32-bit arithmetic: the logistic function s of v
comes from an exponential whose argument v * log2(e) is off by 2 roundings, so
s is off by (|v| + 8) 2^-23 relative at most (4 more roundings and 1 ulp each
of the hardware's exponential and reciprocal, doubled); products of it add
roundings that the 8 covers.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests._ops import DEV, DTYPES, EPS32, case, generator, mg, near, randn

pytestmark = pytest.mark.gpu
GROUP = 128
INNER, CUBIC = math.sqrt(2 / math.pi), 0.044715
SHAPES = [(1, 1), (1, 127), (3, 128), (5, 129), (7, 300), (2, 2731), (33, 512), (4, 4100), (1, 12288), (1000, 65)]


def curve(x, act):
    """(act(x), act'(x), error bound of each) in 64 bits."""
    if act == "silu":
        v, dv = x, torch.ones_like(x)
    else:
        v, dv = 2 * INNER * (x + CUBIC * x**3), 2 * INNER * (1 + 3 * CUBIC * x**2)
    s, t = torch.sigmoid(v), torch.sigmoid(v) * torch.sigmoid(-v)
    a, d = x * s, s + x * t * dv
    err = (v.abs() + 8) * EPS32
    return a, d, a.abs() * err, (s + (x * t * dv).abs()) * err


def checkpoint(x: torch.Tensor):
    """(codes, scales) of the format's definition, in numpy's fp32."""
    a = x.float().cpu().numpy()
    n, h = a.shape
    a = np.pad(a, ((0, 0), (0, -h % GROUP))).reshape(n, -1, GROUP)
    m = np.abs(a).max(-1)
    inv = np.where(m >= 2.0**-119, np.float32(127) / np.maximum(m, np.float32(2.0**-119)), np.float32(0))
    codes = np.rint(a * inv[..., None].astype(np.float32)).astype(np.int8)
    scales = np.where(m >= 2.0**-119, m * np.float32(1 / 127), np.float32(0)).astype(np.float32)
    return codes.reshape(n, -1), scales


def held(saved, i, width):
    codes, scales = saved.codes[i].double(), saved.scales[i].double()
    return (codes.view(*scales.shape, GROUP) * scales[..., None]).flatten(-2)[:, :width]


def inputs(shape, dtype, gated, fused, seed):
    gen = generator(seed)
    n, h = shape
    if fused:
        x = randn(gen, (n, (2 if gated else 1) * h + 3), dtype, 2.0)
        return x[:, 1:h + 1], (x[:, h + 1:2 * h + 1] if gated else None)
    return randn(gen, shape, dtype, 2.0), (randn(gen, shape, dtype) if gated else None)


def check_forward(y, gate, up, act):
    a, _, err, _ = curve(gate.double(), act)
    u = 1.0 if up is None else up.double()
    near(y, a * u, err * (abs(u) if up is None else u.abs()), "y")


def check_backward(grad_out, saved, act, d_gate, d_up, y, width):
    g = held(saved, 0, width)
    a, d, err_a, err_d = curve(g, act)
    dy = grad_out.double()
    u = held(saved, 1, width) if d_up is not None else torch.ones_like(g)
    # the products by dy and u round twice, a relative EPS32 together
    near(d_gate, dy * u * d, (dy * u).abs() * (err_d + d.abs() * EPS32), "d_gate")
    if d_up is not None:
        near(d_up, dy * a, dy.abs() * (err_a + a.abs() * EPS32), "d_up")
    if y is not None:
        near(y, a * u, u.abs() * (err_a + a.abs() * EPS32), "y again")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [True, False])
def test_forward_and_backward(dtype, act, gated):
    for seed, shape in enumerate(SHAPES):
        for fused in (False, True):
            case("gated_act", dtype, act, "gated" if gated else "plain", shape, "fused" if fused else "")
            gate, up = inputs(shape, DTYPES[dtype], gated, fused, seed)
            y, saved = mg.gated_act_pack(gate, up, act=act)
            check_forward(y, gate, up, act)
            assert torch.equal(mg.gated_act(gate, up, act=act), y)
            for i, x in enumerate([gate] if up is None else [gate, up]):
                codes, scales = checkpoint(x)
                assert np.array_equal(saved.codes[i].cpu().numpy(), codes)
                assert np.array_equal(saved.scales[i].cpu().numpy(), scales)
            grad_out = randn(generator(seed + 100), shape, DTYPES[dtype], 0.5)
            d_gate, d_up, again = mg.gated_act_backward(grad_out, saved)
            check_backward(grad_out, saved, act, d_gate, d_up, again, shape[1])
            assert (d_up is None) == (not gated)
            assert mg.gated_act_backward(grad_out, saved, want_y=False)[2] is None


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """d_gate and d_up against central differences, in 64 bits, of the forward
    formula at the checkpoint's values: steps of 1e-4 leave 1e-8 of the third
    derivative (under 2 for both functions) and 1e-12 of rounding."""
    gate, up = inputs((9, 260), torch.float32, True, False, 5)
    grad_out = randn(generator(6), (9, 260), torch.float32)
    _, saved = mg.gated_act_pack(gate, up, act=act)
    d_gate, d_up, _ = mg.gated_act_backward(grad_out, saved)
    g, u, dy, h = held(saved, 0, 260), held(saved, 1, 260), grad_out.double(), 1e-4
    f = lambda x: curve(x, act)[0]  # noqa: E731
    want = dy * u * (f(g + h) - f(g - h)) / (2 * h)
    bound = (dy * u).abs() * (2e-8 + 30 * EPS32)
    near(d_gate, want, bound, "d_gate")
    near(d_up, dy * f(g), dy.abs() * (g.abs() + 1) * 30 * EPS32, "d_up")


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
    """Zeros, tiny values, the type's largest and its infinities and NaN: a
    group with a value that is not finite has NaN gradients, the groups beside
    it have theirs."""
    t = DTYPES[dtype]
    x = randn(generator(1), (2, 6 * GROUP), t)
    x[:, :GROUP] = 0.0
    x[:, GROUP:2 * GROUP] = torch.finfo(t).tiny * 2.0**-2
    x[:, 3 * GROUP] = float("inf")
    x[:, 4 * GROUP + 5] = float("nan")
    x[0, 5 * GROUP] = torch.finfo(t).max
    x[0, 5 * GROUP + 1] = -torch.finfo(t).max
    y, saved = mg.gated_act_pack(x, act="silu")
    finite = torch.isfinite(x)
    a, _, err, _ = curve(torch.where(finite, x.double(), 0.0), "silu")
    near(y[finite], a[finite], err[finite], "y")
    assert bool(y[:, 3 * GROUP].isposinf().all()) and bool(y[:, 4 * GROUP + 5].isnan().all())
    scales = saved.scales[0]
    assert bool(scales[:, [3, 4]].isnan().all()) and bool(scales[:, [0, 2, 5]].isfinite().all())
    codes, want = checkpoint(torch.where(finite, x, torch.zeros_like(x)))
    ok = [0, 1, 2, 5]
    assert np.array_equal(scales[:, ok].cpu().numpy(), want[:, ok])
    if dtype != "f16":        # fp16's smallest values are far above 2^-119
        assert float(scales[0, 1]) == 0.0
    d_gate, _, again = mg.gated_act_backward(torch.ones_like(x), saved)
    d = d_gate.view(2, 6, GROUP)
    assert bool(d[:, [3, 4]].isnan().all()) and bool(d[:, ok].isfinite().all())
    assert bool((d[:, 0] == 0.5).all()) and bool((again.view(2, 6, GROUP)[:, 0] == 0).all())
    x = torch.tensor([[-3e38, 3e38, -1e20, 1e20, -200.0, 200.0]], device=DEV) if dtype == "f32" else \
        torch.tensor([[-6e4, 6e4, -200.0, 200.0]], device=DEV, dtype=t)
    for act in ("silu", "gelu_tanh"):
        y = mg.gated_act(x, act=act)
        assert torch.equal(y, torch.where(x > 0, x, torch.zeros_like(x)))


def test_shapes_and_strides():
    gen = generator(3)
    x = randn(gen, (3, 5, 4, 200), torch.bfloat16)
    up = randn(gen, (3, 5, 4, 200), torch.bfloat16)
    want = mg.gated_act(x, up)
    assert want.shape == x.shape
    # rows that are not evenly spaced, and a last dimension that is not contiguous, are copied
    for view in (lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2),
                 lambda v: torch.cat((v, v), 1)[:, :5]):
        a, b = view(x), view(up)
        assert not a.is_contiguous()
        assert torch.equal(mg.gated_act(a, b), want)
    assert torch.equal(mg.gated_act(x[0, 0, 0], up[0, 0, 0]), want[0, 0, 0])
    one = x[:1, :, :1].expand(3, 5, 4, 200)
    assert torch.equal(mg.gated_act(one, up), mg.gated_act(one.contiguous(), up))
    y, saved = mg.gated_act_pack(x[:0], up[:0])
    assert y.shape == (0, 5, 4, 200)
    d_gate, d_up, again = mg.gated_act_backward(y, saved)
    assert d_gate.shape == d_up.shape == again.shape == (0, 5, 4, 200)


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are those of a small call on them."""
    n, h = (1 << 18) + 5, 8200
    case("gated_act", n, h)
    x = torch.empty((n, h), dtype=torch.bfloat16, device=DEV).fill_(0.25)
    x[-7:] = randn(generator(2), (7, h), torch.bfloat16)
    y, saved = mg.gated_act_pack(x)
    small, kept = mg.gated_act_pack(x[-7:].clone())
    assert torch.equal(y[-7:], small) and torch.equal(saved.codes[:, -7:], kept.codes)
    assert torch.equal(saved.scales[:, -7:], kept.scales)
    assert bool((y[:-7:4096] == y[0, 0]).all())
    d = mg.gated_act_backward(y, saved, want_y=False)[0]
    assert torch.equal(d[-7:], mg.gated_act_backward(small, kept)[0])


def test_autograd_keeps_the_checkpoint_only():
    gen = generator(8)
    gate, up = (randn(gen, (64, 1024), torch.bfloat16).requires_grad_(True) for _ in range(2))
    y = mg.gated_act(gate, up)
    kept = sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors)
    assert kept == 2 * 64 * (1024 + 4 * 1024 // GROUP)
    dy = randn(gen, y.shape, torch.bfloat16)
    y.backward(dy)
    _, saved = mg.gated_act_pack(gate.detach(), up.detach())
    d_gate, d_up, _ = mg.gated_act_backward(dy, saved)
    assert torch.equal(gate.grad, d_gate) and torch.equal(up.grad, d_up)
    with torch.no_grad():
        assert mg.gated_act(gate, up).grad_fn is None
    gate.grad = None
    mg.gated_act(gate, act="gelu_tanh").sum().backward()       # a broadcast gradient
    assert gate.grad.shape == gate.shape


def test_streams_and_graphs():
    gate, up = inputs((65, 777), torch.float16, True, True, 4)
    grad_out = randn(generator(9), (65, 777), torch.float16)
    y, saved = mg.gated_act_pack(gate, up)
    want = (y, *mg.gated_act_backward(grad_out, saved))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, saved = mg.gated_act_pack(gate, up)
        got = (y, *mg.gated_act_backward(grad_out, saved))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, saved = mg.gated_act_pack(gate, up)
        got = (y, *mg.gated_act_backward(grad_out, saved))
    for k in range(3):
        gate.mul_(-1.0)
        graph.replay()
        y, kept = mg.gated_act_pack(gate, up)
        want = (y, *mg.gated_act_backward(grad_out, kept))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_refusals():
    x = torch.ones((4, 256), device=DEV)
    y, saved = mg.gated_act_pack(x, x)
    with pytest.raises(ValueError, match="unknown activation"):
        mg.gated_act(x, act="relu")
    with pytest.raises(ValueError, match="differ in shape"):
        mg.gated_act(x, x[:3])
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        mg.gated_act(x.double())
    with pytest.raises(TypeError, match="beside"):
        mg.gated_act(x, x.half())
    with pytest.raises(RuntimeError, match="no CPU path"):
        mg.gated_act(x.cpu())
    with pytest.raises(RuntimeError, match="no CPU path"):
        mg.gated_act(x, x.cpu())
    with pytest.raises(ValueError, match="last dimension"):
        mg.gated_act(x[:, :0])
    with pytest.raises(ValueError, match="checkpoint is not one"):
        mg.gated_act_backward(y[:3], saved)
    with pytest.raises(ValueError, match="checkpoint is not one"):
        mg.gated_act_backward(y, saved._replace(scales=saved.scales.half()))
