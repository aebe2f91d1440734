"""qk_norm_rope and its backward pass against the formulas in 64 bits.

Bounds, u = 2^-24.  A head's sum of squares is a chain of at most 16 fused
steps and 6 additions, then a product and a sum with eps: 24 u, so
1 / sqrt(...) is off by 14 u relative.  An output adds two products of three
factors: (|a c| + |b s|) 20 u.  The rotated-back gradient g is off by 2 u of
G = |ga c| + |gb s|; with H = G |w|, xhat off by 15 u and M = mean(H |xhat|),
the mean of h xhat is off by (25 + 28 + 4) u M, so dx by
r (22 u H + 75 u |xhat| M).  A weight's gradient is a sum over all tokens and
heads: every lane adds the heads it takes of its tokens, then come at most 6 +
4 + 16 + 6 additions: (steps + 32 + 20) u of the sum of magnitudes.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, near, randn, same_bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
EPS = 1e-6

#: batch, length, q heads, k heads, dim, rotary
SHAPES = [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 128, 128), (3, 7, 12, 12, 64, 32), (1, 5, 32, 8, 128, 128), (2, 9, 3, 1, 80, 80),
          (1, 4, 6, 2, 96, 48), (2, 2, 2, 1, 256, 256), (1, 3, 2, 2, 512, 512), (2, 5, 5, 3, 33, 10), (1, 6, 7, 1, 200, 100),
          (1, 2, 2, 1, 511, 0), (1, 1, 2, 3, 300, 298), (64, 1, 32, 8, 128, 128), (1, 700, 2, 1, 16, 8)]


def make(shape, dtype, seed, fused=False, weight_dtype=None, heads_first=False):
    B, T, Hq, Hk, D, R = shape
    gen, t = generator(seed), DTYPES[dtype]
    s = {}
    if fused:
        x = randn(gen, (B, T, Hq + 2 * Hk, D + 3), t, 1.5)[..., 1:D + 1]
        s["q"], s["k"] = x[:, :, :Hq], x[:, :, Hq:Hq + Hk]
    else:
        s["q"], s["k"] = randn(gen, (B, T, Hq, D), t, 1.5), randn(gen, (B, T, Hk, D), t, 1.5)
    s["wq"], s["wk"] = (randn(gen, (D,), weight_dtype or t, 0.3) + 1 for _ in range(2))
    s["cos"], s["sin"] = mg.rope_tables(T + 40, R, device=DEV) if R else (torch.empty((T + 40, 0), device=DEV),) * 2
    s["positions"] = torch.randint(0, T + 40, (B, T), generator=gen, device=DEV)
    order = (lambda h: (B, h, T, D)) if heads_first else (lambda h: (B, T, h, D))
    s["gq"], s["gk"] = randn(gen, order(Hq), t, 0.5), randn(gen, order(Hk), t, 0.5)
    return s


def pairs(x, R, inter):
    return (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R])


def joined(a, b, rest, inter):
    return torch.cat((torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1), rest), -1)


def turn(x, c, d, R, inter):
    a, b = pairs(x, R, inter)
    return joined(a * c - b * d, b * c + a * d, x[..., R:], inter)


def spread(x, c, d, R, inter):
    """|a c| + |b s| of each rotated element."""
    a, b = pairs(x.abs(), R, inter)
    return joined(a * c.abs() + b * d.abs(), b * c.abs() + a * d.abs(), x[..., R:].abs(), inter)


def tables(s):
    c, d = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    return c[:, :, None], d[:, :, None]


def forward(x, w, c, d, R, inter, eps=EPS):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return turn(x * r * w, c, d, R, inter), r


def check(s, shape, inter, heads_first, outs, grads):
    B, T, Hq, Hk, D, R = shape
    c, d = tables(s)
    order = (lambda v: v.transpose(1, 2)) if heads_first else (lambda v: v)
    for name, heads, i in (("q", Hq, 0), ("k", Hk, 1)):
        x, w = s[name].double(), s["w" + name].double()
        want, r = forward(x, w, c, d, R, inter)
        near(order(outs[i]), want, spread(x * r * w, c, d, R, inter) * 20 * U, name)
        if grads is None:
            continue
        gin = order(s["g" + name]).double()
        g, G = turn(gin, c, -d, R, inter), spread(gin, c, d, R, inter)
        xhat, h, H = x * r, g * w, G * w.abs()
        M = (H * xhat.abs()).mean(-1, keepdim=True)
        near(grads[i], r * (h - xhat * (h * xhat).mean(-1, keepdim=True)), r * (22 * H + 75 * xhat.abs() * M) * U, "d" + name)
        steps = math.ceil(B * T / 800 + 1) * (Hq + Hk)
        near(grads[2 + i], (g * xhat).sum((0, 1, 2)), (G * xhat.abs()).sum((0, 1, 2)) * (steps + 52) * U, "d weight " + name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads_first", [False, True])
def test_forward_and_backward(dtype, inter, heads_first):
    for seed, shape in enumerate(SHAPES):
        case("qk_norm_rope", dtype, shape, "interleaved" if inter else "", "heads first" if heads_first else "")
        s = make(shape, dtype, seed, fused=seed % 2 == 1, heads_first=heads_first,
                 weight_dtype=torch.float32 if seed % 3 == 0 else None)
        given = (s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
        more = {"interleaved": inter, "heads_first": heads_first}
        outs = mg.qk_norm_rope(*given, **more)
        grads = mg.qk_norm_rope_backward(s["gq"], s["gk"], *given, **more)
        assert grads[2].dtype == s["wq"].dtype and grads[0].shape == s["q"].shape
        check(s, shape, inter, heads_first, outs, grads)


def test_many_tokens():
    shape = (2, 4096, 4, 2, 128, 128)
    s = make(shape, "bf16", 4)
    given = (s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    check(s, shape, False, False, mg.qk_norm_rope(*given), mg.qk_norm_rope_backward(s["gq"], s["gk"], *given))
    shape = (1, 9001, 1, 1, 34, 20)         # single elements, an odd number of tokens
    s = make(shape, "f32", 5)
    given = (s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    check(s, shape, False, False, mg.qk_norm_rope(*given), mg.qk_norm_rope_backward(s["gq"], s["gk"], *given))


@pytest.mark.parametrize("inter", [False, True])
def test_gradients_against_differences(inter):
    """Central differences, in 64 bits, of the sum of out * g: steps of 1e-5 leave
    under 1e-8 of the third derivative (x is of size 1 over dim elements) and
    1e-10 of rounding."""
    shape = (1, 2, 2, 1, 12, 8)
    s = make(shape, "f32", 3)
    dq, _, dwq, _ = mg.qk_norm_rope_backward(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                             s["positions"], interleaved=inter)
    c, d = tables(s)
    x, w, g, h = s["q"].double(), s["wq"].double(), s["gq"].double(), 1e-5

    def f(x, w):
        return float((forward(x, w, c, d, 8, inter)[0] * g).sum())

    def differences(v, of):
        out = torch.zeros_like(v)
        for i in range(v.numel()):
            step = torch.zeros_like(v)
            step.view(-1)[i] = h
            out.view(-1)[i] = (of(v + step) - of(v - step)) / (2 * h)
        return out

    want = differences(x, lambda v: f(v, w))
    near(dq, want, torch.full_like(want, 1e-7) + 400 * U * want.abs().amax(), "dq")
    want = differences(w, lambda v: f(x, v))
    near(dwq, want, torch.full_like(want, 1e-7) + 400 * U * want.abs().amax(), "dw")


def test_positions():
    shape = (3, 6, 2, 1, 64, 64)
    s = make(shape, "f32", 6)
    run = lambda p: mg.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], p)  # noqa: E731
    want = run(s["positions"])
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    assert same(run(s["positions"].int()), want)
    wide = torch.zeros((3, 12), dtype=torch.int64, device=DEV)
    wide[:, ::2] = s["positions"]
    assert same(run(wide[:, ::2]), want)
    line = torch.arange(6, device=DEV)
    assert same(run(None), run(line)) and same(run(line), run(line.expand(3, 6))) and same(run(line[None]), run(line))
    off = s["positions"].clone()
    off[1, 2], off[2, 0] = -1, 46            # outside the table
    got = run(off)
    for g, w in zip(got, want):
        bad = torch.zeros((3, 6), dtype=torch.bool, device=DEV)
        bad[1, 2] = bad[2, 0] = True
        assert bool(g[bad].isnan().all()) and torch.equal(g[~bad], w[~bad])


def test_special_values():
    shape = (1, 4, 2, 1, 128, 128)
    for dtype in DTYPES:
        s = make(shape, dtype, 7)
        s["q"][0, 0] = 0.0
        s["q"][0, 1, 0, 5] = float("nan")
        s["q"][0, 2, 1, 9] = float("inf")
        q, k = mg.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
        assert bool((q[0, 0] == 0).all()) and bool(q[0, 1, 0].isnan().all()) and bool(q[0, 1, 1].isfinite().all())
        assert bool(q[0, 3].isfinite().all()) and bool(k.isfinite().all())
        # an infinite element has 1/sqrt 0: the others go to 0 and it to NaN, with its pair
        assert int(q[0, 2, 1].isnan().sum()) == 2 and bool((q[0, 2, 1].nan_to_num() == 0).all())
        dq, dk, dwq, dwk = mg.qk_norm_rope_backward(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                                    s["positions"])
        assert bool(dq[0, 0].isfinite().all()) and bool(dq[0, 1, 0].isnan().all()) and bool(dq[0, 1, 1].isfinite().all())
        assert bool(dk.isfinite().all()) and bool(dwk.isfinite().all()) and bool(dwq.isnan().any())
    # an empty batch, and one of no tokens
    s = make((2, 3, 2, 1, 64, 64), "bf16", 8)
    for cut in (lambda t: t[:0], lambda t: t[:, :0]):
        q, k = cut(s["q"]), cut(s["k"])
        assert mg.qk_norm_rope(q, k, s["wq"], s["wk"], s["cos"], s["sin"])[0].shape == q.shape
        grads = mg.qk_norm_rope_backward(q, k, q, k, s["wq"], s["wk"], s["cos"], s["sin"])
        assert grads[0].shape == q.shape and bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())


def test_strides_and_autograd():
    shape = (2, 5, 4, 2, 64, 64)
    B, T, Hq, Hk, D, R = shape
    s = make(shape, "bf16", 9)
    fixed = (s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    want = mg.qk_norm_rope(s["q"], s["k"], *fixed)
    grads = mg.qk_norm_rope_backward(s["gq"], s["gk"], s["q"], s["k"], *fixed)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    heads_first = lambda v: v.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    last = lambda v: v.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
    for view in (heads_first, last):
        assert same(mg.qk_norm_rope(view(s["q"]), view(s["k"]), *fixed), want)
        got = mg.qk_norm_rope_backward(view(s["gq"]), view(s["gk"]), view(s["q"]), s["k"], *fixed)
        assert same(got, grads)
    first = mg.qk_norm_rope(s["q"], s["k"], *fixed, heads_first=True)
    assert same([v.transpose(1, 2) for v in first], want) and first[0].is_contiguous()
    one = s["gq"][:, :, :1].expand_as(s["gq"])           # a gradient that all heads share
    assert same(mg.qk_norm_rope_backward(one, s["gk"], s["q"], s["k"], *fixed),
                mg.qk_norm_rope_backward(one.contiguous(), s["gk"], s["q"], s["k"], *fixed))
    qkv = torch.cat((s["q"], s["k"], s["k"]), 2).requires_grad_(True)
    wq, wk = s["wq"].clone().requires_grad_(True), s["wk"].clone().requires_grad_(True)
    q, k = mg.qk_norm_rope(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], wq, wk, *fixed[2:])
    ((q.float() * s["gq"].float()).sum() + (k.float() * s["gk"].float()).sum()).backward()
    assert torch.equal(qkv.grad[:, :, :Hq], grads[0]) and torch.equal(qkv.grad[:, :, Hq:Hq + Hk], grads[1])
    assert bool((qkv.grad[:, :, Hq + Hk:] == 0).all()) and torch.equal(wq.grad, grads[2]) and torch.equal(wk.grad, grads[3])


def test_offsets_beyond_32_bits():
    """Heads more than 2^31 elements into their tensor."""
    B, T, H, D = 1, 70_000, 250, 128
    case("qk_norm_rope", B, T, H, D)
    q = torch.ones((B, T, H, D), dtype=torch.bfloat16, device=DEV)
    s = make((1, 3, H, 2, D, D), "bf16", 3)
    q[:, -3:] = s["q"]
    k = torch.ones((B, T, 2, D), dtype=torch.bfloat16, device=DEV)
    p = torch.zeros(T, dtype=torch.int64, device=DEV)
    p[-3:] = s["positions"][0]
    got, _ = mg.qk_norm_rope(q, k, s["wq"], s["wk"], s["cos"], s["sin"], p)
    want, _ = mg.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    assert torch.equal(got[:, -3:], want) and torch.equal(got[:, 1], got[:, -4])
    got.zero_()
    got[:, -3:] = s["gq"]
    d = mg.qk_norm_rope_backward(got, k, q, k, s["wq"], s["wk"], s["cos"], s["sin"], p)
    want = mg.qk_norm_rope_backward(s["gq"], s["k"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    assert torch.equal(d[0][:, -3:], want[0]) and bool((d[0][:, :-3:500] == 0).all())


def test_streams_and_graphs():
    s = make((2, 33, 6, 2, 80, 80), "f16", 4)
    given = (s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"])
    run = lambda: (*mg.qk_norm_rope(*given), *mg.qk_norm_rope_backward(s["gq"], s["gk"], *given))  # noqa: E731
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for k in range(3):
        s["q"].mul_(-0.7)
        s["positions"].add_(1)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert same_bits(got, want), k      # positions that leave the table give NaN


def test_refusals():
    s = make((2, 3, 4, 2, 64, 64), "f32", 1)
    q, k, wq, wk, cos, sin, p = (s[n] for n in ("q", "k", "wq", "wk", "cos", "sin", "positions"))
    run = mg.qk_norm_rope
    for bad in (k[:1], k[:, :2], k[..., :32], k[0]):
        with pytest.raises(ValueError, match="differ in heads only"):
            run(q, bad, wq, wk, cos, sin)
    with pytest.raises(TypeError, match="beside"):
        run(q, k.half(), wq, wk, cos, sin)
    with pytest.raises(TypeError, match="beside"):
        run(q, k, wq, wk.half(), cos, sin)
    with pytest.raises(TypeError, match="expected float32"):
        run(q.double(), k.double(), wq, wk, cos, sin)
    with pytest.raises(ValueError, match="need shape"):
        run(q, k, wq[:5], wk, cos, sin)
    with pytest.raises(ValueError, match="rotary at most dim"):
        run(q[..., :32].contiguous(), k[..., :32].contiguous(), wq[:32], wk[:32], cos, sin)
    with pytest.raises(TypeError, match="float32"):
        run(q, k, wq, wk, cos.double(), sin.double())
    with pytest.raises(TypeError, match="int64 or int32"):
        run(q, k, wq, wk, cos, sin, p.float())
    for bad in (p[:, :2], p[:1, :2], p[0, :2], p[None]):
        with pytest.raises(ValueError, match="positions need shape"):
            run(q, k, wq, wk, cos, sin, bad)
    with pytest.raises(ValueError, match="eps"):
        run(q, k, wq, wk, cos, sin, eps=-1.0)
    wide = torch.ones((1, 1, 1, 514), device=DEV)
    with pytest.raises(ValueError, match="more than 512"):
        run(wide, wide, wide[0, 0, 0], wide[0, 0, 0], cos, sin)
    with pytest.raises(ValueError, match="outputs' shapes"):
        mg.qk_norm_rope_backward(s["gq"].transpose(1, 2), s["gk"], q, k, wq, wk, cos, sin)
    for bad in (3, 0):
        with pytest.raises(ValueError, match="rotary must be even"):
            mg.rope_tables(4, bad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        run(q.cpu(), k.cpu(), wq, wk, cos, sin)
    with pytest.raises(RuntimeError, match="no CPU path"):
        run(q, k, wq, wk, cos.cpu(), sin.cpu())
