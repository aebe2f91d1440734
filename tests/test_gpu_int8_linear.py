"""int8_linear against sums of integers and the formula in 64 bits.

The sum of products is exact; what follows rounds it to 32 bits, multiplies by a
product of scales (two roundings) and adds the bias (one): 3 u of the product's
magnitude and 1 u of the result's, u = 2^-24.
"""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, near, randn, same_bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
#: rows, width, channels: one of each, no multiples of anything, each form's edges, a long contraction
SHAPES = [(1, 1, 1), (1, 768, 2304), (3, 5, 7), (31, 127, 33), (32, 128, 32), (33, 129, 31), (64, 1000, 100), (65, 1001, 63),
          (66, 64, 64), (200, 2731, 321), (129, 4096, 130), (7, 131_071, 5), (70, 20_000, 66), (4133, 130, 4101), (4096, 96, 4096)]


def codes(gen, rows, width, low=-127):
    c = torch.randint(low, 128, (rows, width), generator=gen, device=DEV, dtype=torch.int8)
    return c, torch.rand(rows, generator=gen, device=DEV) * 0.02 + 1e-3


def check(y, x, w, bias, part=slice(None)):
    """Rows `part` of y; the sums in 64-bit floats, which hold them exactly."""
    total = x.codes[part].double() @ w.codes.double().t().contiguous()
    want = total * x.scales[part].double()[:, None] * w.scales.double()
    within = want.abs() * 3.1 * U
    if bias is not None:
        want = want + bias.double()
        within = within + want.abs() * 1.1 * U
    near(y[part], want, within, "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [None, *DTYPES])
def test_products(dtype, bias):
    for seed, (M, K, N) in enumerate(SHAPES):
        case("int8_linear", dtype, "bias", bias, (M, K, N))
        gen = generator(seed)
        x, w = mg.Int8Rows(*codes(gen, M, K)), mg.Int8Rows(*codes(gen, N, K))
        b = None if bias is None else randn(gen, (N,), DTYPES[bias], 3.0)
        y = mg.int8_linear(x, w, b, dtype=DTYPES[dtype])
        assert y.shape == (M, N) and y.dtype == DTYPES[dtype] and y.is_contiguous()
        check(y, x, w, b)


@pytest.mark.parametrize("M, K, N", [(40, 131_071, 40), (300, 70_001, 70), (2100, 131_071, 8200)])
def test_largest_sums(M, K, N):
    """All codes -128: sums up to 131,071 * 2^14, just below 2^31."""
    case("int8_linear", "largest", M, K, N)
    one = torch.ones((), device=DEV)
    x, w = (mg.Int8Rows(torch.full((n, K), -128, dtype=torch.int8, device=DEV), one.expand(n)) for n in (M, N))
    y = mg.int8_linear(x, w, dtype=torch.float32)
    assert float(y.min()) == float(y.max()) == float(torch.tensor(K * 2.0**14, dtype=torch.float32))


def test_rows_apart_and_as_the_norm_leaves_them():
    gen = generator(3)
    x, w = mg.Int8Rows(*codes(gen, 90, 203)), mg.Int8Rows(*codes(gen, 77, 203))
    want = mg.int8_linear(x, w)
    for step, start in ((1, 0), (208, 0), (211, 3), (203, 1)):
        room = torch.full((200 * max(step, 203) + 8,), 99, dtype=torch.int8, device=DEV)
        if step == 1:
            spaced = x.codes[:, None].expand(90, 1, 203)
            got = mg.int8_linear(mg.Int8Rows(spaced, x.scales[:, None]), w)[:, 0]
        else:
            a = room.as_strided((90, 203), (step, 1), start)
            a.copy_(x.codes)
            b = room.clone().as_strided((77, 203), (step, 1), start)
            b.copy_(w.codes)
            got = mg.int8_linear(mg.Int8Rows(a, x.scales), mg.Int8Rows(b, w.scales))
        assert same_bits([got], [want])
    assert same_bits([mg.int8_linear(mg.Int8Rows(x.codes.t().contiguous().t(), x.scales), w)], [want])
    three = mg.Int8Rows(x.codes.view(9, 10, 203), x.scales.view(9, 10))
    assert same_bits([mg.int8_linear(three, w)], [want.view(9, 10, 77)])
    same = mg.Int8Rows(x.codes[:1].expand(90, 203), x.scales[:1].expand(90))       # one row again and again
    assert same_bits([mg.int8_linear(same, w)], [want[:1].expand(90, 77)])
    half = mg.Int8Rows(x.codes[::2], x.scales[::2])
    assert same_bits([mg.int8_linear(half, w)], [want[::2]])
    for empty in (mg.Int8Rows(x.codes[:0], x.scales[:0]),):
        assert mg.int8_linear(empty, w).shape == (0, 77) and mg.int8_linear(x, mg.Int8Rows(w.codes[:0], w.scales[:0])).shape == (90, 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_gives_the_same_bits_in_any_batch(dtype):
    """The sums are integers, so every form's results are the same."""
    gen = generator(4)
    x, w = mg.Int8Rows(*codes(gen, 4200, 389)), mg.Int8Rows(*codes(gen, 4133, 389))
    want = mg.int8_linear(x, w, dtype=DTYPES[dtype])
    check(want, x, w, None, slice(4190, 4200))
    for n in (1, 33, 64, 65, 700):
        case("int8_linear", dtype, "rows", n)
        assert same_bits([mg.int8_linear(mg.Int8Rows(x.codes[:n], x.scales[:n]), w, dtype=DTYPES[dtype])], [want[:n]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_a_layer_in_8_bits(dtype, rows):
    """The norm's rows through a product: near the layer in 64 bits, whose inputs
    and weights round to 8 bits (half a code of the row's largest each)."""
    t, gen = DTYPES[dtype], generator(5)
    x, res, norm = randn(gen, (rows, 640), t), randn(gen, (rows, 640), t, 2.0), randn(gen, (640,), t, 0.1).add_(1.0)
    weight = randn(gen, (200, 640), t, 0.05)
    w = mg.int8_rows(weight)
    a, h = mg.rms_norm_int8(x, norm, residual=res)
    y = mg.int8_linear(a, w, dtype=t)
    check(y, a, w, None)
    f = h.double()
    row = f / torch.sqrt(f.square().mean(-1, keepdim=True) + 1e-6) * norm.double()
    half_x, half_w = row.abs().amax(-1, keepdim=True) / 254, weight.double().abs().amax(-1, keepdim=True) / 254
    off = half_x * weight.double().abs().sum(-1) + row.abs().sum(-1, keepdim=True) * half_w.t() + 640 * half_x * half_w.t()
    near(y, row @ weight.double().t().contiguous(), off * 1.001 + 1e-6, "layer")


def test_scales_that_are_not_finite():
    gen = generator(6)
    for n in (5, 100):
        x, w = mg.Int8Rows(*codes(gen, n, 64)), mg.Int8Rows(*codes(gen, 40, 64))
        want = mg.int8_linear(x, w)
        x.scales[2], w.scales[7] = float("nan"), float("nan")
        y = mg.int8_linear(x, w)
        assert bool(y[2].isnan().all()) and bool(y[:, 7].isnan().all())
        keep_r, keep_c = [i for i in range(n) if i != 2], [i for i in range(40) if i != 7]
        assert same_bits([y[keep_r][:, keep_c]], [want[keep_r][:, keep_c]])


def test_streams_and_graphs():
    gen = generator(7)
    w = mg.int8_rows(randn(gen, (300, 256), torch.bfloat16))
    x, norm = randn(gen, (100, 256), torch.bfloat16), randn(gen, (256,), torch.bfloat16)
    layer = lambda t: mg.int8_linear(mg.rms_norm_int8(t, norm)[0], w)  # noqa: E731
    want = layer(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    assert same_bits([got], [want])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for _ in range(3):
        x.copy_(randn(gen, (100, 256), torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits([y], [layer(x)])


def test_refusals():
    gen = generator(8)
    x, w = mg.Int8Rows(*codes(gen, 4, 16)), mg.Int8Rows(*codes(gen, 6, 16))
    for bad, what in (((mg.Int8Rows(x.codes[:, :15], x.scales), w), "differ in width"),
                      ((mg.Int8Rows(x.codes, x.scales[:3]), w), "a scale for each row"),
                      ((x, mg.Int8Rows(w.codes, w.scales[:, None])), "a scale for each row"),
                      ((x, mg.Int8Rows(w.codes[None], w.scales[None])), "channels, width"),
                      ((x, w, torch.ones(5, device=DEV)), "bias needs shape"),
                      ((mg.Int8Rows(x.codes[:, :0], x.scales), w), "last dimension")):
        with pytest.raises(ValueError, match=what):
            mg.int8_linear(*bad)
    wide = torch.zeros((2, 131_072), dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="131071"):
        mg.int8_linear(mg.Int8Rows(wide, x.scales[:2]), mg.Int8Rows(wide, x.scales[:2]))
    for bad in ((mg.Int8Rows(x.codes.short(), x.scales), w), (x, mg.Int8Rows(w.codes, w.scales.half())),
                (x, w, torch.ones(6, device=DEV, dtype=torch.float64))):
        with pytest.raises(TypeError):
            mg.int8_linear(*bad)
    with pytest.raises(TypeError):
        mg.int8_linear(x, w, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU"):
        mg.int8_linear(x, mg.Int8Rows(w.codes.cpu(), w.scales))
    for bad in ((mg.Int8Rows(x.codes, x.scales.clone().requires_grad_(True)), w),
                (x, w, torch.ones(6, device=DEV, requires_grad=True))):
        with pytest.raises(ValueError, match="no gradient"):
            mg.int8_linear(*bad)
        with torch.no_grad():
            mg.int8_linear(*bad)


@pytest.mark.parametrize("M, K, N", [(1, 1000, 70), (40, 2731, 100), (64, 20, 33), (300, 2731, 300), (70, 250, 66), (2050, 1000, 2060),
                                     (4133, 1000, 4101), (2050, 100, 2060)])
def test_rows_that_start_on_16_bytes(M, K, N):
    """As int8_rows lays them out, and packed: the same bits, in every form."""
    case("int8_linear, aligned", M, K, N)
    gen = generator(9)
    x, w, b = mg.Int8Rows(*codes(gen, M, K, -128)), mg.Int8Rows(*codes(gen, N, K, -128)), randn(gen, (N,), torch.float32)
    want = mg.int8_linear(x, w, b, dtype=torch.float32)
    check(want, x, w, b, slice(max(0, M - 70), M))

    def laid_out(r):
        n, pitch = r.codes.shape[0], (K + 15) // 16 * 16
        room = torch.full((n, pitch), 77, dtype=torch.int8, device=DEV)          # what lies between the rows counts for nothing
        return mg.Int8Rows(room[:, :K].copy_(r.codes), r.scales)

    assert same_bits([mg.int8_linear(laid_out(x), laid_out(w), b, dtype=torch.float32)], [want])
    half = mg.int8_linear(laid_out(x), laid_out(w), b, dtype=torch.bfloat16)
    assert same_bits([half], [want.to(torch.bfloat16)])
