"""policy_loss, policy_loss_grad and token_log_probs against the formulas in 64
bits.

Bounds.  u = 2^-24.  A row's sum s of V exponentials is summed by at least 64
threads, at most V / 64 + 8 terms in a chain where V is at most 2,048 and
V / 256 + 8 or V / 1024 + 8 beyond (at least 4 elements an access), each step
rounding up to 1.4 times (a rescale every 4 elements), and at most 10 joins of 4
roundings: (1.4 chain + 40) u.  An exponential's argument t = (x - m) log2(e) / T
is off by 3 roundings of it and the hardware's exponential by 1 ulp:
(2.1 |t| + 2) u relative.  log s is therefore off by
E = (1.4 chain + 42 + 2.1 sum_j p_j |t_j|) u, and so is logp; the scalars after
it are in 64 bits, and each row's terms are rounded once to 32.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests._ops import DEV, DTYPES, ROUND, case, generator, mg, near, randn

pytestmark = pytest.mark.gpu
U = 2.0**-24
CLIP, KL = (0.2, 0.3), 0.1
VOCABS = [1, 2, 7, 64, 96, 257, 1000, 2049, 5000, 50304, 151_937]


def chain(V):
    return V / (64 if V <= 2048 else 256 if V <= 16384 else 1024) + 8


def make(rows, V, dtype, seed, ref=True, mask=None, spread=2.0):
    gen = generator(seed)
    s = {"logits": randn(gen, (rows, V), DTYPES[dtype], spread),
         "targets": torch.randint(0, V, (rows,), generator=gen, device=DEV)}
    logp = torch.log_softmax(s["logits"].double(), -1).gather(1, s["targets"][:, None])[:, 0]
    # ratios on both sides of the clip and not within 2^-10 of its edges
    offset = torch.round(torch.randn(rows, generator=gen, device=DEV) * 0.3 * 64) / 64 + 2.0**-8
    s["old_logp"] = (logp - offset).float()
    s["ref_logp"] = (logp + torch.randn(rows, generator=gen, device=DEV) * 0.3).float() if ref else None
    s["advantages"] = torch.randn(rows, generator=gen, device=DEV)
    s["mask"] = None
    if mask == "bool":
        s["mask"] = torch.rand(rows, generator=gen, device=DEV) > 0.4
    elif mask == "float":
        s["mask"] = torch.rand(rows, generator=gen, device=DEV) * (torch.rand(rows, generator=gen, device=DEV) > 0.3)
    return s


def reference(s, temperature=1.0, scale=1.0, clip=CLIP, kl_coef=KL):
    """Results in 64 bits, and bounds of their errors before the rounding of the output."""
    x = s["logits"].detach().double() / temperature
    rows, V = x.shape
    w = torch.ones(rows, dtype=torch.float64, device=DEV) if s["mask"] is None else s["mask"].double()
    on = w != 0
    y = torch.where(on, s["targets"].long(), 0)
    logs = torch.log_softmax(x, -1)
    p = logs.exp()
    t = (x.amax(-1, keepdim=True) - x) * math.log2(math.e)
    E = (1.4 * chain(V) + 42 + 2.1 * (p * t).nan_to_num().sum(-1)) * U
    logp = torch.where(on, logs.gather(1, y[:, None])[:, 0], 0.0)
    ratio = (logp - s["old_logp"].double()).exp()
    A = s["advantages"].double()
    s1, s2 = ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A
    held = s2 < s1
    kl, dkl, e = torch.zeros_like(logp), torch.zeros_like(logp), torch.zeros_like(logp)
    if s["ref_logp"] is not None:
        r = s["ref_logp"].double() - logp
        e = r.exp()
        kl, dkl = torch.expm1(r) - r, -torch.expm1(r)
    total = w.sum()
    inv = 0.0 if float(total) == 0 else 1.0 / float(total)
    mean = lambda v: torch.where(on, w * v, 0.0).sum() * inv  # noqa: E731
    policy, kl_mean = mean(-torch.minimum(s1, s2)), mean(kl)
    slope = torch.where(on, w * (torch.where(held, 0.0, -s1) + kl_coef * dkl), 0.0) * inv * scale / temperature
    E_slope = torch.where(on, w * (s1.abs() + kl_coef * e) * (E + logp.abs() * U), 0.0) * inv * scale / temperature
    d = -slope[:, None] * p
    within = (E_slope[:, None] * p + slope[:, None].abs() * p * (E[:, None] + (2.1 * t.nan_to_num() + 8) * U)
              + slope[:, None].abs() * 2.0**-125)
    at = torch.arange(rows, device=DEV)
    d[at, y] += slope
    within[at, y] += E_slope + 2 * slope.abs() * U
    d[~on], within[~on] = 0.0, 0.0
    e_policy, e_kl = mean(s1.abs() * (E + U) + s2.abs() * U), mean((e + 1) * E + kl.abs() * U)
    return {"loss": policy + kl_coef * kl_mean, "log_probs": logp, "policy": policy, "kl": kl_mean,
            "clip_fraction": mean(held.double()), "d": d}, \
           {"loss": e_policy + kl_coef * e_kl, "log_probs": E, "policy": e_policy, "kl": e_kl,
            "clip_fraction": 1e-7, "d": within}


def check(s, result, grad, temperature=1.0, scale=1.0, **more):
    want, within = reference(s, temperature, scale, **more)
    for name in ("loss", "log_probs", "policy", "kl", "clip_fraction"):
        b = within[name]
        near(getattr(result, name), want[name], b if torch.is_tensor(b) else torch.tensor(b, device=DEV), name)
    if grad is not None:
        near(grad, want["d"], within["d"], "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [None, "bool", "float"])
def test_loss_and_gradient(dtype, mask):
    scale = torch.tensor(512.0, device=DEV)
    for seed, V in enumerate(VOCABS):
        rows = 5 if V > 10_000 else 67
        temperature = 1.0 if seed % 2 else 0.7
        case("policy_loss", dtype, "mask", mask, "rows", rows, "vocab", V, "temperature", temperature)
        s = make(rows, V, dtype, seed, ref=seed % 3 != 0, mask=mask)
        given = (s["logits"], s["targets"], s["old_logp"], s["advantages"])
        more = {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL, "temperature": temperature}
        r, grad = mg.policy_loss_grad(*given, grad_scale=scale, **more)
        check(s, r, grad, temperature, 512.0)
        assert torch.equal(mg.token_log_probs(s["logits"], s["targets"], mask=s["mask"], temperature=temperature),
                           r.log_probs)
        s["logits"].requires_grad_(True)
        r = mg.policy_loss(*given, **more)
        (r.loss * scale).backward()
        check(s, r, s["logits"].grad, temperature, 512.0)


def test_gradient_against_differences():
    """Central differences, in 64 bits, of the formula: steps of 1e-5 leave 1e-10
    of the third derivative (under 20 here) and 1e-10 of rounding."""
    s = make(6, 40, "f32", 3)
    given = (s["logits"], s["targets"], s["old_logp"], s["advantages"])
    _, grad = mg.policy_loss_grad(*given, ref_logp=s["ref_logp"], clip=CLIP, kl_coef=KL)
    x, h = s["logits"].double(), 1e-5
    want = torch.zeros_like(x)

    def loss(v):
        return float(reference({**s, "logits": v})[0]["loss"])

    for i in range(x.shape[0]):
        for j in range(x.shape[1]):
            up, down = x.clone(), x.clone()
            up[i, j] += h
            down[i, j] -= h
            want[i, j] = (loss(up) - loss(down)) / (2 * h)
    near(grad, want, torch.full_like(want, 1e-8) + reference(s)[1]["d"], "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [96, 2600, 50_001])
def test_masked_rows_are_not_read(dtype, V):
    s = make(24, V, dtype, 7)
    s["mask"] = torch.arange(24, device=DEV) % 3 == 1
    off = ~s["mask"]
    given = lambda: (s["logits"], s["targets"], s["old_logp"], s["advantages"])  # noqa: E731
    more = lambda: {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL}  # noqa: E731
    r, grad = mg.policy_loss_grad(*given(), **more())
    check(s, r, grad)
    for name, value in (("logits", float("nan")), ("targets", -100), ("old_logp", float("inf")),
                        ("advantages", float("nan")), ("ref_logp", float("-inf"))):
        s[name][off] = value
    r2, grad2 = mg.policy_loss_grad(*given(), **more())
    assert torch.equal(grad, grad2) and all(torch.equal(a, b) for a, b in zip(r, r2))
    assert bool((grad2[off] == 0).all()) and bool((r2.log_probs[off] == 0).all())
    s["targets"][off] = 2**40
    s["logits"].requires_grad_(True)
    loss = mg.policy_loss(*given(), **more()).loss
    loss.backward()
    assert torch.equal(loss, r.loss) and bool((s["logits"].grad[off] == 0).all())
    s["logits"] = s["logits"].detach()
    s["mask"] = torch.zeros(24, dtype=torch.bool, device=DEV)       # a batch that the mask leaves empty
    r, grad = mg.policy_loss_grad(*given(), **more())
    assert all(float(v) == 0 for v in (r.loss, r.policy, r.kl, r.clip_fraction)) and bool((grad == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [70, 3000, 40_000])
def test_infinities_and_lowest_values(dtype, V):
    t = DTYPES[dtype]
    low, inf, nan = torch.finfo(t).min, float("inf"), float("nan")
    s = make(12, V, dtype, 9)
    s["targets"][:] = 3
    x = s["logits"]
    x[0, 10:] = -inf                       # a padded vocabulary
    x[1, 10:] = low                        # masked by the type's lowest value
    x[2, :] = low                          # nothing but that: uniform
    x[3, 5] = -torch.tensor(low, dtype=t)  # the largest value, far above the others
    x[4, :3] = -inf
    x[4, 4:] = -inf                        # the target alone
    x[5, 3] = -inf                         # the target impossible: logp -inf, ratio 0
    x[6, :] = -inf                         # nothing
    x[7, 8] = inf
    x[8, 8] = nan
    s["targets"][9] = V
    s["targets"][10] = -1
    r, grad = mg.policy_loss_grad(x, s["targets"], s["old_logp"], s["advantages"], clip=CLIP)
    assert bool(r.loss.isnan())
    logp, want = r.log_probs, torch.log_softmax(x.double(), -1)[:, 3]
    ok = [0, 1, 2, 3, 4, 11]
    near(logp[ok], want[ok], torch.full_like(want[ok], (1.4 * chain(V) + 42 + 2.1 * math.log2(V)) * U), "log_probs")
    assert float(logp[5]) == -inf and bool(logp[[6, 7, 8, 9, 10]].isnan().all())
    assert bool(grad[[0, 1, 2, 3, 4, 5, 11]].isfinite().all()) and bool(grad[[6, 7, 8, 9, 10]].isnan().all())
    assert bool((grad[0, 10:] == 0).all()) and bool((grad[1, 10:] == 0).all())
    # rows 0 to 5 and 11 by themselves
    keep = [0, 1, 2, 3, 4, 11]
    part = {k: (v[keep].contiguous() if torch.is_tensor(v) else v) for k, v in s.items()}
    part["ref_logp"] = None
    part["old_logp"] = (torch.log_softmax(part["logits"].double(), -1)[:, 3] - 0.1).float()
    r, grad = mg.policy_loss_grad(part["logits"], part["targets"], part["old_logp"], part["advantages"], clip=CLIP)
    check(part, r, grad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, V", [(70, 300), (70, 30_000), (3, 151_937)])
def test_logits_of_large_magnitude_and_small_temperatures(dtype, rows, V):
    """Every result depends on the logits' differences alone, however large the
    logits are: the oracle takes them less the row's largest, which 64 bits hold."""
    t = DTYPES[dtype]
    levels = [(60_000.0, 1e-6), (-60_000.0, 1e-6)] if dtype == "f16" else [(-1e10, 1.0), (-1e30, 1.0), (1e12, 0.7), (3e38, 1.0)]
    for level, temperature in [*levels, (None, 1e-9), (None, 1e-30 if dtype != "f16" else 1e-6), (None, 1e9)]:
        case("policy_loss", dtype, "rows", rows, "vocab", V, "level", level, "temperature", temperature)
        s = make(rows, V, dtype, 17, ref=False)
        if level is not None:  # the level, and in two of three columns a step or two below it
            low = level - abs(level) * 4 * ROUND[t] * (torch.arange(V, device=DEV) % 3).double()
            s["logits"] = low.to(t).expand(rows, V).contiguous()
        s["targets"] = s["logits"].argmax(-1)
        shifted = s["logits"].double() - s["logits"].double().amax(-1, keepdim=True)
        s["old_logp"] = (torch.log_softmax(shifted / temperature, -1).gather(1, s["targets"][:, None])[:, 0] - 0.1).float()
        scale = torch.tensor(temperature, device=DEV)
        given, more = (s["logits"], s["targets"], s["old_logp"], s["advantages"]), {"clip": CLIP, "temperature": temperature}
        oracle = {**s, "logits": shifted}
        r, grad = mg.policy_loss_grad(*given, grad_scale=scale, **more)
        check(oracle, r, grad, temperature, float(scale), kl_coef=0.0)
        assert torch.equal(mg.token_log_probs(s["logits"], s["targets"], temperature=temperature), r.log_probs)
        s["logits"].requires_grad_(True)
        r = mg.policy_loss(*given, **more)
        (r.loss * scale).backward()
        check(oracle, r, s["logits"].grad, temperature, float(scale), kl_coef=0.0)


def test_weights_that_cancel():
    """The weights' sum is 0 without a weight of 0: the means are 0, and their gradient."""
    for rows, V in ((4, 300), (4, 151_937)):
        s = make(rows, V, "bf16", 23)
        mask = torch.tensor([1.0, -1.0, 0.5, -0.5], device=DEV)
        given = (s["logits"], s["targets"], s["old_logp"], s["advantages"])
        more = {"ref_logp": s["ref_logp"], "mask": mask, "clip": CLIP, "kl_coef": KL}
        r, grad = mg.policy_loss_grad(*given, **more)
        s["logits"].requires_grad_(True)
        loss = mg.policy_loss(*given, **more).loss
        loss.backward()
        assert all(float(v) == 0 for v in (r.loss, r.policy, r.kl, r.clip_fraction, loss))
        assert bool((grad == 0).all()) and bool((s["logits"].grad == 0).all())


def test_layouts_types_and_in_place():
    s = make(30, 700, "bf16", 4, mask="bool")
    more = {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL}
    given = (s["targets"], s["old_logp"], s["advantages"])
    want, grad = mg.policy_loss_grad(s["logits"], *given, **more)
    wide = torch.zeros((30, 901), dtype=torch.bfloat16, device=DEV)
    view = wide[:, 100:800]
    view.copy_(s["logits"])
    got, g = mg.policy_loss_grad(view, *given, **more)
    assert torch.equal(g, grad) and all(torch.equal(a, b) for a, b in zip(got, want))
    got, g = mg.policy_loss_grad(view, *given, out=view, **more)          # over the logits
    assert g.data_ptr() == view.data_ptr() and torch.equal(view, grad) and torch.equal(got.loss, want.loss)
    assert bool((wide[:, :100] == 0).all()) and bool((wide[:, 800:] == 0).all())
    three = {k: (v.view(5, 6, *v.shape[1:]) if torch.is_tensor(v) else v) for k, v in s.items()}
    got, g = mg.policy_loss_grad(three["logits"], three["targets"].int(), three["old_logp"], three["advantages"],
                                 ref_logp=three["ref_logp"], mask=three["mask"], clip=CLIP, kl_coef=KL)
    assert g.shape == (5, 6, 700) and torch.equal(g.view(30, 700), grad) and got.log_probs.shape == (5, 6)
    got, g = mg.policy_loss_grad(s["logits"].t().contiguous().t(), *given, **more)   # copied
    assert torch.equal(g, grad)
    one = mg.token_log_probs(s["logits"][3], s["targets"][3:4])
    assert one.shape == () and torch.equal(one, mg.token_log_probs(s["logits"], s["targets"])[3])
    r, g = mg.policy_loss_grad(s["logits"][:0], s["targets"][:0], s["old_logp"][:0], s["advantages"][:0])
    assert g.shape == (0, 700) and float(r.loss) == 0 and r.log_probs.shape == (0,)
    assert mg.token_log_probs(s["logits"][:0], s["targets"][:0]).shape == (0,)


def test_offsets_beyond_32_bits():
    """More than 2^31 logits: the last rows are those of a small call on them."""
    rows, V = 14_200, 151_936
    case("policy_loss", rows, V)
    x = torch.zeros((rows, V), dtype=torch.bfloat16, device=DEV)
    s = make(5, V, "bf16", 2)
    x[-5:] = s["logits"]
    t = torch.zeros(rows, dtype=torch.int64, device=DEV)
    t[-5:] = s["targets"]
    fill = lambda v: torch.cat((torch.zeros(rows - 5, device=DEV), v))  # noqa: E731
    mask = torch.arange(rows, device=DEV) >= rows - 5
    r, grad = mg.policy_loss_grad(x, t, fill(s["old_logp"]), fill(s["advantages"]), mask=mask, out=x)
    want, small = mg.policy_loss_grad(s["logits"], s["targets"], s["old_logp"], s["advantages"])
    assert torch.equal(r.log_probs[-5:], want.log_probs) and torch.equal(grad[-5:], small)
    assert torch.equal(r.loss, want.loss) and bool((grad[:-5:1000] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 7, 127, 128])
def test_few_long_rows(dtype, rows):
    """Rows cut in slices, and one row more than is cut: in place, where one
    slice's gradient overwrites logits that others have read, and by autograd."""
    V = 90_007 if dtype != "f32" else 60_013
    case("policy_loss", dtype, "rows", rows, "vocab", V)
    s = make(rows, V, dtype, rows, mask="bool" if rows > 2 else None)
    given = (s["targets"], s["old_logp"], s["advantages"])
    more = {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL}
    r, grad = mg.policy_loss_grad(s["logits"], *given, **more)
    check(s, r, grad)
    copy = s["logits"].clone()
    again, g = mg.policy_loss_grad(copy, *given, out=copy, **more)
    assert torch.equal(copy, grad) and all(torch.equal(a, b) for a, b in zip(again, r))
    assert torch.equal(mg.token_log_probs(s["logits"], s["targets"], mask=s["mask"]), r.log_probs)
    s["logits"].requires_grad_(True)
    r = mg.policy_loss(s["logits"], *given, **more)
    r.loss.backward()
    check(s, r, s["logits"].grad)


def test_many_rows():
    s = make(40_000, 11, "f32", 5, mask="float")
    r, grad = mg.policy_loss_grad(s["logits"], s["targets"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                                  mask=s["mask"], clip=CLIP, kl_coef=KL)
    check(s, r, grad)


def test_backward_scales_and_repeats():
    s = make(20, 300, "f32", 6)
    s["logits"].requires_grad_(True)
    r = mg.policy_loss(s["logits"], s["targets"], s["old_logp"], s["advantages"], clip=CLIP)
    first, = torch.autograd.grad(r.loss, s["logits"], torch.tensor(2.0, device=DEV), retain_graph=True)
    again, = torch.autograd.grad(r.loss, s["logits"], torch.tensor(2.0, device=DEV), retain_graph=True)
    kept = first.clone()
    other, = torch.autograd.grad(r.loss, s["logits"], torch.tensor(4.0, device=DEV))
    assert torch.equal(first, again) and torch.equal(first, kept) and torch.equal(other, 2 * first)
    assert not r.kl.requires_grad and not r.log_probs.requires_grad and float(r.kl) == 0.0
    with torch.no_grad():
        assert not mg.policy_loss(s["logits"], s["targets"], s["old_logp"], s["advantages"]).loss.requires_grad


def test_streams_and_graphs():
    s = make(50, 2500, "f16", 8, mask="bool")
    given = (s["logits"], s["targets"], s["old_logp"], s["advantages"])
    more = {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL}
    run = lambda: mg.policy_loss_grad(*given, **more)  # noqa: E731
    want, grad = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, g = run()
    side.synchronize()
    assert torch.equal(g, grad) and all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, g = run()
    for k in range(3):
        s["logits"].mul_(0.9)
        s["mask"].logical_not_()
        graph.replay()
        want, grad = run()
        torch.cuda.synchronize()
        assert torch.equal(g, grad) and all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_refusals():
    s = make(8, 50, "f32", 1)
    x, y, o, a = s["logits"], s["targets"], s["old_logp"], s["advantages"]
    run = mg.policy_loss_grad
    with pytest.raises(ValueError, match="values for 8 rows"):
        run(x, y[:5], o, a)
    with pytest.raises(ValueError, match="values for 8 rows"):
        run(x, y, o, a, mask=torch.ones(7, device=DEV))
    with pytest.raises(TypeError, match="int64 or int32"):
        run(x, y.float(), o, a)
    with pytest.raises(TypeError, match="old_logp must be float32"):
        run(x, y, o.double(), a)
    with pytest.raises(TypeError, match="mask must be"):
        run(x, y, o, a, mask=torch.ones(8, device=DEV, dtype=torch.int64))
    with pytest.raises(TypeError, match="expected float32"):
        run(x.double(), y, o, a)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            run(x, y, o, a, temperature=bad)
    with pytest.raises(ValueError, match="clip range"):
        run(x, y, o, a, clip=(-0.1, 0.2))
    with pytest.raises(ValueError, match="grad_scale"):
        run(x, y, o, a, grad_scale=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="out has shape"):
        run(x, y, o, a, out=x[:5])
    wide = torch.empty(9 * 50 + 7, device=DEV)
    with pytest.raises(ValueError, match="overlaps the logits"):
        run(wide[: 8 * 50].view(8, 50), y, o, a, out=wide[7: 8 * 50 + 7].view(8, 50))
    with pytest.raises(ValueError, match="overlaps the logits"):
        run(wide[: 8 * 50].view(8, 50), y, o, a, out=wide.as_strided((8, 50), (51, 1)))
    with pytest.raises(ValueError, match="rows overlap"):
        run(x, y, o, a, out=torch.empty(50, device=DEV).expand(8, 50))
    with pytest.raises(ValueError, match="evenly spaced"):
        run(x, y, o, a, out=torch.empty((50, 8), device=DEV).t())
    with pytest.raises(RuntimeError, match="no CPU path"):
        run(x.cpu(), y, o, a)
    with pytest.raises(RuntimeError, match="no CPU path"):
        run(x, y.cpu(), o, a)
    with pytest.raises(ValueError, match="last dimension"):
        run(x[:, :0], y, o, a)
    with pytest.raises(ValueError, match="no gradient by advantages"):
        mg.policy_loss(x, y, o, a.requires_grad_(True))
