"""What autograd, forward-mode derivatives and traces see of the operators: their
outputs changed in place, tensors that they write in place, dual tensors."""

from __future__ import annotations

import copy
import io

import pytest
import torch
from torch.autograd import forward_ad

from tests._ops import DEV, generator, mg, randn, same_bits
from tests.test_gpu_policy_loss import CLIP, KL, make

pytestmark = pytest.mark.gpu


def _loss_args(rows=24, V=300, dtype="f32"):
    s = make(rows, V, dtype, 31)
    return s["logits"], (s["targets"], s["old_logp"], s["advantages"]), {"ref_logp": s["ref_logp"], "clip": CLIP, "kl_coef": KL}


def test_losses_take_in_place_operations():
    """loss /= n and loss += term before backward, and the other three used as
    accumulators: each is a tensor of its own."""
    x, given, more = _loss_args()
    x.requires_grad_(True)
    r = mg.policy_loss(x, *given, **more)
    before = [v.clone() for v in r]
    want, = torch.autograd.grad(r.loss / 4, x)
    r = mg.policy_loss(x, *given, **more)
    r.kl.div_(2)
    r.policy.add_(1)
    r.clip_fraction.zero_()
    loss, aux = r.loss, torch.tensor(3.0, device=DEV, requires_grad=True)
    loss /= 4
    loss += aux
    loss.backward()
    assert torch.equal(x.grad, want) and float(aux.grad) == 1.0
    assert torch.equal(loss, before[0] / 4 + 3) and torch.equal(r.kl, before[3] / 2)
    assert torch.equal(r.policy, before[2] + 1) and float(r.clip_fraction) == 0
    r, _ = mg.policy_loss_grad(x.detach(), *given, **more)
    total = r.loss
    total += aux
    total.backward()
    assert float(aux.grad) == 2.0 and torch.equal(total, before[0] + 3)
    assert all(torch.equal(a, b) for a, b in zip(r[1:], before[1:]))


def test_a_gradient_over_the_logits_is_seen_by_autograd():
    """What was saved of the logits for another backward pass is gone."""
    x, given, more = _loss_args()
    x.requires_grad_(True)
    logits = x * 2
    z = logits.logsumexp(-1).square().sum()
    mg.policy_loss_grad(logits.detach(), *given, **more)              # reads them
    want, = torch.autograd.grad(z, x, retain_graph=True)
    near = 2 * (2 * logits.logsumexp(-1)[:, None] * logits.softmax(-1))
    assert float((want - near).abs().max()) < 1e-4
    mg.policy_loss_grad(logits.detach(), *given, out=torch.empty_like(logits), **more)
    assert same_bits(torch.autograd.grad(z, x, retain_graph=True), [want])
    mg.policy_loss_grad(logits.detach(), *given, out=logits.detach(), **more)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, x)


def test_an_accumulated_gradient_is_seen_by_autograd():
    gen = generator(1)
    buf, ids = randn(gen, (50, 16), torch.float32).requires_grad_(True), torch.arange(20, device=DEV)
    g = randn(gen, (20, 16), torch.float32)
    for accumulate in (True, False):
        y = (buf * buf).sum()
        mg.embedding_grad_(buf.detach(), ids, g, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():       # tensors without a version
        grad, logits = torch.zeros((50, 16), device=DEV), _loss_args()[0] * 1.0
    mg.embedding_grad_(grad, ids, g)
    assert torch.equal(grad[:20], g)
    _, given, more = _loss_args()
    _, want = mg.policy_loss_grad(logits, *given, **more)
    _, got = mg.policy_loss_grad(logits, *given, out=logits, **more)
    assert got.data_ptr() == logits.data_ptr() and torch.equal(got, want)


def _differentiable():
    """(name, function of its differentiable inputs, those inputs)"""
    gen = generator(2)
    ids = torch.randint(0, 60, (40,), generator=gen, device=DEV)
    q, k = randn(gen, (2, 5, 4, 64), torch.float32), randn(gen, (2, 5, 2, 64), torch.float32)
    wq, wk = randn(gen, (64,), torch.float32), randn(gen, (64,), torch.float32)
    cos, sin = mg.rope_tables(9, 64, device=DEV)
    return [("embedding", lambda w: mg.embedding(ids, w, scale=1.5), (randn(gen, (60, 24), torch.float32),)),
            ("qk_norm_rope", lambda *a: mg.qk_norm_rope(*a, cos, sin), (q, k, wq, wk)),
            ("gated_act", lambda g: mg.gated_act(g, act="gelu_tanh"), (randn(gen, (9, 200), torch.float32),)),
            ("gated_act with a gate", lambda g, u: mg.gated_act(g, u),
             (randn(gen, (9, 200), torch.float32), randn(gen, (9, 200), torch.float32)))]


def _outputs(y):
    return [y] if torch.is_tensor(y) else list(y)


@pytest.mark.parametrize("i", range(4))
def test_forward_mode_derivatives_are_refused(i):
    """A dual tensor asks for no gradient; its tangent is not dropped silently."""
    name, f, inputs = _differentiable()[i]
    want = _outputs(f(*inputs))
    with forward_ad.dual_level():
        assert same_bits(_outputs(f(*inputs)), want)       # no tangent, no change
        for j in range(len(inputs)):
            given = list(inputs)
            given[j] = forward_ad.make_dual(given[j], torch.ones_like(given[j]))
            with pytest.raises(NotImplementedError, match="jvp"):
                f(*given)
    assert same_bits(_outputs(f(*inputs)), want)


@pytest.mark.parametrize("i", range(4))
def test_a_trace_holds_the_operators(i):
    name, f, inputs = _differentiable()[i]
    traced = torch.jit.trace(f, inputs)
    others = tuple(1.5 * x for x in inputs)
    assert same_bits(_outputs(traced(*others)), _outputs(f(*others)))


@pytest.mark.parametrize("dtype, rows, V", [("f32", 4000, 200), ("bf16", 4000, 200), ("bf16", 100, 120_007)])
def test_forward_and_backward_clip_the_same_rows(dtype, rows, V):
    """Ratios that the rounding of old_logp leaves on either side of the clip's
    edge: the backward pass holds the rows that the loss counted, and gives the
    gradient of the one-pass form."""
    s = make(rows, V, dtype, 41, ref=False)
    logp = torch.log_softmax(s["logits"].double(), -1).gather(1, s["targets"][:, None])[:, 0]
    s["old_logp"] = (logp - torch.log1p(torch.tensor(CLIP[1], dtype=torch.float64, device=DEV))).float()
    s["advantages"] = s["advantages"].abs() + 0.1
    given, more = (s["targets"], s["old_logp"], s["advantages"]), {"clip": CLIP}
    one, want = mg.policy_loss_grad(s["logits"], *given, **more)
    x = s["logits"].requires_grad_(True)
    r = mg.policy_loss(x, *given, **more)
    r.loss.backward()
    assert torch.equal(r.clip_fraction, one.clip_fraction) and 0.05 < float(r.clip_fraction) < 0.95
    held = int((x.grad == 0).all(-1).sum())
    assert held == round(float(r.clip_fraction) * rows), (held, float(r.clip_fraction) * rows)
    assert same_bits([x.grad], [want])


def test_losses_as_ordinary_tensors():
    """In inference mode, copied, saved, reshaped: no trace of the shared memory."""
    x, given, more = _loss_args()
    want, grad = mg.policy_loss_grad(x, *given, **more)
    with torch.inference_mode():
        r, g = mg.policy_loss_grad(x, *given, **more)
        r.loss.mul_(2)
        assert same_bits([g], [grad]) and torch.equal(r.loss, want.loss * 2) and torch.equal(r.policy, want.policy)
    for v in (want.loss, want.policy, want.kl, want.clip_fraction):
        assert v.shape == () and v.dtype == torch.float32 and v.is_contiguous() and not v._is_view()
        file = io.BytesIO()
        torch.save(v, file)
        file.seek(0)
        for other in (copy.deepcopy(v), v.clone(), torch.load(file, weights_only=True), v.view(1)[0], v.cpu().to(DEV)):
            assert same_bits([other], [v])
        assert float(v) == v.item() == v.cpu().numpy()
    total = torch.stack([want.loss, want.policy, want.kl, want.clip_fraction])
    assert same_bits([total[0], total[3]], [want.loss, want.clip_fraction])
