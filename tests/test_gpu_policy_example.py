"""The operators together, as examples/policy_tuning.py uses them: its model's
loss and gradients against the same model in plain torch operations, and a run
of optimizer steps."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch
from torch.nn import functional as F

from tests._ops import DEV, mg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "policy_tuning.py"
    spec = importlib.util.spec_from_file_location("policy_tuning", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _norm_rope(x, w, cos, sin):
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    a, b = n.chunk(2, -1)
    c, s = cos[: x.shape[1], None], sin[: x.shape[1], None]
    return torch.cat((a * c - b * s, b * c + a * s), -1).transpose(1, 2)


def _plain_block(block, x, cos, sin):
    B, T, _ = x.shape
    qkv = block.qkv(block.input_norm(x)).view(B, T, -1, block.dim)
    q, k, v = qkv.split((block.q_heads, block.k_heads, block.k_heads), 2)
    q, k = _norm_rope(q, block.q_norm, cos, sin), _norm_rope(k, block.k_norm, cos, sin)
    x = x + block.out(block._attend(q, k, v.transpose(1, 2)))
    h = block.mlp_norm(x)
    return x + block.down(F.silu(block.gate(h)) * block.up(h))


def _plain_loss(model, ids, targets, mask, advantages, old, kl_coef):
    x = model.embed[ids]
    for b in model.blocks:
        x = _plain_block(b, x, model.cos, model.sin)
    logp = torch.log_softmax(model.head(model.norm(x)), -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    ratio = (logp - old).exp()
    policy = -torch.minimum(ratio * advantages, ratio.clamp(0.8, 1.2) * advantages)
    r = old - logp
    return ((policy + kl_coef * (r.exp() - r - 1)) * mask).sum() / mask.sum()


def test_gradients_of_the_whole_model(example):
    """Float32: the forward pass agrees to rounding.  The gradients of the MLP
    come from an 8-bit checkpoint, whose error is a step of a 127th of a group's
    largest magnitude (about 3 standard deviations of 128 values) over sqrt(12),
    0.7 % of a value, and reach every gradient below it: 3 % of each gradient's
    norm, and 0.1 % where only the head's products lie above."""
    torch.manual_seed(3)
    model = example.Policy(vocab=200, width=96, n_layer=2, q_heads=4, k_heads=2, dim=32, inter=200, length=40).to(DEV)
    ids, targets, mask, advantages = example.rollouts(200, 6, 40, 10, 1)
    with torch.no_grad():
        old = mg.token_log_probs(model(ids), targets, mask=mask)
        old = old + 0.1 * torch.randn(old.shape, device=DEV) * mask
    logits = model(ids)
    result, grad = mg.policy_loss_grad(logits.detach(), targets, old, advantages, ref_logp=old, mask=mask, kl_coef=0.02)
    logits.backward(grad)
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    loss = _plain_loss(model, ids, targets, mask, advantages, old, 0.02)
    loss.backward()
    assert math.isclose(float(result.loss), float(loss), rel_tol=1e-4, abs_tol=1e-5)
    for n, p in model.named_parameters():
        off = float((got[n] - p.grad).norm() / p.grad.norm())
        assert off < (1e-3 if n in ("head.weight", "norm.weight") else 0.03), (n, off)
    # the differentiable loss gives the same logits' gradient
    logits = model(ids).detach().requires_grad_(True)
    again, = torch.autograd.grad(mg.policy_loss(logits, targets, old, advantages, ref_logp=old, mask=mask,
                                                kl_coef=0.02).loss, logits)
    near = (again - grad).abs().max() / grad.abs().max()
    assert float(near) < 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_lower_the_loss(example, dtype):
    losses = example.tune(12, batch=4, length=48, dtype=dtype, log=lambda *_: None, vocab=300, width=128, inter=300)
    assert all(math.isfinite(x) for x in losses)
    assert abs(losses[0]) < 0.2 and losses[-1] < losses[0] - 0.02, losses


def test_a_rerun_gives_the_same_bits(example):
    """No operator's result depends on the order of atomics, so two runs of the
    same steps agree exactly (float32, whose products run the same way twice)."""
    a, b = (example.tune(4, batch=2, length=32, dtype=torch.float32, log=lambda *_: None) for _ in range(2))
    assert a == b
