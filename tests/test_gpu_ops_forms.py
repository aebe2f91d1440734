"""Forms of the operators' kernels that only large calls reach, under the bounds
of test_gpu_policy_loss.py and test_gpu_gated_act.py."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests._ops import DEV, DTYPES, case, generator, mg, near, randn, same_bits
from tests.test_gpu_gated_act import check_forward
from tests.test_gpu_policy_loss import CLIP, KL, check, make, reference
from tests.test_ops_host import PolicyArgs

pytestmark = pytest.mark.gpu
#: vectors a row: more than 20,480 are held in part and read again (12,288 of them held); 16,385 to 20,480 fill the registers
LONG_ROWS = [("f32", 100_003), ("bf16", 170_001), ("f16", 163_853), ("f32", 75_001), ("bf16", 150_001), ("f16", 163_840)]


@pytest.mark.parametrize("dtype, V", LONG_ROWS)
@pytest.mark.parametrize("mask", [None, "bool", "float"])
def test_many_long_rows(dtype, V, mask):
    """130 rows, which are not cut in slices: targets in the part that is held,
    in the part that is read again, and in the tail past the last whole vector."""
    case("policy_loss", dtype, "mask", mask, "rows 130, vocab", V)
    s = make(130, V, dtype, 51, mask=mask)
    n = 16 // s["logits"].element_size()
    at = [0, n, 12 * 1024 * n - 1, 12 * 1024 * n, 12 * 1024 * n + n + 1, V // n * n - 1, V - 1]
    s["targets"][:len(at)] = torch.tensor(at, device=DEV).clamp(max=V - 1)
    logp = torch.log_softmax(s["logits"].double(), -1).gather(1, s["targets"][:, None])[:, 0]
    s["old_logp"], s["ref_logp"] = (logp - 0.125).float(), (logp + 0.25).float()
    given = (s["targets"], s["old_logp"], s["advantages"])
    more = {"ref_logp": s["ref_logp"], "mask": s["mask"], "clip": CLIP, "kl_coef": KL, "temperature": 0.7}
    scale = torch.tensor(64.0, device=DEV)
    r, grad = mg.policy_loss_grad(s["logits"], *given, grad_scale=scale, **more)
    check(s, r, grad, 0.7, 64.0)
    assert same_bits([mg.token_log_probs(s["logits"], s["targets"], mask=s["mask"], temperature=0.7)], [r.log_probs])
    wide = torch.full((130, V + 5), 7.0, dtype=DTYPES[dtype], device=DEV)    # over the logits, rows at odd places
    view = wide[:, 3:V + 3]
    view.copy_(s["logits"])
    again, g = mg.policy_loss_grad(view, *given, grad_scale=scale, out=view, **more)
    assert g.data_ptr() == view.data_ptr() and same_bits([view], [grad]) and same_bits(again, r)
    assert bool((wide[:, :3] == 7).all()) and bool((wide[:, V + 3:] == 7).all())
    s["logits"].requires_grad_(True)
    r = mg.policy_loss(s["logits"], *given, **more)
    (r.loss * scale).backward()
    check(s, r, s["logits"].grad, 0.7, 64.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_long_rows_without_a_workspace(dtype):
    """The C entry takes no workspace for log-probabilities: rows are not cut."""
    native = mg._native
    rows, V = 5, 90_007
    s = make(rows, V, dtype, 61, ref=False)
    out = torch.empty(rows, device=DEV)
    a = PolicyArgs(logits=s["logits"].data_ptr(), targets=s["targets"].data_ptr(), log_probs=out.data_ptr(), rows=rows, vocab=V,
                   logits_stride=V, temperature=1.0, target_bytes=8, dtype=native.dtype_code(DTYPES[dtype]))
    stream = ctypes.c_void_p(native.stream_handle(s["logits"].device))
    assert native.lib().mgopt_token_log_probs(ctypes.byref(a), stream) == 0
    want, within = reference(s)
    near(out, want["log_probs"], within["log_probs"], "log_probs")
    near(mg.token_log_probs(s["logits"], s["targets"]), want["log_probs"], within["log_probs"], "in slices")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("pack", [True, False])
def test_streamed_forward(dtype, act, gated, pack):
    """A forward pass that moves more than 256 MiB, rows of an odd width at odd
    places: each row as a small call gives it, and a few against 64 bits."""
    t, h = DTYPES[dtype], 16_411
    b, inputs = torch.empty((), dtype=t).element_size(), 2 if gated else 1
    n = (1 << 28) // (h * (b * (inputs + 1) + (inputs if pack else 0))) + 5
    case("gated_act", dtype, act, "gated" if gated else "plain", "checkpoint" if pack else "", n, h)
    x = randn(generator(71), (n, inputs * h + 3), t, 2.0)
    gate, up = x[:, 1:h + 1], (x[:, h + 1:2 * h + 1] if gated else None)
    run = lambda g, u: mg.gated_act_pack(g, u, act=act) if pack else (mg.gated_act(g, u, act=act), None)  # noqa: E731
    y, saved = run(gate, up)
    ends = [(0, n // 2), (n // 2, n)]
    for lo, hi in ends:
        small, kept = run(gate[lo:hi], None if up is None else up[lo:hi])
        assert same_bits([y[lo:hi]], [small])
        if pack:
            assert torch.equal(saved.codes[:, lo:hi], kept.codes) and same_bits([saved.scales[:, lo:hi]], [kept.scales])
    for lo in (0, n // 2 - 2, n - 4):
        check_forward(y[lo:lo + 4], gate[lo:lo + 4], None if up is None else up[lo:lo + 4], act)
