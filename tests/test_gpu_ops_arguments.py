"""Arguments that the operators refuse: shapes that pair rows wrongly, gradients
that they do not form."""

from __future__ import annotations

import pytest
import torch

from tests._ops import DEV, generator, mg, randn, same_bits
from tests.test_gpu_policy_loss import make

pytestmark = pytest.mark.gpu


def test_values_per_row_in_another_order():
    """(length, batch) beside logits of (batch, length, vocab) has the right count
    and the wrong order."""
    s = make(12, 40, "f32", 3, mask="bool")
    x = s["logits"].view(3, 4, 40)
    y, o, a, ref, mask = (s[k].view(3, 4) for k in ("targets", "old_logp", "advantages", "ref_logp", "mask"))
    turned = lambda v: v.t().contiguous()  # noqa: E731
    for f in (mg.policy_loss, mg.policy_loss_grad):
        for bad in (dict(targets=turned(y)), dict(old_logp=turned(o)), dict(advantages=turned(a)), dict(ref_logp=turned(ref)),
                    dict(mask=turned(mask)), dict(targets=y.reshape(2, 6)), dict(advantages=a.reshape(6, 2))):
            given = {"targets": y, "old_logp": o, "advantages": a, "ref_logp": ref, "mask": mask, **bad}
            with pytest.raises(ValueError, match=f"{next(iter(bad))} has shape"):
                f(x, **given)
    with pytest.raises(ValueError, match="targets has shape"):
        mg.token_log_probs(x, turned(y))
    with pytest.raises(ValueError, match="mask has shape"):
        mg.token_log_probs(x, y, mask=turned(mask))
    # one order only: flat lists, flat logits, dimensions of one
    want = mg.token_log_probs(s["logits"], s["targets"], mask=s["mask"])
    for given in ((x, s["targets"], s["mask"]), (x, y[..., None], mask), (s["logits"], y, mask), (x[:, None], y, mask[None]),
                  (x, y, s["mask"])):
        assert same_bits([mg.token_log_probs(given[0], given[1], mask=given[2]).flatten()], [want])
    assert mg.token_log_probs(x[:0], y[:0]).shape == (0, 4) and mg.token_log_probs(x[:, :0], y[:, :0]).shape == (3, 0)


def test_gradient_in_another_order_than_the_checkpoint():
    """A gradient has to be laid out as the activation was."""
    gen = generator(4)
    x, up = randn(gen, (3, 4, 200), torch.bfloat16), randn(gen, (3, 4, 200), torch.bfloat16)
    dy = randn(gen, (3, 4, 200), torch.bfloat16)
    _, saved = mg.gated_act_pack(x, up)
    want = mg.gated_act_backward(dy, saved)
    for bad in (dy.transpose(0, 1), dy.view(2, 6, 200), dy[..., :130], dy.view(12, 200)[..., :199]):
        with pytest.raises(ValueError, match="the checkpoint is not one"):
            mg.gated_act_backward(bad, saved)
    for good in (dy.view(12, 200), dy[:, None], dy.view(1, 12, 200)):
        got = mg.gated_act_backward(good, saved)
        assert same_bits([g.flatten() for g in got], [w.flatten() for w in want])
    # a checkpoint put together again from its tensors knows its rows only
    got = mg.gated_act_backward(dy, mg.ActCheckpoint(saved.codes, saved.scales, "silu"))
    assert same_bits(got, want)


def test_tables_that_ask_for_a_gradient():
    gen = generator(5)
    q, k = randn(gen, (1, 3, 2, 32), torch.float32), randn(gen, (1, 3, 1, 32), torch.float32)
    w = torch.ones(32, device=DEV)
    cos, sin = mg.rope_tables(3, 32, device=DEV)
    want = mg.qk_norm_rope(q, k, w, w, cos, sin)
    for asks in (False, True):
        q.requires_grad_(asks)
        for name, c, s in (("cos", cos.clone().requires_grad_(True), sin), ("sin", cos, sin.clone().requires_grad_(True))):
            with pytest.raises(ValueError, match=f"no gradient by {name}"):
                mg.qk_norm_rope(q, k, w, w, c, s)
            with torch.no_grad():
                assert same_bits(mg.qk_norm_rope(q, k, w, w, c, s), want)
