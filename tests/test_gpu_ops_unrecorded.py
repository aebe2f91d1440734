"""Calls that record nothing for autograd (attention_lse, rms_norm_int8, int8_rows,
int8_linear) where something watches: a trace holds them, a tangent is not
dropped, and inputs that ask for a gradient give results that do not."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests._ops import generator, mg, randn, same_bits

pytestmark = pytest.mark.gpu


def flat(*results):
    """The results' tensors in one list; codes as float32, so that same_bits takes them."""
    out = []
    for r in results:
        out += flat(*r) if isinstance(r, (tuple, list)) else [r.float() if r.dtype == torch.int8 else r]
    return out


def calls():
    gen = generator(1)
    x, res = randn(gen, (6, 48), torch.bfloat16), randn(gen, (6, 48), torch.bfloat16)
    w, bias = randn(gen, (48,), torch.bfloat16), randn(gen, (20,), torch.bfloat16)
    heads, values = randn(gen, (1, 9, 2, 32), torch.bfloat16), randn(gen, (1, 9, 2, 32), torch.bfloat16)
    w8 = mg.int8_rows(randn(gen, (20, 48), torch.bfloat16))
    x8 = mg.int8_rows(x)
    return {"int8_rows": (lambda t: tuple(mg.int8_rows(t)), (x,)),
            "rms_norm_int8": (lambda t: (*mg.rms_norm_int8(t, w)[0], mg.rms_norm_int8(t, w)[1]), (x,)),
            "rms_norm_int8 with a residual": (lambda t, r: (*mg.rms_norm_int8(t, w, residual=r)[0],
                                                            mg.rms_norm_int8(t, w, residual=r)[1]), (x, res)),
            "int8_linear": (lambda s: mg.int8_linear(mg.Int8Rows(x8.codes, s), w8, bias), (x8.scales,)),
            "a layer": (lambda t: mg.int8_linear(mg.int8_rows(t), w8, dtype=torch.float32), (x,)),
            "attention_lse": (lambda t: mg.attention_lse(t, t, values), (heads,))}


@pytest.mark.parametrize("name", ["int8_rows", "rms_norm_int8", "rms_norm_int8 with a residual", "int8_linear", "a layer",
                                  "attention_lse"])
def test_a_trace_holds_the_call(name):
    f, given = calls()[name]
    with pytest.warns(DeprecationWarning):
        traced = torch.jit.trace(f, given)
    other = tuple(t * 2 + 1 for t in given)
    want, got = flat(f(*other)), flat(traced(*other))
    assert same_bits(got, want) and not same_bits(want, flat(f(*given)))


def test_a_traced_call_runs_on_the_current_stream():
    """Behind what that stream has yet to do, which writes the input."""
    for name, (f, given) in calls().items():
        with pytest.warns(DeprecationWarning):
            traced = torch.jit.trace(f, given)
        other = tuple(t * 2 + 1 for t in given)
        want = flat(f(*other))
        late = tuple(torch.zeros_like(t) for t in given)
        for _ in range(3):
            flat(traced(*late))                 # whatever the first runs of a trace prepare
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            for a, b in zip(late, other):
                a.copy_(b)
            got = traced(*late)
        side.synchronize()
        assert same_bits(flat(got), want), name


@pytest.mark.parametrize("name", ["int8_rows", "rms_norm_int8", "rms_norm_int8 with a residual", "int8_linear", "attention_lse"])
def test_no_tangent_is_dropped(name):
    f, given = calls()[name]
    plain = flat(f(*given))
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            f(*(forward_ad.make_dual(t, torch.ones_like(t)) for t in given))
        assert same_bits(flat(f(*given)), plain)     # inputs without a tangent are served


def test_inputs_that_ask_for_a_gradient():
    """As documented: results that ask for none, the same bits."""
    for name in ("int8_rows", "attention_lse"):
        f, given = calls()[name]
        asks = tuple(t.clone().requires_grad_(True) for t in given)
        got = f(*asks)
        assert not any(t.requires_grad for t in got) and same_bits(flat(got), flat(f(*given)))
