"""The operators together, as a training step and a rollout use them: a decoder
block's loss and gradients against the same block in plain operations in 64
bits; tokens generated one by one over a cache against the whole sequence; the
block's projections in 8 bits."""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from tests._ops import DEV, generator, mg, randn, same_bits

pytestmark = pytest.mark.gpu
V, W, H, HK, D, I = 96, 128, 4, 2, 32, 160


def weights(dtype, seed=1, grad=False):
    gen = generator(seed)
    shapes = {"embed": (V, W), "qkv": ((H + 2 * HK) * D, W), "out": (W, H * D), "up": (2 * I, W), "down": (W, I), "head": (V, W)}
    p = {n: randn(gen, s, dtype, 0.1) for n, s in shapes.items()}
    p |= {n: randn(gen, s, dtype, 0.1).add_(1.0) for n, s in (("n1", (W,)), ("n2", (W,)), ("n3", (W,)), ("qn", (D,)), ("kn", (D,)))}
    return {n: t.requires_grad_(grad) for n, t in p.items()}


def block(p, ids, offsets, positions, cos, sin):
    """(logits, stream) over packed sequences."""
    x = mg.embedding(ids, p["embed"])[None]
    y = mg.rms_norm(x, p["n1"])
    q, k, v = F.linear(y, p["qkv"]).view(1, -1, H + 2 * HK, D).split((H, HK, HK), 2)
    q, k = mg.qk_norm_rope(q, k, p["qn"], p["kn"], cos, sin, positions, heads_first=True)
    a = mg.attention(q, k, v.transpose(1, 2), offsets=offsets, heads_first=True)
    y, x = mg.add_rms_norm(F.linear(a.flatten(2), p["out"]), x, p["n2"])
    gate, up = F.linear(y, p["up"]).chunk(2, -1)
    y, x = mg.add_rms_norm(F.linear(mg.gated_act(gate, up), p["down"]), x, p["n3"])
    return F.linear(y, p["head"]), x


def plain(p, ids, parts, cos, sin):
    """The same in torch's operations, sequence by sequence."""
    norm = lambda x, w: x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731

    def turn(x, w):
        x = norm(x, w)
        a, b = x.chunk(2, -1)
        c, s = cos[: x.shape[0], None].to(x.dtype), sin[: x.shape[0], None].to(x.dtype)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    out = []
    for at in parts:
        x = p["embed"][ids[at]]
        n = x.shape[0]
        q, k, v = F.linear(norm(x, p["n1"]), p["qkv"]).view(n, -1, D).split((H, HK, HK), 1)
        q, k = turn(q, p["qn"]), turn(k, p["kn"]).repeat_interleave(H // HK, 1)
        s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * D**-0.5
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), float("-inf")).softmax(-1)
        a = torch.matmul(s, v.repeat_interleave(H // HK, 1).transpose(0, 1).contiguous()).transpose(0, 1).reshape(n, H * D)
        x = x + F.linear(a, p["out"])
        gate, up = F.linear(norm(x, p["n2"]), p["up"]).chunk(2, -1)
        x = x + F.linear(F.silu(gate) * up, p["down"])
        out.append(F.linear(norm(x, p["n3"]), p["head"]))
    return torch.cat(out)


def test_gradients_of_a_packed_block():
    """Float32.  The forward pass agrees to rounding; the gradients behind the
    activation come from its 8-bit checkpoint (half a code, 1/254 of a group's
    largest, about 3 standard deviations: 0.7 % of a value as a root mean square)
    and are within 3 %, the head's and the last norm's, above it, within 1e-4."""
    lengths = [37, 1, 0, 90, 12]
    at = [0] + torch.tensor(lengths).cumsum(0).tolist()
    parts = [slice(a, b) for a, b in zip(at, at[1:]) if b > a]
    ids = torch.randint(0, V, (at[-1],), generator=generator(2), device=DEV)
    positions = torch.cat([torch.arange(n) for n in lengths]).to(DEV)[None]
    cos, sin = mg.rope_tables(100, D, device=DEV)
    targets = torch.randint(0, V, (at[-1],), generator=generator(3), device=DEV)
    p = weights(torch.float32, grad=True)
    logits, _ = block(p, ids, torch.tensor(at, dtype=torch.int32, device=DEV), positions, cos, sin)
    old = mg.token_log_probs(logits.detach()[0], targets) - 0.05
    adv = randn(generator(4), (at[-1],), torch.float32)
    mg.policy_loss(logits[0], targets, old, adv).loss.backward()
    exact = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    z = plain(exact, ids, parts, cos, sin)
    assert float((z - logits[0]).abs().max()) < 1e-4 * float(z.abs().max())
    logp = torch.log_softmax(z, -1).gather(1, targets[:, None])[:, 0]
    ratio = (logp - old.double()).exp()
    (-torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv).mean()).backward()
    for n, t in p.items():
        off = float((t.grad - exact[n].grad).norm() / exact[n].grad.norm())
        assert off < (1e-4 if n in ("head", "n3") else 0.03), (n, off)


def test_a_step_without_the_checkpoint_is_exact():
    """Without the activation between them, norms and attention alone: 1e-5."""
    ids = torch.randint(0, V, (3, 70), generator=generator(5), device=DEV)
    p, gen = weights(torch.float32, grad=True), generator(6)
    g = randn(gen, (3, 70, W), torch.float32)

    def run(p, norm, attend):
        x = F.embedding(ids, p["embed"])
        q, k, v = F.linear(norm(x, p["n1"]), p["qkv"]).view(3, 70, -1, D).split((H, HK, HK), 2)
        x = x + F.linear(attend(q, k, v).flatten(2), p["out"])
        return norm(x, p["n2"])

    def attend(q, k, v):
        k, v = (t.repeat_interleave(H // HK, 2).transpose(1, 2) for t in (k, v))
        s = torch.matmul(q.transpose(1, 2), k.transpose(-1, -2).contiguous()) * D**-0.5
        s = s.masked_fill(~torch.ones(70, 70, dtype=torch.bool, device=DEV).tril(), float("-inf")).softmax(-1)
        return torch.matmul(s, v.contiguous()).transpose(1, 2)

    run(p, mg.rms_norm, mg.attention).backward(g)
    exact = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    run(exact, lambda x, w: x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w, attend).backward(g.double())
    for n in ("embed", "n1", "qkv", "out", "n2"):
        off = float((p[n].grad - exact[n].grad).norm() / exact[n].grad.norm())
        assert off < 1e-5, (n, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_over_a_cache_give_the_whole_sequence(dtype):
    """A prompt, then one token at a time over the cache: each row's attention is
    near the row of the whole sequence's (the sums run in another order: the
    type's rounding of out, twice, and of the probabilities)."""
    gen, B, N, prompt = generator(7), 3, 40, 25
    q, k, v = randn(gen, (B, N, H, D), dtype), randn(gen, (B, N, HK, D), dtype), randn(gen, (B, N, HK, D), dtype)
    want = mg.attention(q, k, v).float()
    cache = [torch.full((B, 64, HK, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    filled = torch.full((B,), prompt, dtype=torch.int32, device=DEV)
    for c, t in zip(cache, (k, v)):
        c[:, :prompt] = t[:, :prompt]
    bound = 4 * torch.finfo(dtype).eps / 2 * float(v.float().abs().max()) + 1e-5
    got = mg.attention(q[:, :prompt], *cache, key_lengths=filled)
    assert float((got.float() - want[:, :prompt]).abs().max()) < bound
    for i in range(prompt, N):
        for c, t in zip(cache, (k, v)):
            c[:, i] = t[:, i]
        filled += 1
        got = mg.attention(q[:, i:i + 1], *cache, key_lengths=filled)
        assert float((got.float() - want[:, i:i + 1]).abs().max()) < bound


def test_a_block_in_8_bits():
    """A rollout's forward pass with 8-bit projections beside the 16-bit one: each
    product is off by half a code of both factors, 0.7 % of a value each as a root
    mean square, and the five of them in the block by some 3 %."""
    ids = torch.randint(0, V, (8, 33), generator=generator(8), device=DEV)
    p = weights(torch.bfloat16)
    cos, sin = mg.rope_tables(33, D, device=DEV)
    w8 = {n: mg.int8_rows(p[n]) for n in ("qkv", "out", "up", "down", "head")}
    with torch.no_grad():
        x = mg.embedding(ids, p["embed"])
        y, x = mg.rms_norm_int8(x, p["n1"])
        q, k, v = mg.int8_linear(y, w8["qkv"]).view(8, 33, -1, D).split((H, HK, HK), 2)
        q, k = mg.qk_norm_rope(q, k, p["qn"], p["kn"], cos, sin)
        a = mg.attention(q, k, v)
        y, x = mg.rms_norm_int8(mg.int8_linear(mg.int8_rows(a.flatten(2)), w8["out"]), p["n2"], residual=x)
        gate, up = mg.int8_linear(y, w8["up"]).chunk(2, -1)
        y, x = mg.rms_norm_int8(mg.int8_linear(mg.int8_rows(mg.gated_act(gate, up)), w8["down"]), p["n3"], residual=x)
        got = mg.int8_linear(y, w8["head"], dtype=torch.float32)
        again = mg.int8_linear(y, w8["head"], dtype=torch.float32)
        offsets = torch.arange(0, 8 * 33 + 1, 33, device=DEV)
        positions = torch.arange(33, device=DEV).repeat(8)[None]
        want, _ = block(p, ids.flatten(), offsets, positions, cos, sin)
    assert same_bits([got], [again])
    off = float((got.flatten(0, 1) - want[0].float()).norm() / want.float().norm())
    assert off < 0.06, off


def test_two_streams_at_once():
    """Calls of one operator on two streams overlap without sharing anything."""
    gen = generator(9)
    sets = [(randn(gen, (1, 300, 8, 64), torch.bfloat16), randn(gen, (1, 900, 2, 64), torch.bfloat16),
             randn(gen, (1, 900, 2, 64), torch.bfloat16)) for _ in range(2)]
    codes = [mg.int8_rows(randn(gen, (n, 512), torch.bfloat16)) for n in (40, 300, 1000)]

    def work(s):
        out, lse = mg.attention_lse(*s)
        return [out, lse, *mg.attention_backward(out, *s, out, lse), mg.attention(s[0][:, :1], s[1], s[2]),
                mg.int8_linear(codes[0], codes[2]), mg.int8_linear(codes[1], codes[2])]

    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(work(s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(same_bits([a], [b]) for a, b in zip(g, want[i % 2]))
