"""Attention, the norm before it and 8-bit products, as cases to measure.

Each case is one pass through one operator, as a program calls it:

  attention    softmax(q k^T scale) v of grouped heads and its backward pass, over
               a batch, over packed sequences, or of a few new tokens over a cache
  rms_norm     the residual's addition and the RMS norm of the sum, with the
               backward pass ("train") or without ("forward")
  int8_linear  a product of 8-bit integers with a scale per token and per output
               channel; its input comes in 8 bits ("codes"), is rounded to 8 bits
               first ("rows"), or comes out of the norm in 8 bits ("norm")

`own` selects the framework's kernels; otherwise the same results come from
elementary torch operations in 32 bits, rounded once at the end.  exact() is
the definition in 64 bits.
"""

from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _mg():
    return importlib.import_module("minigpt-train-infra_amd")


# ----------------------------------------------------------------- the cases


def listed():
    return [
        # the tiny CPU configuration's attention: 8 sequences of 128 tokens, four heads of 32, fp32, launch-bound
        {"name": "attn_tiny", "op": "attention", "mode": "train", "layout": "batch", "batch": 8, "queries": 128, "keys": 128,
         "q_heads": 4, "k_heads": 4, "dim": 32, "dtype": "f32", "causal": True, "heads_first": True, "fused": False},
        # GPT-2-small over a micro-batch of packed documents of very different lengths, one of them empty
        {"name": "attn_packed", "op": "attention", "mode": "train", "layout": "packed", "batch": 23, "queries": 8183,
         "keys": 8183, "q_heads": 12, "k_heads": 12, "dim": 64, "dtype": "f16", "causal": True, "heads_first": False,
         "fused": True},
        # Qwen3-8B in training: 32 + 8 heads of 128, laid out as the norms and the rotation leave them
        {"name": "attn_qwen3", "op": "attention", "mode": "train", "layout": "batch", "batch": 2, "queries": 4096,
         "keys": 4096, "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "causal": True, "heads_first": True,
         "fused": False},
        # generation for a rollout: 64 sequences, one new token each, caches of up to 4,096 tokens filled unevenly
        {"name": "attn_token", "op": "attention", "mode": "forward", "layout": "cache", "batch": 64, "queries": 1,
         "keys": 4096, "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "causal": True, "heads_first": False,
         "fused": False},
        # one sequence's next token over a long cache
        {"name": "attn_long", "op": "attention", "mode": "forward", "layout": "cache", "batch": 1, "queries": 1,
         "keys": 131_071, "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "causal": True, "heads_first": False,
         "fused": False},
        # the tiny configuration's width
        {"name": "norm_tiny", "op": "rms_norm", "mode": "train", "rows": 1024, "width": 128, "dtype": "f32", "add": True},
        # fp16 rows that do not start on 16 bytes
        {"name": "norm_odd", "op": "rms_norm", "mode": "train", "rows": 2049, "width": 2731, "dtype": "f16", "add": True},
        # Qwen3-8B's residual stream over 8,192 tokens
        {"name": "norm_qwen3", "op": "rms_norm", "mode": "train", "rows": 8192, "width": 4096, "dtype": "bf16", "add": True},
        # one token of one sequence through a GPT-2-small projection with a bias
        {"name": "int8_one", "op": "int8_linear", "input": "rows", "rows": 1, "width": 768, "channels": 2304, "dtype": "f16",
         "bias": True},
        # a rollout's 64 tokens from the residual stream through Qwen3-8B's gate projection
        {"name": "int8_token", "op": "int8_linear", "input": "norm", "rows": 64, "width": 4096, "channels": 12288,
         "dtype": "bf16", "bias": False},
        # sizes that no tile divides, fp32 outputs
        {"name": "int8_odd", "op": "int8_linear", "input": "rows", "rows": 1023, "width": 2731, "channels": 1371,
         "dtype": "f32", "bias": True},
        # the prompts' 8,192 tokens through Qwen3-8B's gate projection
        {"name": "int8_qwen3", "op": "int8_linear", "input": "codes", "rows": 8192, "width": 4096, "channels": 12288,
         "dtype": "bf16", "bias": False},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high, step):
    """A size spread over its logarithm: half of them multiples of `step`, the others as they fall."""
    n = _log_int(rng, low, high)
    return max(step, n // step * step) if rng.random() < 0.5 and high >= step else n


def draw(rng):
    op = rng.choice(["attention", "attention", "rms_norm", "int8_linear"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "attention":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 1, 2, 3, 4, 8])
        layout = rng.choice(["batch", "packed", "cache"])
        case = {"op": op, "mode": "forward" if layout == "cache" else rng.choice(["forward", "train", "train"]),
                "layout": layout}
        if layout == "cache":
            batch = _log_int(rng, 1, 64)
            keys = _log_int(rng, 16, max(16, min(131_071, 250_000_000 // (batch * k_heads * dim * BYTES[dtype]))))
            queries = rng.choice([1, 1, 2, 5])
        else:
            # the plain form's scores: heads * tokens^2 values, with the batch's tokens in one row where they are packed
            most = 1_000_000_000 // q_heads
            if layout == "packed":
                batch, queries = rng.choice([1, 2, 7, 30]), _size(rng, 64, min(8192, int(math.sqrt(most))), 64)
            else:
                batch = rng.choice([1, 2, 3, 8])
                queries = _size(rng, 1, min(4096, int(math.sqrt(most / batch))), 64)
            keys = queries
        return case | {"batch": batch, "queries": queries, "keys": keys, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
                       "dtype": dtype, "causal": layout == "cache" or rng.random() < 0.8, "heads_first": rng.random() < 0.5,
                       "fused": layout != "cache" and rng.random() < 0.5}
    if op == "rms_norm":
        width = _size(rng, 64, 16384, 64)
        return {"op": op, "mode": rng.choice(["forward", "train", "train"]),
                "rows": _log_int(rng, 1, min(16384, 67_000_000 // (width * BYTES[dtype]))), "width": width, "dtype": dtype,
                "add": rng.random() < 0.7}
    width, channels = _size(rng, 64, 12288, 64), _size(rng, 64, 12288, 64)
    rows = _log_int(rng, 1, min(8192, 400_000_000_000 // (width * channels)))
    return {"op": op, "input": rng.choice(["codes", "rows", "norm"]), "rows": rows, "width": width, "channels": channels,
            "dtype": dtype, "bias": rng.random() < 0.5}


def _lengths(case):
    """The lengths of packed sequences (they sum to the tokens), or the filled parts of the caches."""
    n, total = case["batch"], case["keys"]
    rng = random.Random(n * 1_000_003 + total)
    if case["layout"] == "cache":
        return [max(case["queries"], total - rng.randrange(total // 2 + 1)) for _ in range(n)]
    share = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(n)]
    if n > 2:
        share[rng.randrange(n)] = 0.0
    ends = [round(total * sum(share[:i + 1]) / sum(share)) for i in range(n)]
    return [b - a for a, b in zip([0] + ends, ends)]


# ---------------------------------------------------------------- the inputs


def _randn(gen, shape, dtype, sigma=1.0):
    out = torch.empty(shape, dtype=dtype, device=DEV)
    return out.normal_(0.0, sigma, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "attention":
        Hq, Hk, D, first = case["q_heads"], case["k_heads"], case["dim"], case["heads_first"]
        B = 1 if case["layout"] == "packed" else case["batch"]
        N, M = case["queries"], case["keys"]
        if case["fused"]:                   # slices of one projection's output
            x = _randn(gen, (B, N, Hq + 2 * Hk, D), dtype)
            parts = x[:, :, :Hq], x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:]
            s["q"], s["k"], s["v"] = (p.transpose(1, 2) if first else p for p in parts)
        else:
            shape = (lambda n, h: (B, h, n, D)) if first else (lambda n, h: (B, n, h, D))
            s["q"], s["k"], s["v"] = (_randn(gen, shape(n, h), dtype) for n, h in ((N, Hq), (M, Hk), (M, Hk)))
        s["q"].mul_(1.5)
        if case["layout"] == "packed":
            s["offsets"] = torch.tensor([0] + _lengths(case), device=DEV).cumsum(0).to(torch.int32)
        if case["layout"] == "cache":
            s["key_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
        if case["mode"] == "train":
            s["grad_out"] = _randn(gen, (B, N, Hq, D), dtype, 1e-2)
    elif case["op"] == "rms_norm":
        shape = (case["rows"], case["width"])
        s["x"] = _randn(gen, shape, dtype)
        s["residual"] = _randn(gen, shape, dtype, 2.0) if case["add"] else None
        s["weight"] = _randn(gen, shape[1:], dtype, 0.1).add_(1.0)
        if case["mode"] == "train":
            s["grad_y"] = _randn(gen, shape, dtype, 1e-2)
            s["grad_h"] = _randn(gen, shape, dtype, 1e-2) if case["add"] else None
    else:
        M, K, N = case["rows"], case["width"], case["channels"]
        w = _randn(gen, (N, K), torch.float32, 0.02)
        s["w_codes"], s["w_scales"] = _codes(w)
        s["bias"] = _randn(gen, (N,), dtype) if case["bias"] else None
        if case["input"] == "codes":
            s["codes"], s["scales"] = _codes(_randn(gen, (M, K), torch.float32))
        else:
            s["x"] = _randn(gen, (M, K), dtype)
        if case["input"] == "norm":
            s["residual"] = _randn(gen, (M, K), dtype, 2.0)
            s["weight"] = _randn(gen, (K,), dtype, 0.1).add_(1.0)
    return s


def _codes(x):
    """8-bit codes of x (fp32) and a scale for each row; the format is defined in 32 bits."""
    most = x.abs().amax(-1, keepdim=True)
    inv = torch.where(most >= 2.0**-119, torch.div(torch.full_like(most, 127.0), most), 0.0)
    return torch.round(x * inv).to(torch.int8), torch.where(most >= 2.0**-119, most * (1.0 / 127.0), 0.0)[:, 0]


# ----------------------------------------------------------------- one pass


def run(s):
    c = s["case"]
    return {"attention": _attention, "rms_norm": _rms_norm, "int8_linear": _int8_linear}[c["op"]](s, c)


def _attention(s, c):
    more = {"causal": c["causal"], "heads_first": c["heads_first"]}
    if c["layout"] == "packed":
        more["offsets"] = s["offsets"]
    if c["layout"] == "cache":
        more["key_lengths"] = s["key_lengths"]
    if own:
        mg = _mg()
        if c["mode"] == "forward":
            with torch.no_grad():
                return {"out": mg.attention(s["q"], s["k"], s["v"], **more)}
        out, lse = mg.attention_lse(s["q"], s["k"], s["v"], **more)
        dq, dk, dv = mg.attention_backward(s["grad_out"], s["q"], s["k"], s["v"], out, lse, **more)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    Hk, D, N, M = c["k_heads"], c["dim"], c["queries"], c["keys"]
    G, dtype = c["q_heads"] // Hk, DTYPES[c["dtype"]]
    turn = (lambda t: t) if c["heads_first"] else (lambda t: t.transpose(1, 2))
    q, k, v = (turn(s[n]).float().contiguous() for n in ("q", "k", "v"))
    B = q.shape[0]
    q = q.view(B, Hk, G * N, D)                                     # the heads that share keys, below each other
    # which keys a query sees: (sequences, queries, keys)
    row, col = torch.arange(N, device=DEV)[:, None], torch.arange(M, device=DEV)
    if c["layout"] == "packed":
        part = torch.bucketize(torch.arange(N, device=DEV), s["offsets"][1:-1].long(), right=True)
        seen = (part[:, None] == part)[None]
        if c["causal"]:
            seen = seen & (col <= row)
    elif c["layout"] == "cache":
        m = s["key_lengths"].long()[:, None, None]
        seen = (col < m) & ((col <= row + m - N) | (not c["causal"]))
    else:
        seen = (col <= row)[None] if c["causal"] else torch.ones((1, N, M), dtype=torch.bool, device=DEV)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, Hk, G, N, M).mul_(D**-0.5)
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.clamp_(min=-3e38)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30)).view(B, Hk, G * N, M)
    out = torch.matmul(p, v)
    back = lambda t: t.view(B, Hk * G, N, D).transpose(1, 2).to(dtype).contiguous()  # noqa: E731
    if c["mode"] == "forward":
        return {"out": back(out)}
    g = s["grad_out"].float().transpose(1, 2).contiguous().view(B, Hk, G * N, D)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), g)
    dp = torch.matmul(g, v.transpose(-1, -2).contiguous())
    dx = dp.sub_((g * out).sum(-1, keepdim=True)).mul_(p).mul_(D**-0.5)
    dq = torch.matmul(dx, k).view(B, Hk * G, N, D)
    dk = torch.matmul(dx.transpose(-1, -2).contiguous(), q)
    return {"out": back(out), **{n: turn(t).to(dtype).contiguous() for n, t in (("dq", dq), ("dk", dk), ("dv", dv))}}


def _normed(s, dtype):
    """(h, its rounded sum in fp32, 1 / sqrt(mean + eps), the normed row in fp32): the mean in 64 bits, so that the
    8-bit codes of the result do not hang on the order of a sum."""
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype)
    f = h.float()
    r = (f.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    return h, f, r, f * r * s["weight"].float()


def _rms_norm(s, c):
    dtype = DTYPES[c["dtype"]]
    if own:
        mg = _mg()
        with torch.no_grad():
            if c["add"]:
                y, h = mg.add_rms_norm(s["x"], s["residual"], s["weight"], eps=EPS)
            else:
                y, h = mg.rms_norm(s["x"], s["weight"], eps=EPS), s["x"]
            out = {"y": y, "h": h} if c["add"] else {"y": y}
            if c["mode"] == "train":
                out["dx"], out["dweight"] = mg.rms_norm_backward(s["grad_y"], h, s["weight"], grad_h=s["grad_h"], eps=EPS)
        return out
    h, f, r, y = _normed(s, dtype)
    out = {"y": y.to(dtype), "h": h} if c["add"] else {"y": y.to(dtype)}
    if c["mode"] == "train":
        g, xhat = s["grad_y"].float(), f * r
        gw = g * s["weight"].float()
        dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        out["dx"] = (dx + s["grad_h"].float() if c["add"] else dx).to(dtype)
        out["dweight"] = (g * xhat).sum(0).to(dtype)
    return out


def _int8_linear(s, c):
    dtype = DTYPES[c["dtype"]]
    if own:
        mg = _mg()
        weight = mg.Int8Rows(s["w_codes"], s["w_scales"])
        if c["input"] == "norm":
            x, h = mg.rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
            return {"y": mg.int8_linear(x, weight, s["bias"], dtype=dtype), "h": h}
        x = mg.int8_rows(s["x"]) if c["input"] == "rows" else mg.Int8Rows(s["codes"], s["scales"])
        return {"y": mg.int8_linear(x, weight, s["bias"], dtype=dtype)}
    out = {}
    if c["input"] == "norm":
        out["h"], _, _, y = _normed(s, dtype)
        codes, scales = _codes(y)
    else:
        codes, scales = _codes(s["x"].float()) if c["input"] == "rows" else (s["codes"], s["scales"])
    y = torch.matmul(codes.float(), s["w_codes"].float().t().contiguous())
    y.mul_(scales[:, None] * s["w_scales"])
    if c["bias"]:
        y.add_(s["bias"].float())
    return out | {"y": y.to(dtype)}


# ------------------------------------------------------- the smallest traffic


def _pairs(case):
    """(query, key) pairs of one head that count, over all sequences."""
    def one(n, m):
        return sum(max(0, min(m, i + 1 + m - n)) for i in range(n)) if n < 8 else n * m - n * (n - 1) // 2
    if case["layout"] == "batch":
        n = case["queries"]
        return case["batch"] * (n * (n + 1) // 2 if case["causal"] else n * n)
    if case["layout"] == "packed":
        return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
    return sum(one(case["queries"], m) for m in _lengths(case))


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "attention":
        D, rows, keys = case["dim"], case["queries"], case["keys"]
        if case["layout"] == "batch":
            rows, keys = rows * case["batch"], keys * case["batch"]
        if case["layout"] == "cache":
            rows, keys = rows * case["batch"], sum(_lengths(case))
        q, k = rows * case["q_heads"] * D * b, keys * case["k_heads"] * D * b
        pairs = _pairs(case) * case["q_heads"]
        if case["mode"] == "forward":
            return {"bytes": 2 * q + 2 * k, "flops": 4 * D * pairs}
        # forward: q, k, v read, out written; backward: those and the gradient read, three gradients written
        return {"bytes": (2 * q + 2 * k) + (4 * q + 4 * k), "flops": 14 * D * pairs}
    if case["op"] == "rms_norm":
        n, add = case["rows"] * case["width"], 1 if case["add"] else 0
        moved = n * b * (2 + 2 * add) + case["width"] * b
        if case["mode"] == "train":
            moved += n * b * (3 + add) + 2 * case["width"] * b
        return {"bytes": moved, "flops": n * (18 if case["mode"] == "train" else 6)}
    M, K, N = case["rows"], case["width"], case["channels"]
    read = {"codes": M * K + 4 * M, "rows": M * K * b, "norm": 3 * M * K * b}[case["input"]]
    return {"bytes": read + N * K + 4 * N + M * N * b, "flops": 2 * M * N * K}


# ------------------------------------------------------ the results in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rms_norm": _exact_rms_norm, "int8_linear": _exact_int8_linear}[case["op"]](s, case)


def _exact_attention(s, c):
    """Sequence by sequence and head by head; the gradients are autograd's of the definition."""
    group, train = c["q_heads"] // c["k_heads"], c["mode"] == "train"
    place = (lambda t, b, h: t[b, h]) if c["heads_first"] else (lambda t, b, h: t[b, :, h])
    names = ("q", "k", "v")
    grads = {"d" + n: torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) for n in names} if train else {}
    B, N, Hq, D = s["q"].shape[0], c["queries"], c["q_heads"], c["dim"]
    out = torch.zeros((B, N, Hq, D), dtype=torch.float64, device=DEV)
    lengths = _lengths(c) if c["layout"] != "batch" else [c["keys"]] * B
    start = 0
    for i, m in enumerate(lengths):
        b, n = (0, m) if c["layout"] == "packed" else (i, N)
        at, to = (start, start + m) if c["layout"] == "packed" else (0, m)
        start += m
        if m == 0:
            continue
        rows = slice(at, to) if c["layout"] == "packed" else slice(0, N)
        hidden = torch.ones((n, m), dtype=torch.bool, device=DEV).triu(1 + m - n) if c["causal"] else None
        for h in range(Hq):
            q, k, v = (place(s[t], b, h if t == "q" else h // group)[rows if t == "q" else slice(at, to)].double()
                       .requires_grad_(train) for t in names)
            x = (q @ k.t().contiguous()) / math.sqrt(D)
            if hidden is not None:
                x = x.masked_fill(hidden, float("-inf"))
            y = torch.softmax(x, -1) @ v
            out[b, rows, h] = y.detach()
            if train:
                for t, g in zip(names, torch.autograd.grad(y, (q, k, v), s["grad_out"][b, rows, h].double())):
                    place(grads["d" + t], b, h if t == "q" else h // group)[rows] += g
    return {"out": out} | grads


def _exact_rms_norm(s, c):
    with torch.no_grad():
        h = s["x"] if s["residual"] is None else (s["x"] + s["residual"])       # one rounding to the stream's type
        t, w = h.double(), s["weight"].double()
        size = torch.sqrt((t * t).sum(-1, keepdim=True) / c["width"] + EPS)
        out = {"y": t / size * w}
        if c["add"]:
            out["h"] = s["x"].double() + s["residual"].double()
        if c["mode"] == "train":
            g = s["grad_y"].double()
            dx = g * w / size - t * ((g * w * t).sum(-1, keepdim=True) / (c["width"] * size**3))
            out["dx"] = dx + s["grad_h"].double() if c["add"] else dx
            out["dweight"] = (g * t / size).sum(0)
    return out


def _exact_int8_linear(s, c):
    """The codes are as the format defines them, in 32 bits; their product and all after it in 64."""
    out = {}

    def held(x):
        most = x.abs().max(-1, keepdim=True).values
        inv = (127.0 / most.double()).float()
        return (x.double() * inv.double()).float().double().round() * (most * (1.0 / 127.0)).double()

    if c["input"] == "codes":
        x = s["codes"].double() * s["scales"].double()[:, None]
    elif c["input"] == "rows":
        x = held(s["x"].float())
    else:
        h = s["x"] + s["residual"]
        out["h"] = s["x"].double() + s["residual"].double()
        size = (1.0 / torch.sqrt((h.double() ** 2).sum(-1, keepdim=True) / c["width"] + EPS)).float()
        x = held(h.float() * size * s["weight"].float())
    y = x @ (s["w_codes"].double() * s["w_scales"].double()[:, None]).t().contiguous()
    return out | {"y": y + s["bias"].double() if c["bias"] else y}
