"""CPU-only checks of the training-step operators' C ABI and host layer (no GPU
work is launched)."""

from __future__ import annotations

import ctypes
import importlib
import re
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
P = 0x1000      # an address that no call here reaches
E_INVALID, E_ALIGN, E_LIMIT = 10001, 10002, 10003


@pytest.fixture(scope="module")
def native():
    return importlib.import_module("minigpt-train-infra_amd._native")


def test_library_exports_every_declared_operator(native):
    lib = native.load_library()
    header = (ROOT / "include" / "mgopt_ops.h").read_text()
    declared = set(re.findall(r"MGOPT_API\s+[\w\s\*]+?\b(mgopt_\w+)\s*\(", header))
    assert declared == set(native.OPS_EXPORTS)
    for name in declared:
        assert getattr(lib, name) is not None


def test_operator_header_is_c99_and_cxx(tmp_path):
    src = tmp_path / "include.c"
    src.write_text('#include "mgopt_ops.h"\nint main(void) { return 0; }\n')
    inc = str(ROOT / "include")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", inc, "-fsyntax-only", str(src)],
                   check=True)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-x", "c++", "-I", inc,
                    str(src)], check=True)


def _refused(lib, rc, code, text):
    assert rc == code and text in lib.mgopt_last_error(), (rc, lib.mgopt_last_error())


def test_embedding_rejects_bad_arguments(native):
    lib = native.load_library()
    vp, i64, f = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    lib.mgopt_embedding_grad_workspace.restype = i64
    assert lib.mgopt_embedding_grad_workspace(i64(10), i64(10), i64(10)) > 0
    for bad in ((-1, 10, 10), (10, 0, 10), (10, 10, 0)):
        assert lib.mgopt_embedding_grad_workspace(*map(i64, bad)) == -1

    def lookup(ids=P, id_bytes=8, n=4, weight=P, wd=0, rows=5, width=8, scale=1.0, out=P, od=0):
        return lib.mgopt_embedding(vp(ids), id_bytes, i64(n), vp(weight), wd, i64(rows), i64(width), f(scale), vp(out), od,
                                   vp(None))

    def grad(ids=P, id_bytes=8, n=4, grad_out=P, wd=0, dst=P, od=0, rows=5, width=8, scale=1.0, pad=-1, acc=1, work=P):
        return lib.mgopt_embedding_grad(vp(ids), id_bytes, i64(n), vp(grad_out), wd, vp(dst), od, i64(rows), i64(width),
                                        f(scale), i64(pad), acc, vp(work), vp(None))

    for call in (lookup, grad):
        for bad in (dict(id_bytes=2), dict(n=-1), dict(rows=0), dict(width=0), dict(wd=3), dict(od=-1), dict(ids=None),
                    dict(scale=float("nan"))):
            _refused(lib, call(**bad), E_INVALID, b"embedding")
    for bad in (dict(weight=None), dict(out=None)):
        _refused(lib, lookup(**bad), E_INVALID, b"NULL")
    for bad in (dict(grad_out=None), dict(dst=None), dict(pad=5), dict(pad=-2)):
        _refused(lib, grad(**bad), E_INVALID, b"embedding_grad")
    for bad in (dict(work=None), dict(work=P + 8)):
        _refused(lib, grad(**bad), E_ALIGN, b"workspace")
    for bad in (dict(n=2**30), dict(rows=2**31, n=1000), dict(n=2**29, width=2**20)):
        _refused(lib, grad(**bad), E_LIMIT, b"embedding_grad")
    assert lookup(n=0) == 0 and grad(n=0) == 0


def _gated_act(lib, gate=P, up=None, dtype=0, rows=4, width=8, act=0, y=P, codes=None, scales=None):
    vp, i64 = ctypes.c_void_p, ctypes.c_int64
    return lib.mgopt_gated_act(vp(gate), i64(8), vp(up), i64(8), dtype, i64(rows), i64(width), act, vp(y), vp(codes),
                               vp(scales), vp(None))


def test_gated_act_rejects_bad_arguments(native):
    lib = native.load_library()
    for bad in (dict(dtype=7), dict(rows=-1), dict(width=0), dict(act=2), dict(gate=None), dict(y=None),
                dict(codes=P), dict(scales=P)):
        _refused(lib, _gated_act(lib, **bad), E_INVALID, b"gated_act")
    _refused(lib, _gated_act(lib, codes=P + 4, scales=P), E_ALIGN, b"8-byte")
    assert _gated_act(lib, gate=None, rows=0) == 0


class PolicyArgs(ctypes.Structure):            # mgopt_policy_args
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "targets", "old_logp", "advantages", "ref_logp", "mask",
                                               "grad_scale", "log_probs", "d_logits", "workspace")]
    _fields_ += [(n, ctypes.c_int64) for n in ("rows", "vocab", "logits_stride", "d_logits_stride")]
    _fields_ += [(n, ctypes.c_double) for n in ("clip_low", "clip_high", "kl_coef", "temperature")]
    _fields_ += [(n, ctypes.c_int32) for n in ("dtype", "target_bytes", "mask_kind", "reserved")]


def _policy(**more):
    a = PolicyArgs(logits=P, targets=P, old_logp=P, advantages=P, log_probs=P, d_logits=P, workspace=P, rows=4, vocab=8,
                   logits_stride=8, d_logits_stride=8, clip_low=0.2, clip_high=0.2, temperature=1.0, target_bytes=8)
    for k, v in more.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_policy_loss_rejects_bad_arguments(native):
    lib = native.load_library()
    vp = ctypes.c_void_p
    lib.mgopt_policy_workspace.restype = ctypes.c_int64
    assert lib.mgopt_policy_workspace(ctypes.c_int64(100)) >= 2400 and lib.mgopt_policy_workspace(ctypes.c_int64(-1)) == -1
    calls = {"log_probs": lambda a: lib.mgopt_token_log_probs(a, vp(None)),
             "policy_loss": lambda a: lib.mgopt_policy_loss(a, vp(P), vp(P), vp(None)),
             "backward": lambda a: lib.mgopt_policy_loss_backward(a, vp(None))}
    for name, call in calls.items():
        for bad in (dict(dtype=5), dict(rows=-1), dict(vocab=0), dict(target_bytes=2), dict(mask_kind=3),
                    dict(temperature=0.0), dict(temperature=float("nan")), dict(logits=None), dict(targets=None),
                    dict(log_probs=None), dict(mask_kind=1), dict(mask=P)):
            _refused(lib, call(_policy(**bad)), E_INVALID, name.encode())
        _refused(lib, call(None), E_INVALID, b"NULL")
        if name != "log_probs":
            for bad in (dict(clip_low=-0.1), dict(clip_high=float("nan")), dict(old_logp=None), dict(advantages=None)):
                _refused(lib, call(_policy(**bad)), E_INVALID, name.encode())
            for bad in (dict(workspace=None), dict(workspace=P + 8)):
                _refused(lib, call(_policy(**bad)), E_ALIGN, b"workspace")
    _refused(lib, calls["backward"](_policy(d_logits=None)), E_INVALID, b"NULL")
    _refused(lib, lib.mgopt_policy_loss(_policy(), vp(None), vp(P), vp(None)), E_INVALID, b"NULL")
    assert calls["log_probs"](_policy(rows=0)) == 0 and calls["backward"](_policy(rows=0)) == 0


def test_policy_loss_rejects_temperatures_beyond_32_bits(native):
    """log2(e) / T has to be a normal 32-bit number."""
    lib, vp = native.load_library(), ctypes.c_void_p
    for bad in (2.0**-121, 2.0**121, float("inf"), -1.0):
        for rc in (lib.mgopt_token_log_probs(_policy(temperature=bad), vp(None)),
                   lib.mgopt_policy_loss(_policy(temperature=bad), vp(P), vp(P), vp(None)),
                   lib.mgopt_policy_loss_backward(_policy(temperature=bad), vp(None))):
            _refused(lib, rc, E_INVALID, b"temperature")


class Heads(ctypes.Structure):                 # mgopt_heads
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "out", "grad", "d_x", "d_weight")]
    _fields_ += [(n, ctypes.c_int64 * 3) for n in ("x_stride", "out_stride", "grad_stride", "d_x_stride")]
    _fields_ += [("heads", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class QkArgs(ctypes.Structure):                # mgopt_qk_args
    _fields_ = [("q", Heads), ("k", Heads)]
    _fields_ += [(n, ctypes.c_void_p) for n in ("cos", "sin", "positions", "workspace")]
    _fields_ += [(n, ctypes.c_int64) for n in ("table_rows", "position_stride", "batch", "length")]
    _fields_ += [(n, ctypes.c_int32) for n in ("dim", "rotary", "dtype", "weight_dtype", "position_bytes", "interleaved")]
    _fields_ += [("eps", ctypes.c_float), ("reserved", ctypes.c_int32)]


def _qk(side=None, **more):
    heads = dict(x=P, weight=P, out=P, grad=P, d_x=P, d_weight=P, heads=2)
    a = QkArgs(q=Heads(**heads), k=Heads(**heads), cos=P, sin=P, workspace=P, table_rows=4, batch=1, length=2, dim=64,
               rotary=64, eps=1e-6)
    for k, v in more.items():
        setattr(a if side is None else getattr(a, side), k, v)
    return ctypes.byref(a)


def test_qk_norm_rope_rejects_bad_arguments(native):
    lib = native.load_library()
    vp = ctypes.c_void_p
    lib.mgopt_qk_norm_rope_workspace.restype = ctypes.c_int64
    assert lib.mgopt_qk_norm_rope_workspace(64) > 0 and lib.mgopt_qk_norm_rope_workspace(0) == -1
    forward, backward = lib.mgopt_qk_norm_rope, lib.mgopt_qk_norm_rope_backward
    for call in (forward, backward):
        for bad in (dict(dtype=3), dict(weight_dtype=-1), dict(batch=-1), dict(length=-1), dict(dim=0), dict(rotary=63),
                    dict(rotary=66), dict(rotary=-2), dict(eps=-1.0), dict(eps=float("nan")), dict(cos=None), dict(sin=None),
                    dict(positions=P, position_bytes=2)):
            _refused(lib, call(_qk(**bad), vp(None)), E_INVALID, b"qk_norm_rope")
        for bad in (dict(dim=514, rotary=64), dict(batch=2**20, length=2**20)):
            _refused(lib, call(_qk(**bad), vp(None)), E_LIMIT, b"more than")
        for side in ("q", "k"):
            for bad in (dict(heads=0), dict(x=None), dict(weight=None)):
                _refused(lib, call(_qk(side, **bad), vp(None)), E_INVALID, b"qk_norm_rope")
            _refused(lib, call(_qk(side, heads=2**21), vp(None)), E_LIMIT, b"heads")
        _refused(lib, call(None, vp(None)), E_INVALID, b"NULL")
    _refused(lib, forward(_qk("k", out=None), vp(None)), E_INVALID, b"NULL")
    for call in (forward, backward):
        many = _qk(batch=2**10, length=2**18)._obj
        many.q.heads = 2**20
        _refused(lib, call(ctypes.byref(many), vp(None)), E_LIMIT, b"too many heads")
    for bad in (dict(grad=None), dict(d_x=None), dict(d_weight=None)):
        _refused(lib, backward(_qk("q", **bad), vp(None)), E_INVALID, b"NULL")
    _refused(lib, backward(_qk(workspace=None), vp(None)), E_ALIGN, b"workspace")
    assert forward(_qk(batch=0), vp(None)) == 0


def test_argument_structs_match_the_header(tmp_path):
    """The sizes of the structs as gcc lays them out are those declared here."""
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "mgopt_ops.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   "sizeof(mgopt_policy_args), sizeof(mgopt_heads), sizeof(mgopt_qk_args)); return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(c) for c in (PolicyArgs, Heads, QkArgs)]


def test_operators_have_no_cpu_path(mg):
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    with pytest.raises(RuntimeError, match="no CPU"):
        mg.gated_act(torch.ones(3, 4))
    with pytest.raises(RuntimeError, match="no CPU"):
        mg.embedding(torch.zeros(3, dtype=torch.int64), torch.ones(3, 4))
    with pytest.raises(RuntimeError, match="no CPU"):
        mg.token_log_probs(torch.ones(3, 4), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU"):
        x, w = torch.ones(1, 2, 3, 4), torch.ones(4)
        mg.qk_norm_rope(x, x, w, w, *mg.rope_tables(2, 4))
