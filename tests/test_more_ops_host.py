"""CPU-only checks of the C ABI of attention, the residual's norm and the 8-bit
products, and of their host layer (no GPU work is launched)."""

from __future__ import annotations

import ctypes
import importlib
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
P = 0x1000      # an address that no call here reaches
E_INVALID, E_ALIGN, E_LIMIT = 10001, 10002, 10003
vp, i32, i64, f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_double


@pytest.fixture(scope="module")
def lib():
    lib = importlib.import_module("minigpt-train-infra_amd._native").load_library()
    for name in ("mgopt_rms_norm_workspace", "mgopt_attention_workspace"):
        getattr(lib, name).restype = i64
    return lib


def _refused(lib, rc, code, text):
    assert rc == code and text in lib.mgopt_last_error(), (rc, lib.mgopt_last_error())


def _norm(lib, x=P, res=None, weight=P, wd=0, dt=0, rows=4, width=64, eps=1e-6, h=None, y=P, codes=None, pitch=64, scales=None):
    return lib.mgopt_rms_norm(vp(x), i64(width), vp(res), i64(width), vp(weight), wd, dt, i64(rows), i64(width), f64(eps), vp(h),
                              vp(y), vp(codes), i64(pitch), vp(scales), vp(None))


def test_rms_norm_rejects_bad_arguments(lib):
    for bad in (dict(dt=3), dict(wd=-1), dict(rows=-1), dict(width=0), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None),
                dict(weight=None), dict(res=P), dict(h=P), dict(y=None), dict(codes=P, scales=P), dict(y=None, codes=P),
                dict(y=None, codes=P, scales=P, pitch=80)):
        _refused(lib, _norm(lib, **bad), E_INVALID, b"rms_norm")
    _refused(lib, _norm(lib, width=32769), E_LIMIT, b"32768")
    for bad in (dict(codes=P + 8), dict(codes=P, pitch=72), dict(codes=P, pitch=48)):
        _refused(lib, _norm(lib, y=None, scales=P, **bad), E_ALIGN, b"codes")
    assert _norm(lib, rows=0, x=None, y=None) == 0


def test_rms_norm_backward_rejects_bad_arguments(lib):
    assert lib.mgopt_rms_norm_workspace(i64(10), i64(64)) == 10 * 64 * 4
    assert lib.mgopt_rms_norm_workspace(i64(-1), i64(64)) == -1 and lib.mgopt_rms_norm_workspace(i64(1), i64(40000)) == -1

    def call(gy=P, gh=None, h=P, weight=P, wd=0, dt=0, rows=4, width=64, eps=1e-6, dx=P, dw=P, work=P):
        return lib.mgopt_rms_norm_backward(vp(gy), i64(width), vp(gh), i64(width), vp(h), i64(width), vp(weight), wd, dt, i64(rows),
                                           i64(width), f64(eps), vp(dx), vp(dw), vp(work), vp(None))

    for bad in (dict(dt=3), dict(wd=7), dict(rows=-1), dict(width=0), dict(eps=-1.0), dict(gy=None), dict(h=None),
                dict(weight=None), dict(dx=None)):
        _refused(lib, call(**bad), E_INVALID, b"rms_norm_backward")
    _refused(lib, call(width=32769), E_LIMIT, b"32768")
    for bad in (dict(work=None), dict(work=P + 8)):
        _refused(lib, call(**bad), E_ALIGN, b"workspace")
    assert call(rows=0, dw=None, work=None, gy=None) == 0


def test_int8_rejects_bad_arguments(lib):
    def rows(x=P, dt=0, n=4, width=30, codes=P, pitch=32, scales=P):
        return lib.mgopt_int8_rows(vp(x), i64(width), dt, i64(n), i64(width), vp(codes), i64(pitch), vp(scales), vp(None))

    def linear(x=P, sx=P, w=P, sw=P, bias=None, bd=0, n=4, width=32, channels=8, y=P, dt=0):
        return lib.mgopt_int8_linear(vp(x), i64(32), vp(sx), vp(w), i64(32), vp(sw), vp(bias), bd, i64(n), i64(width), i64(channels),
                                     vp(y), dt, vp(None))

    for bad in (dict(dt=4), dict(n=-1), dict(width=0), dict(x=None), dict(codes=None), dict(scales=None), dict(pitch=48)):
        _refused(lib, rows(**bad), E_INVALID, b"int8_rows")
    for bad in (dict(codes=P + 4), dict(pitch=31), dict(pitch=16)):
        _refused(lib, rows(**bad), E_ALIGN, b"int8_rows")
    assert rows(n=0, x=None) == 0
    for bad in (dict(dt=-1), dict(bias=P, bd=9), dict(n=-1), dict(width=0), dict(channels=-1), dict(x=None), dict(sx=None),
                dict(w=None), dict(sw=None), dict(y=None)):
        _refused(lib, linear(**bad), E_INVALID, b"int8_linear")
    _refused(lib, linear(width=131072), E_LIMIT, b"131071")
    _refused(lib, linear(n=2**40, channels=2**40), E_LIMIT, b"int8_linear")
    assert linear(n=0, x=None) == 0 and linear(channels=0, w=None) == 0


class AttentionArgs(ctypes.Structure):         # mgopt_attention_args
    _fields_ = [(n, vp) for n in ("q", "k", "v", "out", "lse", "grad_out", "d_q", "d_k", "d_v", "q_offsets", "k_offsets",
                                  "q_lengths", "k_lengths", "workspace")]
    _fields_ += [(n + "_stride", i64 * 3) for n in ("q", "k", "v", "out", "grad_out", "d_q", "d_k", "d_v")]
    _fields_ += [(n, i64) for n in ("batch", "queries", "keys", "sequences")] + [("scale", f64)]
    _fields_ += [(n, i32) for n in ("q_heads", "k_heads", "dim", "dtype", "offset_bytes", "causal")]


def _attention(**more):
    a = AttentionArgs(**{n: P for n in ("q", "k", "v", "out", "lse", "grad_out", "d_q", "d_k", "d_v", "workspace")}, batch=2,
                      queries=5, keys=7, scale=0.125, q_heads=4, k_heads=2, dim=64, causal=1)
    for k, v in more.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_attention_rejects_bad_arguments(lib):
    for call in (lib.mgopt_attention, lib.mgopt_attention_backward):
        go = lambda a: call(a, vp(None))  # noqa: E731
        for bad in (dict(dtype=3), dict(batch=-1), dict(queries=-1), dict(keys=-1), dict(q_heads=3), dict(k_heads=0), dict(dim=0),
                    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_offsets=P),
                    dict(q_offsets=P, k_offsets=P, offset_bytes=4), dict(batch=1, q_offsets=P, k_offsets=P, offset_bytes=2),
                    dict(batch=1, q_offsets=P, k_offsets=P, offset_bytes=8, q_lengths=P), dict(k_lengths=P), dict(q=None),
                    dict(k=None), dict(v=None), dict(out=None), dict(q_stride=(i64 * 3)(0, -1, 0)), dict(sequences=-1)):
            _refused(lib, go(_attention(**bad)), E_INVALID, b"attention")
        _refused(lib, go(None), E_INVALID, b"NULL")
        for bad in (dict(dim=129), dict(queries=2**30), dict(keys=2**31), dict(k_stride=(i64 * 3)(0, 2**23, 0)),
                    dict(batch=2**28, queries=2**20)):
            _refused(lib, go(_attention(**bad)), E_LIMIT, b"attention")
    for bad in ("grad_out", "lse", "d_q", "d_k", "d_v"):
        _refused(lib, lib.mgopt_attention_backward(_attention(**{bad: None}), vp(None)), E_INVALID, b"NULL")
    for bad in (None, P + 8):
        _refused(lib, lib.mgopt_attention_backward(_attention(workspace=bad), vp(None)), E_ALIGN, b"workspace")
        _refused(lib, lib.mgopt_attention(_attention(workspace=bad, queries=1, keys=4096), vp(None)), E_ALIGN, b"workspace")
    assert lib.mgopt_attention(_attention(batch=0), vp(None)) == 0
    assert lib.mgopt_attention_backward(_attention(batch=0), vp(None)) == 0


def test_attention_workspace(lib):
    """Two floats a row for the backward pass; parts of a row's keys where rows are few and keys many."""
    size = lambda back, **more: lib.mgopt_attention_workspace(_attention(**more), back)  # noqa: E731
    assert size(1) == 2 * 5 * 4 * 8
    assert size(0) == 0 and size(0, queries=1, keys=4096) > 0
    assert size(0, queries=1, keys=4096) % (2 * 4 * (64 + 2) * 4) == 0
    assert size(0, dim=129) == -1 and size(1, dim=129) == -1


def test_argument_struct_matches_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "mgopt_ops.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   "sizeof(mgopt_attention_args), offsetof(mgopt_attention_args, scale), "
                   "offsetof(mgopt_attention_args, workspace_dev)); return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(AttentionArgs), AttentionArgs.scale.offset, AttentionArgs.workspace.offset]


def test_operators_have_no_cpu_path(mg):
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    x, w = torch.ones(2, 4), torch.ones(4)
    codes = mg.Int8Rows(torch.ones((2, 4), dtype=torch.int8), torch.ones(2))
    heads = torch.ones(1, 2, 3, 4)
    for call in (lambda: mg.rms_norm(x, w), lambda: mg.add_rms_norm(x, x, w), lambda: mg.rms_norm_int8(x, w),
                 lambda: mg.int8_rows(x), lambda: mg.int8_linear(codes, codes), lambda: mg.attention(heads, heads, heads)):
        with pytest.raises(RuntimeError, match="no CPU"):
            call()


def test_attention_batches_beyond_a_grid(lib):
    """Batches that no grid takes, or whose rows pass 64 bits, are refused, not taken for empty ones."""
    for batch in (2**24 + 1, 2**62):
        for call in (lib.mgopt_attention, lib.mgopt_attention_backward):
            _refused(lib, call(_attention(batch=batch, queries=1, keys=1), vp(None)), E_LIMIT, b"attention")
        assert lib.mgopt_attention_workspace(_attention(batch=batch, queries=1, keys=1), 1) == -1
