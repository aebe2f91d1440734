"""Builds libmgopt.so (the HIP kernels and C ABI) for gfx950, in-tree.

Run as a script or call build().  The library lands in _build/ next to this
file; the Python host layer loads it from there and nowhere else.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
#: the optimizer step and the training-step operators
SRCS = [HERE / "csrc" / name for name in ("mgopt.hip", "ops_embedding.hip", "ops_gated_act.hip",
                                          "ops_policy_loss.hip", "ops_qk_norm_rope.hip")]
INCLUDE = HERE.parent / "include"
OUT_DIR = HERE / "_build"
LIB = OUT_DIR / "libmgopt.so"

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # every fused multiply-add in the kernels is written out explicitly
    "-ffp-contract=off",
    # no packed-fp32 instructions (v_pk_*_f32) anywhere in the device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fvisibility=hidden",
    "-Wall",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required to build libmgopt.so)")


def build(verbose: bool = False) -> Path:
    OUT_DIR.mkdir(exist_ok=True)
    objects = [OUT_DIR / f"{src.stem}.o" for src in SRCS]
    compile_ = [[hipcc(), *HIPCC_FLAGS, f"-I{INCLUDE}", "-c", str(src), "-o", str(obj)] for src, obj in zip(SRCS, objects)]
    _run(compile_, verbose)
    tmp = LIB.with_suffix(".so.tmp")
    _run([[hipcc(), *HIPCC_FLAGS, "-shared", *map(str, objects), "-o", str(tmp)]], verbose)
    os.replace(tmp, LIB)
    return LIB


def _run(commands: list[list[str]], verbose: bool) -> None:
    """Runs the commands side by side; raises with the output of the first that fails."""
    procs = []
    for cmd in commands:
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    results = [(p, *p.communicate()) for p in procs]
    for p, out, err in results:
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed ({p.returncode}):\n{out}\n{err}")
        noise = [ln for ln in err.splitlines() if "packed-fp32-ops" not in ln and ln.strip()]
        if verbose and noise:
            print("\n".join(noise), file=sys.stderr)


HOST_SRCS = [HERE / "csrc" / name for name in ("host_ptrs.cpp", "host_ops.cpp")]
HOST_DIR = OUT_DIR / "host"


def build_host(verbose: bool = False) -> Path:
    """Builds the host-side helper (a torch C++ extension) into _build/host/."""
    from torch.utils.cpp_extension import load

    if HOST_DIR.exists():
        shutil.rmtree(HOST_DIR)
    HOST_DIR.mkdir(parents=True)
    load(name="mgopt_host", sources=list(map(str, HOST_SRCS)), build_directory=str(HOST_DIR), extra_cflags=["-O2"],
         extra_include_paths=[str(INCLUDE)],
         verbose=verbose)
    return HOST_DIR / "mgopt_host.so"


if __name__ == "__main__":
    print(build(verbose=True))
    print(build_host(verbose=False))
