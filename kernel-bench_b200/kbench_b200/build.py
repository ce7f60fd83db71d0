"""Build ``libkb_solver.so`` (all CUDA kernels + the C ABI) in-tree with nvcc for sm_100a, and the
Python extension ``_kb_host.so`` (host side of the row scores and the fitting step) with g++.

    python kernel-bench_b200/kbench_b200/build.py [--verbose]

Both land next to this file; the Python layer loads ``libkb_solver.so`` with ctypes, imports
``_kb_host``, and fails loudly when one is missing.  The library needs neither torch nor Python headers
and is built first; where the extension cannot be, that is reported and the library stands.
``-Xptxas -v`` output (registers, spills, shared memory per kernel) is written to ``_build/ptxas.txt`` for
inspection.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent.parent
CSRC = PKG / "csrc"
INCLUDE = REPO / "include"
LIB = PKG / "libkb_solver.so"
HOST = PKG / "_kb_host.so"
SOURCES = ["kb_misc.cu", "kb_estep.cu", "kb_params.cu", "kb_dts.cu", "kb_wave_fwd.cu", "kb_wave_bwd.cu", "kb_engine.cu", "kb_tangent.cu", "kb_hvp.cu", "kb_builder.cu", "kb_sched.cu", "kb_score.cu", "kb_fit.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def host_target() -> str:
    """The Python and torch that the host extension is built for, and runs with alone."""
    import torch
    return f"{sysconfig.get_config_var('SOABI')}, torch {torch.__version__}"


def build_host(force: bool = False) -> Path:
    """The host extension, against the installed torch's headers and libraries."""
    src, made_for = CSRC / "kb_host.cpp", REPO / "_build" / "host_target.txt"
    newest = max(src.stat().st_mtime, (INCLUDE / "kb_solver.h").stat().st_mtime)
    target = host_target()
    if HOST.exists() and not force and newest <= HOST.stat().st_mtime and made_for.exists() \
            and made_for.read_text() == target:
        return HOST
    import torch
    base = Path(torch.__file__).resolve().parent
    include = [base / "include", base / "include/torch/csrc/api/include", sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           *(f"-isystem{p}" for p in include), f"-I{INCLUDE}", f'-DKB_TARGET="{target}"', str(src), "-o", str(HOST) + ".tmp", f"-L{base / 'lib'}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        HOST.unlink(missing_ok=True)  # not of this source for this target
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode})")
    os.replace(str(HOST) + ".tmp", HOST)
    made_for.parent.mkdir(exist_ok=True)
    made_for.write_text(target)
    return HOST


def build_library(verbose: bool = False, force: bool = False) -> Path:
    srcs = [CSRC / s for s in SOURCES]
    deps = srcs + list(CSRC.glob("*.cuh")) + [INCLUDE / "kb_solver.h"]
    if LIB.exists() and not force:
        lib_mtime = LIB.stat().st_mtime
        if all(d.stat().st_mtime <= lib_mtime for d in deps):
            return LIB
    build_dir = REPO / "_build"
    build_dir.mkdir(exist_ok=True)
    cmd = [nvcc_path(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
           "-Xptxas", "-v", f"-I{INCLUDE}", f"-I{CSRC}", "-o", str(LIB) + ".tmp", *map(str, srcs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    (build_dir / "ptxas.txt").write_text(res.stdout + res.stderr)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc failed ({res.returncode})")
    os.replace(str(LIB) + ".tmp", LIB)
    if verbose:
        print(res.stderr)
    return LIB


def build(verbose: bool = False, force: bool = False) -> Path:
    """The library, then the host extension; without the latter (reported here) ``scoring`` and ``fitting``
    raise and everything else runs."""
    lib = build_library(verbose=verbose, force=force)
    try:
        build_host(force=force)
    except Exception as e:
        sys.stderr.write(f"kbench_b200: the host extension {HOST.name} was not built ({type(e).__name__}: {e}); "
                         "kbench_b200.scoring and kbench_b200.fitting need it\n")
    return lib


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force))
