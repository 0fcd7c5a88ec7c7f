"""Build libcdb_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and libcdb_torch.so
(PyTorch operators in C++ over it) with g++.

    python -m continuous_depth_batching_b200.csrc.build            # both
    python -m continuous_depth_batching_b200.csrc.build --c-abi    # the first alone: no g++, no torch headers

The libraries land next to the package (``continuous_depth_batching_b200/libcdb_b200.so``) so
they ship with the source tree; ``continuous_depth_batching_b200._lib`` loads them, the first with ctypes.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
REPO = PKG.parent
LIB_NAME = "libcdb_b200.so"
TORCH_LIB_NAME = "libcdb_torch.so"
SOURCES = [
    "attention.cu", "prefill_attention.cu", "elementwise.cu", "gemm.cu", "scheduler.cu", "fused_ops.cu", "kv_swap.cu",
    "kv8_append.cu", "kv8_decode.cu", "kv8_prefill.cu", "gemv_w4.cu", "step_tables.cu",
]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or install the CUDA toolkit")
    return cand


def library_path() -> Path:
    return PKG / LIB_NAME


def _stale(out: Path, inputs: list[Path]) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(p.stat().st_mtime > t for p in inputs)


def build_library(force: bool = False, verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile every ``.cu`` into objects, then link the shared library. Returns its path."""

    nvcc = nvcc_path()
    build_dir = PKG / "_build"
    build_dir.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + list((REPO / "include").glob("*.h"))
    objs = []
    procs = []
    for src in SOURCES:
        src_path = CSRC / src
        obj = build_dir / (src_path.stem + ".o")
        objs.append(obj)
        if force or _stale(obj, [src_path, *headers]):
            cmd = [
                nvcc,
                *ARCH_FLAGS,
                "-O3",
                "-lineinfo",
                "-std=c++17",
                "-Xcompiler",
                "-fPIC",
                "-Xptxas",
                "-v" if verbose else "-O3",
                f"-I{REPO / 'include'}",
                "-c",
                str(src_path),
                "-o",
                str(obj),
            ]
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for src, proc in procs:
        out, _ = proc.communicate()
        if verbose or proc.returncode != 0:
            sys.stdout.write(out)
        if proc.returncode != 0:
            failed.append(src)
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    lib = library_path()
    if force or _stale(lib, objs):
        cmd = [nvcc, *ARCH_FLAGS, "-shared", "-Xlinker", f"-soname={LIB_NAME}", "-o", str(lib), *map(str, objs)]
        subprocess.run(cmd, check=True)
    return lib


def build_torch_ops(lib: Path, force: bool = False) -> Path:
    """Compile ``torch_ops.cpp`` against the installed torch and link it to the CUDA library. The
    result fits that build of torch only, so it is built again for another one."""

    import torch

    src, out = CSRC / "torch_ops.cpp", PKG / TORCH_LIB_NAME
    built_for = PKG / "_build" / "torch_ops.torch"
    this = f"{torch.__version__} {torch.version.git_version} {torch.__file__}"
    same = built_for.exists() and built_for.read_text() == this
    if not force and same and not _stale(out, [src, lib, REPO / "include" / "cdb_b200.h"]):
        return out
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    cmd = [
        "g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}", f"-I{cuda / 'include'}", str(src),
        "-o", str(out), str(lib), f"-L{root / 'lib'}", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
        f"-L{cuda / 'lib64'}", "-lcudart", "-Wl,-rpath,$ORIGIN",
    ]
    subprocess.run(cmd, check=True)
    built_for.parent.mkdir(exist_ok=True)
    built_for.write_text(this)
    return out


if __name__ == "__main__":
    path = build_library(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
    if "--c-abi" not in sys.argv:
        print(build_torch_ops(path, force="--force" in sys.argv))
