"""libcdb_torch.so holds the low-bit operators only: without it, or with one of another torch, the rest of the
package works as it does without them, and the C library is built without torch's headers."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from continuous_depth_batching_b200 import _lib
from continuous_depth_batching_b200.csrc import build

ROOT = Path(__file__).resolve().parent.parent
IMPORT = """
import sys, warnings
from pathlib import Path
import torch
from continuous_depth_batching_b200 import _lib
_lib.TORCH_OPS_PATH = Path(sys.argv[1])
with warnings.catch_warnings(record=True) as said:
    warnings.simplefilter("always")
    import continuous_depth_batching_b200.ops as ops
    import continuous_depth_batching_b200.hf_attention
assert any("no low-bit ops" in str(w.message) for w in said)
for name in ("step_tables", "kv8_append", "kv8_gather", "kv8_decode_attention", "kv8_prefill_attention", "gemv_w4"):
    try:
        getattr(ops, name)(torch.zeros(1))
    except _lib.CDBError as e:
        assert name in str(e) and sys.argv[1] in str(e), e
    else:
        raise AssertionError(name)
"""
CPU = IMPORT + """
try:
    ops.gemm_bf16(torch.zeros(8, 64).bfloat16(), torch.zeros(64, 64).bfloat16(), torch.zeros(8, 64).bfloat16())
except RuntimeError as e:
    assert "CUDA tensors only" in str(e), e
else:
    raise AssertionError("a CPU product")
"""
GPU = IMPORT + """
x, w = torch.randn(8, 64, device="cuda").bfloat16(), torch.randn(64, 64, device="cuda").bfloat16()
out = torch.empty(8, 64, device="cuda").bfloat16()
torch.ops.cdb.gemm_bf16(x, w, out)
want = x.double() @ w.double().t()
assert ((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-18 * (x.double().abs() @ w.double().abs().t())).all()
assert ops.status_code() == 0
"""


def _run(code, path):
    done = subprocess.run([sys.executable, "-c", code, str(path)], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


def _another(tmp_path, what):
    path = tmp_path / "libcdb_torch.so"
    if what == "unloadable":
        path.write_bytes(b"not a library")
    return path


@pytest.mark.parametrize("what", ["missing", "unloadable"])
def test_import_without_it(tmp_path, what):
    _run(CPU, _another(tmp_path, what))


@pytest.mark.gpu
def test_other_operators_run_without_it(tmp_path):
    _run(GPU, _another(tmp_path, "missing"))


def test_the_c_library_alone_needs_no_torch(tmp_path, monkeypatch):
    """build_library() runs nvcc only."""

    ran = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd[0]))
    monkeypatch.setattr(build, "PKG", tmp_path)
    monkeypatch.setattr(build, "SOURCES", [])
    build.build_library()
    assert len(ran) == 1 and ran[0] == build.nvcc_path()


def test_built_again_for_another_torch(tmp_path, monkeypatch):
    ran = []
    monkeypatch.setattr(build, "PKG", tmp_path)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: (ran.append(cmd[0]), (tmp_path / build.TORCH_LIB_NAME).touch()))
    lib = _lib.LIB_PATH
    build.build_torch_ops(lib)
    build.build_torch_ops(lib)
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_torch_ops(lib)
    build.build_torch_ops(lib)
    assert len(ran) == 2
