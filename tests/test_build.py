"""What the native build needs, from make's own plan of it (make -n: nothing is compiled here)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gradient-compression_amd", "csrc")

if shutil.which("make") is None:
    pytest.skip("no make", allow_module_level=True)


def plan(*args):
    r = subprocess.run(["make", "-n", "-C", CSRC, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_everything_is_built(tmp_path):
    out = plan(f"OUT={tmp_path}")
    assert "tensor_list.cpp" in out and f"{tmp_path}/libgcodec.so" in out


def test_the_library_needs_no_python_headers(tmp_path):
    """A C user's machine: libgcodec.so is built, gcodec.clip's list reader is left out, and make says so."""
    for missing in ("PY_INC=/nonexistent", "TORCH=/nonexistent", "TORCH="):
        out = plan(f"OUT={tmp_path}", missing)
        assert f"{tmp_path}/libgcodec.so" in out and "tensor_list.cpp" not in out and "_tensor_list.so" in out


def test_the_list_reader_follows_the_installed_torch():
    """It is compiled against torch's C++ interface: another torch needs another build."""
    assert "tensor_list.cpp" in plan("TORCH_VERSION=0.0")
