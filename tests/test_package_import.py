"""What importing and building the package loads and needs (no GPU)."""
import os
import subprocess
import sys

import pytest
from conftest import PKG_DIR


def _python(code, **env):
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": PKG_DIR, **env}, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    return r.stdout


def test_importing_the_package_loads_no_built_file():
    """build() imports the package first: what an earlier build left must not be in the process by then."""
    if not os.path.exists(os.path.join(PKG_DIR, "vitfp4", "_fast.so")):
        pytest.skip("vitfp4/_fast.so is not built")
    out = _python("""
import sys
import vitfp4
from vitfp4 import _build, nvfp4
from vitfp4.nvfp4 import ops
assert "vitfp4._fast" not in sys.modules
loaded = lambda: [l for l in open("/proc/self/maps") if "libvitfp4" in l or "_fast.so" in l]
assert not loaded(), loaded()
assert ops._fast_module is sys.modules["vitfp4._fast"] and loaded()
print("fine")
""")
    assert "fine" in out


@pytest.mark.parametrize("missing", ["compiler", "headers", "toolkit"])
def test_a_module_that_cannot_be_built_is_done_without(missing, tmp_path, monkeypatch):
    from vitfp4 import _build
    old = tmp_path / "_fast.so"
    old.write_bytes(b"")
    monkeypatch.setattr(_build, "FAST", str(old))
    if missing == "headers":
        gxx = tmp_path / "g++"
        gxx.write_text("#!/bin/sh\necho no headers; exit 1\n")
        gxx.chmod(0o755)
    elif missing == "toolkit":
        def none():
            raise RuntimeError("nvcc not found")
        monkeypatch.setattr(_build, "_nvcc", none)
    monkeypatch.setenv("PATH", str(tmp_path))
    with pytest.warns(UserWarning, match="Python path"):
        assert _build.build_fast(force=True) is None
    assert not old.exists()


def test_a_module_built_for_another_torch_is_neither_kept_nor_loaded(tmp_path, monkeypatch):
    import torch

    from vitfp4 import _build
    if not os.path.exists(_build.FAST):
        pytest.skip("vitfp4/_fast.so is not built")
    here = _build.build_fast()
    stamp = os.stat(here).st_mtime_ns
    assert _build.build_fast() == here and os.stat(here).st_mtime_ns == stamp      # nothing to do
    code = "import torch\ntorch.__version__ = '9.9.0'\nfrom vitfp4.nvfp4 import ops\nassert ops._fast_module is None"
    _python(code)
    other = tmp_path / "_fast.so"
    other.write_bytes(open(here, "rb").read())
    monkeypatch.setattr(_build, "FAST", str(other))
    monkeypatch.setattr(_build, "_fast_command", lambda out: ["touch", out])       # stands in for the compiler
    assert _build.build_fast() == str(other) and other.stat().st_size > 0
    monkeypatch.setattr(torch, "__version__", "9.9.0")
    assert _build.build_fast() == str(other) and other.stat().st_size == 0         # built anew


def test_the_package_imports_where_torch_has_no_cuda():
    """A torch built without CUDA lacks the functions that name the current device and stream; the format's helpers need
    neither."""
    _python("""
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from vitfp4 import _lib
from vitfp4.nvfp4 import cross_sdpa, dequantize_fp8_block, quantize_to_fp8_block
assert dequantize_fp8_block(torch.ones(2, 130).to(torch.float8_e4m3fn), torch.full((2, 2), 3.0)).eq(3).all()
try:
    quantize_to_fp8_block(torch.zeros(2, 128))
except _lib.VitFp4Error as e:
    assert "CUDA" in str(e)
else:
    raise AssertionError
""")
