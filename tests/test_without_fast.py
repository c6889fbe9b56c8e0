"""The package without its C fast path (an interpreter it was not built for): it imports, and
the Python checks alone accept and refuse what they always do. Child processes, CPU only."""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

import pytest

from conftest import ROOT

PKG = os.path.join(ROOT, "wgblas_b200")
SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")


def child(code, cwd):
    env = dict(os.environ, PYTHONPATH=cwd)
    return subprocess.run([sys.executable, "-c", code], cwd=cwd, env=env, capture_output=True, text=True, timeout=300)


@pytest.fixture()
def copy(tmp_path):
    """The package's Python files and its library, no extension."""
    dst = tmp_path / "wgblas_b200"
    dst.mkdir()
    for name in os.listdir(PKG):
        if name.endswith(".py"):
            shutil.copy(os.path.join(PKG, name), dst / name)
    os.symlink(os.path.join(PKG, "libwgblas_b200.so"), dst / "libwgblas_b200.so")
    return str(tmp_path)


CALL = '''
import ctypes as ct
import wgblas_b200 as wg
assert wg.__file__.startswith({root!r}), wg.__file__

class Tensor:
    is_cuda = True
    def __init__(self, n, dtype, ptr): self.n, self.dtype, self.ptr = n, dtype, ptr
    def data_ptr(self): return self.ptr
    def get_device(self): return 0
    def is_contiguous(self): return True
    def numel(self): return self.n

block = (ct.c_char * 65536)()
dev = wg.Device(ct.cast(block, ct.c_void_p), 0, False, {{}}, "stand-in")
args = [dev, "transpose", 3, 10, 6, 8, 1.0, Tensor(80, "bfloat16", 1 << 32), 8, Tensor(144, "bfloat16", 2 << 32), 8, 48,
        Tensor(4, "int32", 3 << 32), 0.0, Tensor(60, "bfloat16", 4 << 32), 6]
try:
    wg.gemmGrouped(*args)
    raise SystemExit("not reached")
except wg._native.NativeError as e:  # every check passed; the stand-in is no sm_100 device
    assert e.status == wg._native.WG_ERR_NOT_SUPPORTED
args[5] = -1
try:
    wg.gemmGrouped(*args)
    raise SystemExit("not refused")
except wg.Error as e:
    assert "non-negative" in str(e)
q = wg.GpuMxMatrix.wrap(dev, Tensor(40 * 32, "uint8", 1 << 32), Tensor(512, "uint8", 2 << 32), 40, 50)
try:
    wg.mxQuantize(dev, "no-transpose", 40, 50, Tensor(2000, "bfloat16", 3 << 32), 50, q)
    raise SystemExit("not reached")
except wg._native.NativeError as e:
    assert e.status == wg._native.WG_ERR_NOT_SUPPORTED
print("fast" if wg._native.has_fast else "plain")
'''


def test_the_package_works_without_the_extension(copy):
    r = child(CALL.format(root=copy), copy)
    assert r.returncode == 0 and r.stdout.strip() == "plain", r.stderr


def test_an_extension_of_another_interpreter_is_not_loaded(copy):
    """A file without this interpreter's tag (here: no extension at all) is passed over, not loaded."""
    for name in ("_fast.so", "_fast.cpython-38-x86_64-linux-gnu.so"):
        with open(os.path.join(copy, "wgblas_b200", name), "wb") as f:
            f.write(b"another interpreter's")
    r = child(CALL.format(root=copy), copy)
    assert r.returncode == 0 and r.stdout.strip() == "plain", r.stderr


def test_the_build_names_the_interpreter(copy):
    """The extension that was built here is this interpreter's, and it is the one in use."""
    assert os.path.exists(os.path.join(PKG, "_fast" + SUFFIX)) and "cpython" in SUFFIX
    shutil.copy(os.path.join(PKG, "_fast" + SUFFIX), os.path.join(copy, "wgblas_b200"))
    r = child(CALL.format(root=copy), copy)
    assert r.returncode == 0 and r.stdout.strip() == "fast", r.stderr


def test_the_build_does_without_an_extension_that_cannot_be_built(tmp_path, monkeypatch, capsys):
    """No headers of this interpreter: the rest is built all the same, and the build says so."""
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setattr(b, "FAST", str(tmp_path / "_fast.so"))
    monkeypatch.setattr(b, "PYTHON_INCLUDE", str(tmp_path))
    assert b.build_fast() is None
    assert "not built" in capsys.readouterr().err
