"""CPU tests: the package without its native binding (_binding.so), which only shortens the way to
the 4-bit calls: it imports, plans, and refuses with the checks in Python."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

import fufft_amd as ff

PKG = Path(ff.__file__).resolve().parent

USE = """
import numpy as np
import fufft_amd as ff
assert ff.plan_filter(np.ones(256, np.complex64), 256).shape == (256,)
assert ff._binding is None
if ff.torch is None:
    x, what = np.zeros((4, 200), np.float32), TypeError
    c = s = np.zeros(512, np.uint8)
else:
    x, (c, s), what = ff.torch.zeros(4, 200), ff.mx4_empty(4, 200, device="cpu"), ValueError
for call in (lambda: ff.mx4_quantize(x, c, s), lambda: ff.mx4_dequantize(c, s, x), lambda: ff.mx4_linear(x, c, s, x),
             lambda: ff.mx4_matmul(c, s, c, s, x, 200), lambda: ff.mx4_cache_write(x, c, c, s),
             lambda: ff.mx4_cache_read(c, s, c, c, x), lambda: ff.mx4_cache_conv(c, s, c, c, x, x)):
    try:
        call()
    except what:
        pass
    else:
        raise AssertionError("not refused")
"""
NO_TORCH = "import sys; sys.modules['torch'] = None\n"


def copy_of_package(tmp_path, binding):
    root = tmp_path / "fufft_amd"
    root.mkdir()
    for name in ("__init__.py", "libfufft_amd.so"):
        shutil.copy(PKG / name, root / name)
    if binding is not None:
        (root / "_binding.so").write_bytes(binding)
    return tmp_path


def run(code, where):
    return subprocess.run([sys.executable, "-W", "always", "-c", code], cwd=where, capture_output=True, text=True, timeout=120)


@pytest.mark.parametrize("first", ["", NO_TORCH])
def test_import_without_the_binding(tmp_path, first):
    r = run(first + USE, copy_of_package(tmp_path, None))
    assert r.returncode == 0, r.stderr
    assert "_binding.so" not in r.stderr


def test_import_without_torch_and_with_the_binding(tmp_path):
    r = run(NO_TORCH + USE, copy_of_package(tmp_path, b"of no use"))
    assert r.returncode == 0, r.stderr


def test_import_with_a_binding_that_does_not_load(tmp_path):
    r = run(USE, copy_of_package(tmp_path, b"not a library"))
    assert r.returncode == 0, r.stderr
    assert "RuntimeWarning" in r.stderr and "_binding.so is not used" in r.stderr


def test_import_with_a_binding_for_another_torch(tmp_path):
    """Told by the version that it was built for, as its code reads tensors inline."""
    if ff._binding is None:
        pytest.skip("the native binding is not built")
    where = copy_of_package(tmp_path, (PKG / "_binding.so").read_bytes())
    r = run("import torch; torch.__version__ = '9.9.9'\n" + USE, where)
    assert r.returncode == 0, r.stderr
    assert "built for torch" in r.stderr


def test_the_binding_is_used_where_it_is_built():
    if not (PKG / "_binding.so").exists():
        pytest.skip("the native binding is not built")
    assert ff._binding is not None
