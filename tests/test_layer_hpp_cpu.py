"""The norm, 8-bit and decaying-attention part of include/fufft/fufft.hpp: built with g++ and run without a GPU."""
import shutil
import subprocess
from pathlib import Path

import pytest


def test_cpp_header(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    root = Path(__file__).resolve().parent.parent
    exe, lib = tmp_path / "layer_hpp_check", root / "fufft_amd"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{root / 'include'}",
                    str(root / "tests" / "cpp" / "layer_hpp_check.cpp"), f"-L{lib}", "-lfufft_amd", f"-Wl,-rpath,{lib}",
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0
