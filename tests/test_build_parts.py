"""CPU test of the build's parts: without torch or without g++ the native binding is left out and the rest
is built."""
import importlib.util
import shutil
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(monkeypatch):
    """The build module, its compilers not run; `ran` holds the parts and commands that were."""
    spec = importlib.util.spec_from_file_location("_build_parts", ROOT / "fufft_amd" / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.ran = []
    for name in ("build_oracle", "build_library", "build_cpp_checks"):
        monkeypatch.setattr(b, name, lambda *a, name=name: b.ran.append(name))
    monkeypatch.setattr(b, "_run", lambda cmd: b.ran.append(cmd[0]))
    monkeypatch.setattr(b.os, "replace", lambda *a: None)
    return b


def test_all_parts(build):
    build.build()
    assert build.ran == ["build_oracle", "build_library", "g++", "build_cpp_checks"]


def test_without_torch(build, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    build.build()
    assert build.ran == ["build_oracle", "build_library", "build_cpp_checks"]


def test_without_a_host_compiler(build, monkeypatch):
    which = shutil.which
    monkeypatch.setattr(build.shutil, "which", lambda name, *a: None if name == "g++" else which(name, *a))
    build.build()
    assert build.ran == ["build_oracle", "build_library"]
