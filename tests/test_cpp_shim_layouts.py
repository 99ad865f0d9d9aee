"""What the C++ classes for attention between cells refuse: compiled and linked without a GPU, run on one."""
import shutil
import subprocess

import pytest

from test_cpp_shim import _compile


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_layouts_compile_and_link(tmp_path):
    _compile(tmp_path / "shim_layouts_check", "shim_layouts_check.cpp")


@pytest.mark.gpu
def test_layouts(tmp_path):
    exe = _compile(tmp_path / "shim_layouts_check", "shim_layouts_check.cpp")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "shim_layouts_check OK" in r.stdout, r.stdout + r.stderr
