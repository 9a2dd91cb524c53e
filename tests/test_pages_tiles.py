"""The rows that the paged attention's tiles read, on the CPU (tests/cpp/pages_tiles_check.cpp): in the table, in
the page that was looked up, each cached row once. The kernels use the same functions."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not on PATH")
def test_pages_tiles(tmp_path):
    exe = str(tmp_path / "pages_tiles_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I",
                    os.path.join(ROOT, "neuralnet.cpp_amd", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "cpp", "pages_tiles_check.cpp")], check=True)
    out = subprocess.run([exe], check=False, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip().endswith("wrong 0"), out.stdout + out.stderr
