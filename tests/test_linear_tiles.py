"""The tile arithmetic of the tensor-core linear layers (csrc/linear_tiles.cuh), compiled for the
host with undefined behaviour trapped: tests/c/linear_tiles.cpp."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tiles_on_the_host(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no C++ compiler")
    out = str(tmp_path / "linear_tiles")
    r = subprocess.run([gxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined",
                        "-fsanitize-undefined-trap-on-error", "-I",
                        os.path.join(ROOT, "cuda-triton-scala_b200", "csrc"),
                        os.path.join(ROOT, "tests", "c", "linear_tiles.cpp"), "-o", out],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "warning" not in r.stderr, r.stderr
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, f"{r.returncode} {r.stdout}"
    assert "ok" in r.stdout
