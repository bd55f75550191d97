"""Runs the C++ mirror's test program of attention over a context in two parts (tests/cpp/test_host_mirror_context.cpp, built by floneum_amd/build.py)
on the GPU."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpp_host_mirror():
    exe = os.path.join(ROOT, "tests", "cpp", "test_host_mirror_context")
    assert os.path.exists(exe), "tests/cpp/test_host_mirror_context is missing: run floneum_amd/build.py"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
