"""Runs tests/cpp/test_step.cpp: heads normed and turned, a cache in 8 bits and drafted trees through the C++ host mirror."""
import os
import subprocess

import pytest

from adrastea_amd import build


def test_cpp_step_cpu():
    r = subprocess.run([build.build_step_test()], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr


@pytest.mark.gpu
def test_cpp_step_gpu():
    assert os.path.exists(build.STEP_TEST_BIN), "build the test first: python -m adrastea_amd.build"
    r = subprocess.run([build.STEP_TEST_BIN, "gpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("OK"), r.stdout + r.stderr
