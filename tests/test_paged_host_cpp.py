"""The C++ host API's paged-cache operators (tests/host_cpp/paged_test.cpp)."""
import os
import subprocess

import pytest

PAGED_TEST = os.path.join(os.path.dirname(__file__), "host_cpp", "paged_test")


def _run(what):
    assert os.path.exists(PAGED_TEST), "build() compiles tests/host_cpp/paged_test"
    r = subprocess.run([PAGED_TEST, what], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "ALL PASS" in r.stdout, r.stdout + r.stderr


def test_cpu_cases():
    _run("cpu")


@pytest.mark.gpu
def test_gpu_cases():
    _run("gpu")
