"""The C++ host API's operators of a decoder block in microscaled types (tests/host_cpp/mx_test.cpp)."""
import os
import subprocess

import pytest

MX_TEST = os.path.join(os.path.dirname(__file__), "host_cpp", "mx_test")


def _run(what):
    assert os.path.exists(MX_TEST), "build() compiles tests/host_cpp/mx_test"
    r = subprocess.run([MX_TEST, what], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    assert r.returncode == 0 and "ALL PASS" in r.stdout, r.stdout + r.stderr


def test_cpu_cases():
    _run("cpu")


@pytest.mark.gpu
def test_gpu_cases():
    _run("gpu")
