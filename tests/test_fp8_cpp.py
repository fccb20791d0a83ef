"""The C++ host mirror's 8-bit products, norms and log probabilities (tests/cpp/fp8_calls.cpp): built on the CPU, run on the GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "fp8_calls")


def test_the_program_is_built():
    from staleynet_amd import build as builder

    if not os.path.exists(BINARY):
        builder.build_cpp_tests()
    assert os.path.exists(BINARY)


@pytest.mark.gpu
def test_the_mirror_matches():
    proc = subprocess.run([BINARY], capture_output=True, text=True, timeout=100)
    assert proc.returncode == 0, proc.stdout + proc.stderr
