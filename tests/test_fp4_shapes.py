"""4-bit operands whose sizes pass 64 bits are refused by the bindings, which would else make small ones of what
is left of the size: in Python on the CPU, in the C++ host mirror (tests/cpp/fp4_shapes.cpp) on the GPU."""
import os
import subprocess

import pytest

from staleynet_amd import gemm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "fp4_shapes")


@pytest.mark.parametrize("rows,inner", [((1 << 64) + 3, 64), (3, (1 << 64) + 64), (-1, 0), (3, -32), ((1 << 32) * (1 << 32), 1)])
def test_sizes_past_64_bits_are_refused(rows, inner):
    with pytest.raises(gemm.GpuError) as error:
        gemm.fp4_sizes(rows, inner)
    assert error.value.status == gemm.SN_ERR_OVERFLOW


def test_the_program_is_built():
    from staleynet_amd import build as builder

    if not os.path.exists(BINARY):
        builder.build_cpp_tests()
    assert os.path.exists(BINARY)


@pytest.mark.gpu
def test_the_mirror_refuses_them():
    proc = subprocess.run([BINARY], capture_output=True, text=True, timeout=100)
    assert proc.returncode == 0, proc.stdout + proc.stderr
