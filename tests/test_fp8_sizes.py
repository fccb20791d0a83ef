"""8-bit operands whose sizes pass 64 bits are refused by the Python binding, which would else pass the C ABI the lower 64
bits: a smaller matrix than was asked for."""
import pytest

from staleynet_amd import gemm
from staleynet_amd.gemm import ByteBuffer, Fp8Matrix


@pytest.mark.parametrize("rows,inner", [((1 << 64) + 3, 64), (3, (1 << 64) + 64), (-1, 64), (3, -32)])
def test_a_matrix_past_64_bits_is_refused(rows, inner):
    none = ByteBuffer(None, 0, 0)
    with pytest.raises(gemm.GpuError) as error:
        Fp8Matrix(rows, inner, none, none)
    assert error.value.status == gemm.SN_ERR_OVERFLOW
    assert Fp8Matrix((1 << 64) - 1, 0, none, none).rows == (1 << 64) - 1
