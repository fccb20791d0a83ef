"""The ends of the range of attention over a 4-bit cache (``sn_fp4_attention``), as its header states them."""
import numpy as np
import pytest

import fp4_reference as ref
from test_fp4_attention_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("queries", [1, 5])
def test_the_values_of_a_single_key_come_back_exactly(gpu, head_dim, queries):
    """Its weight is 1: every code at every scale byte, subnormals and the largest among them. Queries ahead of
    the key see nothing."""
    case = Case(256, 2, 1, queries, 3, head_dim, [1] * 256, seed=head_dim)
    case.codes[1][:, 0, 0] = np.tile(np.arange(16, dtype=np.uint8) * 0x10 + np.arange(16, dtype=np.uint8)[::-1], head_dim // 32)
    case.scales[1][:, 0, 0] = np.arange(256, dtype=np.uint8)[:, None]
    got = case.run(gpu)
    values = ref.dequantize(case.codes[1][:, 0, 0], case.scales[1][:, 0, 0])
    assert not got[:, :, :queries - 1].any()
    for head in range(2):
        assert np.array_equal(got[:253, head, -1], values[:253].astype(np.float32))
        assert np.isnan(got[253:, head, -1]).all()


@pytest.mark.parametrize("head_dim,heads,queries,length", [(32, 2, 1, 250), (64, 4, 40, 250), (128, 2, 1, 8000)])
@pytest.mark.parametrize("spread", [1.0, 6.0])
def test_large_values(gpu, head_dim, heads, queries, length, spread):
    """Just under 2^119 by their number: 250 of up to 6 x 2^108, 8000 of up to 6 x 2^103. Sums stay finite."""
    case = Case(2, heads, 2, queries, length, head_dim, [length, length - 3], seed=length, spread=spread)
    case.scales[1][:, :, :length - 3] = 127 + (108 if length == 250 else 103)
    case.check(case.run(gpu))
