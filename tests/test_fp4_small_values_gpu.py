"""GPU parity of products with 4-bit weights where x is so small that three bf16 parts do not hold it: under
2^-110 a value's last bits are under 2^-133, bf16's smallest subnormal. Weights go up to 6 x 2^125, so those
bits reach outputs of ordinary size.

Tolerance: the products' own (test_fp4_matmul_gpu), which counts a chain of ceil(inner / 32) additions for each of
the three parts. What they leave is at most 16 bits of a value, a further sum of two parts with the same chain, in
place of parts that are 0 or a few bits there; its power of two is exact and it is added to the output with one rounding
more, so ceil(inner / 32) + 64 steps more are allowed. A value at 2^-121 cut at 2^-133 is off by up to 2^-12 of itself,
which 64 to 400 steps of 2^-23 do not hide."""
import numpy as np
import pytest

import fp4_reference as ref
from bench import HipGraph
from staleynet_amd.gemm import Fp4Matrix, MatmulSpec, Precision, Shape
from test_fp4_matmul_gpu import run, to_bf16

pytestmark = pytest.mark.gpu

BANDS = (-112, -117, -121, -126, -131, -140, -149)


def small(rng, count, exponent):
    """Values of 2^exponent to 2^(exponent + 1) with every fraction bit that fp32 has there, both signs."""
    return np.ldexp(rng.uniform(1, 2, count) * rng.choice([-1, 1], count), exponent).astype(np.float32)


def operands(rows, inner, cols, shift, seed):
    """Rows of one band each; in every other one, ordinary values stand in the odd blocks, whose weights are as much
    smaller, so that both kinds reach the sum."""
    rng = np.random.default_rng(seed)
    blocks = ref.blocks_of(inner)
    codes = rng.integers(0, 256, (cols, blocks * 16), dtype=np.uint8)
    scales = rng.integers(240, 253, (cols, blocks), dtype=np.uint8)
    scales[:, 1::2] = rng.integers(1, 9, scales[:, 1::2].shape)
    x = np.zeros((rows, inner), np.float32)
    odd = np.arange(inner) // 32 % 2 == 1
    for r in range(rows):
        band = BANDS[(r + shift) % len(BANDS)]
        x[r] = small(rng, inner, band)
        x[r, odd] = small(rng, odd.sum(), band + 238) if r % 2 else 0
    return x, codes, scales, ref.dequantize(codes, scales, inner)


def check(got, x, w, inner, scale=1.0, before=None, bias=None):
    x = x.astype(np.float64)
    expected = scale * (x @ w.T)
    steps = 4 * -(-inner // 32) + 128
    bound = steps * 2.0 ** -23 * abs(scale) * (np.abs(x) @ np.abs(w).T) + 2.0 ** -24 * np.abs(expected)
    for more in (before, bias):
        if more is not None:
            expected = expected + more
            bound = bound + 2 * 2.0 ** -24 * np.abs(expected)
    wrong = np.abs(got - expected) > bound
    assert np.isfinite(bound).all() and np.isfinite(got).all()
    assert not wrong.any(), (np.argwhere(wrong)[:4], got[wrong][:4], expected[wrong][:4], wrong.mean())


@pytest.mark.parametrize("rows,inner,cols", [
    (1, 300, 50), (1, 33, 5201), (1, 300, 12301), (2, 64, 50), (5, 300, 50), (5, 96, 12301), (10, 130, 50), (16, 300, 50),
    (16, 96, 5201), (16, 64, 12301),                            # few rows: one, two and four column tiles a wave
    (16, 3, 40), (40, 300, 77), (40, 2100, 100), (130, 33, 70), # tiles of 32 x 128, sliced among them
    (1990, 64, 4001)])                                          # tiles of 128 x 256
def test_small_values_count_in_full(gpu, rows, inner, cols):
    for shift in range(len(BANDS) if rows < len(BANDS) else 1):
        x, codes, scales, w = operands(rows, inner, cols, shift, rows + shift)
        got = run(gpu, MatmulSpec.new(rows, cols, inner), x, codes, scales, offset=rows % 2)
        check(got, x, w, inner)
    assert np.array_equal(got, run(gpu, MatmulSpec.new(rows, cols, inner), x, codes, scales, offset=rows % 2))


@pytest.mark.parametrize("rows,inner,cols", [(1, 300, 50), (16, 300, 50), (40, 300, 77), (40, 2100, 100)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_small_values_scaled_accumulated_and_with_bias(gpu, rows, inner, cols, with_bias):
    rng = np.random.default_rng(rows)
    x, codes, scales, w = operands(rows, inner, cols, 2, rows)
    magnitude = np.abs(x.astype(np.float64)) @ np.abs(w).T
    before = (magnitude * rng.standard_normal((rows, cols))).astype(np.float32)
    bias = (magnitude[0] * rng.standard_normal(cols)).astype(np.float32) if with_bias else None
    spec = MatmulSpec.new(rows, cols, inner).scaled(-0.375)
    check(run(gpu, spec, x, codes, scales, bias=bias), x, w, inner, -0.375, None, bias)
    check(run(gpu, spec.accumulate(), x, codes, scales, bias=bias, before=before), x, w, inner, -0.375, before, bias)


@pytest.mark.parametrize("rows,inner,cols", [(3, 300, 50), (16, 300, 50), (40, 300, 77), (40, 2100, 100),
                                             (1990, 64, 4001)])
def test_rows_without_small_values_keep_their_bits(gpu, rows, inner, cols):
    """Beside a row of small values: ordinary rows, one of zeros (whose results here are -0), and one with an infinity;
    a NaN block is its column's alone."""
    rng = np.random.default_rng(inner)
    _, codes, scales, _ = operands(rows, inner, cols, 0, inner)
    scales[:, :] = rng.integers(118, 128, scales.shape)
    scales[5, 0] = 255
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    x[1] = 0
    x[rows - 1, 7] = np.inf
    spec = MatmulSpec.new(rows, cols, inner).scaled(-0.375)
    expected = run(gpu, spec, x, codes, scales)
    x[0] = small(rng, inner, -126)
    got = run(gpu, spec, x, codes, scales)
    assert np.array_equal(got[1:].view(np.uint32), expected[1:].view(np.uint32))
    assert np.signbit(got[1, :5]).all() and np.isnan(got[:, 5]).all() and not np.isnan(got[0, :5]).any()


@pytest.mark.parametrize("rows,inner,cols", [(1, 300, 50), (20, 300, 50), (40, 300, 77), (1100, 64, 3900)])
def test_small_values_rounded_to_bf16(gpu, rows, inner, cols):
    """Rounded once, to bf16's subnormals where they lie among them."""
    for shift in range(len(BANDS) if rows < len(BANDS) else 1):
        x, codes, scales, w = operands(rows, inner, cols, shift, rows + shift)
        got = run(gpu, MatmulSpec.new(rows, cols, inner).with_precision(Precision.Bf16), x, codes, scales)
        check(got, to_bf16(x), w, inner)


@pytest.mark.parametrize("rows,inner,cols", [(1, 300, 50), (16, 300, 50), (40, 2100, 100)])
def test_a_captured_product_meets_small_values_later(gpu, rows, inner, cols):
    """Captured on ordinary values and replayed on small ones, on ordinary ones again and on both: the eager bits."""
    x, codes, scales, w = operands(rows, inner, cols, 2, rows)
    ordinary = np.random.default_rng(rows).standard_normal(x.shape).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner)
    matrix = Fp4Matrix(cols, inner, gpu.upload_bytes(codes), gpu.upload_bytes(scales))
    left, out = gpu.upload(Shape(rows, inner), ordinary), gpu.zeros(Shape(rows, cols))
    call = lambda: gpu.matmul_fp4(spec.right_transposed(), left, matrix, out)
    call()
    gpu.synchronize()
    graph = HipGraph(gpu.stream, call)
    try:
        for values in (x, ordinary, np.where(np.arange(inner) % 2, x, ordinary), x):
            gpu.copy_from_host(left, values)
            graph.launch()
            got = gpu.download(out).reshape(rows, cols)
            eager = run(gpu, spec, values, codes, scales)  # infinities and NaN among the ordinary ones'
            assert np.array_equal(got.view(np.uint32), eager.view(np.uint32))
        check(got, x, w, inner)
    finally:
        gpu.synchronize()
        graph.close()
