"""GPU parity of products with 4-bit weights (``sn_matmul_fp4``) against 64 bits.

Tolerance. Products are exact; what differs from the 64-bit result is the fp32 summation. An output's
sum is a chain of at most ceil(inner / 32) additions into a matrix accumulator for each of the three
parts, 32 terms added inside each instruction, and at most 16 waves' sums and two part sums added
after; each rounding is at most 2^-23 (were additions to cut off) of a partial sum, which the sum of
magnitudes S bounds: (3 ceil(inner / 32) + 64) 2^-23 S. The scale, the previous output and the bias add
a rounding of half a step each: 3 x 2^-24 of what they meet."""
import numpy as np
import pytest

import fp4_reference as ref
from fp4_reference import View
from staleynet_amd.gemm import Fp4Matrix, Gpu, MatmulKernel, MatmulPanic, MatmulSpec, Precision, Shape, Storage

pytestmark = pytest.mark.gpu


def weights(cols, inner, seed):
    """Codes and scale bytes as a quantized N(0, 1) operand has them (values are drawn as codes, so that
    large operands are quick), and the values."""
    rng = np.random.default_rng(seed)
    blocks = ref.blocks_of(inner)
    codes = rng.integers(0, 256, (cols, blocks * 16), dtype=np.uint8)
    scales = rng.integers(121, 128, (cols, blocks), dtype=np.uint8)
    return codes, scales, ref.dequantize(codes, scales, inner)


def to_bf16(x):
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def run(gpu, spec, x, codes, scales, bias=None, before=None, offset=0, guard=9):
    """The product with x `offset` floats into its buffer; the output's surroundings must keep theirs."""
    rows, cols = spec.rows, spec.cols
    left = gpu.upload(Shape.vector(x.size + offset), np.concatenate([np.zeros(offset, np.float32), x.ravel()]))
    filled = np.full(offset + rows * cols + guard, 123.0, np.float32)
    if before is not None:
        filled[offset:offset + rows * cols] = before.ravel()
    out = gpu.upload(Shape.vector(filled.size), filled)
    matrix = Fp4Matrix(cols, spec.inner, gpu.upload_bytes(codes), gpu.upload_bytes(scales))
    bias_t = None if bias is None else gpu.upload(Shape.vector(cols), bias)
    gpu.matmul_fp4(spec.right_transposed(), View(left, offset, x.size), matrix, View(out, offset, rows * cols), bias_t)
    got = gpu.download(out)
    assert (got[:offset] == 123).all() and (got[offset + rows * cols:] == 123).all()
    return got[offset:offset + rows * cols].reshape(rows, cols)


def check(got, x, w, inner, scale=1.0, before=None, bias=None):
    x = x.astype(np.float64)
    total, magnitude = x @ w.T, np.abs(x) @ np.abs(w).T
    expected = scale * total
    bound = (3 * -(-inner // 32) + 64) * 2.0 ** -23 * abs(scale) * magnitude + 2.0 ** -24 * np.abs(expected)
    for more in (before, bias):
        if more is not None:
            expected = expected + more
            bound = bound + 2.0 ** -24 * np.abs(expected)
    wrong = np.abs(got - expected) > bound + 1e-37
    assert not wrong.any(), (np.argwhere(wrong)[:4], got[wrong][:4], expected[wrong][:4])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 6, 15, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("inner,cols", [(1, 1), (31, 17), (32, 16), (33, 15), (129, 130), (1001, 77), (768, 250)])
def test_product(gpu, rows, inner, cols, bf16):
    rng = np.random.default_rng(rows * 7 + inner)
    codes, scales, w = weights(cols, inner, rows + inner)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner).with_precision(Precision.Bf16 if bf16 else Precision.F32)
    got = run(gpu, spec, x, codes, scales, offset=rows % 2)
    check(got, to_bf16(x) if bf16 else x, w, inner)


@pytest.mark.parametrize("rows,inner,cols", [(1, 8192, 300), (4, 4100, 1000), (16, 6000, 700), (40, 3000, 333),
                                             (300, 2052, 520), (513, 640, 1030), (257, 96, 2500)])
def test_long_and_wide(gpu, rows, inner, cols):
    rng = np.random.default_rng(rows)
    codes, scales, w = weights(cols, inner, rows)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    bias = rng.standard_normal(cols).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner)
    got = run(gpu, spec, x, codes, scales, bias=bias)
    check(got, x, w, inner, bias=bias)
    assert np.array_equal(got, run(gpu, spec, x, codes, scales, bias=bias))  # the same bits again
    # Few-row, or accumulated, or scaled: the fp32 tolerance of the framework holds besides.
    error = np.abs(got - (x.astype(np.float64) @ w.T + bias)).max() / np.abs(got).max()
    assert error < MatmulKernel.MfmaF32.tolerance()


@pytest.mark.parametrize("cols", [50, 5201, 12301])
@pytest.mark.parametrize("inner", [4, 33, 300, 1100])
@pytest.mark.parametrize("rows,bf16", [(1, False), (2, True), (5, False), (7, True), (9, False), (16, False), (17, True),
                                       (25, True), (32, True)])
def test_few_rows_of_wide_weights(gpu, rows, bf16, inner, cols):
    """One, two and four column tiles a wave, the last ones partial; blocks that end inside a step."""
    rng = np.random.default_rng(inner)
    codes, scales, w = weights(cols, inner, inner)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner).with_precision(Precision.Bf16 if bf16 else Precision.F32)
    check(run(gpu, spec, x, codes, scales, offset=rows % 2), to_bf16(x) if bf16 else x, w, inner)


@pytest.mark.parametrize("rows,inner,cols,bf16", [
    (2000, 203, 3900, False),   # tiles of 128 x 256, quads shifted at the rows' ends
    (1990, 64, 4001, False),    # the same, one stage
    (1100, 130, 3900, True),    # tiles of 64 x 128
    (1100, 3, 3900, True),      # values read one by one
    (70, 2, 300, False),
    (300, 1000, 200, True)])    # sliced
def test_tiles(gpu, rows, inner, cols, bf16):
    rng = np.random.default_rng(rows)
    codes, scales, w = weights(cols, inner, rows)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    bias = rng.standard_normal(cols).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner).with_precision(Precision.Bf16 if bf16 else Precision.F32)
    check(run(gpu, spec, x, codes, scales, bias=bias, offset=1), to_bf16(x) if bf16 else x, w, inner, bias=bias)


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("offset", [1, 2, 7])
def test_scales_at_any_byte(gpu, rows, offset):
    """Scale bytes need no alignment, and none past the last is read: what surrounds them is NaN's."""
    rng = np.random.default_rng(offset)
    inner, cols = 700, 65
    codes, scales, w = weights(cols, inner, offset)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    around = gpu.upload_bytes(np.concatenate([np.full(offset, 255, np.uint8), scales.ravel(), np.full(40, 255, np.uint8)]))
    matrix = Fp4Matrix(cols, inner, gpu.upload_bytes(codes), View(around, offset, scales.size, 1))
    out = gpu.zeros(Shape.new(rows, cols))
    gpu.matmul_fp4(MatmulSpec.new(rows, cols, inner).right_transposed(), gpu.upload(Shape.new(rows, inner), x), matrix, out)
    check(gpu.download(out).reshape(rows, cols), x, w, inner)


@pytest.mark.parametrize("rows", [1, 5, 9, 40, 100])
@pytest.mark.parametrize("with_bias", [False, True])
def test_scale_accumulate_and_bias(gpu, rows, with_bias):
    rng = np.random.default_rng(rows)
    inner, cols = 200, 50
    codes, scales, w = weights(cols, inner, 5)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    before = rng.standard_normal((rows, cols)).astype(np.float32)
    bias = rng.standard_normal(cols).astype(np.float32) if with_bias else None
    spec = MatmulSpec.new(rows, cols, inner).scaled(-0.375)
    check(run(gpu, spec, x, codes, scales, bias=bias), x, w, inner, -0.375, None, bias)
    check(run(gpu, spec.accumulate(), x, codes, scales, bias=bias, before=before), x, w, inner, -0.375, before, bias)


@pytest.mark.parametrize("rows", [1, 4, 7, 20, 70])
def test_infinities_nan_and_large_values_follow_ieee(gpu, rows):
    """Each stays in its row (x) or column (a NaN block); inf times 0 is NaN, inf times others inf; the
    largest float times a code is exact."""
    rng = np.random.default_rng(rows)
    inner, cols = 96, 40
    codes, scales, _ = weights(cols, inner, 6)
    scales[3, 1] = 255
    scales[7, 2] = 253
    w = ref.dequantize(codes, scales, inner)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    x[0, 40] = np.inf
    if rows > 1:
        x[1, 5] = np.nan
        x[1, 6] = np.array([0x7F800001], np.uint32).view(np.float32)[0]  # a NaN with low bits only
        x[rows - 1, :] = 0
        x[rows - 1, 70] = np.finfo(np.float32).max * (0.25 if rows % 2 else -0.25)
    got = run(gpu, MatmulSpec.new(rows, cols, inner), x, codes, scales)
    with np.errstate(invalid="ignore", over="ignore"):
        expected = x.astype(np.float64) @ w.T
        expected = np.where(np.abs(expected) > np.finfo(np.float32).max, np.sign(expected) * np.inf, expected)
    assert np.array_equal(np.isnan(got), np.isnan(expected))
    assert np.array_equal(np.isinf(got), np.isinf(expected))
    finite = np.isfinite(expected)
    with np.errstate(invalid="ignore"):
        magnitude = np.abs(x.astype(np.float64)) @ np.abs(w).T
    assert (np.abs(got - expected)[finite] <= 73 * 2.0 ** -23 * magnitude[finite]).all()


def test_every_scale_byte(gpu):
    """One block a column, its scale byte the column's number: exact for one row of one value."""
    codes = np.tile(np.arange(16, dtype=np.uint8) * 0x11, (256, 1))
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    w = ref.dequantize(codes, scales)
    for k in (1, 14, 15):  # codes 0, 7 and 7's neighbour: 0.5 .. 6
        x = np.zeros((1, 32), np.float32)
        x[0, k] = 1
        got = run(gpu, MatmulSpec.new(1, 256, 32), x, codes, scales)[0]
        assert np.array_equal(got[:253], w[:253, k].astype(np.float32))
        assert np.isnan(got[253:]).all()


def test_precision_goes_by_the_context_and_the_spec():
    gpu = Gpu(0, workspace_bytes=0)
    try:
        rng = np.random.default_rng(2)
        codes, scales, w = weights(48, 128, 3)
        for rows in (3, 30, 200):
            x = rng.standard_normal((rows, 128)).astype(np.float32)
            spec = MatmulSpec.new(rows, 48, 128)
            f32 = run(gpu, spec, x, codes, scales)
            check(f32, x, w, 128)
            gpu.matmul_kernel = MatmulKernel.Simple
            assert np.array_equal(run(gpu, spec, x, codes, scales), f32)
            gpu.matmul_kernel = MatmulKernel.MfmaBf16
            bf16 = run(gpu, spec, x, codes, scales)
            check(bf16, to_bf16(x), w, 128)
            assert np.array_equal(run(gpu, spec.with_precision(Precision.F32), x, codes, scales), f32)
            gpu.matmul_kernel = MatmulKernel.MfmaF32
            assert np.array_equal(run(gpu, spec.with_precision(Precision.Bf16), x, codes, scales), bf16)
    finally:
        gpu.close()


@pytest.mark.parametrize("rows", [2, 9, 20])
def test_codes_past_32_bits(gpu, rows):
    """5 GB of codes, zeros but for the last 40 columns."""
    cols, inner, some = 300_000, 32_768, 40
    rng = np.random.default_rng(rows)
    matrix = gpu.fp4_matrix(cols, inner)
    w = rng.standard_normal((some, inner)).astype(np.float32)
    blocks = inner // 32
    part = Fp4Matrix(some, inner, View(matrix.codes, (cols - some) * blocks * 16, some * blocks * 16, 1),
                     View(matrix.scales, (cols - some) * blocks, some * blocks, 1))
    gpu.quantize_fp4(gpu.upload(Shape.vector(w.size), w), part, Storage.Transposed)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    out = gpu.upload(Shape(rows, cols), np.ones(rows * cols))
    gpu.matmul_fp4(MatmulSpec.new(rows, cols, inner).right_transposed(), gpu.upload(Shape(rows, inner), x), matrix, out)
    got = gpu.download(out).reshape(rows, cols)
    assert not got[:, :-some].any()
    values = ref.dequantize(gpu.download_bytes(part.codes).reshape(some, -1),
                            gpu.download_bytes(part.scales).reshape(some, -1), inner)
    check(got[:, -some:], x, values, inner)


def test_empty_products_and_refusals_on_the_device(gpu):
    codes, scales, _ = weights(4, 32, 1)
    x = np.ones((2, 32), np.float32)
    assert run(gpu, MatmulSpec.new(0, 4, 32), x[:0], codes, scales).size == 0
    empty = run(gpu, MatmulSpec.new(2, 4, 0), x[:, :0], codes[:, :0], scales[:, :0], bias=np.arange(4.0))
    assert np.array_equal(empty, np.tile(np.arange(4.0), (2, 1)))
    left = gpu.upload(Shape(2, 32), x)
    out = gpu.zeros(Shape(2, 4))
    shifted = Fp4Matrix(3, 32, View(gpu.upload_bytes(codes), 4, 60, 1), gpu.upload_bytes(scales))
    with pytest.raises(MatmulPanic, match="unsupported"):
        gpu.matmul_fp4(MatmulSpec.new(2, 3, 32).right_transposed(), left, shifted, out)
    matrix = Fp4Matrix(4, 32, gpu.upload_bytes(codes), gpu.upload_bytes(scales))
    with pytest.raises(MatmulPanic, match="overlaps"):
        gpu.matmul_fp4(MatmulSpec.new(2, 4, 32).right_transposed(), left, matrix, View(left, 3, 8))
    with pytest.raises(MatmulPanic, match="right operand"):
        gpu.matmul_fp4(MatmulSpec.new(2, 5, 32).right_transposed(), left, matrix, out)
