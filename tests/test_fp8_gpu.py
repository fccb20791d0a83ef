"""GPU parity of 8-bit operands (``sn_quantize_fp8``, ``sn_dequantize_fp8``) with their numpy form, bit for bit, and of
their products (``sn_matmul_fp8``) with 64 bits.

Tolerance of a product. Products are exact; what differs from the 64-bit result is the fp32 summation. An output's sum
is a chain of at most ceil(inner / 32) additions into a matrix accumulator, 32 terms added inside each instruction, and at
most 32 slices' sums added after; each rounding is at most 2^-23 (were additions to cut off) of a partial sum, which the
sum of magnitudes S bounds: (ceil(inner / 32) + 64) 2^-23 S. The scale, the previous output and the bias add a rounding
of half a step each: 2^-24 of what they meet."""
import numpy as np
import pytest

import fp8_reference as ref
from bench import HipGraph
from fp4_reference import View
from staleynet_amd.gemm import Fp8Matrix, Gpu, GpuError, MatmulPanic, MatmulSpec, Shape, Storage

pytestmark = pytest.mark.gpu


def upload(gpu, values, offset=0):
    """Values in a device buffer from its element `offset` on."""
    flat = np.ascontiguousarray(values, np.float32).ravel()
    return View(gpu.upload(Shape.vector(flat.size + offset), np.concatenate([np.zeros(offset, np.float32), flat])), offset,
                flat.size)


def quantized(gpu, values, storage=Storage.RowMajor, offset=0, guard=64):
    """Codes and scales from the GPU; what lies behind them has to keep its bytes."""
    rows, inner = values.shape
    codes, scales = rows * ref.blocks_of(inner) * 128, rows * ref.scale_stride(inner)
    held = [gpu.upload_bytes(np.full(n + guard, 77, np.uint8)) for n in (codes, scales)]
    matrix = Fp8Matrix(rows, inner, View(held[0], 0, codes, 1), View(held[1], 0, scales, 1))
    source = values if storage == Storage.RowMajor else values.T
    gpu.quantize_fp8(upload(gpu, source, offset), matrix, storage)
    got = [gpu.download_bytes(b) for b in held]
    assert (got[0][codes:] == 77).all() and (got[1][scales:] == 77).all()
    return got[0][:codes].reshape(rows, -1), got[1][:scales].reshape(rows, -1), matrix


def same_as_reference(gpu, values, **kw):
    codes, scales, matrix = quantized(gpu, values, **kw)
    want_codes, want_scales = ref.quantize(values)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes), np.argwhere(codes != want_codes)[:4]
    return codes, scales, matrix


@pytest.mark.parametrize("storage", list(Storage))
@pytest.mark.parametrize("rows,inner", [(1, 1), (1, 127), (3, 128), (2, 129), (65, 300), (70, 512), (130, 513), (7, 1001),
                                        (257, 768)])
def test_quantize_and_back(gpu, rows, inner, storage):
    rng = np.random.default_rng(rows + inner)
    values = rng.standard_normal((rows, inner)) * 10.0 ** rng.integers(-3, 4, (rows, 1))
    values[rng.random(values.shape) < 0.05] = 0
    codes, scales, matrix = same_as_reference(gpu, values.astype(np.float32), storage=storage, offset=inner % 3)
    want = ref.dequantize(codes, scales, inner).astype(np.float32)
    shape = (rows, inner) if storage == Storage.RowMajor else (inner, rows)
    filled = np.full(rows * inner + 12, 5, np.float32)
    out = gpu.upload(Shape.vector(filled.size), filled)
    gpu.dequantize_fp8(matrix, View(out, 3, rows * inner), storage)
    got = gpu.download(out)
    assert (got[:3] == 5).all() and (got[3 + rows * inner:] == 5).all()
    got = got[3:3 + rows * inner].reshape(shape)
    assert np.array_equal(got if storage == Storage.RowMajor else got.T, want)


@pytest.mark.parametrize("storage", list(Storage))
def test_every_tie_and_its_neighbours(gpu, storage):
    """Each code's value, each middle of two codes and the floats next to it, both signs, at factors from the least to
    the largest; the block's largest magnitude (448, or 464 at which it still is the factor) fixes the factor."""
    middles = (ref.MAGNITUDES[:126] + ref.MAGNITUDES[1:127]) / 2
    values = np.concatenate([ref.MAGNITUDES[:127], middles]).astype(np.float32)
    values = np.concatenate([values, np.nextafter(values, np.float32(0)), np.nextafter(values, np.float32(1e9))])
    values = values[values <= 464]
    values = np.concatenate([values, -values, [0.0, -0.0]]).astype(np.float32)
    values = np.pad(values, (0, -values.size % 127)).reshape(-1, 127)
    rows = []
    for largest in (448, 464):
        block = np.concatenate([np.full((len(values), 1), largest, np.float32), values], 1)
        for e in (-124, -123, -100, -1, 0, 1, 60, 118):
            with np.errstate(under="ignore"):
                rows.append((block.astype(np.float64) * 2.0 ** e).astype(np.float32))
    same_as_reference(gpu, np.concatenate(rows), storage=storage)


@pytest.mark.parametrize("storage", list(Storage))
def test_the_edges_of_the_range(gpu, storage):
    """Blocks of zeros, of subnormals, past 448 of the largest factor, with infinities and NaN; 464 and the next float."""
    largest = np.finfo(np.float32).max
    rng = np.random.default_rng(4)
    rows = np.zeros((12, 300), np.float32)
    rows[0, 5] = -0.0
    rows[1] = rng.integers(0, 1 << 23, 300).astype(np.uint32).view(np.float32)      # subnormal floats
    rows[2] = 2.0 ** -126
    rows[3] = rng.standard_normal(300) * 2.0 ** -118
    rows[4] = rng.uniform(-1, 1, 300) * largest
    rows[5, ::2] = largest
    rows[5, 1::2] = -largest
    rows[6] = rng.standard_normal(300)
    rows[6, 130] = np.inf
    rows[7] = rng.standard_normal(300)
    rows[7, 2] = -np.inf
    rows[7, 299] = np.nan
    rows[8, 140] = np.array([0x7F800001], np.uint32).view(np.float32)[0]            # a NaN of low bits only
    rows[9, 0], rows[9, 128] = 464, np.nextafter(np.float32(464), np.float32(465))
    rows[10, 0], rows[10, 128] = 463.99997, 465
    rows[11] = 448 * 2.0 ** 119 * rng.choice([1, 0.5, 0.53, 1.0 / 900], 300)
    _, scales, _ = same_as_reference(gpu, rows, storage=storage)
    assert list(scales[0]) == [3, 3, 3, 0] and list(scales[7]) == [255, scales[7, 1], 255, 0]


def test_every_code_and_scale_byte(gpu):
    """All 256 codes under all 256 scale bytes, read back and as a product with one (both operands): exact, or NaN."""
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.zeros((256, 4), np.uint8)
    scales[:, :2] = np.arange(256)[:, None]
    want = ref.dequantize(codes, scales)
    matrix = Fp8Matrix(256, 256, gpu.upload_bytes(codes), gpu.upload_bytes(scales))
    out = gpu.zeros(Shape(256, 256))
    gpu.dequantize_fp8(matrix, out)
    got = gpu.download(out).reshape(256, 256)
    assert np.array_equal(got, want.astype(np.float32), equal_nan=True)
    assert np.signbit(got[:247, 128]).all()  # -0 (a NaN block has no sign)
    # Column c of `one` is 1 at k = c: a product picks each value out of its row.
    one = np.zeros((256, 256), np.uint8)
    np.fill_diagonal(one, 0x38)
    ones = np.zeros((256, 4), np.uint8)
    ones[:, :2] = 127
    identity = Fp8Matrix(256, 256, gpu.upload_bytes(one), gpu.upload_bytes(ones))
    finite = codes.copy()
    finite[:, [127, 255]] = 0  # a NaN code makes all of its row NaN
    matrix = Fp8Matrix(256, 256, gpu.upload_bytes(finite), gpu.upload_bytes(scales))
    want = ref.dequantize(finite, scales).astype(np.float32)
    spec = MatmulSpec.new(256, 256, 256).right_transposed()
    gpu.matmul_fp8(spec, matrix, identity, out)
    assert np.array_equal(gpu.download(out).reshape(256, 256), want, equal_nan=True)
    gpu.matmul_fp8(spec, identity, matrix, out)
    assert np.array_equal(gpu.download(out).reshape(256, 256).T, want, equal_nan=True)


def operand(rows, inner, seed, spread=3):
    """Codes and scales drawn as such (quick for large operands), without NaN codes, and their values."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (rows, ref.blocks_of(inner) * 128), dtype=np.uint8)
    codes[(codes & 127) == 127] = 0x30
    codes[:, inner:] = 0
    scales = np.zeros((rows, ref.scale_stride(inner)), np.uint8)
    scales[:, :ref.blocks_of(inner)] = rng.integers(120 - spread, 120 + spread, (rows, ref.blocks_of(inner)))
    return codes, scales, ref.dequantize(codes, scales, inner)


def matrix_of(gpu, codes, scales, inner):
    return Fp8Matrix(len(codes), inner, gpu.upload_bytes(codes), gpu.upload_bytes(scales))


def run(gpu, spec, left, right, bias=None, before=None, guard=9):
    """The product; what lies around the output has to keep its values."""
    count = spec.rows * spec.cols
    filled = np.full(count + 2 * guard, 123.0, np.float32)
    if before is not None:
        filled[guard:guard + count] = before.ravel()
    out = gpu.upload(Shape.vector(filled.size), filled)
    bias_t = None if bias is None else gpu.upload(Shape.vector(spec.cols), bias)
    gpu.matmul_fp8(spec.right_transposed(), matrix_of(gpu, *left[:2], spec.inner), matrix_of(gpu, *right[:2], spec.inner),
                   View(out, guard, count), bias_t)
    got = gpu.download(out)
    assert (got[:guard] == 123).all() and (got[guard + count:] == 123).all()
    return got[guard:guard + count].reshape(spec.rows, spec.cols)


def check(got, x, w, inner, scale=1.0, before=None, bias=None):
    total, magnitude = x @ w.T, np.abs(x) @ np.abs(w).T
    expected = scale * total
    bound = (-(-inner // 32) + 64) * 2.0 ** -23 * abs(scale) * magnitude + 2.0 ** -24 * np.abs(expected)
    for more in (before, bias):
        if more is not None:
            expected = expected + more
            bound = bound + 2.0 ** -24 * np.abs(expected)
    wrong = np.abs(got - expected) > bound + 1e-37
    assert not wrong.any(), (np.argwhere(wrong)[:4], got[wrong][:4], expected[wrong][:4])


@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 130])
@pytest.mark.parametrize("inner,cols", [(1, 1), (127, 17), (128, 16), (129, 15), (513, 130), (1001, 77), (768, 250)])
def test_product(gpu, rows, inner, cols):
    left, right = operand(rows, inner, rows), operand(cols, inner, cols)
    check(run(gpu, MatmulSpec.new(rows, cols, inner), left, right), left[2], right[2], inner)


@pytest.mark.parametrize("rows,inner,cols", [(1, 8192, 300), (4, 4100, 1000), (16, 6000, 700), (40, 3000, 333),
                                             (64, 5000, 520), (80, 2500, 2049), (300, 2052, 520), (513, 640, 1030),
                                             (257, 96, 2500), (1100, 130, 3900), (200, 9000, 200)])
def test_long_and_wide(gpu, rows, inner, cols):
    left, right = operand(rows, inner, rows), operand(cols, inner, cols)
    bias = np.random.default_rng(rows).standard_normal(cols).astype(np.float32)
    spec = MatmulSpec.new(rows, cols, inner)
    got = run(gpu, spec, left, right, bias=bias)
    check(got, left[2], right[2], inner, bias=bias)
    assert np.array_equal(got, run(gpu, spec, left, right, bias=bias))  # the same bits again


@pytest.mark.parametrize("rows,inner,cols", [
    (16, 300, 4300), (9, 1000, 6201), (16, 1200, 12301), (3, 130, 12300), (20, 1500, 4097), (32, 1100, 16500), (17, 260, 16401),
    (16, 9000, 500), (20, 10000, 300), (50, 9000, 700), (64, 2100, 4096), (40, 1500, 4097), (64, 900, 9001),  # of few rows, then tiles of each size
    (80, 260, 16400), (333, 2000, 3000), (69, 6252, 4186), (1000, 1200, 3001), (520, 9000, 3900), (1500, 1000, 3001)])
def test_each_form(gpu, rows, inner, cols):
    left, right = operand(rows, inner, rows), operand(cols, inner, cols)
    check(run(gpu, MatmulSpec.new(rows, cols, inner), left, right), left[2], right[2], inner)


@pytest.mark.parametrize("inner", [1, 130, 300, 500, 640, 700, 900])
@pytest.mark.parametrize("rows,cols", [(4090, 4081), (2500, 4095)])
def test_the_largest_tiles(gpu, rows, cols, inner):
    """One to eight blocks: whole rounds of steps and each remainder."""
    left, right = operand(rows, inner, rows), operand(cols, inner, cols)
    got = run(gpu, MatmulSpec.new(rows, cols, inner).accumulate(), left, right, before=np.ones((rows, cols), np.float32))
    check(got, left[2], right[2], inner, before=np.ones((rows, cols), np.float32))


@pytest.mark.parametrize("rows", [1, 5, 16, 40, 100, 300])
@pytest.mark.parametrize("with_bias", [False, True])
def test_scale_accumulate_and_bias(gpu, rows, with_bias):
    rng = np.random.default_rng(rows)
    inner, cols = 2000, 50
    left, right = operand(rows, inner, rows), operand(cols, inner, 5)
    before = rng.standard_normal((rows, cols)).astype(np.float32)
    bias = rng.standard_normal(cols).astype(np.float32) if with_bias else None
    spec = MatmulSpec.new(rows, cols, inner).scaled(-0.375)
    check(run(gpu, spec, left, right, bias), left[2], right[2], inner, -0.375, None, bias)
    check(run(gpu, spec.accumulate(), left, right, bias, before), left[2], right[2], inner, -0.375, before, bias)


@pytest.mark.parametrize("rows", [1, 20, 100])
def test_an_empty_inner_dimension(gpu, rows):
    before, bias = np.full((rows, 30), 2, np.float32), np.arange(30, dtype=np.float32)
    empty = np.zeros((rows, 0), np.uint8), np.zeros((rows, 0), np.uint8)
    other = np.zeros((30, 0), np.uint8), np.zeros((30, 0), np.uint8)
    spec = MatmulSpec.new(rows, 30, 0)
    assert np.array_equal(run(gpu, spec, empty, other, bias), np.tile(bias, (rows, 1)))
    assert np.array_equal(run(gpu, spec.accumulate(), empty, other, bias, before), before + bias)
    assert np.array_equal(run(gpu, spec, empty, other), np.zeros((rows, 30)))


@pytest.mark.parametrize("rows", [3, 20, 70, 300])
def test_nan_blocks_and_codes_stay_in_their_row_or_column(gpu, rows):
    inner, cols = 600, 90
    left, right = operand(rows, inner, 1), operand(cols, inner, 2)
    left[1][1, 2] = 255
    left[0][rows - 1, 599] = 0x7F
    right[1][40, 4] = 247
    right[0][89, 0] = 0xFF
    x, w = ref.dequantize(*left[:2], inner), ref.dequantize(*right[:2], inner)
    got = run(gpu, MatmulSpec.new(rows, cols, inner), left, right)
    bad = np.isnan(x).any(1)[:, None] | np.isnan(w).any(1)[None]
    assert np.array_equal(np.isnan(got), bad)
    x, w = np.nan_to_num(x), np.nan_to_num(w)
    check(np.where(bad, x @ w.T, got), x, w, inner)


@pytest.mark.parametrize("rows", [1, 33, 100])
def test_extreme_factors(gpu, rows):
    """Large factors meet small ones, sums overflow to infinities and fall to subnormals as the formula has it."""
    rng = np.random.default_rng(rows)
    inner, cols = 384, 64
    left, right = operand(rows, inner, 3), operand(cols, inner, 4)
    left[1][:, :3], right[1][:, :3] = [3, 246, 130], [246, 3, 120]
    w = ref.dequantize(*right[:2], inner)
    check(run(gpu, MatmulSpec.new(rows, cols, inner), left, right), ref.dequantize(*left[:2], inner), w, inner)
    left[1][:, :3], right[1][:, :3] = 70, rng.integers(50, 60, (cols, 1))  # of 2^-134 .. 2^-100
    x, w = ref.dequantize(*left[:2], inner), ref.dequantize(*right[:2], inner)
    got = run(gpu, MatmulSpec.new(rows, cols, inner), left, right)
    # Each of the 12 + 64 roundings is a subnormal's half step besides.
    assert (np.abs(got - x @ w.T) <= 76 * (2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -149)).all()
    left[1][:, :3], right[1][:, :3] = 246, 200
    x, w = np.abs(ref.dequantize(*left[:2], inner)), np.abs(ref.dequantize(*right[:2], inner))
    got = run(gpu, MatmulSpec.new(rows, cols, inner), (left[0] & 127, left[1]), (right[0] & 127, right[1]))
    assert (got[x @ w.T > 1e39] == np.inf).all() and (x @ w.T > 1e39).any()


@pytest.mark.parametrize("rows,cols,inner", [(1, 300, 4000), (50, 64, 9000), (300, 200, 4000)])
def test_a_small_workspace(gpu, rows, cols, inner):
    left, right = operand(rows, inner, 5), operand(cols, inner, 6)
    for bytes_ in (0, 1 << 16):
        other = Gpu(0, workspace_bytes=bytes_)
        try:
            check(run(other, MatmulSpec.new(rows, cols, inner), left, right), left[2], right[2], inner)
        finally:
            other.close()


def test_rows_do_not_depend_on_others(gpu):
    """A row's bits are the same whatever the other rows hold."""
    for rows in (1, 12, 40, 200):
        left, right = operand(rows, 3000, 7), operand(210, 3000, 8)
        spec = MatmulSpec.new(rows, 210, 3000)
        got = run(gpu, spec, left, right)
        changed = left[0].copy()
        changed[1:] = 0x7E
        assert np.array_equal(run(gpu, spec, (changed, left[1]), right)[0], got[0])


def test_offsets_past_32_bits(gpu):
    """5 GB of codes: the last four blocks of an operand's last two rows, and of another's, among zeros."""
    inner, rows, cols = 1 << 20, 5000, 40
    rng = np.random.default_rng(10)
    left, right = gpu.fp8_matrix(rows, inner), gpu.fp8_matrix(cols, inner)

    def fill(matrix, row):
        values = rng.standard_normal((1, 512)).astype(np.float32)
        end, scales = (row + 1) * inner, (row + 1) * (inner // 128)
        part = Fp8Matrix(1, 512, View(matrix.codes, end - 512, 512, 1), View(matrix.scales, scales - 4, 4, 1))
        gpu.quantize_fp8(upload(gpu, values), part)
        return ref.dequantize(*ref.quantize(values))[0]

    x = np.stack([fill(left, rows - 2), fill(left, rows - 1)])
    w = np.stack([fill(right, c) for c in range(cols)])
    out = gpu.zeros(Shape(rows, cols))
    gpu.matmul_fp8(MatmulSpec.new(rows, cols, inner).right_transposed(), left, right, out)
    got = gpu.download(out).reshape(rows, cols)
    assert not got[:-2].any()
    check(got[-2:], x, w, inner)
    few = Fp8Matrix(2, inner, View(left.codes, (rows - 2) * inner, 2 * inner, 1),
                    View(left.scales, (rows - 2) * (inner // 128), inner // 64, 1))
    out = gpu.zeros(Shape(2, rows))
    gpu.matmul_fp8(MatmulSpec.new(2, rows, inner).right_transposed(), few, left, out)
    got = gpu.download(out).reshape(2, rows)
    assert not got[:, :-2].any()
    check(got[:, -2:], x, x, inner)


def test_refusals_on_the_device(gpu):
    matrix, out = gpu.fp8_matrix(4, 128), gpu.zeros(Shape(4, 4))
    spec = MatmulSpec.new(4, 4, 128).right_transposed()
    gpu.matmul_fp8(spec, matrix, matrix, out)  # the same operand twice is allowed
    for bad in (Fp8Matrix(4, 128, View(gpu.zeros_bytes(600), 8, 512, 1), matrix.scales),
                Fp8Matrix(4, 128, matrix.codes, View(gpu.zeros_bytes(32), 2, 16, 1))):
        for left, right in ((bad, matrix), (matrix, bad)):
            with pytest.raises(MatmulPanic):
                gpu.matmul_fp8(spec, left, right, out)
        with pytest.raises(MatmulPanic):
            gpu.quantize_fp8(gpu.zeros(Shape(4, 128)), bad)
    overlapping = Fp8Matrix(4, 128, View(out, 0, 512, 1), matrix.scales)
    with pytest.raises((MatmulPanic, GpuError)):
        gpu.matmul_fp8(spec, overlapping, matrix, View(out, 0, 16))
    with pytest.raises(MatmulPanic):
        gpu.matmul_fp8(MatmulSpec.new(4, 5, 128).right_transposed(), matrix, matrix, out)


def test_captured_products_replay(gpu):
    """Few rows, sliced and tiled products and the quantizing ahead of them in one graph: each replay leaves the eager
    bits, with eager work and synchronizations between the replays."""
    rng = np.random.default_rng(9)
    calls = []
    for rows, cols, inner in ((1, 700, 2000), (50, 64, 9000), (300, 400, 700)):
        x = gpu.upload(Shape(rows, inner), rng.standard_normal((rows, inner)))
        w = gpu.upload(Shape(inner, cols), rng.standard_normal((inner, cols)))
        left, right, out = gpu.fp8_matrix(rows, inner), gpu.fp8_matrix(cols, inner), gpu.zeros(Shape(rows, cols))
        calls.append((MatmulSpec.new(rows, cols, inner).right_transposed(), x, w, left, right, out))

    def step():
        for spec, x, w, left, right, out in calls:
            gpu.quantize_fp8(x, left)
            gpu.quantize_fp8(w, right, Storage.Transposed)
            gpu.matmul_fp8(spec, left, right, out)

    step()
    want = [gpu.download(c[-1]) for c in calls]
    for (spec, x, w, *_), got in zip(calls, want):
        a = ref.dequantize(*ref.quantize(gpu.download(x).reshape(spec.rows, spec.inner)), spec.inner)
        b = ref.dequantize(*ref.quantize(gpu.download(w).reshape(spec.inner, spec.cols).T), spec.inner)
        check(got.reshape(spec.rows, spec.cols), a, b, spec.inner)
    graph = HipGraph(gpu.stream, step)
    try:
        for _ in range(3):
            for c in calls:
                gpu.fill_zero(c[-1])
            graph.launch()
            gpu.synchronize()
            for c, expected in zip(calls, want):
                assert np.array_equal(gpu.download(c[-1]), expected)
            gpu.matmul_fp8(calls[1][0], calls[1][3], calls[1][4], calls[1][5])
    finally:
        graph.close()


@pytest.mark.parametrize("rows,inner", [(70, 33000), (1, 40001), (130, 32897)])
def test_columns_of_more_blocks_than_a_grid_holds(gpu, rows, inner):
    """Transposed operands of more than 256 blocks, as a batch's tokens are a weight gradient's inner dimension."""
    test_quantize_and_back(gpu, rows, inner, Storage.Transposed)


@pytest.mark.parametrize("rows,inner,cols", [(2701, 2348, 68), (129, 9077, 6403), (4109, 4929, 932)])
def test_slices_of_the_other_tiles(gpu, rows, inner, cols):
    """Tiles of 64 x 128, 192 x 256 and 256 x 256 with the inner dimension in slices."""
    left, right = operand(rows, inner, rows), operand(cols, inner, cols)
    rng = np.random.default_rng(rows)
    before, bias = (rng.standard_normal(n).astype(np.float32) for n in ((rows, cols), cols))
    spec = MatmulSpec.new(rows, cols, inner).scaled(0.25).accumulate()
    check(run(gpu, spec, left, right, bias, before), left[2], right[2], inner, 0.25, before, bias)


@pytest.mark.parametrize("tokens,width,cols", [(1, 40, 70), (333, 200, 300), (1100, 768, 130), (4099, 96, 513)])
def test_a_weight_gradient(gpu, tokens, width, cols):
    """dW += X^T dY: both operands transposed to 8-bit blocks along the tokens."""
    rng = np.random.default_rng(tokens)
    x, d_y = (rng.standard_normal((tokens, n)).astype(np.float32) for n in (width, cols))
    before = rng.standard_normal((width, cols)).astype(np.float32)
    left, right = (same_as_reference(gpu, np.ascontiguousarray(v.T), storage=Storage.Transposed) for v in (x, d_y))
    out = gpu.upload(Shape(width, cols), before)
    gpu.matmul_fp8(MatmulSpec.new(width, cols, tokens).right_transposed().accumulate(), left[2], right[2], out)
    a, b = (ref.dequantize(*m[:2], tokens) for m in (left, right))
    check(gpu.download(out).reshape(width, cols), a, b, tokens, before=before)
