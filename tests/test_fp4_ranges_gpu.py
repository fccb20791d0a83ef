"""The ends of the ranges that the header of the 4-bit operators states: values, strides, lengths, the capacity of a cache
and the inner dimension of a product."""
import numpy as np
import pytest

import fp4_reference as ref
from fp4_reference import View
from staleynet_amd.gemm import Fp4Matrix, Gpu, GpuError, MatmulSpec, Precision, Shape, Storage
from test_fp4_attention_gpu import Case
from test_fp4_matmul_gpu import check as check_product
from test_fp4_matmul_gpu import to_bf16

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


@pytest.mark.parametrize("strides,accepted", [
    ((192, 32, 64), True), ((192, 32, 63), False), ((191, 32, 64), False), ((192, 31, 64), False),  # (time, head)
    ((96, 192, 32), True), ((95, 192, 32), False), ((96, 191, 32), False),                          # (head, sequence, time)
    ((400, 96, 64), False)])  # heads at 0, 96, rows at 0, 64, 128: shares nothing but does not nest
def test_output_strides_nest(gpu, strides, accepted):
    """Two sequences of two heads and three queries, 32 floats each: the least strides, one under them, and strides that
    interleave. Accepted ones leave what lies between the outputs as it was."""
    case = Case(2, 2, 2, 3, 9, 32, [9, 5], seed=1)
    q = gpu.upload(Shape.vector(case.q.size), case.q)
    filled = np.full(1000, 7, np.float32)
    out = gpu.upload(Shape.vector(1000), filled)
    call = lambda: gpu.fp4_attention(case.cache(gpu), q, out, 2, 3, case.scale, 0, gpu.upload_tokens(case.lengths),
                                     out_strides=strides)
    if not accepted:
        with pytest.raises(GpuError, match="overlaps"):
            call()
        assert (gpu.download(out) == 7).all()
        return
    call()
    at = sum(np.arange(n).reshape([-1 if i == j else 1 for j in range(4)]) * s
             for i, (n, s) in enumerate(zip((2, 2, 3, 32), (*strides, 1))))
    got = gpu.download(out)
    case.check(got[at])
    filled[at] = got[at]
    assert np.array_equal(got, filled)


def test_strides_of_single_counts_are_not_used(gpu):
    case = Case(1, 1, 1, 1, 9, 32, [9], seed=2)
    out = gpu.zeros(Shape.vector(32))
    gpu.fp4_attention(case.cache(gpu), gpu.upload(Shape.vector(32), case.q), out, 1, 1, case.scale, 9, q_strides=(0, 0, 0),
                      out_strides=(0, 0, 0))
    case.check(gpu.download(out).reshape(case.q.shape))


def test_weights_of_a_very_long_cache_are_all_counted():
    """3 x 2^28 positions that one workgroup takes (no workspace), 3 x 2^23 a lane: the sum of their equal weights, which
    are 1, is exact, so the output is within a few roundings of the values' sum by the positions."""
    gpu = Gpu(0, workspace_bytes=0)
    try:
        capacity, time = 3 << 28, 40
        cache = gpu.fp4_cache(1, 1, capacity, 32)
        packed = np.random.default_rng(31).standard_normal((time, 64)).astype(np.float32)
        gpu.fp4_cache_append(cache, gpu.upload(Shape(time, 64), packed), time, 64, 0, 32, position=capacity - time)
        values = ref.dequantize(*ref.quantize(packed[:, 32:]))
        q, out = gpu.zeros(Shape(1, 32)), gpu.zeros(Shape(1, 32))
        gpu.fp4_attention(cache, q, out, 1, 1, 1.0, keys=capacity)
        want = values.sum(0) / capacity
        assert (np.abs(gpu.download(out) - want) <= 2.0 ** -19 * np.abs(values).sum(0) / capacity).all()
        del cache, q, out
    finally:
        gpu.close()


def test_the_largest_capacity(gpu):
    """2^30 - 1 positions, all held, and so many rows that each tile's keys are one workgroup's share: a share of the
    capacity and the keys held are together 2^31. Positions never written hold zeros, so a query's result is known from
    the 40 that all queries see and that are written."""
    capacity, head_dim, heads, queries, time = (1 << 30) - 1, 32, 4, 1028, 40
    rng = np.random.default_rng(30)
    cache = gpu.fp4_cache(1, 1, capacity, head_dim)
    packed = rng.standard_normal((time, 64)).astype(np.float32)
    first = capacity - queries - time
    gpu.fp4_cache_append(cache, gpu.upload(Shape(time, 64), packed), time, 64, 0, 32, position=first)
    k, v = (ref.dequantize(*ref.quantize(packed[:, i:i + 32])) for i in (0, 32))
    q = rng.standard_normal((heads * queries, head_dim)).astype(np.float32)
    q[::4] = 0
    out = gpu.upload(Shape(heads * queries, head_dim), np.full(q.size, 7, np.float32))
    gpu.fp4_attention(cache, gpu.upload(Shape(heads * queries, head_dim), q), out, heads, queries, 6.0,
                      lengths=gpu.upload_tokens([capacity]))
    got = gpu.download(out).reshape(q.shape)
    s = q.astype(np.float64) @ k.T * 6
    top = np.maximum(s.max(1, keepdims=True), 0)
    p = np.exp(s - top)
    seen = capacity - queries + 1 + np.arange(heads * queries) % queries  # head by head
    others = (seen[:, None] - time) * np.exp(-top)
    total = p.sum(1, keepdims=True) + others
    # Queries of zeros have weights of 1, whose sums are exact. A score of the others is a sum of magnitudes of under 300, so off
    # by (3 + 66) 2^-23 of that, 2^-8.6, which numerator and sum each have; equal weights that are no powers of two are
    # chains of 2^22 additions a lane, each off by 2^-24 of the sum so far: by 2^-2 of their share.
    assert 6 * (np.abs(q) @ np.abs(k).T).max() < 300
    off = np.where(q.any(1, keepdims=True), 2.0 ** -6 + 2.0 ** -2 * others / total, 2.0 ** -18)
    # And each of the 40 weights counts as 0 where it is under 2^-118 of the largest: where the
    # largest one's value is 0, that may be all there is of an output.
    bound = off * (p @ np.abs(v)) / total + time * 2.0 ** -118 * np.abs(v).max()
    assert (np.abs(got - p @ v / total) <= bound).all()


@pytest.mark.parametrize("rows,bf16", [(1, False), (5, False), (16, False), (30, True), (40, False), (40, True)])
def test_the_longest_inner_dimension(gpu, rows, bf16):
    """2^25 - 1 values a column, 5 GB of codes, zeros but for the first and the last two blocks of some columns: a product of 95
    values, as exact as that."""
    inner, cols = (1 << 25) - 1, 300
    blocks = ref.blocks_of(inner)
    rng = np.random.default_rng(rows)
    matrix = gpu.fp4_matrix(cols, inner)
    w = np.zeros((cols, 95))
    for c in (0, 1, 63, 64, 127, 255, 256, 299):
        for first, at, count in ((0, 0, 32), (blocks - 2, 32, 63)):
            place, size = c * blocks + first, -(-count // 32)
            part = Fp4Matrix(1, count, View(matrix.codes, place * 16, size * 16, 1), View(matrix.scales, place, size, 1))
            gpu.quantize_fp4(gpu.upload(Shape.vector(count), rng.standard_normal(count)), part, Storage.Transposed)
            w[c, at:at + count] = ref.dequantize(gpu.download_bytes(part.codes), gpu.download_bytes(part.scales), count)
    x = gpu.zeros(Shape(rows, inner))
    values = rng.standard_normal((rows, 95)).astype(np.float32)
    for r in range(rows):
        gpu.copy_from_host(View(x, r * inner, 32), values[r, :32])
        gpu.copy_from_host(View(x, (r + 1) * inner - 63, 63), values[r, 32:])
    spec = MatmulSpec.new(rows, cols, inner).right_transposed()
    out = gpu.upload(Shape(rows, cols), np.full(rows * cols, 9, np.float32))
    gpu.matmul_fp4(spec.with_precision(Precision.Bf16 if bf16 else Precision.F32), x, matrix, out)
    check_product(gpu.download(out).reshape(rows, cols), to_bf16(values) if bf16 else values, w, 95)
