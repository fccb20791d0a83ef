"""Each bit of an fp32 operand of the 4-bit products and attention: results that are off if one of the three bf16 parts
that stand for it is dropped or misplaced, which the tolerances of long sums would hide; and every code at every
scale byte, in each form of the product.

A value's third part is what lies under 2^-16 of its power of two. Products here have one nonzero weight a column, a
power of two: the output is the value itself, to the bit. For attention there are the two tests below, with their
tolerances; that a dropped third part exceeds them is tested on the CPU (the tests without the gpu mark)."""
import numpy as np
import pytest

import fp4_reference as ref
from staleynet_amd.gemm import MatmulSpec, Precision
from test_fp4_attention_gpu import Case
from test_fp4_matmul_gpu import run

# One form of the product each: operands of 16 parts and column tiles a wave, then tiles and slices.
FORMS = [(1, 300, 50), (2, 100, 5201), (1, 70, 12301), (5, 300, 50), (4, 70, 12301), (9, 300, 50), (10, 64, 5201),
         (8, 40, 12301), (16, 300, 50), (11, 64, 5201), (13, 40, 12301), (16, 3, 50), (17, 300, 50), (40, 2100, 100),
         (130, 33, 70), (1990, 64, 4001), (1990, 61, 4001)]
BF16_FORMS = [(1, 300, 50), (2, 64, 12301), (9, 64, 5201), (16, 40, 12301), (20, 64, 50), (31, 40, 12301), (40, 300, 77),
              (40, 2100, 100), (1100, 64, 3900)]


def full_mantissas(rng, shape, exponents=(-40, 40)):
    """The last bit set, and the one that starts the second part, so that the last is the third part's."""
    bits = rng.integers(0, 1 << 23, shape, dtype=np.uint32) | 0x8001
    exponent = rng.integers(*exponents, shape).astype(np.uint32) + np.uint32(127)
    sign = rng.integers(0, 2, shape, dtype=np.uint32)
    return (sign << np.uint32(31) | exponent << np.uint32(23) | bits).view(np.float32)


def one_weight_a_column(inner, cols, rng):
    """1 at row c % inner of column c, -1 in every third column, at scales around 1."""
    blocks = ref.blocks_of(inner)
    codes = np.zeros((cols, blocks * 16), np.uint8)
    at = np.arange(cols) % inner
    code = np.where(np.arange(cols) % 3 == 2, 10, 2)
    codes[np.arange(cols), at // 2] = code << 4 * (at % 2)
    scales = rng.integers(120, 135, (cols, blocks), dtype=np.uint8)
    return codes, scales, at


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,cols", FORMS)
def test_products_keep_every_bit(gpu, rows, inner, cols):
    rng = np.random.default_rng(rows + inner)
    codes, scales, at = one_weight_a_column(inner, cols, rng)
    x = full_mantissas(rng, (rows, inner))
    got = run(gpu, MatmulSpec.new(rows, cols, inner), x, codes, scales, offset=rows % 2)
    weight = ref.dequantize(codes, scales, inner)[np.arange(cols), at]
    assert np.array_equal(got, (x[:, at] * weight).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,cols,bf16", [(*f, False) for f in FORMS] + [(*f, True) for f in BF16_FORMS])
def test_every_code_at_every_scale_byte(gpu, rows, inner, cols, bf16):
    """Index k of a column has code k % 16 and its block the column's number as scale byte (the blocks after the first
    other ones); a row picks one index. Exact, subnormals too; a NaN block is its column's."""
    blocks = ref.blocks_of(inner)
    codes = np.tile(np.arange(8, dtype=np.uint8) * 0x22 + 0x10, (cols, 2 * blocks))
    scales = ((np.arange(cols)[:, None] + 37 * np.arange(blocks)[None, :]) % 256).astype(np.uint8)
    w = ref.dequantize(codes, scales, inner)
    column_nan = (scales > ref.LARGEST_SCALE).any(1)
    spec = MatmulSpec.new(rows, cols, inner).with_precision(Precision.Bf16 if bf16 else Precision.F32)
    for first in range(0, min(inner, 16), min(rows, 16)):
        picked = (first + np.arange(rows) * (1 if rows <= 16 else 7)) % inner
        x = np.zeros((rows, inner), np.float32)
        x[np.arange(rows), picked] = 1
        got = run(gpu, spec, x, codes, scales)
        assert np.isnan(got[:, column_nan]).all()
        assert np.array_equal(got[:, ~column_nan], w[:, picked].T[:, ~column_nan].astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,cols", [(11, 96, 40), (16, 96, 12301), (16, 96, 5201), (1990, 96, 4001)])
def test_infinities_and_nan_in_every_form(gpu, rows, inner, cols):
    """As test_infinities_nan_and_large_values_follow_ieee, in operands of 48 parts and tiles of 128 x 256."""
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 256, (cols, 48), dtype=np.uint8)
    scales = rng.integers(121, 128, (cols, 3), dtype=np.uint8)
    scales[3, 1], scales[cols - 1, 2] = 255, 253
    w = ref.dequantize(codes, scales)
    x = rng.standard_normal((rows, inner)).astype(np.float32)
    x[0, 40], x[rows // 2, 95] = np.inf, -np.inf
    x[1, 5] = np.nan
    x[2, 6] = np.array([0x7F800001], np.uint32).view(np.float32)[0]  # a NaN with low bits only
    x[rows - 1] = 0
    x[rows - 1, 70] = np.finfo(np.float32).max * 0.25
    got = run(gpu, MatmulSpec.new(rows, cols, inner), x, codes, scales).astype(np.float64)
    with np.errstate(invalid="ignore"):
        expected = x.astype(np.float64) @ w.T
        expected = np.where(np.abs(expected) > np.finfo(np.float32).max, np.sign(expected) * np.inf, expected)
        magnitude = np.abs(x.astype(np.float64)) @ np.abs(w).T
    assert np.array_equal(np.isnan(got), np.isnan(expected))
    assert np.array_equal(np.isinf(got), np.isinf(expected)) and (np.isinf(got) <= (np.sign(got) == np.sign(expected))).all()
    finite = np.isfinite(expected)
    assert (np.abs(got[finite] - expected[finite]) <= 73 * 2.0 ** -23 * magnitude[finite]).all()


class QueryBits:
    """Two keys with scores near 4112 (in units of ln 2), of one dim of q each; all others score 0, so their weights are
    2^-4096, nothing. The values are 1 for the one and -1 for the other: the output is p1 - p2 = tanh((s1 - s2) / 2).

    Tolerance: q times the scale's log2 e (which is 1 to a rounding) is off by 3 x 2^-24 of 4113 at most, a score's
    parts sum exactly, or to two roundings of 2^-24; the difference of two scores is then off by 2 x 4113 x 5 x 2^-24 =
    2^-8.6 in units of ln 2, the output by half of that times ln 2: under 2^-9.9. The first part of q is 4096, the second
    what follows down to 2^-3 of such a unit, and the third up to 2^-3 of it, 2^-4.5 of the output."""

    TOLERANCE = 2.0 ** -9.9

    def __init__(self, head_dim, heads, queries, length, seed):
        pairs = head_dim // 2
        rng = np.random.default_rng(seed)
        self.case = case = Case(pairs, heads, 1, queries, length, head_dim, [length] * pairs, seed=seed)
        case.scale = float(np.float32(np.log(2)))
        for codes in case.codes:
            codes[:] = 0
        for scales in case.scales:
            scales[:] = 127
        dims = rng.permutation(head_dim).reshape(2, pairs)
        # Seen by every query, in any step and workgroup.
        self.at = np.stack([rng.permutation(length - queries + 1)[:2] for _ in range(pairs)], 1)
        for j in range(2):
            case.codes[0][np.arange(pairs), 0, self.at[j], dims[j] // 2] = 2 << 4 * (dims[j] % 2)
            case.codes[1][np.arange(pairs), 0, self.at[j]] = 0x22 if j == 0 else 0xAA
        bits = rng.integers(0, 1 << 23, case.q.shape, dtype=np.uint32)
        # 4112 to 4113, every bit under those.
        case.q[:] = ((127 + 12 << 23) + (16 << 11) + (bits & 0x7FF)).astype(np.uint32).view(np.float32)
        self.s = [case.q[np.arange(pairs), :, :, dims[j]].astype(np.float64) for j in range(2)]

    def output(self, scores):
        return np.tanh((scores[0] - scores[1]) * np.log(2) / 2)[..., None]


class WeightBits:
    """One key has values and a score between -1 and 0 in units of ln 2, so a weight with all its bits; the others'
    scores and values are 0, their weights 1: the output is v p / (p + n - 1), p = 2^score.

    Tolerance, relative: the score is off by 3 x 2^-24 and the exponential by 2^-23, so p by under 2^-22; the weights'
    sum by 2^-24 for each of at most 24 additions after p, the division and two products by 2^-23 together. In all
    under 32 x 2^-24 = 2^-19. The third part of p is up to 2^-16 of its power of two."""

    TOLERANCE = 2.0 ** -19

    def __init__(self, head_dim, heads, queries, length, seed):
        batch = 64
        rng = np.random.default_rng(seed)
        self.case = case = Case(batch, heads, 1, queries, length, head_dim, [length] * batch, seed=seed)
        case.scale = float(np.float32(np.log(2)))
        for scales in case.scales:
            scales[:] = 127
        self.length = length
        at = np.arange(batch) % (length - queries + 1)
        held = case.codes[1][np.arange(batch), 0, at]
        for codes in case.codes:
            codes[:] = 0
        case.codes[0][np.arange(batch), 0, at, 0] = 2  # 1 in the first dim
        case.codes[1][np.arange(batch), 0, at] = held
        self.v = ref.dequantize(held, case.scales[1][np.arange(batch), 0, at])[:, None, None, :]
        case.q[:] = 0
        case.q[..., 0] = -rng.uniform(0.01, 0.99, case.q.shape[:-1])
        self.p = np.exp2(case.q[..., 0].astype(np.float64) * np.log2(np.e) * case.scale)

    def output(self, p):
        seen = self.length - self.case.queries + 1 + np.arange(self.case.queries)  # by each query
        return self.v * (p / (self.p + seen - 1))[..., None]


def without_third_part(x):
    bits = x.astype(np.float32).view(np.uint32)
    first = (bits & 0xFFFF0000).astype(np.uint32).view(np.float32)
    second = ((x.astype(np.float32) - first).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    return first.astype(np.float64) + second


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("heads,queries,length", [(4, 1, 2), (4, 1, 60), (2, 1, 700), (2, 1, 5000), (2, 5, 40), (3, 40, 90)])
def test_attention_uses_every_bit_of_q(gpu, head_dim, heads, queries, length):
    t = QueryBits(head_dim, heads, queries, length, length)
    want = np.broadcast_to(t.output(t.s), t.case.q.shape)
    assert np.abs(t.case.run(gpu) - want).max() <= t.TOLERANCE


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("heads,queries,length", [(4, 1, 32), (4, 1, 64), (17, 1, 64), (2, 5, 40), (3, 20, 60)])
def test_attention_uses_every_bit_of_a_weight(gpu, head_dim, heads, queries, length):
    t = WeightBits(head_dim, heads, queries, length, length)
    want = t.output(t.p)
    assert (np.abs(t.case.run(gpu) - want) <= t.TOLERANCE * np.abs(want)).all()


@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_a_dropped_third_part_of_q_is_seen(head_dim):
    t = QueryBits(head_dim, 4, 1, 60, 60)
    off = np.abs(t.output([without_third_part(s) for s in t.s]) - t.output(t.s))
    assert (off > 2 * t.TOLERANCE).mean() > 0.5


@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_a_dropped_third_part_of_a_weight_is_seen(head_dim):
    t = WeightBits(head_dim, 4, 1, 64, 64)
    off, want = np.abs(t.output(without_third_part(t.p)) - t.output(t.p)), np.abs(t.output(t.p))
    assert ((off > 2 * t.TOLERANCE * want) | (want == 0)).mean() > 0.5


def test_a_dropped_part_of_x_is_seen():
    x = full_mantissas(np.random.default_rng(1), (1000,))
    assert (without_third_part(x) != x).all()
