"""GPU parity of the 8-bit operators, the norm and the log probabilities at the largest sizes that their headers allow and a
GPU holds. Most of a buffer is zeros, so that sums have few terms: adding a zero is exact, and tolerances count the others."""
import numpy as np
import pytest

import fp8_reference as ref
import test_norm_gpu as norm
from fp4_reference import View
from staleynet_amd.gemm import Fp8Matrix, LogprobHeads, MatmulSpec, Shape, Storage
from test_fp8_gpu import check, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(3, 40), (20, 5), (300, 33), (33, 300)])
def test_the_longest_inner_dimension(gpu, rows, cols):
    """2^23 - 1: the last four blocks of each row and column, the last of them one value short, among zeros."""
    inner, padded = (1 << 23) - 1, 1 << 23
    rng = np.random.default_rng(rows)
    left, right = gpu.fp8_matrix(rows, inner), gpu.fp8_matrix(cols, inner)

    def fill(matrix, row):
        values = rng.standard_normal((1, 511)).astype(np.float32)
        part = Fp8Matrix(1, 511, View(matrix.codes, (row + 1) * padded - 512, 512, 1),
                         View(matrix.scales, (row + 1) * (padded // 128) - 4, 4, 1))
        gpu.quantize_fp8(upload(gpu, values), part)
        return ref.dequantize(*ref.quantize(values))[0]

    x, w = (np.stack([fill(m, r) for r in range(m.rows)]) for m in (left, right))
    out = gpu.upload(Shape.vector(rows * cols + 9), np.full(rows * cols + 9, 5))
    gpu.matmul_fp8(MatmulSpec.new(rows, cols, inner).right_transposed(), left, right, View(out, 0, rows * cols))
    got = gpu.download(out)
    assert (got[rows * cols:] == 5).all()
    check(got[:rows * cols].reshape(rows, cols), x, w, 512)


@pytest.mark.parametrize("storage", list(Storage))
def test_the_longest_row_to_quantize(gpu, storage):
    """2^31 - 1 values: the last of them, and back."""
    inner = (1 << 31) - 1
    source, matrix = gpu.zeros(Shape(1, inner)), gpu.fp8_matrix(1, inner)
    values = np.random.default_rng(3).standard_normal(383).astype(np.float32)
    gpu.copy_from_host(View(source, inner - 383, 383), values)
    gpu.quantize_fp8(source, matrix, storage)
    codes, scales = ref.quantize(values[None])
    blocks = ref.blocks_of(inner)
    assert np.array_equal(gpu.download_bytes(View(matrix.codes, 128 * blocks - 384, 384, 1)), codes[0])
    assert np.array_equal(gpu.download_bytes(View(matrix.scales, blocks - 4, 4, 1)), [3, *scales[0, :3]])
    gpu.fill_zero(source)
    gpu.dequantize_fp8(matrix, source, storage)
    assert np.array_equal(gpu.download(View(source, inner - 400, 400)),
                          np.pad(ref.dequantize(codes, scales, 383)[0], (17, 0)).astype(np.float32))


def test_the_widest_norm(gpu):
    rows, width = 2, (1 << 25) - 1
    x, residual, weight = norm.inputs(rows, width, 4)
    total, y, inverse = (norm.place(gpu, np.zeros(n)) for n in (x.size, x.size, rows))
    xt, rt, wt = norm.place(gpu, x), norm.place(gpu, residual), norm.place(gpu, weight)
    gpu.rms_norm(xt, wt, y, norm.EPSILON, rows, rt, total, inverse)
    s = x + residual
    assert np.array_equal(norm.fetch(gpu, total, s.shape), s)
    got, factors = norm.fetch(gpu, y, s.shape), norm.fetch(gpu, inverse, rows)
    want, want_inverse = norm.expected(s, weight)
    # As norm.check_forward, but a lane's 64-bit sum has up to 2^16 + 16 terms: 2^-36 of it.
    assert (np.abs(got - want) <= (norm.U + 2.0 ** -36) * np.abs(want) + 2.0 ** -150).all()
    assert (np.abs(factors - want_inverse) <= (norm.U + 2.0 ** -36) * want_inverse).all()
    matrix = gpu.fp8_matrix(rows, width)
    gpu.rms_norm(xt, wt, matrix, norm.EPSILON, rows, rt, xt)
    assert np.array_equal(norm.fetch(gpu, xt, s.shape), s)
    rounded = gpu.fp8_matrix(rows, width)
    gpu.quantize_fp8(y, rounded)
    for name in ("codes", "scales"):
        assert np.array_equal(*(gpu.download_bytes(getattr(m, name)) for m in (matrix, rounded)))
    # d_out is one value a row, so that the row's dot product has one term.
    d_out = np.zeros(s.shape, np.float32)
    d_out[0, width - 1], d_out[1, 7] = 2.0, -3.0
    before = np.ones(width, np.float32)
    got, got_w = norm.gradients(gpu, s, factors, weight, d_out, None, before)
    i = factors.astype(np.float64)[:, None]
    n, g = s * i, weight.astype(np.float64) * d_out
    mean = (g * n).sum(1, keepdims=True) / width
    # n, g and their product, 1 / width and the mean; then n mean, the difference, its product with i, and the sum's zero.
    off = np.abs(i) * (9 * norm.U * (np.abs(g) + np.abs(n * mean)))
    assert (np.abs(got - i * (g - n * mean)) <= off + 2.0 ** -149).all()
    want = before + (d_out * n).sum(0)
    assert (np.abs(got_w - want) <= 4 * norm.U * (1 + np.abs(want))).all()


@pytest.mark.parametrize("top", [0, 5, 32])
def test_a_row_of_many_classes(gpu, top):
    """2^28 + 77 classes, equal but for some in the lead: the last ones, others in far parts, and two equal ones."""
    classes = (1 << 28) + 77
    logits = gpu.zeros(Shape(1, classes))
    lead = {classes - 1: 9.0, 0: 7.5, 1 << 27: 8.0, (1 << 28) - 1: 8.0, 123456789: 11.0, classes - 2: 6.0}
    for c, v in lead.items():
        gpu.copy_from_host(View(logits, c, 1), [v])
    out = [gpu.zeros(Shape.vector(n)) for n in (1, 1, 2, 32)]
    ids = gpu.upload_tokens(np.zeros(32, np.uint32))
    token = gpu.upload_tokens([classes - 1])
    gpu.token_logprobs(logits, LogprobHeads(classes), token, *out[:3], top, ids, out[3])
    order = sorted(lead, key=lambda c: (-lead[c], c)) + [c for c in range(1, 40)]
    assert list(gpu.download_tokens(ids)[:top]) == order[:top]
    logprob, entropy, stats, best = (gpu.download(t) for t in out)
    z = np.array([v - 11.0 for v in lead.values()])
    e, rest = np.exp(z), (classes - len(lead)) * np.exp(-11.0)
    total = np.log(e.sum() + rest)
    h = total + ((e * -z).sum() + rest * 11) / (e.sum() + rest)
    # A term's e^z: 2^-22 (1 + 11). A wave adds 32 values a lane and 64 lanes, a chunk after the other, 2^28 / 2048 chunks in
    # at most 2048 parts (fewer with a list: 64), the merge 32 parts a lane and 64 lanes; three roundings a step.
    steps = 32 + 6 + 3 * (2 ** 17 / (2048 if top == 0 else min(2048, 2048 // top)) + 1 + 32 + 6)
    off = 12 * 2.0 ** -22 + steps * 2.0 ** -24
    assert stats[0] == 11 and abs(stats[1] - total) <= off + 2.0 ** -22 * total
    assert abs(logprob[0] - (-2 - total)) <= off + 2.0 ** -21 * total
    assert abs(entropy[0] - h) <= 3 * off * h + 2.0 ** -22 * h
    assert (np.abs(best[:top] - ([lead.get(c, 0.0) - 11 for c in order[:top]] - total)) <= off + 2.0 ** -21 * (total + 11)).all()
    # The gradient, over the logits: d_logprob 1 and d_entropy 0.5.
    stats64, h32 = stats.astype(np.float64), float(entropy[0])
    gpu.token_logprobs_backward(logits, LogprobHeads(classes), out[2], logits, token, gpu.upload(Shape.vector(1), [1.0]), out[1],
                                gpu.upload(Shape.vector(1), [0.5]))
    for c in order[:8]:
        log_p = lead.get(c, 0.0) - stats64[0] - stats64[1]
        p = np.exp(log_p)
        want = (c == classes - 1) - p * (1 + 0.5 * (log_p + h32))
        # log p: two roundings of up to 2^5; p: 2^-22 (1 + |log p|) and that; the products' six.
        assert abs(gpu.download(View(logits, c, 1))[0] - want) <= 2.0 ** -24 * abs(want) + \
            p * (1 + 0.5 * abs(log_p + h32)) * (2.0 ** -18 + 2.0 ** -22 * 20 + 6 * 2.0 ** -24) + p * 2.0 ** -18
