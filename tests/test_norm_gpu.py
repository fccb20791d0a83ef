"""GPU parity of the residual addition with the norm (``sn_rms_norm``, ``sn_rms_norm_fp8``) and of its gradients
(``sn_rms_norm_backward``) with 64 bits.

Tolerances. The sum is one fp32 addition: the same bits. y and the inverse are formed in 64 bits and rounded once: 2^-24
of the value, and 2^-40 of it for the 64-bit roundings. The 8-bit rows are the quantized fp32 ones, bit for bit.
Gradients are fp32: n = s i, g = w dy and their product are off by 3 x 2^-24 of it, a sum of `width` such terms by
(width / 64 + 64) 2^-24 of the sum of magnitudes more (a lane's chain, then a tree over lanes and waves); d_x has
that times |n i|, its own five roundings of 2^-24 of |i g| and |i n mean|, and one of the result. d_weight is a sum of
`rows` terms in any order: (rows + 4) 2^-24 of the sum of magnitudes, and a rounding of what it is added to."""
import numpy as np
import pytest

import fp8_reference as ref
from bench import HipGraph
from fp4_reference import View
from staleynet_amd.gemm import CRmsNormShape, Fp8Matrix, Gpu, GpuError, Shape

pytestmark = pytest.mark.gpu

EPSILON = float(np.float32(1e-5))
U = 2.0 ** -24


def place(gpu, values, offset=0, guard=5):
    """Values in a device buffer from its element `offset` on, `guard` more behind them."""
    flat = np.ascontiguousarray(values, np.float32).ravel()
    buffer = gpu.upload(Shape.vector(offset + flat.size + guard), np.pad(flat, (offset, guard), constant_values=77))
    return View(buffer, offset, flat.size)


def fetch(gpu, view, shape):
    """A placed tensor's values; its surroundings have to be as they were."""
    all_ = gpu.download(view.owner)
    first = (view.pointer - view.owner.pointer) // 4
    assert (all_[:first] == 77).all() and (all_[first + len(view):] == 77).all()
    return all_[first:first + len(view)].reshape(shape)


def inputs(rows, width, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, width)).astype(np.float32)
    residual = (3 * rng.standard_normal((rows, width))).astype(np.float32)
    return x, residual, (1 + 0.1 * rng.standard_normal(width)).astype(np.float32)


def expected(s, weight, epsilon=EPSILON):
    s, weight = s.astype(np.float64), weight.astype(np.float64)
    inverse = 1 / np.sqrt((s * s).mean(1) + epsilon)
    return s * inverse[:, None] * weight, inverse


def check_forward(y, inverse, s, weight, epsilon=EPSILON):
    want, want_inverse = expected(s, weight, epsilon)
    assert (np.abs(y - want) <= (U + 2.0 ** -40) * np.abs(want) + 2.0 ** -150).all()
    assert (np.abs(inverse - want_inverse) <= (U + 2.0 ** -40) * want_inverse).all()


WIDTHS = [1, 7, 32, 127, 128, 129, 500, 512, 513, 768, 1000, 1025, 2048, 2049, 4100, 5121, 8192, 9001, 16384, 20000, 33000]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 70])
@pytest.mark.parametrize("with_residual", [True, False])
def test_forward(gpu, rows, width, with_residual):
    x, residual, weight = inputs(rows, width, width + rows)
    offset = rows % 4
    xt, rt, wt = place(gpu, x, offset), place(gpu, residual, offset) if with_residual else None, place(gpu, weight, offset)
    total, y, inverse = (place(gpu, np.zeros(n), offset) for n in (x.size, x.size, rows))
    gpu.rms_norm(xt, wt, y, EPSILON, rows, rt, total, inverse)
    s = x + residual if with_residual else x
    assert np.array_equal(fetch(gpu, total, s.shape), s)
    got = fetch(gpu, y, s.shape)
    check_forward(got, fetch(gpu, inverse, rows), s, weight)
    # Without the optional outputs, and in 8 bits.
    again = place(gpu, np.zeros(x.size))
    gpu.rms_norm(xt, wt, again, EPSILON, rows, rt)
    assert np.array_equal(fetch(gpu, again, s.shape), got)
    codes, scales = rows * ref.blocks_of(width) * 128, rows * ref.scale_stride(width)
    held = [gpu.upload_bytes(np.full(n + 64, 99, np.uint8)) for n in (codes, scales)]
    matrix = Fp8Matrix(rows, width, View(held[0], 0, codes, 1), View(held[1], 0, scales, 1))
    total = place(gpu, np.zeros(x.size), offset)
    gpu.rms_norm(xt, wt, matrix, EPSILON, rows, rt, total)
    assert np.array_equal(fetch(gpu, total, s.shape), s)
    got_codes, got_scales = (gpu.download_bytes(b) for b in held)
    assert (got_codes[codes:] == 99).all() and (got_scales[scales:] == 99).all()
    want_codes, want_scales = ref.quantize(got)
    assert np.array_equal(got_scales[:scales].reshape(rows, -1), want_scales)
    assert np.array_equal(got_codes[:codes].reshape(rows, -1), want_codes)


@pytest.mark.parametrize("width", [100, 768, 5000, 40000])
@pytest.mark.parametrize("onto", ["x", "residual", "both"])
def test_the_stream_updated_in_place(gpu, width, onto):
    x, residual, weight = inputs(6, width, width)
    if onto == "both":
        residual = x
    xt, wt = place(gpu, x), place(gpu, weight)
    rt = xt if onto == "both" else place(gpu, residual)
    total = rt if onto == "residual" else xt
    y, inverse = place(gpu, np.zeros(x.size)), place(gpu, np.zeros(6))
    gpu.rms_norm(xt, wt, y, EPSILON, 6, rt, total, inverse)
    s = x + residual
    assert np.array_equal(fetch(gpu, total, s.shape), s)
    check_forward(fetch(gpu, y, s.shape), fetch(gpu, inverse, 6), s, weight)
    matrix = gpu.fp8_matrix(6, width)
    xt = place(gpu, x)
    rt = xt if onto == "both" else place(gpu, residual)
    total = rt if onto == "residual" else xt
    gpu.rms_norm(xt, wt, matrix, EPSILON, 6, rt, total)
    assert np.array_equal(fetch(gpu, total, s.shape), s)
    assert np.array_equal(gpu.download_bytes(matrix.codes).reshape(6, -1), ref.quantize(fetch(gpu, y, s.shape))[0])


@pytest.mark.parametrize("rows,width", [(1, 64), (1, 512), (3, 200), (1027, 512), (1025, 1000), (4099, 768)])
def test_rows_updated_in_place_are_read_once(gpu, rows, width):
    """Fewer rows than the workgroups' waves are for: none is read again after its sum was written over it."""
    x, residual, weight = inputs(rows, width, rows)
    rt, wt, y = place(gpu, residual), place(gpu, weight), place(gpu, np.zeros(x.size))
    s, xt = x, place(gpu, x)
    for _ in range(24):
        gpu.rms_norm(xt, wt, y, EPSILON, rows, rt, xt)
        s = s + residual
    assert np.array_equal(fetch(gpu, xt, s.shape), s)
    want, _ = expected(s, weight)
    assert (np.abs(fetch(gpu, y, s.shape) - want) <= (U + 2.0 ** -40) * np.abs(want) + 2.0 ** -150).all()


@pytest.mark.parametrize("width", [130, 3000, 50000])
def test_values_at_the_edges(gpu, width):
    """Rows of zeros, of subnormals, of the largest floats; NaN and infinities stay in their row."""
    x, _, weight = inputs(8, width, 3)
    x[0] = 0
    x[1] *= 1e-40
    x[2] = np.finfo(np.float32).max * np.sign(x[2])
    x[3] *= 1e-20
    x[4, width // 2] = np.nan
    x[5, width - 1] = np.inf
    wt, y, inverse = place(gpu, weight), place(gpu, np.zeros(x.size)), place(gpu, np.zeros(8))
    gpu.rms_norm(place(gpu, x), wt, y, EPSILON, 8, inverse=inverse)
    got, factors = fetch(gpu, y, x.shape), fetch(gpu, inverse, 8)
    good = [0, 1, 2, 3, 6, 7]
    check_forward(got[good], factors[good], x[good], weight)
    assert np.isnan(got[4]).all()
    assert np.isnan(got[5, -1]) and not got[5, :-1].any()  # inf * 0, and finite values times 0
    matrix = gpu.fp8_matrix(8, width)
    gpu.rms_norm(place(gpu, x), wt, matrix, EPSILON, 8)
    codes, scales = ref.quantize(got)
    assert np.array_equal(gpu.download_bytes(matrix.codes).reshape(8, -1), codes)
    assert np.array_equal(gpu.download_bytes(matrix.scales).reshape(8, -1), scales)
    # Without epsilon a row of zeros has no direction, others have a mean square of one.
    gpu.rms_norm(place(gpu, x), wt, y, 0.0, 8, inverse=inverse)
    got, factors = fetch(gpu, y, x.shape), fetch(gpu, inverse, 8)
    assert np.isnan(got[0]).all() and factors[0] == np.inf
    check_forward(got[[2, 3, 6]], factors[[2, 3, 6]], x[[2, 3, 6]], weight, 0.0)


def backward(s, inverse, weight, d_out, d_sum):
    """The gradients in 64 bits, and how far fp32 ones may be off."""
    s, i, w, dy = (a.astype(np.float64) for a in (s, inverse[:, None], weight, d_out))
    before = 0.0 if d_sum is None else d_sum.astype(np.float64)
    width = s.shape[1]
    n, g = s * i, w * dy
    mean = (g * n).mean(1, keepdims=True)
    d_x = before + i * (g - n * mean)
    off = (width / 64 + 67) * U * np.abs(g * n).mean(1, keepdims=True)
    d_x_off = np.abs(i) * (np.abs(n) * off + 5 * U * (np.abs(g) + np.abs(n * mean))) + U * np.abs(d_x)
    d_w = (dy * n).sum(0)
    d_w_off = (len(s) + 4) * U * np.abs(dy * n).sum(0)
    return d_x, d_x_off, d_w, d_w_off


def gradients(gpu, s, inverse, weight, d_out, d_sum, d_weight, offset=0, onto=False):
    st, it, wt, dt = (place(gpu, a, offset) for a in (s, inverse, weight, d_out))
    ds = None if d_sum is None else place(gpu, d_sum, offset)
    d_x = ds if onto else place(gpu, np.zeros(s.size), offset)
    dw = None if d_weight is None else place(gpu, d_weight, offset)
    gpu.rms_norm_backward(st, it, wt, dt, d_x, len(s), ds, dw)
    return fetch(gpu, d_x, s.shape), None if dw is None else fetch(gpu, dw, weight.shape)


def grad_inputs(rows, width, seed):
    x, residual, weight = inputs(rows, width, seed)
    s = x + residual
    rng = np.random.default_rng(seed + 1)
    d_out, d_sum = (rng.standard_normal((rows, width)).astype(np.float32) for _ in range(2))
    return s, expected(s, weight)[1].astype(np.float32), weight, d_out, d_sum


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_backward(gpu, rows, width):
    s, inverse, weight, d_out, d_sum = grad_inputs(rows, width, width + rows)
    before = np.random.default_rng(1).standard_normal(width).astype(np.float32)
    for with_sum, with_weight in ((True, True), (False, True), (True, False)):
        got, got_w = gradients(gpu, s, inverse, weight, d_out, d_sum if with_sum else None,
                               before if with_weight else None, rows % 4)
        d_x, d_x_off, d_w, d_w_off = backward(s, inverse, weight, d_out, d_sum if with_sum else None)
        assert (np.abs(got - d_x) <= d_x_off).all()
        if with_weight:
            assert (np.abs(got_w - (before + d_w)) <= d_w_off + 2 * U * np.abs(before + d_w)).all()
    in_place, _ = gradients(gpu, s, inverse, weight, d_out, d_sum, None, onto=True)
    assert np.array_equal(in_place, got)


@pytest.mark.parametrize("rows,width", [(3000, 64), (5000, 768), (1500, 4096), (2500, 130), (700, 9000)])
def test_backward_of_many_rows(gpu, rows, width):
    s, inverse, weight, d_out, d_sum = grad_inputs(rows, width, width)
    before = np.zeros(width, np.float32)
    got, got_w = gradients(gpu, s, inverse, weight, d_out, d_sum, before)
    d_x, d_x_off, d_w, d_w_off = backward(s, inverse, weight, d_out, d_sum)
    assert (np.abs(got - d_x) <= d_x_off).all()
    assert (np.abs(got_w - d_w) <= d_w_off).all()
    again = gradients(gpu, s, inverse, weight, d_out, d_sum, before)
    assert np.array_equal(again[0], got) and np.array_equal(again[1], got_w)
    for bytes_ in (0, 4 * width + 64, 1 << 18):
        other = Gpu(0, workspace_bytes=bytes_)
        try:
            small, small_w = gradients(other, s, inverse, weight, d_out, d_sum, before)
        finally:
            other.close()
        assert np.array_equal(small, got)
        assert (np.abs(small_w - d_w) <= d_w_off).all()


def test_gradients_against_differences(gpu):
    """Central differences in 64 bits of a loss sum(y * d_out) + sum(s * d_sum), over x and the weight."""
    rows, width, h = 3, 40, 1e-6
    x, residual, weight = inputs(rows, width, 5)
    s, inverse, _, d_out, d_sum = grad_inputs(rows, width, 5)

    def loss(s, weight):
        return (expected(s, weight)[0] * d_out).sum() + (s * d_sum.astype(np.float64)).sum()

    base = s.astype(np.float64)
    d_x, d_w = np.zeros(s.shape), np.zeros(width)
    for at in np.ndindex(s.shape):
        step = np.zeros(s.shape)
        step[at] = h
        d_x[at] = (loss(base + step, weight) - loss(base - step, weight)) / (2 * h)
    for k in range(width):
        step = np.zeros(width)
        step[k] = h
        d_w[k] = (loss(base, weight + step) - loss(base, weight - step)) / (2 * h)
    got, got_w = gradients(gpu, s, inverse, weight, d_out, d_sum, np.zeros(width, np.float32))
    # A difference of losses of up to 200 in 64 bits is off by 2^-45 / 2h and h^2 of the third derivative: under 1e-5.
    _, d_x_off, _, d_w_off = backward(s, inverse, weight, d_out, d_sum)
    assert (np.abs(got - d_x) <= d_x_off + 1e-5).all()
    assert (np.abs(got_w - d_w) <= d_w_off + 1e-5).all()


def test_no_rows_and_no_width(gpu):
    buffer = gpu.zeros(Shape(1, 4))
    gpu.rms_norm(buffer, buffer, View(buffer, 0, 0), EPSILON, 0)
    gpu.rms_norm(buffer, View(buffer, 0, 0), buffer, EPSILON, 4)
    gpu.rms_norm_backward(buffer, buffer, buffer, buffer, buffer, 0)
    assert not gpu.download(buffer).any()


def test_overlaps_are_refused(gpu):
    t = [gpu.zeros(Shape(4, 100)) for _ in range(6)]
    w, inverse = gpu.zeros(Shape.vector(100)), gpu.zeros(Shape.vector(4))
    matrix = gpu.fp8_matrix(4, 100)
    shifted = View(gpu.zeros(Shape.vector(401)), 1, 400)
    for kw in (dict(out=t[0]), dict(out=t[1]), dict(out=t[2]), dict(inverse=View(t[3], 0, 4)), dict(inverse=View(t[0], 0, 4)),
               dict(sum=View(shifted.owner, 0, 400), x=shifted), dict(inverse=View(w, 0, 4))):
        args = dict(dict(x=t[0], weight=w, out=t[3], epsilon=0.1, rows=4, residual=t[1], sum=t[2], inverse=inverse), **kw)
        with pytest.raises(GpuError):
            gpu.rms_norm(**args)
    with pytest.raises(GpuError):
        gpu.rms_norm(t[0], w, Fp8Matrix(4, 100, View(t[0], 0, 512, 1), matrix.scales), 0.1, 4)
    with pytest.raises(GpuError):
        gpu.rms_norm(t[0], w, Fp8Matrix(4, 100, View(gpu.zeros_bytes(600), 4, 512, 1), matrix.scales), 0.1, 4)
    with pytest.raises(AssertionError):
        gpu.rms_norm(t[0], w, gpu.fp8_matrix(4, 99), 0.1, 4)
    with pytest.raises(AssertionError):
        gpu.rms_norm(t[0], w, t[1], 0.1, 5)
    for d_x, d_w in ((t[0], None), (t[3], None), (t[4], t[0]), (t[4], w), (t[4], View(t[4], 0, 100)), (t[4], View(t[5], 0, 100))):
        with pytest.raises(GpuError):
            gpu.rms_norm_backward(t[0], inverse, w, t[3], d_x, 4, t[5], d_w)
    assert CRmsNormShape(4, 100, 0.0).rows == 4


def test_captured_norms_replay(gpu):
    """Forward, 8-bit forward and backward in one graph: each replay leaves the eager bits."""
    sets = []
    for rows, width in ((1, 768), (600, 300), (40, 9000)):
        x, residual, weight = inputs(rows, width, 8)
        d_out = inputs(rows, width, 9)[0]
        t = [gpu.upload(Shape(rows, width), a) for a in (x, residual, d_out)] + [gpu.upload(Shape.vector(width), weight)]
        out = [gpu.zeros(Shape(rows, width)) for _ in range(3)] + [gpu.zeros(Shape.vector(n)) for n in (rows, width)]
        sets.append((rows, t, out, gpu.fp8_matrix(rows, width)))

    def step():
        for rows, (x, residual, d_out, weight), (total, y, d_x, inverse, d_w), matrix in sets:
            gpu.rms_norm(x, weight, y, EPSILON, rows, residual, total, inverse)
            gpu.rms_norm(x, weight, matrix, EPSILON, rows, residual, total)
            gpu.rms_norm_backward(total, inverse, weight, d_out, d_x, rows, None, d_w)

    def results():
        return [gpu.download(o) for _, _, out, _ in sets for o in out] + \
            [gpu.download_bytes(b) for *_, m in sets for b in (m.codes, m.scales)]

    step()
    want = results()
    graph = HipGraph(gpu.stream, step)
    try:
        for _ in range(3):
            for _, _, out, _ in sets:
                for o in out:
                    gpu.fill_zero(o)
            graph.launch()
            gpu.synchronize()
            assert all(np.array_equal(a, b) for a, b in zip(results(), want))
            rows, t, out, _ = sets[1]
            gpu.rms_norm_backward(out[0], out[3], t[3], t[2], out[2], rows, None, out[4])
    finally:
        graph.close()


@pytest.mark.parametrize("rows,width", [(1, 300), (9, 500), (3, 768), (4097, 768), (5, 2000), (1025, 1500)])
def test_gradients_in_place_of_groups_that_are_not_full(gpu, rows, width):
    """d_x over d_sum, with d_weight, where the last workgroup has more row groups than rows: the bits of other buffers."""
    s, inverse, weight, d_out, d_sum = grad_inputs(rows, width, rows)
    before = np.ones(width, np.float32)
    want, want_w = gradients(gpu, s, inverse, weight, d_out, d_sum, before)
    d_x, d_x_off, _, _ = backward(s, inverse, weight, d_out, d_sum)
    assert (np.abs(want - d_x) <= d_x_off).all()
    for _ in range(3):
        got, got_w = gradients(gpu, s, inverse, weight, d_out, d_sum, before, onto=True)
        assert np.array_equal(got, want) and np.array_equal(got_w, want_w)


@pytest.mark.parametrize("rows,width", [(1100, 768), (1027, 1000), (1025, 513), (1999, 1024)])
@pytest.mark.parametrize("in_place", [False, True])
def test_many_rows_in_8_bits(gpu, rows, width, in_place):
    """Rows of two vectors a lane, more of them than four a CU: the quantized fp32 output's bits."""
    x, residual, weight = inputs(rows, width, rows)
    wt, y = place(gpu, weight), place(gpu, np.zeros(x.size))
    gpu.rms_norm(place(gpu, x), wt, y, EPSILON, rows, place(gpu, residual))
    codes, scales = rows * ref.blocks_of(width) * 128, rows * ref.scale_stride(width)
    held = [gpu.upload_bytes(np.full(n + 64, 99, np.uint8)) for n in (codes, scales)]
    matrix = Fp8Matrix(rows, width, View(held[0], 0, codes, 1), View(held[1], 0, scales, 1))
    xt = place(gpu, x)
    total = xt if in_place else place(gpu, np.zeros(x.size))
    gpu.rms_norm(xt, wt, matrix, EPSILON, rows, place(gpu, residual), total)
    s = x + residual
    assert np.array_equal(fetch(gpu, total, s.shape), s)
    got = fetch(gpu, y, s.shape)
    want, _ = expected(s, weight)
    assert (np.abs(got - want) <= (U + 2.0 ** -40) * np.abs(want) + 2.0 ** -150).all()
    got_codes, got_scales = (gpu.download_bytes(b) for b in held)
    assert (got_codes[codes:] == 99).all() and (got_scales[scales:] == 99).all()
    want_codes, want_scales = ref.quantize(got)
    assert np.array_equal(got_scales[:scales].reshape(rows, -1), want_scales)
    assert np.array_equal(got_codes[:codes].reshape(rows, -1), want_codes)


def test_captured_8_bit_norms_replay(gpu):
    """The codes and scales of captured norms, overwritten before each replay."""
    sets = []
    for rows, width in ((1, 768), (600, 300), (1100, 768), (40, 9000), (2, 20000)):
        x, _, weight = inputs(rows, width, 15)
        matrix = gpu.fp8_matrix(rows, width)
        other = gpu.upload(Shape(rows, width), 1 - x)
        sets.append((rows, gpu.upload(Shape(rows, width), x), gpu.upload(Shape.vector(width), weight), matrix, other))

    def step():
        for rows, x, weight, matrix, _ in sets:
            gpu.rms_norm(x, weight, matrix, EPSILON, rows)

    def results():
        return [gpu.download_bytes(b) for s in sets for b in (s[3].codes, s[3].scales)]

    step()
    want = results()
    graph = HipGraph(gpu.stream, step)
    try:
        for _ in range(3):
            for rows, _, weight, matrix, other in sets:
                gpu.rms_norm(other, weight, matrix, 1e30, rows)  # other codes, and factors far smaller
            assert not any(np.array_equal(a, b) for a, b in zip(results(), want))
            graph.launch()
            gpu.synchronize()
            assert all(np.array_equal(a, b) for a, b in zip(results(), want))
    finally:
        graph.close()
