"""GPU parity of the 4-bit format: weights to blocks and back (``sn_quantize_fp4``,
``sn_dequantize_fp4``), cache rows appended and read (``sn_fp4_cache_append``, ``sn_fp4_cache_read``).
All bit for bit against the numpy form of the definition (fp4_reference)."""
import numpy as np
import pytest

import fp4_reference as ref
from fp4_reference import View
from staleynet_amd.gemm import Fp4Cache, Fp4Matrix, GpuError, Shape, Storage

pytestmark = pytest.mark.gpu


def awkward(count):
    """Rows of 32 values: ties and their neighbours, largest magnitudes around 7 factors, zeros of
    both signs, subnormals, the largest floats, infinities and NaN."""
    rng = np.random.default_rng(7)
    rows = []
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    near = np.concatenate([ties, np.nextafter(ties, np.float32(0)), np.nextafter(ties, np.float32(9))])
    for e in (0, -3, 40, -100, 124, -126):
        row = np.zeros(32, np.float32)
        row[:21] = near * np.float32(2.0) ** e
        row[21:31] = -row[:10]
        row[31] = np.float32(6.0) * np.float32(2.0) ** min(e, 124)
        rows.append(row)
    for top in (3.9999998, 4, 6.9999995, 7, 7.0000005, 7.9999995, 8):
        row = (rng.standard_normal(32) * 0.5).astype(np.float32)
        row[5] = -top
        rows.append(row)
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, -0.0, np.float32))
    tiny = np.zeros(32, np.float32)
    tiny[:6] = [1e-45, -1e-40, 1e-38, 5e-39, -3e-39, 2.9e-39]
    rows.append(tiny)
    rows.append((tiny * np.float32(0.1)).astype(np.float32))
    huge = (rng.standard_normal(32) * 1e38).astype(np.float32)
    huge[3], huge[9] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    rows.append(huge)
    for bad in (np.inf, -np.inf, np.nan):
        row = rng.standard_normal(32).astype(np.float32)
        row[17] = bad
        rows.append(row)
    while len(rows) < count:
        rows.append((rng.standard_normal(32) * np.float32(2.0) ** rng.integers(-120, 120)).astype(np.float32))
    return np.stack(rows)


def check_weights(gpu, w, storage, offset=0):
    """w [cols][inner]; the fp32 side `offset` floats into its buffer (unaligned)."""
    cols, inner = w.shape
    side = w if storage == Storage.Transposed else w.T
    buffer = gpu.upload(Shape.vector(w.size + offset), np.concatenate([np.zeros(offset, np.float32), side.ravel()]))
    matrix = gpu.fp4_matrix(cols, inner)
    gpu.quantize_fp4(View(buffer, offset, w.size), matrix, storage)
    codes, scales = ref.quantize(w)
    got_codes, got_scales = gpu.download_bytes(matrix.codes), gpu.download_bytes(matrix.scales)
    assert np.array_equal(got_scales, scales.ravel())
    assert np.array_equal(got_codes, codes.ravel())
    back = gpu.upload(Shape.vector(w.size + 2 + offset), np.full(w.size + 2 + offset, 77, np.float32))
    gpu.dequantize_fp4(matrix, View(back, offset, w.size), storage)
    values = ref.dequantize(codes, scales, inner)
    want = values if storage == Storage.Transposed else values.T
    got = gpu.download(back)
    assert np.array_equal(got[offset:-2], want.ravel().astype(np.float32), equal_nan=True)
    assert (got[:offset] == 77).all() and (got[-2:] == 77).all()


@pytest.mark.parametrize("storage", list(Storage))
def test_awkward_blocks(gpu, storage):
    check_weights(gpu, awkward(300), storage)


@pytest.mark.parametrize("storage", list(Storage))
@pytest.mark.parametrize("cols,inner", [(1, 1), (1, 32), (3, 31), (17, 33), (300, 65), (5, 1001), (64, 768)])
def test_odd_sizes(gpu, cols, inner, storage):
    w = np.random.default_rng(cols * 1000 + inner).standard_normal((cols, inner)).astype(np.float32)
    check_weights(gpu, w, storage)
    check_weights(gpu, w, storage, offset=1)


def test_nothing_to_do_and_refusals_on_the_device(gpu):
    gpu.quantize_fp4(gpu.zeros(Shape.vector(0)), gpu.fp4_matrix(0, 5))
    gpu.dequantize_fp4(gpu.fp4_matrix(5, 0), gpu.zeros(Shape.vector(0)))
    source = gpu.zeros(Shape.vector(64))
    matrix = gpu.fp4_matrix(3, 32)
    shifted = Fp4Matrix(2, 32, View(matrix.codes, 8, 40, 1), matrix.scales)
    with pytest.raises(AssertionError, match="unsupported"):
        gpu.quantize_fp4(source, shifted)
    inside = Fp4Matrix(2, 32, View(source, 0, 64, 1), matrix.scales)
    with pytest.raises(AssertionError, match="overlaps"):
        gpu.quantize_fp4(source, inside)


def dense(cache, gpu):
    """The cache's codes and scales, [batch, kv_heads, capacity, ..], keys then values."""
    shape = (cache.batch, cache.kv_heads, cache.capacity, -1)
    return [gpu.download_bytes(b).reshape(shape) for b in (cache.k_codes, cache.k_scales, cache.v_codes,
                                                           cache.v_scales)]


def filled(gpu, batch, kv_heads, capacity, head_dim, seed):
    rng = np.random.default_rng(seed)
    sizes = [batch * kv_heads * capacity * n for n in (head_dim // 2, head_dim // 32)] * 2
    return Fp4Cache(batch, kv_heads, capacity, head_dim,
                    *(gpu.upload_bytes(rng.integers(0, 256, n, dtype=np.uint8)) for n in sizes))


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("batch,kv_heads,time,capacity,extra,offset", [
    (1, 1, 1, 1, 0, 0), (1, 12, 1, 40, 0, 0), (3, 2, 5, 11, 4, 0), (2, 3, 7, 9, 3, 0), (4, 5, 3, 64, 0, 1)])
def test_append_and_read(gpu, head_dim, batch, kv_heads, time, capacity, extra, offset):
    """Every position of a ragged batch, the last sequences' rows past the capacity: those are not
    written and read back as zeros; everything else in the cache keeps its bytes."""
    rng = np.random.default_rng(head_dim + batch)
    columns = kv_heads * head_dim
    width, key, value = 3 * columns + extra, columns + extra, 2 * columns + extra
    packed = rng.standard_normal((batch * time, width)).astype(np.float32)
    buffer = gpu.upload(Shape.vector(packed.size + offset), np.concatenate([np.zeros(offset), packed.ravel()]))
    where = [int(rng.integers(0, capacity)) for _ in range(batch)]
    if batch > 2:
        where[-1] = 0xFFFFFFFF  # a free place's position: nothing of it is written
    cache = filled(gpu, batch, kv_heads, capacity, head_dim, seed=batch)
    want = dense(cache, gpu)
    positions = gpu.upload_tokens(where)
    gpu.fp4_cache_append(cache, View(buffer, offset, packed.size), time, width, key, value, positions=positions)
    read = np.zeros((2, batch, kv_heads, time, head_dim), np.float32)
    for part, first in enumerate((key, value)):
        for b in range(batch):
            for t in range(time):
                if where[b] + t >= capacity:
                    continue
                heads = packed[b * time + t, first:first + columns].reshape(kv_heads, head_dim)
                codes, scales = ref.quantize(heads)
                want[2 * part][b, :, where[b] + t] = codes
                want[2 * part + 1][b, :, where[b] + t] = scales
                read[part, b, :, t] = ref.dequantize(codes, scales)
    for got, expected in zip(dense(cache, gpu), want):
        assert np.array_equal(got, expected)
    keys, values = (gpu.upload(Shape.vector(read[0].size + 1 + offset), np.full(read[0].size + 1 + offset, 5.0))
                    for _ in range(2))
    gpu.fp4_cache_read(cache, time, View(keys, offset, read[0].size), View(values, offset, read[0].size),
                       positions=positions)
    for got, expected in ((keys, read[0]), (values, read[1])):
        got = gpu.download(got)
        assert np.array_equal(got[offset:-1], expected.ravel()) and got[-1] == 5 and (got[:offset] == 5).all()


def test_append_at_one_position_and_its_refusals(gpu):
    batch, heads, time, capacity, head_dim = 2, 2, 3, 8, 32
    packed = np.random.default_rng(3).standard_normal((batch * time, 192)).astype(np.float32)
    cache = gpu.fp4_cache(batch, heads, capacity, head_dim)
    p = gpu.upload(Shape(batch * time, 192), packed)
    gpu.fp4_cache_append(cache, p, time, 192, 64, 128, position=5)
    codes, scales = ref.quantize(packed[:, 128:].reshape(-1, head_dim))
    got = dense(cache, gpu)
    assert np.array_equal(got[2][:, :, 5:].transpose(0, 2, 1, 3).reshape(-1, 16), codes)
    assert np.array_equal(got[3][:, :, 5:].transpose(0, 2, 1, 3).reshape(-1, 1), scales)
    assert not got[2][:, :, :5].any()
    with pytest.raises(AssertionError, match="do not fit"):
        gpu.fp4_cache_append(cache, p, time, 192, 64, 128, position=6)
    same = Fp4Cache(batch, heads, capacity, head_dim, cache.k_codes, cache.k_scales, cache.k_codes, cache.v_scales)
    with pytest.raises(GpuError, match="overlaps"):
        gpu.fp4_cache_append(same, p, time, 192, 64, 128)
    gpu.fp4_cache_append(cache, p, 0, 192, 64, 128, position=8)  # no rows: nothing
    empty = gpu.fp4_cache(0, heads, capacity, head_dim)
    gpu.fp4_cache_append(empty, p, time, 192, 64, 128)
