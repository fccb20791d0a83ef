"""GPU parity of attention over a 4-bit cache (``sn_fp4_attention``) against 64 bits.

Tolerance, for an output o = sum p v / sum p with V = sum p |v| / sum p. A score, in units of e, is off by
at most d = (3 h / 32 + 64) 2^-23 A, A the largest scale |q| |k| of the visible keys (the sums of a
score as in the products' test; the scale and log2 e are two roundings of q, within it), and by 2^-23
of the scores' range, under 2 A, where the maximum is subtracted. Each probability is then off by e^(2 d) - 1
relative to the sum, under 4 (d + 2^-22 A) for numerator and sum, the exponential's own 2^-22 and a rounding
of each rescaling (one every 32 keys at most) added; the sums of n keys are chains of n / 32 additions,
merged over waves and splits:
    |error| <= (4 (3 h / 32 + 66) 2^-23 A + (3 n / 32 + 128) 2^-22) V + n 2^-126 max |v|.
The last term: the exponential is 0 under 2^-126, fp32's smallest normal number, so each of n numerators may lose
that much, and the sum they are divided by is 1 or more, since the largest score's own term is 1."""
import numpy as np
import pytest

import fp4_reference as ref
from fp4_reference import View
from staleynet_amd.gemm import Fp4Cache, Gpu, GpuError, Shape

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, batch, heads, kv_heads, queries, capacity, head_dim, lengths, seed=0, spread=1.0):
        rng = np.random.default_rng(seed)
        self.__dict__.update(batch=batch, heads=heads, kv_heads=kv_heads, queries=queries, capacity=capacity,
                             head_dim=head_dim, lengths=list(lengths), scale=spread * head_dim ** -0.5)
        rows = (batch, kv_heads, capacity)
        self.codes = [rng.integers(0, 256, rows + (head_dim // 2,), dtype=np.uint8) for _ in range(2)]
        self.scales = [rng.integers(124, 127, rows + (head_dim // 32,), dtype=np.uint8) for _ in range(2)]
        self.q = rng.standard_normal((batch, heads, queries, head_dim)).astype(np.float32)
        # What positions past a sequence's length hold is not defined: NaN blocks among them.
        for b, n in enumerate(self.lengths):
            for s in self.scales:
                s[b, :, min(n, capacity):] = rng.choice([0, 100, 253, 255], s[b, :, min(n, capacity):].shape)

    def cache(self, gpu):
        k, v = self.codes
        ks, vs = self.scales
        return Fp4Cache(self.batch, self.kv_heads, self.capacity, self.head_dim,
                        *(gpu.upload_bytes(a) for a in (k, ks, v, vs)))

    def run(self, gpu, uniform=None, packed=False, cache=None):
        b, n, t, h = self.q.shape
        cache = cache or self.cache(gpu)
        lengths = None if uniform is not None else gpu.upload_tokens(self.lengths)
        guard = 5
        if packed:  # columns 3 .. of rows of width n h + 7; the output's rows are n h + 2 wide
            width, out_width = n * h + 7, n * h + 2
            rows = np.zeros((b * t, width), np.float32)
            rows[:, 3:3 + n * h] = self.q.transpose(0, 2, 1, 3).reshape(b * t, n * h)
            q_all = gpu.upload(Shape.vector(rows.size), rows)
            q = View(q_all, 3, rows.size - 3)
            out = gpu.upload(Shape.vector(b * t * out_width + guard), np.full(b * t * out_width + guard, 9.0))
            strides = (t * width, h, width), (t * out_width, h, out_width)
        else:
            q = gpu.upload(Shape.vector(self.q.size), self.q)
            out = gpu.upload(Shape.vector(self.q.size + guard), np.full(self.q.size + guard, 9.0))
            strides = None, None
        gpu.fp4_attention(cache, q, out, n, t, self.scale, uniform or 0, lengths, *strides)
        got = gpu.download(out)
        if packed:
            assert (got[b * t * out_width:] == 9).all()
            rows = got[:b * t * out_width].reshape(b * t, out_width)
            assert (rows[:, n * h:] == 9).all()
            return rows[:, :n * h].reshape(b, t, n, h).transpose(0, 2, 1, 3)
        assert (got[self.q.size:] == 9).all()
        return got[:self.q.size].reshape(self.q.shape)

    def check(self, got):
        b, n, t, h = self.q.shape
        group = n // self.kv_heads
        for i in range(b):
            length = min(self.lengths[i], self.capacity)
            seen = np.arange(max(length, 0))[None, :] <= (length - t + np.arange(t))[:, None]
            for head in range(n):
                at = (i, head // group, slice(0, length))
                k, v = (ref.dequantize(c[at], s[at]) for c, s in zip(self.codes, self.scales))
                q = self.q[i, head].astype(np.float64)
                largest = np.where(seen, np.abs(q) @ np.abs(np.nan_to_num(k)).T, 0).max(initial=0) * self.scale
                s = np.where(seen, q @ k.T * self.scale, -np.inf)
                top = s.max(1, initial=-np.inf, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                total = np.where(p.sum(1, keepdims=True) > 0, p.sum(1, keepdims=True), 1) + 0 * s.sum(1, keepdims=True, where=seen)
                p = p / total
                visible_v = [np.where(seen[j][:, None], v, 0) for j in range(t)]
                want = np.stack([p[j] @ visible_v[j] for j in range(t)])
                size = np.stack([p[j] @ np.abs(visible_v[j]) for j in range(t)])
                bound = (4 * (3 * h / 32 + 66) * 2.0 ** -23 * largest + (3 * length / 32 + 128) * 2.0 ** -22) * size + \
                    length * 2.0 ** -126 * np.abs(np.nan_to_num(v)).max(initial=0)
                result = got[i, head]
                assert np.array_equal(np.isnan(result), np.isnan(want)), (i, head)
                with np.errstate(invalid="ignore"):
                    wrong = np.abs(result - want) > bound
                assert not wrong.any(), (i, head, np.argwhere(wrong)[:4], result[wrong][:4], want[wrong][:4])


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (8, 2), (3, 1), (20, 1), (34, 2)])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 130, 700])
def test_one_token(gpu, head_dim, heads, kv_heads, length):
    case = Case(2, heads, kv_heads, 1, length + 3, head_dim, [length, max(0, length - 7)], seed=length)
    case.check(case.run(gpu, packed=length % 2 == 0))


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,queries", [(2, 2, 5), (4, 2, 17), (3, 1, 40), (8, 1, 100), (2, 1, 150)])
def test_chunk(gpu, head_dim, heads, kv_heads, queries):
    """A chunk at the start of its sequence, one behind cached positions, a shorter one padded in front."""
    lengths = [queries, queries + 83, queries // 2]
    case = Case(3, heads, kv_heads, queries, queries + 90, head_dim, lengths, seed=queries)
    got = case.run(gpu, packed=queries % 2 == 1)
    case.check(got)
    assert not got[2, :, :queries - queries // 2].any()  # those see nothing


def test_many_rows(gpu):
    """More tiles of 16 rows than the CUs take at once (four waves each)."""
    case = Case(2, 24, 6, 333, 400, 64, [333, 390], seed=4)
    case.check(case.run(gpu))


@pytest.mark.parametrize("queries", [1, 3])
def test_lengths_of_zero_and_past_the_capacity(gpu, queries):
    case = Case(4, 4, 2, queries, 50, 64, [0, 50, 0xFFFFFFFF, 1], seed=1)
    got = case.run(gpu)
    case.check(got)
    assert not got[0].any()


@pytest.mark.parametrize("head_dim,heads,kv_heads,queries,length", [
    (128, 8, 1, 1, 5000), (64, 12, 12, 1, 3001), (32, 2, 2, 1, 9000), (128, 4, 2, 2, 2500), (64, 40, 2, 1, 4097),
    (64, 2, 1, 30, 3000)])
def test_long_caches_and_every_workspace(gpu, head_dim, heads, kv_heads, queries, length):
    """Split over workgroups, split less, not split: the same result within the tolerance; with one
    workspace the same bits again."""
    case = Case(2, heads, kv_heads, queries, length + 100, head_dim, [length, length // 3], seed=length)
    case.check(case.run(gpu))
    assert np.array_equal(case.run(gpu), case.run(gpu))
    for workspace in (0, 100_000):
        other = Gpu(0, workspace_bytes=workspace)
        try:
            case.check(case.run(other))
        finally:
            other.close()


@pytest.mark.parametrize("batch,longest,head_dim", [(150, 3000, 32), (65, 9000, 64), (300, 700, 32)])
def test_many_sequences(gpu, batch, longest, head_dim):
    """More sequences than a wave has lanes, lengths from 0 to long: the shares of every one are found."""
    rng = np.random.default_rng(batch)
    lengths = np.minimum(longest, np.exp(rng.uniform(0, np.log(longest + 1), batch)).astype(int) - 1)
    lengths[[0, 63, 64, batch - 1]] = [longest, 0, longest, longest - 1]
    case = Case(batch, 2, 1, 1, longest, head_dim, lengths, seed=batch)
    case.check(case.run(gpu))


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("queries,length", [(1, 900), (40, 200)])
def test_a_cache_inside_larger_buffers(gpu, head_dim, queries, length):
    """Codes at any multiple of 16 bytes, scales at any byte."""
    case = Case(2, 6, 2, queries, length + 5, head_dim, [length, length // 2], seed=head_dim)
    buffers = []
    for codes, scales in zip(case.codes, case.scales):
        for a, ahead in ((codes, 48), (scales, 3)):
            whole = gpu.upload_bytes(np.concatenate([np.full(ahead, 255, np.uint8), a.ravel()]))
            buffers.append(View(whole, ahead, a.size, 1))
    case.check(case.run(gpu, cache=Fp4Cache(2, 2, length + 5, head_dim, *buffers)))


def test_one_length_for_all(gpu):
    case = Case(3, 6, 3, 4, 77, 64, [60, 60, 60], seed=8)
    got = case.run(gpu, uniform=60)
    case.check(got)
    assert np.array_equal(got, case.run(gpu))
    with pytest.raises(AssertionError, match="do not fit"):
        case.run(gpu, uniform=78)


@pytest.mark.parametrize("spread", [0.0, 30.0, 400.0])
def test_flat_and_peaked_scores(gpu, spread):
    case = Case(2, 4, 2, 3, 300, 64, [300, 211], seed=2, spread=spread)
    case.check(case.run(gpu))


@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_nan_reaches_only_the_queries_that_see_it(gpu, head_dim):
    """NaN blocks of keys and of values among the chunk's own positions, a query with NaN, one with inf."""
    case = Case(2, 6, 3, 40, 120, head_dim, [100, 40], seed=3)
    ks, vs = case.scales
    ks[0, 0, 75, 0] = 255                  # seen from the chunk's 16th query on
    vs[0, 1, 81, -1] = 254                 # in the last block only
    vs[0, 1, 99, 0] = 255                  # by the last query alone
    vs[0, 2, 10, 0] = 253                  # by every query
    case.q[1, 2, 7, 3] = np.nan
    case.q[1, 4, 9, 0] = np.inf
    got = case.run(gpu)
    with np.errstate(invalid="ignore"):
        case.check(got)
    assert np.isnan(got[0, 0, 15:]).all() and not np.isnan(got[0, 0, :15]).any()
    assert np.isnan(got[0, 2, 39, :32]).all() and not np.isnan(got[0, 2, 38, :min(32, head_dim - 32)]).any()


@pytest.mark.parametrize("length", [40, 3000])
def test_scores_that_are_all_minus_infinity(gpu, length):
    """q is infinite where every key is -1: no softmax, NaN; a query that sees no key is zeros all the same."""
    case = Case(2, 2, 1, 4, length, 32, [length, 2], seed=length)
    case.codes[0][..., 0] = case.codes[0][..., 0] & 0xF0 | 0xA  # -1 in the first place
    case.q[:, 0, :, 0] = np.inf
    got = case.run(gpu)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 0, 2:]).all()
    assert not got[1, :, :2].any()
    case.q[:, 0] = 0
    got[:, 0] = case.run(gpu)[:, 0]
    case.check(got)


def test_a_cache_whose_offsets_pass_32_bits(gpu):
    """4.3 GB of codes a buffer. Positions never written hold zeros: their scores and values are 0, so
    a query's result is known from the last 40 positions alone."""
    batch, kv_heads, capacity, head_dim, time = 2, 8, 1 << 22, 128, 40
    rng = np.random.default_rng(12)
    cache = gpu.fp4_cache(batch, kv_heads, capacity, head_dim)
    columns = kv_heads * head_dim
    packed = rng.standard_normal((batch * time, 2 * columns)).astype(np.float32)
    rows = gpu.upload(Shape(batch * time, 2 * columns), packed)
    first = [capacity - time, capacity - time - 1000]
    positions = gpu.upload_tokens(first)
    gpu.fp4_cache_append(cache, rows, time, 2 * columns, 0, columns, positions=positions)
    keys, values = (gpu.zeros(Shape.vector(batch * kv_heads * time * head_dim)) for _ in range(2))
    gpu.fp4_cache_read(cache, time, keys, values, positions=positions)
    held = [ref.dequantize(*ref.quantize(packed[:, i * columns:(i + 1) * columns].reshape(-1, head_dim)))
            .reshape(batch, time, kv_heads, head_dim).transpose(0, 2, 1, 3) for i in range(2)]
    for got, expected in zip((keys, values), held):
        assert np.array_equal(gpu.download(got), expected.astype(np.float32).ravel())
    q = rng.standard_normal((batch, kv_heads, 1, head_dim)).astype(np.float32)
    out = gpu.zeros(Shape.vector(q.size))
    lengths = [n + time for n in first]
    scale = 1.5 * head_dim ** -0.5 * 4
    gpu.fp4_attention(cache, gpu.upload(Shape.vector(q.size), q), out, kv_heads, 1, scale,
                      lengths=gpu.upload_tokens(lengths))
    got = gpu.download(out).reshape(batch, kv_heads, head_dim)
    for b in range(batch):
        for head in range(kv_heads):
            s = held[0][b, head] @ q[b, head, 0].astype(np.float64) * scale
            top = max(s.max(), 0.0)
            p = np.exp(s - top)
            expected = p @ held[1][b, head] / (p.sum() + first[b] * np.exp(-top))
            # Within the module's bound: A under 100, chains of 4e6 / 32 / 8 / 32 keys a wave, V under 6.
            assert np.abs(got[b, head] - expected).max() <= 1e-3 * np.abs(expected).max() + 1e-6


def test_two_contexts_do_not_share_their_splits(gpu):
    """Split caches on two contexts at once: each merges its own records."""
    case = Case(2, 8, 2, 1, 5000, 64, [5000, 3000], seed=9)
    expected = case.run(gpu)
    other = Gpu(0, workspace_bytes=64 << 20)
    try:
        cases = [Case(2, 8, 2, 1, 5000, 64, [5000, 3000], seed=9) for _ in range(2)]
        runs = []
        for context, c in zip((gpu, other), cases):
            cache = c.cache(context)
            q = context.upload(Shape.vector(c.q.size), c.q)
            out = context.zeros(Shape.vector(c.q.size))
            lengths = context.upload_tokens(c.lengths)
            runs.append((context, c, cache, q, out, lengths))
        for _ in range(20):
            for context, c, cache, q, out, lengths in runs:
                context.fp4_attention(cache, q, out, c.heads, 1, c.scale, lengths=lengths)
        for context, c, cache, q, out, lengths in runs:
            assert np.array_equal(context.download(out).reshape(c.q.shape), expected)
        del runs, cache, q, out, lengths
    finally:
        other.close()


def test_an_empty_cache(gpu):
    cache = gpu.fp4_cache(2, 2, 0, 64)
    q = gpu.upload(Shape.vector(256), np.ones(256))
    out = gpu.upload(Shape.vector(256), np.ones(256))
    gpu.fp4_attention(cache, q, out, 2, 1, 1.0, lengths=gpu.upload_tokens([7, 0]))
    assert not gpu.download(out).any()


def test_refusals_on_the_device(gpu):
    case = Case(1, 2, 2, 2, 8, 32, [8])
    cache = case.cache(gpu)
    q = gpu.zeros(Shape.vector(case.q.size))
    out = gpu.zeros(Shape.vector(case.q.size))
    with pytest.raises(GpuError, match="overlaps"):
        gpu.fp4_attention(cache, q, q, 2, 2, 1.0, 8)
    with pytest.raises(GpuError, match="overlaps"):  # both heads' outputs in one place
        gpu.fp4_attention(cache, q, out, 2, 2, 1.0, 8, out_strides=(128, 0, 32))
    with pytest.raises(AssertionError, match="too small"):
        gpu.fp4_attention(cache, q, out, 2, 3, 1.0, 8)
    gpu.fp4_attention(cache, q, out, 2, 0, 1.0, 8)  # no queries: nothing
    gpu.fp4_attention(cache, q, out, 2, 2, 1.0, 0)  # no positions: zeros
    assert not gpu.download(out).any()
