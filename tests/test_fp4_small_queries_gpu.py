"""GPU parity of attention over a 4-bit cache where q is so small that three bf16 parts do not hold it (under 2^-110),
against keys of up to 6 x 2^125, which make ordinary scores of it.

Tolerance: the attention tests' own (test_fp4_attention_gpu), with two additions to a score's error d. q times scale
log2 e is rounded to fp32, whose steps are 2^-149 there: half a step a term, 2^-150 sum |k| in units of 2, which is less
in units of e. And what the three parts leave is a sum of two more parts: h / 32 additions and two roundings."""
import numpy as np
import pytest

import fp4_reference as ref
from staleynet_amd.gemm import Gpu
from test_fp4_attention_gpu import Case

pytestmark = pytest.mark.gpu

BANDS = (-112, -118, -122, -126, -131)


class SmallCase(Case):
    """A sequence for each band, its keys as large as its queries are small; every third query is zeros."""

    def __init__(self, heads, kv_heads, queries, capacity, head_dim, lengths, seed):
        super().__init__(len(BANDS), heads, kv_heads, queries, capacity, head_dim, lengths, seed=seed)
        rng = np.random.default_rng(seed)
        for b, band in enumerate(BANDS):
            n = min(lengths[b], capacity)
            self.scales[0][b, :, :n] = min(252, 126 - band) - rng.integers(0, 2, self.scales[0][b, :, :n].shape)
            shape = self.q[b].shape
            self.q[b] = np.ldexp(rng.uniform(1, 2, shape) * rng.choice([-1, 1], shape), band).astype(np.float32)
        if queries > 1:
            self.q[:, :, ::3] = 0

    def check(self, got):
        batch, heads, t, h = self.q.shape
        group = heads // self.kv_heads
        for i in range(batch):
            length = min(self.lengths[i], self.capacity)
            seen = np.arange(length)[None, :] <= (length - t + np.arange(t))[:, None]
            for head in range(heads):
                at = (i, head // group, slice(0, length))
                k, v = (ref.dequantize(c[at], s[at]) for c, s in zip(self.codes, self.scales))
                q = self.q[i, head].astype(np.float64)
                largest = np.where(seen, np.abs(q) @ np.abs(k).T, 0).max() * self.scale
                s = np.where(seen, q @ k.T * self.scale, -np.inf)
                p = np.exp(s - s.max(1, keepdims=True))
                p = p / p.sum(1, keepdims=True)
                want, size = p @ v, p @ np.abs(v)
                d = (4 * h / 32 + 70) * 2.0 ** -23 * largest + 2.0 ** -150 * np.abs(k).sum(1).max()
                assert d < 0.01
                bound = (4 * d + (3 * length / 32 + 128) * 2.0 ** -22) * size + length * 2.0 ** -126 * np.abs(v).max()
                wrong = np.abs(got[i, head] - want) > bound
                assert not wrong.any(), (i, head, np.argwhere(wrong)[:4], got[i, head][wrong][:4], want[wrong][:4])


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,queries,length", [
    (3, 1, 1, 40), (8, 2, 1, 700), (4, 2, 1, 3000),  # a token: one step, a few, shared by workgroups
    (4, 2, 17, 50), (3, 1, 40, 200)])                # a chunk
def test_small_queries_count_in_full(gpu, head_dim, heads, kv_heads, queries, length):
    lengths = [length, length - 1, length, length - 7, length]
    case = SmallCase(heads, kv_heads, queries, length + 3, head_dim, lengths, seed=length + head_dim)
    got = case.run(gpu)
    case.check(got)
    assert np.array_equal(got, case.run(gpu))
    if length == 3000:
        other = Gpu(0, workspace_bytes=0)  # each tile by one workgroup
        try:
            case.check(case.run(other))
        finally:
            other.close()


def test_small_queries_of_many_rows(gpu):
    """More tiles of 16 rows than the CUs take at once."""
    case = SmallCase(24, 6, 150, 160, 64, [160, 150, 155, 157, 160], seed=4)
    case.check(case.run(gpu))


@pytest.mark.parametrize("queries", [1, 40])
def test_other_queries_keep_their_bits(gpu, queries):
    """One query of a tile is small: the others, and one with an infinity, give what they give without it; what they do
    not see (NaN blocks past a length, a NaN key behind some) does not reach them."""
    case = Case(2, 4, 1, queries, 120, 64, [100, 60], seed=queries)
    case.scales[0][0, 0, 99, 0] = 255
    case.q[1, 2, 0, 3] = np.inf
    expected = case.run(gpu)
    case.q[:, 1, 0] = 2.0 ** -126 * (1 + 2.0 ** -22)
    got = case.run(gpu)
    for head in (0, 2, 3):
        assert np.array_equal(got[:, head].view(np.uint32), expected[:, head].view(np.uint32))
    assert np.array_equal(got[:, 1, 1:].view(np.uint32), expected[:, 1, 1:].view(np.uint32))
