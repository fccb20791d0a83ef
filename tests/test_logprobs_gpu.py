"""GPU parity of log probabilities, entropies, the likeliest classes and the gradient (``sn_token_logprobs``,
``sn_token_logprobs_backward``) with 64 bits.

Tolerances. z = a (x - m) is off by 2^-23 of |z| (two roundings). A term e^z is off by that, the rounding of z log2 e and
of log2 e (2^-23 of |z| together) and 2^-22 (the exponential's ulp, twice): r = 2^-22 |z| + 2^-22 of it; a sum of n terms by (n / 64 + 64)
2^-24 of it more (a lane's chain, trees, and merged parts with a factor each). T = log(1 + rest) is off by what rest is
off over 1 + rest, and 2^-22 of itself (the logarithm). So log p: T's, 2^-23 |z| and 2^-23 of the result. H = T + W / (1 + rest): T's, W's
terms off by r + 2^-22 each and the sum's, 1 + rest's relative error of W / (1 + rest), and 2^-22 of H. In the gradient, log p is off by
2^-23 |z| and 2^-23 of the largest of it and T, p by that and r; the rest are six roundings of products."""
import numpy as np
import pytest

import logprobs_reference as ref
from bench import HipGraph
from fp4_reference import View
from logprobs_reference import EMPTY
from staleynet_amd.gemm import Gpu, GpuError, LogprobHeads, Shape

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23


class Placed:
    """A device buffer `offset` words in, with words of 77 around it; shaped for the calls that ask."""

    def __init__(self, gpu, values, offset=0, guard=5, shape=None):
        flat = np.ascontiguousarray(values).ravel()
        self.tokens = flat.dtype == np.uint32
        padded = np.pad(flat if self.tokens else flat.astype(np.float32), (offset, guard), constant_values=77)
        self.owner = gpu.upload_tokens(padded) if self.tokens else gpu.upload(Shape.vector(padded.size), padded)
        self.pointer, self.offset, self.count, self.gpu = self.owner.pointer + 4 * offset, offset, flat.size, gpu
        self.dims = np.shape(values) if shape is None else shape

    def __len__(self):
        return self.count

    def shape(self):
        return Shape(self.dims[0], int(np.prod(self.dims[1:])))

    def fetch(self):
        got = self.gpu.download_tokens(self.owner) if self.tokens else self.gpu.download(self.owner)
        got = np.asarray(got)
        assert (got[:self.offset] == 77).all() and (got[self.offset + self.count:] == 77).all()
        return got[self.offset:self.offset + self.count].reshape(self.dims)


class Case:
    def __init__(self, rows, heads, classes, column_offset=0, after=0, scale=1.0, seed=0, std=3.0, stride=None, token_offset=0):
        rng = np.random.default_rng(seed)
        self.rows, self.heads_count, self.classes, self.offset, self.scale = rows, heads, classes, column_offset, float(np.float32(scale))
        self.cols = column_offset + heads * classes + after
        self.logits = (std * rng.standard_normal((rows, self.cols))).astype(np.float32)
        self.stride = heads if stride is None else stride
        self.token_rows = rng.integers(0, classes, (rows, max(self.stride, token_offset + heads)), dtype=np.uint32)
        self.token_offset = token_offset
        self.heads = LogprobHeads(classes, heads, column_offset, stride, token_offset, scale)
        self.d_logprobs, self.d_entropies = (rng.standard_normal((rows, heads)).astype(np.float32) for _ in range(2))

    @property
    def z(self):
        return self.logits[:, self.offset:self.offset + self.heads_count * self.classes].reshape(
            self.rows, self.heads_count, self.classes)

    @property
    def tokens(self):
        return self.token_rows[:, self.token_offset:self.token_offset + self.heads_count]

    def forward(self, gpu, top, offset=0, want=("logprobs", "entropies", "stats", "top_tokens", "top_logprobs")):
        places = (self.rows, self.heads_count)
        logits, tokens = Placed(gpu, self.logits, offset), Placed(gpu, self.token_rows, offset)
        dims = dict(logprobs=places, entropies=places, stats=places + (2,), top_tokens=places + (top,),
                    top_logprobs=places + (top,))
        out = {n: Placed(gpu, np.zeros(dims[n], np.uint32 if n == "top_tokens" else np.float32), offset) for n in want}
        gpu.token_logprobs(logits, self.heads, tokens if "logprobs" in want else None, top=top, **out)
        return {n: o.fetch() for n, o in out.items()}

    def check(self, got, top):
        z = self.z
        logprobs, entropies, stats, ids, listed = ref.forward(z, self.tokens, self.scale, top)
        m, total = stats[..., 0], stats[..., 1]
        with np.errstate(all="ignore"):
            shifted = (z.astype(np.float64) - m[..., None]) * self.scale
            p = np.exp(shifted)
            r = 2.0 ** -22 * np.abs(shifted) + 2.0 ** -22
            chain = (self.classes / 64 + 64) * 2.0 ** -24
            terms = np.where((shifted < 0) & (p > 0), p * r, 0)
            others = np.where(shifted < 0, p, 0).sum(-1) + (shifted == 0).sum(-1) - 1
            rest_off = terms.sum(-1) + chain * others
            total_off = rest_off / (1 + others) + 2.0 ** -22 * total
            weights = np.where(p > 0, -p * shifted, 0)
            w_off = np.where(p > 0, weights * (r + 2.0 ** -22), 0).sum(-1) + chain * weights.sum(-1)
            w = weights.sum(-1) / (1 + others)
            entropy_off = total_off + w_off / (1 + others) + w * rest_off / (1 + others) + 2.0 ** -22 * entropies

            def lp_off(lp):
                away = np.abs(lp + (total if lp.ndim == 2 else total[..., None]))
                return (total_off if lp.ndim == 2 else total_off[..., None]) + ULP * away + ULP * np.abs(lp)

            def close(a, b, off):
                b = np.where(np.abs(b) > np.finfo(np.float32).max, np.sign(b) * np.inf, b)
                same = (a == b) | (np.isnan(a) & np.isnan(b))
                ok = same | (np.abs(a - b) <= off + 2.0 ** -140)
                assert ok.all(), (np.argwhere(~ok)[:4], a[~ok][:4], b[~ok][:4])

            if "logprobs" in got:
                close(got["logprobs"], logprobs, lp_off(logprobs))
            if "entropies" in got:
                close(got["entropies"], entropies, entropy_off)
            if "stats" in got:
                nan = np.isnan(m)
                assert np.array_equal(np.isnan(got["stats"][..., 0]), nan)
                assert np.array_equal(got["stats"][..., 0][~nan], m[~nan].astype(np.float32))
                close(got["stats"][..., 1], total, total_off)
            if "top_tokens" in got:
                assert np.array_equal(got["top_tokens"], ids)
            if "top_logprobs" in got:
                close(got["top_logprobs"], listed, lp_off(listed))


SIZES = [(1, 1, 1), (3, 2, 5), (2, 3, 64), (5, 16, 100), (3, 16, 1024), (2, 1, 1000), (4, 1, 2047), (3, 2, 2049), (2, 1, 4096),
         (3, 1, 5003), (1, 1, 16385), (2, 1, 50001), (1, 1, 131072), (70, 3, 333)]


@pytest.mark.parametrize("rows,heads,classes", SIZES)
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_forward(gpu, rows, heads, classes, top):
    case = Case(rows, heads, classes, column_offset=top % 3, after=top % 2, scale=(1.0, 0.7)[top % 2], seed=classes + top)
    got = case.forward(gpu, top, offset=rows % 4)
    case.check(got, top)
    again = case.forward(gpu, top)
    assert all(np.array_equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("scale", [3.3e38, 1e-40])
@pytest.mark.parametrize("rows,heads,classes", [(3, 2, 50), (4, 1, 3000), (2, 1, 40000)])
def test_scales_at_the_ends(gpu, rows, heads, classes, scale):
    """The largest logit, which several classes have, has log probability -log of their number; or all are alike."""
    case = Case(rows, heads, classes, scale=scale, seed=classes)
    case.logits = np.minimum(np.rint(case.logits), 4).astype(np.float32)
    case.check(case.forward(gpu, 9), 9)


@pytest.mark.parametrize("rows,heads,classes", [(3, 2, 50), (4, 1, 3000), (2, 1, 40000)])
def test_any_of_the_outputs(gpu, rows, heads, classes):
    case = Case(rows, heads, classes, seed=1, stride=heads + 3, token_offset=2)
    everything = case.forward(gpu, 4)
    case.check(everything, 4)
    for name in everything:
        alone = case.forward(gpu, 4, want=(name,))
        assert np.array_equal(alone[name], everything[name])
    assert case.forward(gpu, 4, want=()) == {}


@pytest.mark.parametrize("classes", [70, 1024, 3001, 20000])
def test_equal_logits_go_by_class(gpu, classes):
    """All equal, few distinct values, zeros of both signs, and equal values in each part of a split row."""
    case = Case(6, 1, classes, seed=2)
    rng = np.random.default_rng(3)
    case.logits[0] = 1.5
    case.logits[1] = rng.integers(0, 3, classes)
    case.logits[2] = np.where(rng.random(classes) < 0.5, 0.0, -0.0)
    case.logits[3] = -np.inf
    case.logits[3, classes // 2:classes // 2 + 20] = 2
    case.logits[4] = -2
    case.logits[4, ::max(1, classes // 25)] = 3
    case.logits[5] = np.arange(classes) % 7 == 0
    for top in (1, 9, 32):
        case.check(case.forward(gpu, top), top)


@pytest.mark.parametrize("classes", [60, 1000, 2048, 4097, 6200, 20000, 200000])
@pytest.mark.parametrize("top", [1, 10, 32])
def test_close_logits(gpu, classes, top):
    """All within a hundredth of each other, rising, falling, and with few in the lead."""
    case = Case(4, 1, classes, seed=classes)
    rng = np.random.default_rng(classes)
    case.logits[0] = 100 + rng.random(classes) / 100
    case.logits[1] = -100 + np.arange(classes) * 2.0 ** -14
    case.logits[2] = 50 - np.arange(classes) * 2.0 ** -14
    case.logits[3] = np.where(np.arange(classes) % 97 == 0, 3 + rng.random(classes) / 1000, -7)
    case.check(case.forward(gpu, top), top)


@pytest.mark.parametrize("classes", [3, 40, 1024, 2500, 30000])
def test_masks_infinities_and_nan(gpu, classes):
    case = Case(12, 2, classes, seed=4)
    lowest = np.finfo(np.float32).min
    z = case.logits.reshape(12, 2, classes)
    rng = np.random.default_rng(5)
    z[0][rng.random((2, classes)) < 0.9] = -np.inf
    z[0, :, 0] = 1
    z[1] = -np.inf                                   # no class may be answered
    z[2] = -np.inf
    z[2, :, classes - 1] = -5                        # only one
    z[3] = lowest                                    # masks of the type's lowest value
    z[4] = lowest
    z[4, :, classes // 2] = 0.25
    z[5, 0, classes // 3] = np.nan                   # NaN and inf stay in their head
    z[6, 1, classes - 1] = np.inf
    z[7, 0] = np.inf
    z[8, 0] = np.nan
    z[9] = np.finfo(np.float32).max
    z[10, :, 0] = np.finfo(np.float32).max
    z[10, :, 1:] = lowest
    z[11, 0, :2] = [np.nan, np.inf]
    case.token_rows[2] = classes - 1
    case.token_rows[4, 0] = EMPTY
    case.token_rows[6, 0] = classes                  # no class
    case.token_rows[0, 1] = 0x80000000
    case.token_rows[1, 0] = EMPTY
    for top in (0, 2, 20):
        got = case.forward(gpu, top)
        case.check(got, top)
        assert np.isnan(got["logprobs"][6, 0]) and got["logprobs"][4, 0] == 0 and got["logprobs"][1, 0] == 0
        assert np.isnan(got["entropies"][1]).all() and (got["entropies"][2] == 0).all() and (got["logprobs"][2] == 0).all()


@pytest.mark.parametrize("classes", [8, 1024, 9000])
def test_nearly_certain_answers_keep_their_digits(gpu, classes):
    """One class far ahead: log probabilities of -1e-4 to -1e-30 and their entropies to 2^-15 relative, at an offset
    of 20 that a log partition rounded with the largest logit would drown them in. The terms' z is up to 71, their relative error
    2^-22 (71 + 1) and the chain's: under 2^-15."""
    case = Case(30, 1, classes, seed=6, std=0.3)
    case.logits += 20
    case.logits[:, 0] = 20 + np.linspace(10, 70, 30).astype(np.float32)
    case.token_rows[:] = 0
    got = case.forward(gpu, 1)
    case.check(got, 1)
    logprobs, entropies, *_ = ref.forward(case.z, case.tokens)
    assert (np.abs(got["logprobs"] / logprobs - 1) < 2.0 ** -15).all()
    assert (np.abs(got["entropies"] / entropies - 1) < 2.0 ** -15).all()
    assert (np.abs(got["top_logprobs"][..., 0] / logprobs - 1) < 2.0 ** -15).all()


def run_backward(gpu, case, stats, entropies, which=("logprobs", "entropies"), offset=0, in_place=False):
    logits, tokens = Placed(gpu, case.logits, offset), Placed(gpu, case.token_rows, offset)
    grad = logits if in_place else Placed(gpu, np.full(case.logits.shape, 55, np.float32), offset)
    kw = {}
    if "logprobs" in which:
        kw.update(tokens=tokens, d_logprobs=Placed(gpu, case.d_logprobs, offset))
    if "entropies" in which:
        kw.update(entropies=Placed(gpu, entropies, offset), d_entropies=Placed(gpu, case.d_entropies, offset))
    gpu.token_logprobs_backward(logits, case.heads, Placed(gpu, stats, offset), grad, **kw)
    got = grad.fetch()
    end = case.offset + case.heads_count * case.classes
    around = case.logits if in_place else np.full(case.logits.shape, 55, np.float32)
    assert np.array_equal(got[:, :case.offset], around[:, :case.offset]) and np.array_equal(got[:, end:], around[:, end:])
    return got[:, case.offset:end].reshape(case.z.shape)


def check_backward(got, case, stats, entropies, which=("logprobs", "entropies")):
    d_lp = case.d_logprobs if "logprobs" in which else None
    d_h = case.d_entropies if "entropies" in which else None
    want = ref.backward(case.z, stats, entropies, case.tokens, d_lp, d_h, case.scale)
    with np.errstate(all="ignore"):
        s = stats.astype(np.float64)
        z = (case.z - s[..., :1]) * case.scale
        log_p = z - s[..., 1:]
        p = np.where(np.isfinite(log_p), np.exp(log_p), 0)
        log_p, z = np.where(p > 0, log_p, 0), np.where(p > 0, z, 0)
        lp_off = ULP * np.abs(z) + ULP * np.maximum(np.abs(log_p), np.abs(s[..., 1:]))
        p_rel = lp_off + 2.0 ** -22 * np.abs(log_p) + 2.0 ** -22
        a = 0 if d_lp is None else np.where(case.tokens == EMPTY, 0, np.abs(d_lp))[..., None]
        h = 0 if d_h is None else np.abs(d_h)[..., None]
        inner = np.abs(log_p) + (0 if d_h is None else np.abs(entropies)[..., None])
        off = p * (a + h * inner) * (p_rel + 6 * ULP) + p * h * lp_off + ULP * np.abs(want / case.scale) + 2.0 ** -126
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    ok = same | (np.abs(got - want) <= case.scale * off)
    assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4])


@pytest.mark.parametrize("rows,heads,classes", SIZES)
@pytest.mark.parametrize("which", [("logprobs", "entropies"), ("logprobs",), ("entropies",), ()])
def test_backward(gpu, rows, heads, classes, which):
    case = Case(rows, heads, classes, column_offset=len(which), after=rows % 2, scale=(0.7, 1.0)[len(which) % 2], seed=classes)
    case.token_rows[0, 0] = EMPTY
    forward = case.forward(gpu, 0, want=("entropies", "stats"))
    got = run_backward(gpu, case, forward["stats"], forward["entropies"], which, offset=rows % 4)
    check_backward(got, case, forward["stats"], forward["entropies"], which)
    again = run_backward(gpu, case, forward["stats"], forward["entropies"], which, in_place=True)
    assert np.array_equal(got, again, equal_nan=True)


@pytest.mark.parametrize("classes", [40, 1024, 30000])
def test_backward_of_masks_and_odd_tokens(gpu, classes):
    case = Case(6, 2, classes, column_offset=3, seed=7)
    z = case.z
    z = case.logits[:, 3:].reshape(6, 2, classes)
    z[0][np.random.default_rng(8).random((2, classes)) < 0.5] = -np.inf
    z[0, :, 3] = 2
    z[1] = -np.inf
    z[2, 0, 5] = np.nan
    z[3, :, 1:] = np.finfo(np.float32).min
    case.logits[:, 3:] = z.reshape(6, -1)
    case.token_rows[0], case.token_rows[3] = 3, 0
    case.token_rows[4, 0], case.token_rows[5, 1] = classes, EMPTY
    forward = case.forward(gpu, 0, want=("entropies", "stats"))
    got = run_backward(gpu, case, forward["stats"], forward["entropies"])
    check_backward(got, case, forward["stats"], forward["entropies"])
    assert np.isnan(got[1]).all() and np.isnan(got[2, 0]).all() and np.isfinite(got[2, 1]).all()


def test_gradient_against_differences(gpu):
    """Central differences in 64 bits of sum(d_logprob logprob + d_entropy H) over the logits."""
    case = Case(3, 2, 17, scale=1.3, seed=9, std=1.0)
    case.token_rows[1, 0] = EMPTY
    forward = case.forward(gpu, 0, want=("entropies", "stats"))
    got = run_backward(gpu, case, forward["stats"], forward["entropies"])
    base, h = case.z.astype(np.float64), 1e-5

    def loss(z):
        logprobs, entropies, *_ = ref.forward(z, case.tokens, case.scale)
        return (logprobs * case.d_logprobs).sum() + (entropies * case.d_entropies).sum()

    for at in np.ndindex(base.shape):
        step = np.zeros(base.shape)
        step[at] = h
        # Losses of up to 50: a difference is off by 2^-46 / 2h and by h^2 of the third derivative, under 1e-8; the
        # stats and the entropy that the gradient takes are fp32.
        assert abs((loss(base + step) - loss(base - step)) / (2 * h) - got[at]) < 2e-5


@pytest.mark.parametrize("rows,classes,top", [(1, 60000, 32), (3, 20000, 5), (9, 5000, 0)])
def test_a_small_workspace(gpu, rows, classes, top):
    case = Case(rows, 1, classes, seed=10)
    want = case.forward(gpu, top)
    for bytes_ in (0, 64, 1 << 12):
        other = Gpu(0, workspace_bytes=bytes_)
        try:
            got = case.forward(other, top)
        finally:
            other.close()
        case.check(got, top)
        assert np.array_equal(got["top_tokens"], want["top_tokens"])


def test_offsets_past_32_bits(gpu):
    """17 GB of logits: the last row's head, forward and backward, in place."""
    rows, cols, classes = 70000, 61000, 500
    logits = gpu.zeros(Shape(rows, cols))
    case = Case(1, 1, classes, seed=11)
    at = rows * cols - classes
    gpu.copy_from_host(View(logits, at, classes), case.logits[0])
    heads = LogprobHeads(classes, 1, cols - classes)
    tokens = np.zeros(rows, np.uint32)
    tokens[-1] = case.token_rows[0, 0]
    t = gpu.upload_tokens(tokens)
    lp, h, stats, best = (gpu.zeros(Shape.vector(n * rows)) for n in (1, 1, 2, 3))
    ids = gpu.upload_tokens(np.zeros(3 * rows, np.uint32))
    gpu.token_logprobs(logits, heads, t, lp, h, stats, 3, ids, best)
    got = dict(logprobs=gpu.download(lp)[-1:], entropies=gpu.download(h)[-1:], stats=gpu.download(stats)[-2:],
               top_tokens=np.asarray(gpu.download_tokens(ids))[-3:], top_logprobs=gpu.download(best)[-3:])
    case.check({n: v.reshape((1, 1, -1) if n[:3] in ("sta", "top") else (1, 1)) for n, v in got.items()}, 3)
    gpu.token_logprobs_backward(logits, heads, stats, logits, t, gpu.upload(Shape.vector(rows), np.full(rows, case.d_logprobs[0, 0])),
                                h, gpu.upload(Shape.vector(rows), np.full(rows, case.d_entropies[0, 0])))
    grad = gpu.download(View(logits, at, classes)).reshape(1, 1, classes)
    check_backward(grad, case, got["stats"].reshape(1, 1, 2), got["entropies"].reshape(1, 1))


def test_nothing_to_do(gpu):
    out = gpu.zeros(Shape(2, 4))
    gpu.token_logprobs(gpu.zeros(Shape(0, 4)), LogprobHeads(4), entropies=out)
    gpu.token_logprobs(out, LogprobHeads(4, heads=0), entropies=gpu.zeros(Shape(2, 4)))
    gpu.token_logprobs_backward(out, LogprobHeads(4, heads=0), out, out)
    assert not gpu.download(out).any()


def test_refusals(gpu):
    case = Case(3, 2, 10)
    logits, tokens = Placed(gpu, case.logits), Placed(gpu, case.token_rows)
    out = [gpu.zeros(Shape.vector(60)) for _ in range(4)]
    for kw in (dict(logprobs=View(logits, 0, 60)), dict(logprobs=out[0], entropies=out[0]), dict(entropies=out[1], stats=out[1]),
               dict(top_logprobs=out[2], top_tokens=out[2], top=3), dict(logprobs=tokens)):
        with pytest.raises(GpuError):
            gpu.token_logprobs(logits, case.heads, tokens, **kw)
    with pytest.raises(AssertionError):  # no tokens: too short
        gpu.token_logprobs(logits, case.heads, None, logprobs=out[0])
    with pytest.raises(AssertionError):
        gpu.token_logprobs(logits, LogprobHeads(10, 3), entropies=out[0])
    with pytest.raises(GpuError):
        gpu.token_logprobs(logits, LogprobHeads(10, 2, scale=0.0), entropies=out[0])
    with pytest.raises(AssertionError):
        gpu.token_logprobs(logits, case.heads, stats=View(out[0], 0, 11))
    grad = Placed(gpu, case.logits)
    for kw in (dict(grad=View(logits, 1, 59)), dict(stats=View(grad, 0, 12)), dict(tokens=tokens, d_logprobs=View(grad, 0, 6)),
               dict(d_entropies=out[0]), dict(d_logprobs=out[0])):
        with pytest.raises((GpuError, AssertionError)):
            gpu.token_logprobs_backward(**dict(dict(logits=logits, heads=case.heads, stats=out[3], grad=grad), **kw))


def test_captured_calls_replay(gpu):
    """Split and unsplit rows, forward and backward, in one graph: each replay leaves the eager bits."""
    sets = []
    for rows, heads, classes in ((4, 16, 1024), (2, 1, 30000)):
        case = Case(rows, heads, classes, seed=12)
        n = rows * heads
        t = [Placed(gpu, case.logits), Placed(gpu, case.token_rows), Placed(gpu, case.d_logprobs), Placed(gpu, case.d_entropies)]
        out = [gpu.zeros(Shape.vector(k * n)) for k in (1, 1, 2, 6)] + [gpu.zeros(Shape(rows, case.cols))]
        sets.append((case, t, out, gpu.upload_tokens(np.zeros(6 * n, np.uint32))))

    def step():
        for case, (logits, tokens, d_lp, d_h), (lp, h, stats, best, grad), ids in sets:
            gpu.token_logprobs(logits, case.heads, tokens, lp, h, stats, 6, ids, best)
            gpu.token_logprobs_backward(logits, case.heads, stats, grad, tokens, d_lp, h, d_h)

    def results():
        return [gpu.download(o) for _, _, out, _ in sets for o in out] + [np.asarray(gpu.download_tokens(s[3])) for s in sets]

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
            case, t, out, ids = sets[1]
            gpu.token_logprobs(t[0], case.heads, t[1], out[0], out[1], out[2], 2, ids, out[3])
    finally:
        graph.close()


@pytest.mark.parametrize("classes", [1, 40, 513, 1024, 1027, 30000])
def test_places_without_a_term_have_no_gradient(gpu, classes):
    """An empty token, or no d_logprobs, with no d_entropy: zeros, in heads without a finite logit or with NaN and
    infinities too. The other places are the same bits as without such rows."""
    case = Case(9, 2, classes, column_offset=1, after=2, seed=13, scale=0.7)
    bad = case.logits[:, 1:-2].reshape(9, 2, classes).copy()
    bad[0] = -np.inf
    bad[1, :, classes // 2] = np.nan
    bad[2, 0, classes - 1], bad[2, 1] = np.inf, np.inf
    bad[3] = np.nan
    good = case.logits.copy()
    case.token_rows[:5] = EMPTY
    case.token_rows[5, 0], case.token_rows[6, 1] = EMPTY, classes
    case.d_entropies[:5], case.d_entropies[4, 1] = 0.0, -0.0
    case.d_logprobs[0], case.d_logprobs[1] = np.nan, np.inf  # an empty token's is not used
    for which in (("logprobs", "entropies"), ("logprobs",), ("entropies",), ()):
        case.logits = good
        forward = case.forward(gpu, 0, want=("entropies", "stats"))
        want = run_backward(gpu, case, forward["stats"], forward["entropies"], which)
        case.logits = good.copy()
        case.logits[:4, 1:-2] = bad.reshape(9, -1)[:4]
        forward = case.forward(gpu, 0, want=("entropies", "stats"))
        assert np.isnan(forward["stats"][:4, :, 0]).all()
        for in_place in (False, True):
            got = run_backward(gpu, case, forward["stats"], forward["entropies"], which, in_place=in_place)
            assert (got[:5] == 0).all()
            assert np.array_equal(got, want)
        if not which:
            assert not got.any()


def test_captured_lists_replay(gpu):
    """The listed classes of split and unsplit rows, overwritten before each replay."""
    sets = []
    for rows, heads, classes in ((4, 16, 1024), (2, 1, 30000)):
        case = Case(rows, heads, classes, seed=14)
        n = 6 * rows * heads
        sets.append((case, Placed(gpu, case.logits), gpu.upload_tokens(np.zeros(n, np.uint32)), gpu.zeros(Shape.vector(n))))

    def step():
        for case, logits, ids, best in sets:
            gpu.token_logprobs(logits, case.heads, top=6, top_tokens=ids, top_logprobs=best)

    def results():
        return [np.asarray(gpu.download_tokens(s[2])) for s in sets] + [gpu.download(s[3]) for s in sets]

    step()
    want = results()
    graph = HipGraph(gpu.stream, step)
    try:
        for _ in range(3):
            for case, logits, ids, best in sets:  # other lists: of the negated logits
                gpu.token_logprobs(Placed(gpu, -case.logits), case.heads, top=6, top_tokens=ids, top_logprobs=best)
            assert not any(np.array_equal(a, b) for a, b in zip(results(), want))
            graph.launch()
            gpu.synchronize()
            assert all(np.array_equal(a, b) for a, b in zip(results(), want))
    finally:
        graph.close()
