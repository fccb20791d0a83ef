"""The 8-bit operators as they are used together: a step that adds to the residual stream, norms it to 8 bits, multiplies by
the head's 8-bit weight and scores tokens, and the way back through the same products to the norm's gradients. Each stage
is held to 64 bits on what the stage before left, within the stages' own tolerances (tests/test_fp8_gpu.py,
test_norm_gpu.py and test_logprobs_gpu.py derive them); then the whole step captured into a graph, and on two contexts."""
import numpy as np
import pytest

import fp8_reference as fp8
import test_fp8_gpu as product
import test_norm_gpu as norm
from bench import HipGraph
from test_logprobs_gpu import Case, check_backward
from staleynet_amd.gemm import Gpu, LogprobHeads, MatmulSpec, Shape, Storage

pytestmark = pytest.mark.gpu

EPSILON = norm.EPSILON


class Step:
    """One head over `rows` tokens: buffers, weights and the calls of a scored step and of its gradients."""

    def __init__(self, gpu, rows, width, heads, classes, seed, top=4):
        rng = np.random.default_rng(seed)
        self.gpu, self.rows, self.width, self.heads, self.classes, self.top = gpu, rows, width, heads, classes, top
        self.cols = heads * classes
        self.layout = LogprobHeads(classes, heads)
        self.host_weight = (0.05 * rng.standard_normal((width, self.cols))).astype(np.float32)
        self.norm_weight = gpu.upload(Shape.vector(width), 1 + 0.1 * rng.standard_normal(width))
        self.bias = gpu.upload(Shape.vector(self.cols), 0.1 * rng.standard_normal(self.cols))
        weight = gpu.upload(Shape(width, self.cols), self.host_weight)
        # The head's columns for the product, its rows for the gradient of the product's input.
        self.columns, self.rows8 = gpu.fp8_matrix(self.cols, width), gpu.fp8_matrix(width, self.cols)
        gpu.quantize_fp8(weight, self.columns, Storage.Transposed)
        gpu.quantize_fp8(weight, self.rows8)
        n = rows * heads
        zeros = lambda *shape: gpu.zeros(Shape(*shape))
        self.x, self.stream = zeros(rows, width), zeros(rows, width)
        self.tokens = gpu.upload_tokens(rng.integers(0, classes, n))
        self.d_logprobs, self.d_entropies = (gpu.upload(Shape(rows, heads), rng.standard_normal(n)) for _ in range(2))
        self.normed = gpu.fp8_matrix(rows, width)
        self.logits, self.y, self.inverse = zeros(rows, self.cols), zeros(rows, width), zeros(1, rows)
        self.logprobs, self.entropies, self.stats = zeros(rows, heads), zeros(rows, heads), zeros(rows, 2 * heads)
        self.best, self.best_logprobs = gpu.upload_tokens(np.zeros(n * top)), zeros(rows, heads * top)
        self.grad, self.grad8 = zeros(rows, self.cols), gpu.fp8_matrix(rows, self.cols)
        self.d_y, self.d_x, self.d_norm = zeros(rows, width), zeros(rows, width), zeros(1, width)
        self.fill(seed)

    def fill(self, seed):
        """The next step's inputs, into the same buffers."""
        rng = np.random.default_rng(1000 + seed)
        for t, std in ((self.x, 1), (self.stream, 3)):
            self.gpu.copy_from_host(t, std * rng.standard_normal(self.rows * self.width))
        self.gpu.copy_from_host(self.d_norm, np.zeros(self.width))

    def run(self):
        gpu = self.gpu
        # The stream updated in place, normed once to 8 bits and once for the backward.
        gpu.rms_norm(self.x, self.norm_weight, self.normed, EPSILON, self.rows, self.stream, self.stream)
        gpu.rms_norm(self.stream, self.norm_weight, self.y, EPSILON, self.rows, inverse=self.inverse)
        spec = MatmulSpec.new(self.rows, self.cols, self.width).right_transposed()
        gpu.matmul_fp8(spec, self.normed, self.columns, self.logits, self.bias)
        gpu.token_logprobs(self.logits, self.layout, self.tokens, self.logprobs, self.entropies, self.stats, self.top,
                           self.best, self.best_logprobs)
        gpu.token_logprobs_backward(self.logits, self.layout, self.stats, self.grad, self.tokens, self.d_logprobs,
                                    self.entropies, self.d_entropies)
        gpu.quantize_fp8(self.grad, self.grad8)
        gpu.matmul_fp8(MatmulSpec.new(self.rows, self.width, self.cols).right_transposed(), self.grad8, self.rows8, self.d_y)
        gpu.rms_norm_backward(self.stream, self.inverse, self.norm_weight, self.d_y, self.d_x, self.rows, None, self.d_norm)

    OUTPUTS = ("stream", "y", "inverse", "logits", "logprobs", "entropies", "stats", "best_logprobs", "grad", "d_y", "d_x",
               "d_norm")

    def results(self):
        got = {name: self.gpu.download(getattr(self, name)) for name in self.OUTPUTS}
        got["best"] = np.asarray(self.gpu.download_tokens(self.best))
        for name in ("normed", "grad8"):
            matrix = getattr(self, name)
            got[name], got[name + "_scales"] = self.gpu.download_bytes(matrix.codes), self.gpu.download_bytes(matrix.scales)
        return got

    def check(self, x, stream):
        """Every stage against 64 bits on what the stage before left."""
        got, rows, width, cols = self.results(), self.rows, self.width, self.cols
        weight = self.gpu.download(self.norm_weight)
        s = x + stream
        assert np.array_equal(got["stream"], s)
        s = s.reshape(rows, width)
        norm.check_forward(got["y"].reshape(rows, width), got["inverse"], s, weight)
        codes, scales = fp8.quantize(got["y"].reshape(rows, width))
        assert np.array_equal(got["normed"].reshape(rows, -1), codes)
        assert np.array_equal(got["normed_scales"].reshape(rows, -1), scales)
        w = fp8.dequantize(*fp8.quantize(self.host_weight.T), width)
        logits = got["logits"].reshape(rows, cols)
        product.check(logits, fp8.dequantize(codes, scales, width), w, width, bias=self.gpu.download(self.bias))
        case = Case(rows, self.heads, self.classes)
        case.logits, case.token_rows = logits, np.asarray(self.gpu.download_tokens(self.tokens)).reshape(rows, -1)
        case.d_logprobs, case.d_entropies = (self.gpu.download(t).reshape(rows, -1) for t in (self.d_logprobs, self.d_entropies))
        places = (rows, self.heads)
        case.check(dict(logprobs=got["logprobs"].reshape(places), entropies=got["entropies"].reshape(places),
                        stats=got["stats"].reshape(places + (2,)), top_tokens=got["best"].reshape(places + (-1,)),
                        top_logprobs=got["best_logprobs"].reshape(places + (-1,))), self.top)
        grad = got["grad"].reshape(rows, cols)
        check_backward(grad.reshape(case.z.shape), case, got["stats"].reshape(places + (2,)),
                       got["entropies"].reshape(places))
        codes, scales = fp8.quantize(grad)
        assert np.array_equal(got["grad8"].reshape(rows, -1), codes)
        rows8 = fp8.dequantize(*fp8.quantize(self.host_weight), cols)
        d_y = got["d_y"].reshape(rows, width)
        product.check(d_y, fp8.dequantize(codes, scales, cols), rows8, cols)
        d_x, d_x_off, d_w, d_w_off = norm.backward(s, got["inverse"], weight, d_y, None)
        assert (np.abs(got["d_x"].reshape(rows, width) - d_x) <= d_x_off).all()
        assert (np.abs(got["d_norm"] - d_w) <= d_w_off).all()


@pytest.mark.parametrize("rows,width,heads,classes", [(1, 768, 16, 1024), (5, 512, 3, 100), (70, 200, 2, 333), (40, 300, 1, 5000),
                                                      (600, 256, 4, 250)])
def test_a_step(gpu, rows, width, heads, classes):
    step = Step(gpu, rows, width, heads, classes, rows)
    for seed in (1, 2):
        step.fill(seed)
        x, stream = gpu.download(step.x), gpu.download(step.stream)
        step.run()
        step.check(x, stream)


def test_a_captured_step(gpu):
    """Replayed on other inputs each time, with an eager step of another size on the same context between."""
    step, other = Step(gpu, 30, 300, 2, 3000, 1), Step(gpu, 3, 512, 4, 128, 2)
    step.run()
    graph = HipGraph(gpu.stream, step.run)
    try:
        for seed in range(3):
            step.fill(seed)
            eager_inputs = gpu.download(step.x), gpu.download(step.stream)
            graph.launch()
            gpu.synchronize()
            step.check(*eager_inputs)
            replayed = step.results()
            other.run()
            step.fill(seed)
            step.run()
            eager = step.results()
            assert all(np.array_equal(replayed[n], eager[n]) for n in eager)
    finally:
        graph.close()


def test_two_contexts_at_once(gpu):
    """Steps in flight on two contexts, each with a stream and a workspace of its own, leave what each leaves alone."""
    second = Gpu(0)
    try:
        steps = [Step(gpu, 200, 700, 2, 9000, 3), Step(second, 50, 9000, 1, 3000, 4)]
        alone = []
        for step in steps:
            step.run()
            alone.append(step.results())
        for _ in range(3):
            for step, seed in zip(steps, (3, 4)):
                step.fill(seed)
            for step in steps:
                step.gpu.synchronize()
            for _ in range(2):
                for step in steps:
                    step.gpu.fill_zero(step.d_norm)
                    step.run()
                for step, seed in zip(steps, (3, 4)):
                    step.fill(seed)
            for step in steps:
                step.run()
            for step, want in zip(steps, alone):
                got = step.results()
                assert all(np.array_equal(got[n], want[n]) for n in want)
    finally:
        second.close()
