"""The 4-bit operators together, as a program serves a model with them: one block's attention half,
prompt chunks and then single tokens of a ragged batch, and the same step captured into a graph."""
import ctypes

import numpy as np
import pytest

import fp4_reference as ref
from bench import HipGraph
from staleynet_amd import gemm
from staleynet_amd.gemm import MatmulSpec, Shape

pytestmark = pytest.mark.gpu

BATCH, HEADS, KV_HEADS, HEAD_DIM, CAPACITY = 3, 8, 2, 64, 96
WIDTH = HEADS * HEAD_DIM
PACKED = WIDTH + 2 * KV_HEADS * HEAD_DIM


class Layer:
    """x -> packed QKV -> cache -> attention -> output projection added to x, on the GPU and in 64 bits."""

    def __init__(self, gpu, time):
        rng = np.random.default_rng(11)
        self.gpu, self.time = gpu, time
        self.weights, self.values, self.bias, self.b = {}, {}, {}, {}
        for name, inner, cols in (("qkv", WIDTH, PACKED), ("out", WIDTH, WIDTH)):
            w = (rng.standard_normal((inner, cols)) * 0.05).astype(np.float32)
            self.bias[name] = (rng.standard_normal(cols) * 0.05).astype(np.float32)
            self.weights[name] = gpu.fp4_matrix(cols, inner)
            gpu.quantize_fp4(gpu.upload(Shape(inner, cols), w), self.weights[name])
            self.values[name] = ref.dequantize(*ref.quantize(w.T), inner)
            self.b[name] = gpu.upload(Shape.vector(cols), self.bias[name])
        self.cache = gpu.fp4_cache(BATCH, KV_HEADS, CAPACITY, HEAD_DIM)
        self.buffers(time)

    def buffers(self, time):
        self.time = time
        gpu, rows = self.gpu, BATCH * time
        self.x, self.y = gpu.zeros(Shape(rows, WIDTH)), gpu.zeros(Shape(rows, WIDTH))
        self.qkv, self.context = gpu.zeros(Shape(rows, PACKED)), gpu.zeros(Shape(rows, WIDTH))

    def step(self, positions, lengths):
        gpu, t, rows = self.gpu, self.time, BATCH * self.time
        gpu.matmul_fp4(MatmulSpec.new(rows, PACKED, WIDTH).right_transposed(), self.x, self.weights["qkv"], self.qkv,
                       self.b["qkv"])
        gpu.fp4_cache_append(self.cache, self.qkv, t, PACKED, WIDTH, WIDTH + KV_HEADS * HEAD_DIM, positions=positions)
        gpu.fp4_attention(self.cache, self.qkv, self.context, HEADS, t, HEAD_DIM ** -0.5, lengths=lengths,
                          q_strides=(t * PACKED, HEAD_DIM, PACKED), out_strides=(t * WIDTH, HEAD_DIM, WIDTH))
        gpu.matmul_fp4(MatmulSpec.new(rows, WIDTH, WIDTH).right_transposed().accumulate(), self.context,
                       self.weights["out"], self.y, self.b["out"])

    def expected(self, x, keys, values, lengths):
        """In 64 bits from the cache as the GPU left it (its rounding to 4 bits is tested bit for bit on its
        own; here a value next to a tie may go either way), which the new keys must be within half a step of."""
        t = self.time
        qkv = x.astype(np.float64) @ self.values["qkv"].T + self.bias["qkv"]
        out = np.zeros((BATCH * t, WIDTH))
        for b in range(BATCH):
            n = lengths[b]
            for i in range(t):
                last = n - t + i
                for head in range(HEADS):
                    q = qkv[b * t + i, head * HEAD_DIM:(head + 1) * HEAD_DIM]
                    kv = head * KV_HEADS // HEADS
                    s = keys[b, kv, :last + 1] @ q * HEAD_DIM ** -0.5
                    p = np.exp(s - s.max())
                    out[b * t + i, head * HEAD_DIM:(head + 1) * HEAD_DIM] = p @ values[b, kv, :last + 1] / p.sum()
        return qkv, out @ self.values["out"].T + self.bias["out"]

    def held(self):
        cache, shape = self.cache, (BATCH, KV_HEADS, CAPACITY, -1)
        codes = [self.gpu.download_bytes(b).reshape(shape) for b in (cache.k_codes, cache.k_scales, cache.v_codes,
                                                                     cache.v_scales)]
        return ref.dequantize(codes[0], codes[1]), ref.dequantize(codes[2], codes[3])


def check_step(layer, x, before, starts, lengths):
    gpu, t = layer.gpu, layer.time
    keys, values = layer.held()
    qkv, added = layer.expected(x, keys, values, lengths)
    got_qkv = gpu.download(layer.qkv).reshape(-1, PACKED)
    scale = np.abs(qkv).max()
    assert np.abs(got_qkv - qkv).max() <= 1e-5 * scale
    for part, held in ((0, keys), (1, values)):
        first = WIDTH + part * KV_HEADS * HEAD_DIM
        new = got_qkv[:, first:first + KV_HEADS * HEAD_DIM].reshape(BATCH, t, KV_HEADS, HEAD_DIM)
        for b in range(BATCH):
            here = new[b].transpose(1, 0, 2).reshape(-1, HEAD_DIM)
            rounded = ref.dequantize(*ref.quantize(here)).reshape(KV_HEADS, t, HEAD_DIM)
            assert np.array_equal(held[b, :, starts[b]:starts[b] + t], rounded)
    got = gpu.download(layer.y).reshape(-1, WIDTH)
    expected = before + added
    # Two products and an attention, each within the fp32 tolerance of its operands.
    assert np.abs(got - expected).max() <= 3e-5 * np.abs(expected).max()


def test_prompt_then_tokens(gpu):
    rng = np.random.default_rng(5)
    layer = Layer(gpu, 7)
    held = [0, 0, 0]
    for time in (7, 20, 1, 1, 1):
        layer.buffers(time)
        x = rng.standard_normal((BATCH * time, WIDTH)).astype(np.float32)
        before = rng.standard_normal((BATCH * time, WIDTH)).astype(np.float32)
        gpu.copy_from_host(layer.x, x)
        gpu.copy_from_host(layer.y, before)
        lengths = [n + time for n in held]
        layer.step(gpu.upload_tokens(held), gpu.upload_tokens(lengths))
        check_step(layer, x, before, held, lengths)
        held = lengths
        held[1] = max(0, held[1] - 5)  # a sequence that takes some tokens back


def write_tokens(gpu, buffer, host):
    words = np.asarray(host, np.uint32).view(np.float32)
    gpu._check(gemm.library().sn_copy_from_host(gpu._ctx, ctypes.c_void_p(buffer.pointer),
                                                words.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), words.size),
               "copy_from_host")


def test_a_captured_step_replays(gpu):
    """Positions and lengths are read on the device: one captured step serves every token. Eager work and
    synchronisations go between the replays, and each is checked."""
    rng = np.random.default_rng(6)
    layer = Layer(gpu, 1)
    positions, lengths = gpu.upload_tokens([0, 0, 0]), gpu.upload_tokens([1, 1, 1])
    layer.step(positions, lengths)
    gpu.synchronize()
    graph = HipGraph(gpu.stream, lambda: layer.step(positions, lengths))
    try:
        held = [0, 30, 0]
        for _ in range(4):
            x = rng.standard_normal((BATCH, WIDTH)).astype(np.float32)
            before = rng.standard_normal((BATCH, WIDTH)).astype(np.float32)
            gpu.copy_from_host(layer.x, x)
            gpu.copy_from_host(layer.y, before)
            after = [n + 1 for n in held]
            write_tokens(gpu, positions, held)
            write_tokens(gpu, lengths, after)
            graph.launch()
            gpu.synchronize()
            check_step(layer, x, before, held, after)
            eager = gpu.upload(Shape(64, 64), rng.standard_normal((64, 64)))
            gpu.matmul(MatmulSpec.new(64, 64, 64), eager, eager, gpu.zeros(Shape(64, 64)))
            held = after
    finally:
        gpu.synchronize()
        graph.close()


def test_two_graphs_on_one_context(gpu):
    """A sliced product and a decode step whose keys workgroups share both keep partial sums in the context's
    workspace: captured apart and replayed in turn, each replay leaves the eager bits."""
    rng = np.random.default_rng(8)
    rows, inner, cols, n = 40, 4096, 320, 3000
    w = gpu.fp4_matrix(cols, inner)
    gpu.quantize_fp4(gpu.upload(Shape(inner, cols), rng.standard_normal((inner, cols))), w)
    x, y = gpu.upload(Shape(rows, inner), rng.standard_normal((rows, inner))), gpu.zeros(Shape(rows, cols))
    cache = gpu.fp4_cache(2, 2, n, 64)
    packed = gpu.upload(Shape(2 * n, 256), rng.standard_normal((2 * n, 256)))
    gpu.fp4_cache_append(cache, packed, n, 256, 0, 128)
    q, out = gpu.upload(Shape(8, 64), rng.standard_normal((8, 64))), gpu.zeros(Shape(8, 64))
    lengths = gpu.upload_tokens([n, n // 2])
    calls = (lambda: gpu.matmul_fp4(MatmulSpec.new(rows, cols, inner).right_transposed(), x, w, y),
             lambda: gpu.fp4_attention(cache, q, out, 4, 1, 0.125, lengths=lengths))
    eager = []
    for call, result in zip(calls, (y, out)):
        call()
        eager.append(gpu.download(result))
    assert all(np.isfinite(e).all() and e.any() for e in eager)
    graphs = [HipGraph(gpu.stream, call) for call in calls]
    try:
        for _ in range(3):
            for buffer in (y, out):
                gpu.fill_zero(buffer)
            for graph in graphs:
                graph.launch()
            for result, expected in zip((y, out), eager):
                assert np.array_equal(gpu.download(result), expected)
            gpu.matmul(MatmulSpec.new(64, 64, 2), q, q, gpu.zeros(Shape(64, 64)))
    finally:
        gpu.synchronize()
        for graph in graphs:
            graph.close()
