"""CPU checks of the 4-bit entry points (include/staleynet_fp4.h): every refusal that the host makes
before it touches the device, sizes, and the format's numpy form that the GPU tests compare with."""
import ctypes
import os
import re

import numpy as np
import pytest

import fp4_reference as ref
from staleynet_amd import gemm
from staleynet_amd.gemm import MatmulSpec

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 40  # addresses that are never read


def ptr(i):
    return ctypes.c_void_p(A * i)


def test_sizes():
    assert gemm.fp4_sizes(3, 64) == (96, 6)
    assert gemm.fp4_sizes(3, 65) == (144, 9)
    assert gemm.fp4_sizes(3, 1) == (48, 3)
    assert gemm.fp4_sizes(0, 5) == (0, 0) and gemm.fp4_sizes(5, 0) == (0, 0)
    with pytest.raises(gemm.GpuError):
        gemm.fp4_sizes(1 << 40, 1 << 40)
    assert gemm.library().sn_fp4_sizes(1, 1, None, None) == gemm.SN_ERR_NULL_ARGUMENT
    header = open(os.path.join(ROOT, "include", "staleynet_fp4.h")).read()
    for name, value in re.findall(r"#define SN_(FP4_\w+) (\d+)u", header):
        assert getattr(gemm, name) == int(value)


def test_structures_have_the_layout_the_library_pins():
    assert ctypes.sizeof(gemm.CFp4CacheShape) == 32
    assert ctypes.sizeof(gemm.CFp4CacheRows) == 40
    assert ctypes.sizeof(gemm.CFp4AttentionShape) == 80 and gemm.CFp4AttentionShape.scale.offset == 72


def weight(function, cols=40, inner=70, storage=0, first=2800, second=40 * 48, third=40 * 3, at=(1, 2, 3)):
    args = [None, cols, inner, storage]
    for i, n in zip(at, (first, second, third)):
        args += [ptr(i), n]
    return getattr(gemm.library(), function)(*args)


def test_quantize_and_dequantize_refusals():
    for function in ("sn_quantize_fp4", "sn_dequantize_fp4"):
        quantize = function == "sn_quantize_fp4"
        sizes = dict(first=2800, second=1920, third=120) if quantize else dict(first=1920, second=120, third=2800)
        assert weight(function, **sizes) == gemm.SN_ERR_NULL_ARGUMENT  # everything but the context
        assert weight(function, storage=2, **sizes) == gemm.SN_ERR_UNSUPPORTED
        assert weight(function, cols=1 << 40, inner=1 << 40, **sizes) == gemm.SN_ERR_OVERFLOW
        assert weight(function, cols=1 << 31, inner=1, **sizes) == gemm.SN_ERR_OVERFLOW
        inputs = ("first",) if quantize else ("first", "second")
        for name in sizes:
            got = weight(function, **dict(sizes, **{name: sizes[name] - 1}))
            assert got == (gemm.SN_ERR_RIGHT_TOO_SMALL if name in inputs else gemm.SN_ERR_OUTPUT_TOO_SMALL), name


def product(spec, left_len=210, codes_len=40 * 48, scales_len=120, bias=None, bias_len=0, out_len=120):
    c = spec.to_c()
    return gemm.library().sn_matmul_fp4(None, ctypes.byref(c), ptr(1), left_len, ptr(2), codes_len, ptr(3),
                                        scales_len, bias, bias_len, ptr(4), out_len)


def test_product_refusals():
    spec = MatmulSpec.new(3, 40, 70).right_transposed()
    assert product(spec) == gemm.SN_ERR_NULL_ARGUMENT
    assert product(spec, left_len=209) == gemm.SN_ERR_LEFT_TOO_SMALL
    assert product(spec, codes_len=1919) == gemm.SN_ERR_RIGHT_TOO_SMALL
    assert product(spec, scales_len=119) == gemm.SN_ERR_RIGHT_TOO_SMALL
    assert product(spec, out_len=119) == gemm.SN_ERR_OUTPUT_TOO_SMALL
    assert product(spec, bias=ptr(5), bias_len=39) == gemm.SN_ERR_LENGTH_MISMATCH
    assert product(MatmulSpec.new(3, 40, 70)) == gemm.SN_ERR_UNSUPPORTED  # columns not contiguous
    assert product(spec.left_transposed()) == gemm.SN_ERR_UNSUPPORTED
    assert product(spec.causal_left()) == gemm.SN_ERR_UNSUPPORTED
    assert product(spec.batched(gemm.BatchStrides(2, 0, 0, 0))) == gemm.SN_ERR_UNSUPPORTED
    assert product(MatmulSpec.new(1 << 31, 1, 1).right_transposed()) == gemm.SN_ERR_OVERFLOW
    assert gemm.library().sn_matmul_fp4(None, None, None, 0, None, 0, None, 0, None, 0, None, 0) == \
        gemm.SN_ERR_NULL_ARGUMENT


CACHE = dict(batch=2, kv_heads=3, capacity=10, head_dim=64)
CODES, SCALES = 2 * 3 * 10 * 32, 2 * 3 * 10 * 2


def append(cache=None, time=4, position=6, width=400, key=0, value=200, packed=3200, positions=None, count=0,
           codes=CODES, scales=SCALES, buffers=(2, 3, 4, 5)):
    shape = gemm.CFp4CacheShape(**dict(CACHE, **(cache or {})))
    rows = gemm.CFp4CacheRows(time, position, width, key, value)
    args = [None, ctypes.byref(shape), ctypes.byref(rows), ptr(1), packed, positions, count]
    for i, b in enumerate(buffers):
        args += [ptr(b), codes if i % 2 == 0 else scales]
    return gemm.library().sn_fp4_cache_append(*args)


def test_append_refusals():
    assert append() == gemm.SN_ERR_NULL_ARGUMENT
    assert append(cache=dict(head_dim=48)) == gemm.SN_ERR_UNSUPPORTED
    assert append(cache=dict(capacity=1 << 62)) == gemm.SN_ERR_OVERFLOW
    assert append(position=7) == gemm.SN_ERR_SHAPE           # 7 + 4 > 10
    assert append(value=209) == gemm.SN_ERR_SHAPE            # 209 + 3 * 64 > 400
    assert append(key=(1 << 64) - 1) == gemm.SN_ERR_OVERFLOW
    assert append(packed=3199) == gemm.SN_ERR_LENGTH_MISMATCH
    assert append(positions=ptr(6), count=1) == gemm.SN_ERR_LENGTH_MISMATCH
    assert append(time=1 << 60) == gemm.SN_ERR_OVERFLOW


def attention(cache=None, heads=6, queries=4, keys=10, q=None, out=None, q_len=2 * 6 * 4 * 64, out_len=2 * 6 * 4 * 64,
              lengths=None, count=0):
    shape = gemm.CFp4CacheShape(**dict(CACHE, **(cache or {})))
    h = CACHE["head_dim"]
    dense = (6 * 4 * h, 4 * h, h)
    s = gemm.CFp4AttentionShape(heads, queries, keys, *(q or dense), *(out or dense), 0.125)
    args = [None, ctypes.byref(shape), ctypes.byref(s), ptr(1), q_len]
    for i in range(4):
        args += [ptr(2 + i), CODES if i % 2 == 0 else SCALES]
    return gemm.library().sn_fp4_attention(*args, lengths, count, ptr(8), out_len)


def test_attention_refusals():
    assert attention() == gemm.SN_ERR_NULL_ARGUMENT
    assert attention(heads=7) == gemm.SN_ERR_SHAPE
    assert attention(keys=11) == gemm.SN_ERR_SHAPE
    assert attention(cache=dict(head_dim=96)) == gemm.SN_ERR_UNSUPPORTED
    assert attention(q_len=2 * 6 * 4 * 64 - 1) == gemm.SN_ERR_LENGTH_MISMATCH
    assert attention(out_len=2 * 6 * 4 * 64 - 1) == gemm.SN_ERR_LENGTH_MISMATCH
    assert attention(lengths=ptr(7), count=1) == gemm.SN_ERR_LENGTH_MISMATCH
    assert attention(queries=1 << 40) == gemm.SN_ERR_OVERFLOW
    assert attention(q=(1 << 62, 64, 64)) == gemm.SN_ERR_OVERFLOW


def test_limits():
    """Sizes whose counts the kernels or their grids would not hold; the largest below are not refused as such."""
    over = gemm.SN_ERR_OVERFLOW
    assert product(MatmulSpec.new(1, 1, 1 << 25).right_transposed(), left_len=1 << 25) == over
    assert product(MatmulSpec.new(1, 1, (1 << 25) - 1).right_transposed(),
                   left_len=1 << 25) == gemm.SN_ERR_RIGHT_TOO_SMALL
    assert product(MatmulSpec.new(1, 1 << 28, 1).right_transposed(), out_len=1 << 28) == over
    assert product(MatmulSpec.new(1, (1 << 28) - 1, 1).right_transposed(),
                   out_len=1 << 28) == gemm.SN_ERR_RIGHT_TOO_SMALL
    for call in (append, attention):
        assert call(cache=dict(batch=1 << 20, kv_heads=2)) == over
        assert call(cache=dict(capacity=1 << 30)) == over
        assert call(cache=dict(capacity=(1 << 30) - 1)) == gemm.SN_ERR_NULL_ARGUMENT  # the context
    assert attention(queries=1 << 24) == over  # 2 * 6 heads
    assert attention(queries=1 << 23) == gemm.SN_ERR_LENGTH_MISMATCH


def test_the_reference_form_on_known_blocks():
    block = np.zeros((1, 32), np.float32)
    block[0, :8] = [6, -6, 0.25, 0.75, 5, -0.1, -0.0, 3.5]
    codes, scales = ref.quantize(block)
    assert scales[0, 0] == 127
    assert list(codes[0, :4]) == [0x7 | 0xF << 4, 0x0 | 0x2 << 4, 0x6 | 0x8 << 4, 0x8 | 0x6 << 4]
    assert list(ref.dequantize(codes, scales)[0, :8]) == [6, -6, 0, 1, 4, -0.0, -0.0, 4]
    block[0, 0] = 7
    codes, scales = ref.quantize(block)
    assert scales[0, 0] == 128 and codes[0, 0] & 15 == 6  # 3.5 factors: 4
    values = np.random.default_rng(1).standard_normal((5, 100)).astype(np.float32)
    codes, scales = ref.quantize(values)
    back = ref.dequantize(codes, scales, 100)
    factor = np.repeat(2.0 ** (scales.astype(float) - 127), 32, 1)[:, :100]
    step = np.where(np.abs(values) < 2 * factor, 0.5, np.where(np.abs(values) < 4 * factor, 1, 2)) * factor
    assert (np.abs(back - values) <= step / 2).all()
    again = ref.quantize(back)
    assert np.array_equal(ref.dequantize(*again), ref.dequantize(codes, scales))


def test_the_rust_binding_matches_the_header():
    """INTEGRATION.md's second -sys file restates this header: constants, structures, functions."""
    header = re.sub(r"/\*.*?\*/", " ", open(os.path.join(ROOT, "include", "staleynet_fp4.h")).read(), flags=re.S)
    blocks = re.findall(r"```rust\n(.*?)```", open(os.path.join(ROOT, "INTEGRATION.md")).read(), flags=re.S)
    block = re.sub(r"//[^\n]*", "", next(b for b in blocks if "staleynet-gemm-sys/src/fp4.rs" in b))
    types = {"size_t": "usize", "uint32_t": "u32", "uint8_t": "u8", "float": "f32", "int": "c_int"}

    def rust_type(c_type):
        stars, const = c_type.count("*"), "const " in c_type
        base = c_type.replace("const ", "").replace("*", "").strip()
        inner = ("*const " if const else "*mut ") if stars else ""
        return "*mut " * max(0, stars - 1) + inner + types.get(base, base)

    for name, value in re.findall(r"#define (SN_FP4_\w+) (\d+)u", header):
        assert re.search(rf"pub const {name}: u32 = {value};", block), name
    for name, body in re.findall(r"typedef struct (sn_\w+) \{(.*?)\}", header, flags=re.S):
        fields = [(f.split()[1], types[f.split()[0]]) for f in body.split(";") if f.strip()]
        got = re.search(rf"#\[repr\(C\)\][^{{]*pub struct {name} \{{(.*?)\}}", block, flags=re.S).group(1)
        assert re.findall(r"pub (\w+): (\w+)", got) == fields, name
    functions = re.findall(r"^int (sn_\w+)\(([^;]*?)\);", header, flags=re.M | re.S)
    assert len(functions) == 11
    for name, params in functions:
        want = [rust_type(re.fullmatch(r"(.*?)(\w+)", p.strip()).group(1)) for p in " ".join(params.split()).split(",")]
        got = re.search(rf"pub fn {name}\((.*?)\)\s*->\s*c_int;", block, flags=re.S).group(1)
        assert [" ".join(p.split(":", 1)[1].split()) for p in " ".join(got.split()).split(",")] == want, name
