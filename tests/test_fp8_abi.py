"""CPU checks of the 8-bit operands, the norm and the log probabilities (include/staleynet_fp8.h, staleynet_norm.h,
staleynet_logprobs.h): every refusal that the host makes before it touches the device, sizes, layouts, the Rust
binding, and the format's numpy form that the GPU tests compare with."""
import ctypes
import os
import re

import numpy as np
import pytest

import fp8_reference as ref
from staleynet_amd import gemm
from staleynet_amd.gemm import MatmulSpec

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 40  # addresses that are never read
HEADERS = ("fp8", "norm", "logprobs")


def header(name):
    return open(os.path.join(ROOT, "include", f"staleynet_{name}.h")).read()


def ptr(i):
    return ctypes.c_void_p(A * i)


def call(name, *args):
    """The library's function without a context; an argument (i, n) is buffer i with n elements."""
    flat = [None]
    for a in args:
        flat += [None if a[0] is None else ptr(a[0]), a[1]] if isinstance(a, tuple) else \
            [ctypes.byref(a) if isinstance(a, ctypes.Structure) else a]
    return getattr(gemm.library(), name)(*flat)


def refusals(call, sizes, status):
    """Each size one short gives its status."""
    for name, short in status.items():
        i, n = sizes[name]
        assert call(**{name: (i, n - 1)}) == short, name


def test_sizes():
    assert gemm.fp8_sizes(3, 128) == (384, 12)
    assert gemm.fp8_sizes(3, 129) == (768, 12)
    assert gemm.fp8_sizes(3, 513) == (1920, 24)
    assert gemm.fp8_sizes(3, 1) == (384, 12)
    assert gemm.fp8_sizes(0, 5) == (0, 0) and gemm.fp8_sizes(5, 0) == (0, 0)
    with pytest.raises(gemm.GpuError):
        gemm.fp8_sizes(1 << 40, 1 << 40)
    assert gemm.library().sn_fp8_sizes(1, 1, None, None) == gemm.SN_ERR_NULL_ARGUMENT
    for name, value in re.findall(r"#define SN_(FP8_\w+|LOGPROBS_\w+) (\d+)u", "".join(map(header, HEADERS))):
        assert getattr(gemm, name) == int(value)


@pytest.mark.parametrize("rows,inner", [((1 << 64) + 3, 64), (3, (1 << 64) + 64), (-1, 0), (3, -32)])
def test_sizes_past_64_bits_are_refused(rows, inner):
    with pytest.raises(gemm.GpuError) as error:
        gemm.fp8_sizes(rows, inner)
    assert error.value.status == gemm.SN_ERR_OVERFLOW
    with pytest.raises(gemm.GpuError):
        gemm.LogprobHeads(classes=inner).to_c(rows, 100)


def test_structures_have_the_layout_the_library_pins():
    assert ctypes.sizeof(gemm.CRmsNormShape) == 24 and gemm.CRmsNormShape.epsilon.offset == 16
    assert ctypes.sizeof(gemm.CLogprobShape) == 72 and gemm.CLogprobShape.scale.offset == 64


def test_quantize_and_dequantize_refusals():
    sizes = dict(values=(1, 2800), codes=(2, 40 * 128), scales=(3, 160))

    def operand(function, rows=40, inner=70, storage=0, **changed):
        got = dict(sizes, **changed)
        order = ("values", "codes", "scales") if function == "sn_quantize_fp8" else ("codes", "scales", "values")
        return call(function, rows, inner, storage, *(got[name] for name in order))

    for function, inputs in (("sn_quantize_fp8", ("values",)), ("sn_dequantize_fp8", ("codes", "scales"))):
        assert operand(function) == gemm.SN_ERR_NULL_ARGUMENT  # everything but the context
        assert operand(function, storage=2) == gemm.SN_ERR_UNSUPPORTED
        assert operand(function, rows=1 << 40, inner=1 << 40) == gemm.SN_ERR_OVERFLOW
        assert operand(function, rows=1 << 31, inner=1) == gemm.SN_ERR_OVERFLOW
        refusals(lambda **c: operand(function, **c), sizes,
                 {n: gemm.SN_ERR_RIGHT_TOO_SMALL if n in inputs else gemm.SN_ERR_OUTPUT_TOO_SMALL for n in sizes})


def test_product_refusals():
    sizes = dict(x=(1, 3 * 128), x_scales=(2, 12), w=(3, 40 * 128), w_scales=(4, 160), bias=(None, 0), out=(6, 120))

    def product(spec=MatmulSpec.new(3, 40, 70).right_transposed(), **changed):
        return call("sn_matmul_fp8", spec.to_c(), *dict(sizes, **changed).values())

    assert product() == gemm.SN_ERR_NULL_ARGUMENT
    refusals(product, sizes, dict(x=gemm.SN_ERR_LEFT_TOO_SMALL, x_scales=gemm.SN_ERR_LEFT_TOO_SMALL,
                                  w=gemm.SN_ERR_RIGHT_TOO_SMALL, w_scales=gemm.SN_ERR_RIGHT_TOO_SMALL,
                                  out=gemm.SN_ERR_OUTPUT_TOO_SMALL))
    assert product(bias=(5, 39)) == gemm.SN_ERR_LENGTH_MISMATCH
    assert product(bias=(5, 41)) == gemm.SN_ERR_LENGTH_MISMATCH
    spec = MatmulSpec.new(3, 40, 70)
    for other in (spec, spec.right_transposed().left_transposed(), spec.right_transposed().causal_left(),
                  spec.right_transposed().batched(gemm.BatchStrides(2, 0, 0, 0))):
        assert product(other) == gemm.SN_ERR_UNSUPPORTED
    for rows, cols, inner in ((1 << 28, 1, 1), (1, 1 << 25, 1), (1, 1, 1 << 23), (1 << 31, 1, 1)):
        assert product(MatmulSpec.new(rows, cols, inner).right_transposed(), out=(6, 1 << 31)) == gemm.SN_ERR_OVERFLOW
    assert product(MatmulSpec.new(1, 1, (1 << 23) - 1).right_transposed()) == gemm.SN_ERR_LEFT_TOO_SMALL
    assert gemm.library().sn_matmul_fp8(None, None, *[None, 0] * 6) == gemm.SN_ERR_NULL_ARGUMENT
    assert product(MatmulSpec.new(1, 1 << 24, 1).right_transposed(), out=(6, 1 << 24)) == gemm.SN_ERR_OVERFLOW
    assert product(MatmulSpec.new(1, (1 << 24) - 1, 1).right_transposed(), out=(6, 1 << 24)) == gemm.SN_ERR_RIGHT_TOO_SMALL


def test_norm_refusals():
    common = dict(x=(1, 210), residual=(2, 210), weight=(3, 70), sum=(4, 210))
    tails = dict(sn_rms_norm=dict(out=(5, 210), inverse=(6, 3)), sn_rms_norm_fp8=dict(codes=(5, 384), scales=(6, 12)))

    for function, tail in tails.items():
        def norm(rows=3, width=70, epsilon=1e-5, **changed):
            return call(function, gemm.CRmsNormShape(rows, width, epsilon), *{**common, **tail, **changed}.values())

        assert norm() == gemm.SN_ERR_NULL_ARGUMENT
        refusals(norm, {**common, **tail}, dict.fromkeys({**common, **tail}, gemm.SN_ERR_LENGTH_MISMATCH))
        for epsilon in (-1e-5, float("nan"), float("inf")):
            assert norm(epsilon=epsilon) == gemm.SN_ERR_UNSUPPORTED
        for rows, width in ((1 << 31, 1), (1, 1 << 25), (1 << 40, 1 << 40)):
            assert norm(rows=rows, width=width) == gemm.SN_ERR_OVERFLOW
        assert norm(residual=(None, 0), sum=(None, 0)) == gemm.SN_ERR_NULL_ARGUMENT  # the context
    assert gemm.library().sn_rms_norm(None, None, *[None, 0] * 6) == gemm.SN_ERR_NULL_ARGUMENT


def test_norm_backward_refusals():
    sizes = dict(sum=(1, 210), inverse=(2, 3), weight=(3, 70), d_out=(4, 210), d_sum=(5, 210), d_x=(6, 210),
                 d_weight=(7, 70))

    def backward(rows=3, width=70, **changed):
        return call("sn_rms_norm_backward", gemm.CRmsNormShape(rows, width, 0.0), *dict(sizes, **changed).values())

    assert backward() == gemm.SN_ERR_NULL_ARGUMENT
    assert backward(d_sum=(None, 0), d_weight=(None, 0)) == gemm.SN_ERR_NULL_ARGUMENT
    refusals(backward, sizes, dict.fromkeys(sizes, gemm.SN_ERR_LENGTH_MISMATCH))
    assert backward(rows=1 << 31) == gemm.SN_ERR_OVERFLOW


SHAPE = dict(rows=5, cols=100, column_offset=10, classes=30, heads=3, token_stride=4, token_offset=1, top=7, scale=1.0)


def logprob_call(function, sizes, shape=None, **changed):
    return call(function, gemm.CLogprobShape(**dict(SHAPE, **(shape or {}))), *dict(sizes, **changed).values())


LOGPROBS = dict(logits=(1, 500), tokens=(2, 20), logprobs=(3, 15), entropies=(4, 15), stats=(5, 30), top_tokens=(6, 105),
                top_logprobs=(7, 105))
GRADS = dict(logits=(1, 500), tokens=(2, 20), stats=(3, 30), entropies=(4, 15), d_logprobs=(5, 15), d_entropies=(6, 15),
             grad=(7, 500))


@pytest.mark.parametrize("function,sizes", [("sn_token_logprobs", LOGPROBS), ("sn_token_logprobs_backward", GRADS)])
def test_logprob_refusals(function, sizes):
    def logprobs(shape=None, **changed):
        return logprob_call(function, sizes, shape, **changed)

    assert logprobs() == gemm.SN_ERR_NULL_ARGUMENT
    refusals(logprobs, sizes, dict.fromkeys(sizes, gemm.SN_ERR_LENGTH_MISMATCH))
    assert logprobs(dict(column_offset=11)) == gemm.SN_ERR_SHAPE
    assert logprobs(dict(classes=0)) == gemm.SN_ERR_SHAPE
    assert logprobs(dict(heads=4)) == gemm.SN_ERR_SHAPE
    assert logprobs(dict(top=33)) == gemm.SN_ERR_UNSUPPORTED
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert logprobs(dict(scale=scale)) == gemm.SN_ERR_UNSUPPORTED
    for shape in (dict(rows=1 << 31), dict(classes=1 << 30), dict(rows=1 << 40, cols=1 << 40), dict(rows=1 << 20, cols=1 << 20),
                  dict(token_stride=1 << 60), dict(column_offset=(1 << 64) - 1)):
        assert logprobs(shape) == gemm.SN_ERR_OVERFLOW
    assert gemm.library().sn_token_logprobs(None, None, *[None, 0] * 7) == gemm.SN_ERR_NULL_ARGUMENT
    # The row stride's rest after the last row's tokens need not be there.
    assert logprobs(dict(token_offset=0), tokens=(2, 19)) == gemm.SN_ERR_NULL_ARGUMENT


def test_unused_buffers_need_not_be_given():
    none = (None, 0)
    only = dict.fromkeys(LOGPROBS, none)
    assert logprob_call("sn_token_logprobs", dict(only, logits=(1, 500))) == gemm.SN_ERR_NULL_ARGUMENT
    only = dict.fromkeys(GRADS, none)
    assert logprob_call("sn_token_logprobs_backward", dict(only, logits=(1, 500), stats=(3, 30), grad=(7, 500))) == \
        gemm.SN_ERR_NULL_ARGUMENT  # the context


def test_the_reference_form_on_known_blocks():
    block = np.zeros((1, 128), np.float32)
    block[0, :9] = [448, -448, 464, 17, 19, 1 / 512, 1 / 1024, 3 / 1024, -0.0]
    codes, scales = ref.quantize(block)
    assert list(scales[0]) == [127, 0, 0, 0]
    assert list(codes[0, :9]) == [0x7E, 0xFE, 0x7E, 0x58, 0x5A, 1, 0, 2, 0x80]  # 17: between 16 and 18, to 16; 19: to 20
    block[0, 2] = np.nextafter(np.float32(464), np.float32(500))
    codes, scales = ref.quantize(block)
    assert scales[0, 0] == 128 and codes[0, 0] == 0x76 and codes[0, 2] == 0x77  # just past 232, the middle of 224 and 240
    values = np.random.default_rng(1).standard_normal((5, 300)).astype(np.float32)
    codes, scales = ref.quantize(values)
    back = ref.dequantize(codes, scales, 300)
    factor = np.repeat(ref.factors_of(scales)[:, :3], 128, 1)[:, :300]
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(values) / factor, 2.0 ** -6))) - 3) * factor
    assert (np.abs(back - values) <= step / 2).all()
    again = ref.quantize(back)
    assert np.array_equal(ref.dequantize(*again), ref.dequantize(codes, scales))


def test_the_rust_binding_matches_the_headers():
    """INTEGRATION.md's third -sys file restates these headers: constants, structures, functions."""
    text = re.sub(r"/\*.*?\*/", " ", "".join(map(header, HEADERS)), flags=re.S)
    blocks = re.findall(r"```rust\n(.*?)```", open(os.path.join(ROOT, "INTEGRATION.md")).read(), flags=re.S)
    block = re.sub(r"//[^\n]*", "", next(b for b in blocks if "staleynet-gemm-sys/src/fp8.rs" in b))
    types = {"size_t": "usize", "uint32_t": "u32", "uint8_t": "u8", "float": "f32", "int": "c_int"}

    def rust_type(c_type):
        stars, const = c_type.count("*"), "const " in c_type
        base = c_type.replace("const ", "").replace("*", "").strip()
        return (("*const " if const else "*mut ") if stars else "") + types.get(base, base)

    for name, value in re.findall(r"#define (SN_\w+) (\d+)u", text):
        assert re.search(rf"pub const {name}: u32 = {value};", block), name
    for name, body in re.findall(r"typedef struct (sn_\w+) \{(.*?)\}", text, flags=re.S):
        fields = [(f.split()[1], types[f.split()[0]]) for f in body.split(";") if f.strip()]
        got = re.search(rf"#\[repr\(C\)\][^{{]*pub struct {name} \{{(.*?)\}}", block, flags=re.S).group(1)
        assert re.findall(r"pub (\w+): (\w+)", got) == fields, name
    functions = re.findall(r"^int (sn_\w+)\(([^;]*?)\);", text, flags=re.M | re.S)
    assert len(functions) == 9
    for name, params in functions:
        if name == "sn_fp8_sizes":
            assert "pub fn sn_fp8_sizes(rows: usize, inner: usize, codes_bytes: *mut usize, scales_bytes: *mut usize)" in \
                " ".join(block.split())
            continue
        want = [rust_type(re.fullmatch(r"(.*?)(\w+)", p.strip()).group(1)) for p in " ".join(params.split()).split(",")]
        got = re.search(rf"pub fn {name}\((.*?)\)\s*->\s*c_int;", block, flags=re.S).group(1)
        assert [" ".join(p.split(":", 1)[1].split()) for p in " ".join(got.split()).split(",")] == want, name


def test_products_of_more_tiles_than_a_launch_holds_are_refused():
    """2^24 tiles of 256 x 256 outputs and 256 threads each would be 2^32 threads."""
    def product(rows, cols):
        spec = MatmulSpec.new(rows, cols, 1).right_transposed()
        (x, x_scales), (w, w_scales) = gemm.fp8_sizes(rows, 1), gemm.fp8_sizes(cols, 1)
        return call("sn_matmul_fp8", spec.to_c(), (1, x), (2, x_scales), (3, w), (4, w_scales), (None, 0), (6, rows * cols))

    assert product(4096 * 256, 4095 * 256) == gemm.SN_ERR_NULL_ARGUMENT  # the context
    assert product(4096 * 256, 4095 * 256 + 1) == gemm.SN_ERR_OVERFLOW
    assert product(4095 * 256 + 1, 4096 * 256) == gemm.SN_ERR_OVERFLOW
    assert product((1 << 28) - 1, (1 << 24) - 1) == gemm.SN_ERR_OVERFLOW
    assert product((1 << 28) - 1, 64) == gemm.SN_ERR_NULL_ARGUMENT
    assert product(64, (1 << 24) - 1) == gemm.SN_ERR_NULL_ARGUMENT
