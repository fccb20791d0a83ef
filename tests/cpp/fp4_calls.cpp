// The C++ host mirror's 4-bit calls on the GPU (staleynet_cuda.hpp over staleynet_fp4.h), each held
// to the framework's fp32 call on the values the 4-bit operands stand for: a product to matmul_bias,
// the cache's rows to split_heads' columns, attention over the cache to causal_attention.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "staleynet_cuda.hpp"

extern "C" void oracle_random_values(size_t count, uint64_t seed, float* out);

using namespace staleynet_cuda;

static int failures = 0;
static void expect(bool ok, const char* what) {
    if (!ok) {
        ++failures;
        std::printf("FAILED: %s\n", what);
    }
}

static std::vector<float> values(size_t count, uint64_t seed) {
    std::vector<float> v(count);
    oracle_random_values(count, seed, v.data());
    return v;
}

static float relative_error(const std::vector<float>& a, const std::vector<float>& b) {
    float worst = 0.f, largest = 0.f;
    for (size_t i = 0; i < a.size(); ++i) {
        worst = std::max(worst, std::fabs(a[i] - b[i]));
        largest = std::max(largest, std::fabs(a[i]));
    }
    return a.size() != b.size() || largest == 0.f ? 1.f : worst / largest;
}

int main() {
    const Gpu gpu = Gpu::new_(0);
    {
        const size_t inner = 200, cols = 72;
        const Tensor w = gpu.upload(Shape::new_(inner, cols), values(inner * cols, 1));
        const Tensor bias = gpu.upload(Shape::vector(cols), values(cols, 2));
        Fp4Matrix matrix = gpu.fp4_matrix(cols, inner);
        gpu.quantize_fp4(w, matrix);
        Tensor back = gpu.zeros(Shape::new_(inner, cols));
        gpu.dequantize_fp4(matrix, back);
        expect(relative_error(gpu.download(w), gpu.download(back)) < 0.2f, "rounded weights are near the weights");
        for (size_t rows : {size_t(1), size_t(7), size_t(50)}) {
            const Tensor x = gpu.upload(Shape::new_(rows, inner), values(rows * inner, 3));
            Tensor expected = gpu.zeros(Shape::new_(rows, cols)), got = gpu.zeros(Shape::new_(rows, cols));
            gpu.matmul_bias(MatmulSpec::new_(rows, cols, inner), x, back, bias, expected);
            gpu.matmul_fp4(MatmulSpec::new_(rows, cols, inner).right_transposed(), x, matrix, got, &bias);
            expect(relative_error(gpu.download(expected), gpu.download(got)) < 1e-5f, "matmul_fp4");
        }
        Tensor x = gpu.zeros(Shape::new_(1, inner)), y = gpu.zeros(Shape::new_(1, cols));
        bool refused = false;
        try {
            gpu.matmul_fp4(MatmulSpec::new_(1, cols, inner), x, matrix, y);
        } catch (const Panic& panic) {
            refused = panic.status == SN_ERR_UNSUPPORTED;
        }
        expect(refused, "a right operand that is not transposed is refused");
    }
    {
        const size_t batch = 2, heads = 4, head_dim = 64, time = 40, width = 3 * heads * head_dim;
        Fp4Cache cache = gpu.fp4_cache(sn_fp4_cache_shape{batch, heads, time, head_dim});
        const Tensor packed = gpu.upload(Shape::new_(batch * time, width), values(batch * time * width, 4));
        const sn_fp4_cache_rows rows{time, 0, width, heads * head_dim, 2 * heads * head_dim};
        gpu.fp4_cache_append(cache, rows, packed);
        const Shape major = Shape::new_(batch * heads * time, head_dim);
        Tensor keys = gpu.zeros(major), vals = gpu.zeros(major), split = gpu.zeros(major), q = gpu.zeros(major);
        gpu.fp4_cache_read(cache, rows, keys, vals);
        gpu.split_heads(packed, split, HeadLayout::dense(batch, time, heads, head_dim, width, 2 * heads * head_dim));
        expect(relative_error(gpu.download(split), gpu.download(vals)) < 0.2f, "cached values are near split_heads'");
        gpu.split_heads(packed, q, HeadLayout::dense(batch, time, heads, head_dim, width, 0));
        Tensor expected = gpu.zeros(major), got = gpu.zeros(major);
        const float scale = 0.125f;
        gpu.causal_attention(q, keys, vals, expected,
                             sn_attention_shape{batch * heads, time, time, head_dim, time * head_dim, time * head_dim,
                                                0, scale});
        const sn_fp4_attention_shape shape{heads, time, time, heads * time * head_dim, time * head_dim, head_dim,
                                           heads * time * head_dim, time * head_dim, head_dim, scale};
        gpu.fp4_attention(cache, shape, q, got);
        expect(relative_error(gpu.download(expected), gpu.download(got)) < 1e-5f, "fp4_attention");
        const TokenBuffer lengths = gpu.upload_tokens({uint32_t(time), 0u});
        gpu.fp4_attention(cache, shape, q, got, &lengths);
        std::vector<float> ragged = gpu.download(got), whole = gpu.download(expected);
        std::fill(whole.begin() + std::ptrdiff_t(whole.size() / 2), whole.end(), 0.f);
        expect(relative_error(whole, ragged) < 1e-5f, "a sequence of length 0 gives zeros");
    }
    std::printf(failures == 0 ? "fp4 calls ok\n" : "%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
