// The C++ host mirror's 8-bit products, norms and log probabilities on the GPU (staleynet_cuda.hpp over
// staleynet_fp8.h, staleynet_norm.h and staleynet_logprobs.h): products held to the framework's fp32 call on the
// values the 8-bit operands stand for, the others to loops in 64 bits.
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
    const size_t inner = 200, cols = 72;
    const Tensor w = gpu.upload(Shape::new_(inner, cols), values(inner * cols, 1));
    const Tensor bias = gpu.upload(Shape::vector(cols), values(cols, 2));
    Fp8Matrix weights = gpu.fp8_matrix(cols, inner);
    gpu.quantize_fp8(w, weights, Storage::Transposed);
    Tensor back = gpu.zeros(Shape::new_(inner, cols));
    gpu.dequantize_fp8(weights, back, Storage::Transposed);
    expect(relative_error(gpu.download(w), gpu.download(back)) <= 0.0625f, "rounded weights are near the weights");
    for (size_t rows : {size_t(1), size_t(7), size_t(130)}) {
        const Tensor x = gpu.upload(Shape::new_(rows, inner), values(rows * inner, 3));
        const Tensor residual = gpu.upload(Shape::new_(rows, inner), values(rows * inner, 4));
        const Tensor scale = gpu.upload(Shape::vector(inner), values(inner, 5));
        const sn_rms_norm_shape shape{rows, inner, 1e-5f};
        Tensor sum = gpu.zeros(Shape::new_(rows, inner)), y = gpu.zeros(Shape::new_(rows, inner));
        Tensor inverse = gpu.zeros(Shape::vector(rows));
        gpu.rms_norm(shape, x, &residual, scale, &sum, y, &inverse);
        const std::vector<float> hx = gpu.download(x), hr = gpu.download(residual), hw = gpu.download(scale);
        std::vector<float> expected(rows * inner);
        for (size_t r = 0; r < rows; ++r) {
            double squares = 0;
            for (size_t k = 0; k < inner; ++k) squares += std::pow(double(hx[r * inner + k] + hr[r * inner + k]), 2);
            const double factor = 1.0 / std::sqrt(squares / double(inner) + double(shape.epsilon));
            for (size_t k = 0; k < inner; ++k)
                expected[r * inner + k] = float((hx[r * inner + k] + hr[r * inner + k]) * factor * hw[k]);
        }
        expect(relative_error(expected, gpu.download(y)) < 1e-6f, "rms_norm");

        // The 8-bit rows into a product, against the fp32 product of what they stand for.
        Fp8Matrix rounded = gpu.fp8_matrix(rows, inner);
        gpu.rms_norm_fp8(shape, x, &residual, scale, nullptr, rounded);
        Tensor values8 = gpu.zeros(Shape::new_(rows, inner));
        gpu.dequantize_fp8(rounded, values8);
        expect(relative_error(expected, gpu.download(values8)) <= 0.0625f, "rms_norm_fp8");
        Tensor wanted = gpu.zeros(Shape::new_(rows, cols)), got = gpu.zeros(Shape::new_(rows, cols));
        gpu.matmul_bias(MatmulSpec::new_(rows, cols, inner), values8, back, bias, wanted);
        gpu.matmul_fp8(MatmulSpec::new_(rows, cols, inner).right_transposed(), rounded, weights, got, &bias);
        expect(relative_error(gpu.download(wanted), gpu.download(got)) < 1e-5f, "matmul_fp8");

        // Those logits' log probabilities, two heads of 36 classes, and gradients back to the norm's input.
        const size_t heads = 2, classes = cols / heads, top = 3;
        const sn_logprob_shape logprob{rows, cols, 0, classes, heads, heads, 0, top, 1.f};
        std::vector<uint32_t> ids(rows * heads);
        for (size_t i = 0; i < ids.size(); ++i) ids[i] = uint32_t(7 * i % classes);
        const TokenBuffer tokens = gpu.upload_tokens(ids);
        TokenBuffer best = gpu.upload_tokens(std::vector<uint32_t>(rows * heads * top));
        Tensor lp = gpu.zeros(Shape::new_(rows, heads)), entropy = gpu.zeros(Shape::new_(rows, heads));
        Tensor stats = gpu.zeros(Shape::new_(rows, 2 * heads)), best_lp = gpu.zeros(Shape::new_(rows, heads * top));
        gpu.token_logprobs(logprob, got, &tokens, &lp, &entropy, &stats, &best, &best_lp);
        const std::vector<float> logits = gpu.download(got), hlp = gpu.download(lp), hbest = gpu.download(best_lp);
        std::vector<float> lp_wanted(rows * heads), best_wanted(rows * heads);
        for (size_t i = 0; i < rows * heads; ++i) {
            const float* z = &logits[i * classes];
            const double largest = *std::max_element(z, z + classes);
            double total = 0;
            for (size_t c = 0; c < classes; ++c) total += std::exp(double(z[c]) - largest);
            lp_wanted[i] = float(double(z[ids[i]]) - largest - std::log(total));
            best_wanted[i] = float(-std::log(total));
        }
        std::vector<float> first(rows * heads);
        for (size_t i = 0; i < rows * heads; ++i) first[i] = hbest[i * top];
        expect(relative_error(lp_wanted, hlp) < 1e-6f, "token_logprobs");
        expect(relative_error(best_wanted, first) < 1e-6f, "the likeliest class");

        const Tensor d_lp = gpu.upload(Shape::new_(rows, heads), std::vector<float>(rows * heads, 1.f));
        Tensor grad = gpu.zeros(Shape::new_(rows, cols));
        gpu.token_logprobs_backward(logprob, got, &tokens, stats, nullptr, &d_lp, nullptr, grad);
        std::vector<float> row_sums(rows * heads), ones(rows * heads);
        const std::vector<float> hgrad = gpu.download(grad);
        for (size_t i = 0; i < rows * heads; ++i) {
            for (size_t c = 0; c < classes; ++c) row_sums[i] += hgrad[i * classes + c];
            ones[i] = hgrad[i * classes + ids[i]] + std::exp(hlp[i]);
        }
        expect(*std::max_element(row_sums.begin(), row_sums.end()) < 1e-5f, "a head's gradient sums to zero");
        expect(relative_error(std::vector<float>(rows * heads, 1.f), ones) < 1e-5f, "the token's gradient is 1 - p");
        Tensor d_y = gpu.zeros(Shape::new_(rows, inner)), d_x = gpu.zeros(Shape::new_(rows, inner));
        Tensor d_scale = gpu.zeros(Shape::vector(inner));
        gpu.matmul(MatmulSpec::new_(rows, inner, cols).right_transposed(), grad, back, d_y);
        gpu.rms_norm_backward(shape, sum, inverse, scale, d_y, nullptr, d_x, &d_scale);
        // y does not change along the sum: its gradient is orthogonal to it, but for epsilon.
        const std::vector<float> hs = gpu.download(sum), hd = gpu.download(d_x);
        for (size_t r = 0; r < rows; ++r) {
            double along = 0, length = 0;
            for (size_t k = 0; k < inner; ++k) {
                along += double(hs[r * inner + k]) * hd[r * inner + k];
                length += std::fabs(double(hs[r * inner + k]) * hd[r * inner + k]);
            }
            expect(std::fabs(along) <= 1e-4 * length, "rms_norm_backward");
        }
    }
    bool refused = false;
    try {
        Fp8Matrix x = gpu.fp8_matrix(1, inner);
        Tensor y = gpu.zeros(Shape::new_(1, cols));
        gpu.matmul_fp8(MatmulSpec::new_(1, cols, inner), x, weights, y);
    } catch (const Panic& panic) {
        refused = panic.status == SN_ERR_UNSUPPORTED;
    }
    expect(refused, "a right operand that is not transposed is refused");
    std::printf(failures == 0 ? "fp8 calls ok\n" : "%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
