// The C ABI of the norm (include/staleynet_norm.h): checks of the arguments,
// then the kernels of norm.hip on the context's stream.
#include "staleynet_norm.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "abi_checks.h"
#include "context_internal.h"
#include "fp8_internal.h"

// The struct's layout is part of the ABI (x86-64 / aarch64 LP64).
static_assert(sizeof(sn_rms_norm_shape) == 24 && offsetof(sn_rms_norm_shape, epsilon) == 16,
              "sn_rms_norm_shape layout");

namespace {

using namespace sn::abi;

constexpr size_t kMaxRows = size_t(1) << 31;
constexpr size_t kMaxWidth = size_t(1) << 25;

int check_shape(const sn_rms_norm_shape* shape, size_t* elements) {
    if (shape == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (!product(shape->rows, shape->width, elements) || shape->rows >= kMaxRows || shape->width >= kMaxWidth)
        return SN_ERR_OVERFLOW;
    if (!(shape->epsilon >= 0.f) || !std::isfinite(shape->epsilon)) return SN_ERR_UNSUPPORTED;
    return SN_OK;
}

// A sum in place of x or the residual is no overlap with it.
const void* other_than(const void* data, const void* in_place) { return data == in_place ? nullptr : data; }

// `out` and `inverse`, or `codes` and `scales`.
int forward(sn_context* ctx, const sn_rms_norm_shape* shape, const float* x, size_t x_len, const float* residual,
            size_t residual_len, const float* weight, size_t weight_len, float* sum, size_t sum_len, float* out,
            size_t out_len, float* inverse, size_t inverse_len, bool eight, uint8_t* codes, size_t codes_len,
            uint8_t* scales, size_t scales_len) {
    size_t elements, codes_need = 0, scales_need = 0;
    const int rc = check_shape(shape, &elements);
    if (rc != SN_OK) return rc;
    if (eight && sn_fp8_sizes(shape->rows, shape->width, &codes_need, &scales_need) != SN_OK) return SN_ERR_OVERFLOW;
    if (x_len < elements || (residual != nullptr && residual_len < elements) || weight_len < shape->width ||
        (sum != nullptr && sum_len < elements) || (inverse != nullptr && inverse_len < shape->rows) ||
        (!eight && out_len < elements) || codes_len < codes_need || scales_len < scales_need)
        return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (elements == 0) return SN_OK;
    if (x == nullptr || weight == nullptr || (eight ? codes == nullptr || scales == nullptr : out == nullptr))
        return SN_ERR_NULL_ARGUMENT;
    if (eight && (!aligned<16>(codes) || !aligned<4>(scales))) return SN_ERR_UNSUPPORTED;
    const size_t bytes = elements * sizeof(float);
    const Span sum_span{sum, bytes}, x_span{x, bytes}, residual_span{residual, bytes},
        weight_span{weight, shape->width * sizeof(float)};
    const Span sum_inputs[] = {{other_than(x, sum), bytes}, {other_than(residual, sum), bytes}, weight_span};
    const Span sum_only[] = {sum_span};
    const Span others[] = {{out, eight ? 0 : bytes},
                           {inverse, shape->rows * sizeof(float)},
                           {codes, codes_need},
                           {scales, scales_need}};
    const Span inputs[] = {x_span, residual_span, weight_span, sum_span};
    if (any_overlap(sum_inputs, sum_only) || any_overlap(inputs, others)) return SN_ERR_ALIASING;
    sn::RmsNormArgs args;
    args.x = x;
    args.residual = residual;
    args.weight = weight;
    args.sum = sum;
    args.out = out;
    args.inverse = inverse;
    args.codes = codes;
    args.scales = scales;
    args.rows = int64_t(shape->rows);
    args.width = int64_t(shape->width);
    args.epsilon = shape->epsilon;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = sn::launch_rms_norm(args, ctx->stream);
    return status(err);
}

}  // namespace

extern "C" {

int sn_rms_norm(sn_context* ctx, const sn_rms_norm_shape* shape, const float* x, size_t x_len, const float* residual,
                size_t residual_len, const float* weight, size_t weight_len, float* sum, size_t sum_len, float* out,
                size_t out_len, float* inverse, size_t inverse_len) {
    return forward(ctx, shape, x, x_len, residual, residual_len, weight, weight_len, sum, sum_len, out, out_len,
                   inverse, inverse_len, false, nullptr, 0, nullptr, 0);
}

int sn_rms_norm_fp8(sn_context* ctx, const sn_rms_norm_shape* shape, const float* x, size_t x_len,
                    const float* residual, size_t residual_len, const float* weight, size_t weight_len, float* sum,
                    size_t sum_len, uint8_t* codes, size_t codes_len, uint8_t* scales, size_t scales_len) {
    return forward(ctx, shape, x, x_len, residual, residual_len, weight, weight_len, sum, sum_len, nullptr, 0, nullptr,
                   0, true, codes, codes_len, scales, scales_len);
}

int sn_rms_norm_backward(sn_context* ctx, const sn_rms_norm_shape* shape, const float* sum, size_t sum_len,
                         const float* inverse, size_t inverse_len, const float* weight, size_t weight_len,
                         const float* d_out, size_t d_out_len, const float* d_sum, size_t d_sum_len, float* d_x,
                         size_t d_x_len, float* d_weight, size_t d_weight_len) {
    size_t elements;
    const int rc = check_shape(shape, &elements);
    if (rc != SN_OK) return rc;
    if (sum_len < elements || inverse_len < shape->rows || weight_len < shape->width || d_out_len < elements ||
        (d_sum != nullptr && d_sum_len < elements) || d_x_len < elements ||
        (d_weight != nullptr && d_weight_len < shape->width))
        return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (elements == 0) return SN_OK;
    if (sum == nullptr || inverse == nullptr || weight == nullptr || d_out == nullptr || d_x == nullptr)
        return SN_ERR_NULL_ARGUMENT;
    const size_t bytes = elements * sizeof(float), row = shape->width * sizeof(float);
    const Span inputs[] = {{sum, bytes},
                           {inverse, shape->rows * sizeof(float)},
                           {weight, row},
                           {d_out, bytes},
                           {other_than(d_sum, d_x), bytes}};
    const Span outputs[] = {{d_x, bytes}, {d_weight, row}};
    const Span d_sum_input[] = {{d_sum, bytes}};
    const Span weight_output[] = {{d_weight, row}};
    if (any_overlap(inputs, outputs) || any_overlap(d_sum_input, weight_output)) return SN_ERR_ALIASING;
    sn::RmsNormBackwardArgs args;
    args.sum = sum;
    args.inverse = inverse;
    args.weight = weight;
    args.d_out = d_out;
    args.d_sum = d_sum;
    args.d_x = d_x;
    args.d_weight = d_weight;
    args.rows = int64_t(shape->rows);
    args.width = int64_t(shape->width);
    args.workspace = ctx->env.workspace;
    args.workspace_bytes = ctx->env.workspace_bytes;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = sn::launch_rms_norm_backward(args, ctx->stream);
    return status(err);
}

}  // extern "C"
