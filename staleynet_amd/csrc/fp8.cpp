// The C ABI of the 8-bit operands (include/staleynet_fp8.h): checks of the
// arguments, then the kernels of fp8_*.hip on the context's stream.
#include "staleynet_fp8.h"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "abi_checks.h"
#include "context_internal.h"
#include "fp8_internal.h"
#include "gemm_internal.h"

namespace {

using namespace sn::abi;
using namespace sn::fp8;

constexpr size_t kMaxDimension = size_t(1) << 31;
constexpr size_t kMaxRows = size_t(1) << 28;   // of a product; its tiles are counted in the call
constexpr size_t kMaxCols = size_t(1) << 24;   // of a product: 32 rows of outputs are less than 2^31 bytes
constexpr size_t kMaxInner = size_t(1) << 23;  // of a product: 256 rows of codes lie within 32-bit offsets

int operand_call(sn_context* ctx, bool quantize, size_t rows, size_t inner, uint32_t storage, const float* values,
                 size_t values_len, const uint8_t* codes, size_t codes_len, const uint8_t* scales,
                 size_t scales_len) {
    if (storage > SN_TRANSPOSED) return SN_ERR_UNSUPPORTED;
    size_t codes_need, scales_need, elements;
    if (sn_fp8_sizes(rows, inner, &codes_need, &scales_need) != SN_OK || !product(rows, inner, &elements) ||
        rows >= kMaxDimension || inner >= kMaxDimension)
        return SN_ERR_OVERFLOW;
    const bool short_bytes = codes_len < codes_need || scales_len < scales_need;
    if (quantize ? values_len < elements : short_bytes) return SN_ERR_RIGHT_TOO_SMALL;
    if (quantize ? short_bytes : values_len < elements) return SN_ERR_OUTPUT_TOO_SMALL;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (elements == 0) return SN_OK;
    if (values == nullptr || codes == nullptr || scales == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (!aligned<16>(codes) || !aligned<4>(scales)) return SN_ERR_UNSUPPORTED;
    const Span value_span{values, elements * sizeof(float)}, code_span{codes, codes_need},
        scale_span{scales, scales_need};
    if (overlaps(value_span, code_span) || overlaps(value_span, scale_span) ||
        (quantize && overlaps(code_span, scale_span)))
        return SN_ERR_ALIASING;
    OperandArgs args;
    args.source = values;
    args.output = const_cast<float*>(values);
    args.codes = const_cast<uint8_t*>(codes);
    args.scales = const_cast<uint8_t*>(scales);
    args.rows = int64_t(rows);
    args.inner = int64_t(inner);
    args.transposed = storage == SN_TRANSPOSED;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = launch_operand(args, quantize, ctx->stream);
    return status(err);
}

}  // namespace

extern "C" {

int sn_fp8_sizes(size_t rows, size_t inner, size_t* codes_bytes, size_t* scales_bytes) {
    if (codes_bytes == nullptr || scales_bytes == nullptr) return SN_ERR_NULL_ARGUMENT;
    *codes_bytes = *scales_bytes = 0;
    const size_t blocks = inner / SN_FP8_BLOCK + (inner % SN_FP8_BLOCK != 0);
    size_t scales, codes, count;
    if (!product(rows, blocks, &count) || !product(count, SN_FP8_BLOCK, &codes) ||
        !product(rows, (blocks + 3) / 4 * 4, &scales))
        return SN_ERR_OVERFLOW;
    *codes_bytes = codes;
    *scales_bytes = scales;
    return SN_OK;
}

int sn_quantize_fp8(sn_context* ctx, size_t rows, size_t inner, uint32_t storage, const float* source,
                    size_t source_len, uint8_t* codes, size_t codes_len, uint8_t* scales, size_t scales_len) {
    return operand_call(ctx, true, rows, inner, storage, source, source_len, codes, codes_len, scales, scales_len);
}

int sn_dequantize_fp8(sn_context* ctx, size_t rows, size_t inner, uint32_t storage, const uint8_t* codes,
                      size_t codes_len, const uint8_t* scales, size_t scales_len, float* output, size_t output_len) {
    return operand_call(ctx, false, rows, inner, storage, output, output_len, codes, codes_len, scales, scales_len);
}

int sn_matmul_fp8(sn_context* ctx, const sn_matmul_spec* spec, const uint8_t* left_codes, size_t left_codes_len,
                  const uint8_t* left_scales, size_t left_scales_len, const uint8_t* right_codes,
                  size_t right_codes_len, const uint8_t* right_scales, size_t right_scales_len, const float* bias,
                  size_t bias_len, float* output, size_t output_len) {
    // The operands' elements are counted as sn_matmul counts them, their bytes below.
    const int rc = sn_matmul_validate(spec, SIZE_MAX, SIZE_MAX, output_len);
    if (rc != SN_OK) return rc;
    if (spec->left_storage != SN_ROW_MAJOR || spec->right_storage != SN_TRANSPOSED || spec->batch_count != 1 ||
        spec->mask != SN_MASK_NONE)
        return SN_ERR_UNSUPPORTED;
    size_t left_codes_need, left_scales_need, right_codes_need, right_scales_need;
    if (sn_fp8_sizes(spec->rows, spec->inner, &left_codes_need, &left_scales_need) != SN_OK ||
        sn_fp8_sizes(spec->cols, spec->inner, &right_codes_need, &right_scales_need) != SN_OK ||
        spec->inner >= kMaxInner || spec->rows >= kMaxRows || spec->cols >= kMaxCols ||
        (spec->rows + kLargestTile - 1) / kLargestTile * ((spec->cols + kLargestTile - 1) / kLargestTile) >= kMaxTiles)
        return SN_ERR_OVERFLOW;
    if (left_codes_len < left_codes_need || left_scales_len < left_scales_need) return SN_ERR_LEFT_TOO_SMALL;
    if (right_codes_len < right_codes_need || right_scales_len < right_scales_need) return SN_ERR_RIGHT_TOO_SMALL;
    if (bias != nullptr && bias_len != spec->cols) return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (spec->rows == 0 || spec->cols == 0) return SN_OK;
    if (output == nullptr || (spec->inner > 0 && (left_codes == nullptr || left_scales == nullptr ||
                                                  right_codes == nullptr || right_scales == nullptr)))
        return SN_ERR_NULL_ARGUMENT;
    if (!aligned<16>(left_codes) || !aligned<16>(right_codes) || !aligned<4>(left_scales) ||
        !aligned<4>(right_scales))
        return SN_ERR_UNSUPPORTED;
    const Span inputs[] = {{left_codes, left_codes_need},   {left_scales, left_scales_need},
                           {right_codes, right_codes_need}, {right_scales, right_scales_need},
                           {bias, bias_len * sizeof(float)}};
    const Span outputs[] = {{output, spec->rows * spec->cols * sizeof(float)}};
    if (any_overlap(inputs, outputs)) return SN_ERR_ALIASING;
    ProductArgs args;
    args.x = left_codes;
    args.x_scales = left_scales;
    args.w = right_codes;
    args.w_scales = right_scales;
    args.bias = bias;
    args.y = output;
    args.rows = int64_t(spec->rows);
    args.cols = int64_t(spec->cols);
    args.inner = int64_t(spec->inner);
    args.blocks = blocks_of(args.inner);
    args.scale = spec->scale;
    args.accumulate = spec->write == SN_ACCUMULATE;
    args.workspace = ctx->env.workspace;
    args.workspace_bytes = ctx->env.workspace_bytes;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = launch_product(args, ctx->stream);
    return status(err);
}

}  // extern "C"
