// Interface between the 8-bit entry points (fp8.cpp, norm_abi.cpp) and their kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "staleynet_fp8.h"

namespace sn {
namespace fp8 {

// Values (and bytes) of a block; the scale bytes of the least and the largest factor.
constexpr int64_t kBlock = SN_FP8_BLOCK;
constexpr uint32_t kLeastScale = 3;
constexpr uint32_t kLargestScale = 246;

constexpr int64_t blocks_of(int64_t inner) { return (inner + kBlock - 1) / kBlock; }
// Bytes of a row's scales.
constexpr int64_t scale_stride(int64_t blocks) { return (blocks + 3) / 4 * 4; }

// An operand to 8 bits and back (fp8_quantize.hip): `rows` rows of the format of
// `inner` values; the fp32 side is [rows, inner], or transposed [inner, rows].
struct OperandArgs {
    const float* source = nullptr;  // to quantize
    float* output = nullptr;        // else
    uint8_t* codes = nullptr;
    uint8_t* scales = nullptr;
    int64_t rows = 0, inner = 0;
    bool transposed = false;
};
hipError_t launch_operand(const OperandArgs& args, bool quantize, hipStream_t stream);

// Products of two 8-bit operands (fp8_matmul.hip): less than kMaxTiles tiles of 256 threads, as a launch is less than 2^32
// threads; the largest tiles are kLargestTile rows by as many columns.
constexpr int64_t kMaxTiles = int64_t(1) << 24, kLargestTile = 256;
struct ProductArgs {
    const uint8_t* x = nullptr;
    const uint8_t* x_scales = nullptr;
    const uint8_t* w = nullptr;
    const uint8_t* w_scales = nullptr;
    const float* bias = nullptr;  // null: none
    float* y = nullptr;
    int64_t rows = 0, cols = 0, inner = 0, blocks = 0;
    float scale = 1.f;
    bool accumulate = false;
    float* workspace = nullptr;
    size_t workspace_bytes = 0;
    int cu_count = 256;
};
hipError_t launch_product(const ProductArgs& args, hipStream_t stream);

}  // namespace fp8

// The norm (norm.hip): codes and scales, or out.
struct RmsNormArgs {
    const float* x = nullptr;
    const float* residual = nullptr;  // null: none
    const float* weight = nullptr;
    float* sum = nullptr;             // null: not wanted
    float* out = nullptr;
    float* inverse = nullptr;         // null: not wanted
    uint8_t* codes = nullptr;
    uint8_t* scales = nullptr;
    int64_t rows = 0, width = 0;
    float epsilon = 0.f;
    int cu_count = 256;
};
hipError_t launch_rms_norm(const RmsNormArgs& args, hipStream_t stream);

struct RmsNormBackwardArgs {
    const float* sum = nullptr;
    const float* inverse = nullptr;
    const float* weight = nullptr;
    const float* d_out = nullptr;
    const float* d_sum = nullptr;  // null: none
    float* d_x = nullptr;
    float* d_weight = nullptr;     // null: not wanted
    int64_t rows = 0, width = 0;
    float* workspace = nullptr;
    size_t workspace_bytes = 0;
    int cu_count = 256;
};
hipError_t launch_rms_norm_backward(const RmsNormBackwardArgs& args, hipStream_t stream);

}  // namespace sn
