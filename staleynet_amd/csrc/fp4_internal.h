// Interface between the 4-bit entry points (fp4.cpp) and their kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "staleynet_fp4.h"

namespace sn {
namespace fp4 {

// Values and bytes of codes of a block; the largest scale byte that is not NaN's.
constexpr int64_t kBlock = SN_FP4_BLOCK;
constexpr int64_t kBlockBytes = kBlock / 2;
constexpr uint32_t kLargestScale = 252;

constexpr int64_t blocks_of(int64_t inner) { return (inner + kBlock - 1) / kBlock; }

// Weights to 4 bits and back (fp4_quantize.hip): `cols` rows of the format with
// `inner` values each; the fp32 side is [inner, cols], or transposed [cols, inner].
struct WeightArgs {
    const float* source = nullptr;  // to quantize
    float* output = nullptr;        // else
    uint8_t* codes = nullptr;
    uint8_t* scales = nullptr;
    int64_t cols = 0, inner = 0;
    bool transposed = false;
};
hipError_t launch_weights(const WeightArgs& args, bool quantize, hipStream_t stream);

// Rows of a cache from packed fp32 rows, and back to dense fp32.
struct CacheRowsArgs {
    const float* packed = nullptr;        // append
    float* keys = nullptr;                // read
    float* values = nullptr;
    const uint32_t* positions = nullptr;  // null: `position` for every sequence
    uint8_t* k_codes = nullptr;
    uint8_t* k_scales = nullptr;
    uint8_t* v_codes = nullptr;
    uint8_t* v_scales = nullptr;
    int64_t batch = 0, kv_heads = 0, capacity = 0, head_dim = 0;
    int64_t time = 0, position = 0, width = 0, key_column = 0, value_column = 0;
};
hipError_t launch_cache_append(const CacheRowsArgs& args, hipStream_t stream);
hipError_t launch_cache_read(const CacheRowsArgs& args, hipStream_t stream);

// Products with 4-bit weights (fp4_matmul.hip).
struct ProductArgs {
    const float* x = nullptr;
    const uint8_t* codes = nullptr;
    const uint8_t* scales = nullptr;
    const float* bias = nullptr;  // null: none
    float* y = nullptr;
    int64_t rows = 0, cols = 0, inner = 0, blocks = 0;
    float scale = 1.f;
    bool accumulate = false;
    bool bf16 = false;  // x rounded to bf16
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
    int cu_count = 256;
};
hipError_t launch_product(const ProductArgs& args, hipStream_t stream);

// Attention over a 4-bit cache (fp4_attention.hip).
struct AttentionArgs {
    const float* q = nullptr;
    const uint8_t* k_codes = nullptr;
    const uint8_t* k_scales = nullptr;
    const uint8_t* v_codes = nullptr;
    const uint8_t* v_scales = nullptr;
    const uint32_t* lengths = nullptr;  // null: `keys` for every sequence
    float* out = nullptr;
    int64_t batch = 0, heads = 0, kv_heads = 0, capacity = 0, head_dim = 0, queries = 0, keys = 0;
    int64_t q_sequence = 0, q_head = 0, q_row = 0, out_sequence = 0, out_head = 0, out_row = 0;
    float scale = 1.f;
    float* workspace = nullptr;
    size_t workspace_bytes = 0;
    uint32_t* counters = nullptr;  // zero between calls
    size_t counter_count = 0;
    int cu_count = 256;
};
hipError_t launch_attention(const AttentionArgs& args, hipStream_t stream);

}  // namespace fp4
}  // namespace sn
