// The C ABI of the 4-bit weights and cache (include/staleynet_fp4.h): checks of
// the arguments, then the kernels of fp4_*.hip on the context's stream.
#include "staleynet_fp4.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "context_internal.h"
#include "fp4_internal.h"
#include "gemm_internal.h"

// The structs' layouts are part of the ABI (x86-64 / aarch64 LP64).
static_assert(sizeof(sn_fp4_cache_shape) == 32 && offsetof(sn_fp4_cache_shape, head_dim) == 24,
              "sn_fp4_cache_shape layout");
static_assert(sizeof(sn_fp4_cache_rows) == 40 && offsetof(sn_fp4_cache_rows, value_column) == 32,
              "sn_fp4_cache_rows layout");
static_assert(sizeof(sn_fp4_attention_shape) == 80 && offsetof(sn_fp4_attention_shape, out_row) == 64 &&
                  offsetof(sn_fp4_attention_shape, scale) == 72,
              "sn_fp4_attention_shape layout");

namespace {

using namespace sn::fp4;

// Sizes and offsets stay below this, so that byte offsets fit the kernels' signed arithmetic.
constexpr size_t kLimit = size_t(1) << 60;
constexpr size_t kMaxDimension = size_t(1) << 31;
constexpr size_t kMaxCols = size_t(1) << 28;       // of a product: 2^32 threads a launch
constexpr size_t kMaxInner = size_t(1) << 25;      // of a product: its kernels count blocks in 32 bits
// Query rows of an attention call and heads of a cache, over their sequences: at most 2^23 + 2^21 tiles of
// 16 rows, of 256 threads each, where a launch holds 2^32.
constexpr size_t kMaxRows = size_t(1) << 27;
constexpr size_t kMaxHeads = size_t(1) << 21;
constexpr size_t kMaxPositions = size_t(1) << 30;  // of a cache: attention counts them in 32 bits

int status(hipError_t err) { return err == hipSuccess ? SN_OK : int(err); }

// a * b, or false where it reaches the limit.
bool product(size_t a, size_t b, size_t* out) { return !__builtin_mul_overflow(a, b, out) && *out < kLimit; }
bool sum(size_t a, size_t b, size_t* out) { return !__builtin_add_overflow(a, b, out) && *out < kLimit; }

bool overlaps(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    if (a == nullptr || b == nullptr || a_bytes == 0 || b_bytes == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    return a0 < b0 + b_bytes && b0 < a0 + a_bytes;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A byte buffer an entry point takes, with what it needs of it.
struct Bytes {
    const uint8_t* data;
    size_t len, need;
};

int weight_call(sn_context* ctx, bool quantize, size_t cols, size_t inner, uint32_t storage, const float* values,
                size_t values_len, const uint8_t* codes, size_t codes_len, const uint8_t* scales, size_t scales_len) {
    if (storage > SN_TRANSPOSED) return SN_ERR_UNSUPPORTED;
    size_t codes_need, scales_need, elements;
    if (sn_fp4_sizes(cols, inner, &codes_need, &scales_need) != SN_OK || !product(cols, inner, &elements) ||
        cols >= kMaxDimension || inner >= kMaxDimension)
        return SN_ERR_OVERFLOW;
    const bool short_bytes = codes_len < codes_need || scales_len < scales_need;
    if (quantize ? values_len < elements : short_bytes) return SN_ERR_RIGHT_TOO_SMALL;
    if (quantize ? short_bytes : values_len < elements) return SN_ERR_OUTPUT_TOO_SMALL;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (elements == 0) return SN_OK;
    if (values == nullptr || codes == nullptr || scales == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (!aligned16(codes)) return SN_ERR_UNSUPPORTED;
    const size_t value_bytes = elements * sizeof(float);
    if (overlaps(values, value_bytes, codes, codes_need) || overlaps(values, value_bytes, scales, scales_need) ||
        (quantize && overlaps(codes, codes_need, scales, scales_need)))
        return SN_ERR_ALIASING;
    WeightArgs args;
    args.source = values;
    args.output = const_cast<float*>(values);
    args.codes = const_cast<uint8_t*>(codes);
    args.scales = const_cast<uint8_t*>(scales);
    args.cols = int64_t(cols);
    args.inner = int64_t(inner);
    args.transposed = storage == SN_TRANSPOSED;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = launch_weights(args, quantize, ctx->stream);
    return status(err);
}

// What a cache's four buffers need, and the checks that they have it. `codes` and
// `scales` are the bytes of one of the two buffers of each kind.
int cache_need(const sn_fp4_cache_shape& c, size_t* codes, size_t* scales) {
    if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return SN_ERR_UNSUPPORTED;
    size_t heads, rows, values;
    if (!product(c.batch, c.kv_heads, &heads) || !product(heads, c.capacity, &rows) ||
        !product(rows, c.head_dim, &values) || heads >= kMaxHeads || c.capacity >= kMaxPositions)
        return SN_ERR_OVERFLOW;
    *codes = values / 2;
    *scales = values / SN_FP4_BLOCK;
    return SN_OK;
}

int check_buffers(const Bytes (&buffers)[4]) {
    for (const Bytes& b : buffers)
        if (b.len < b.need) return SN_ERR_LENGTH_MISMATCH;
    for (const Bytes& b : buffers)
        if (b.data == nullptr && b.need > 0) return SN_ERR_NULL_ARGUMENT;
    if (!aligned16(buffers[0].data) || !aligned16(buffers[2].data)) return SN_ERR_UNSUPPORTED;
    return SN_OK;
}

int cache_rows_call(sn_context* ctx, bool append, const sn_fp4_cache_shape* cache, const sn_fp4_cache_rows* rows,
                    const float* packed, size_t packed_len, const uint32_t* positions, size_t positions_len,
                    const uint8_t* k_codes, size_t k_codes_len, const uint8_t* k_scales, size_t k_scales_len,
                    const uint8_t* v_codes, size_t v_codes_len, const uint8_t* v_scales, size_t v_scales_len,
                    float* keys, size_t keys_len, float* values, size_t values_len) {
    if (cache == nullptr || rows == nullptr) return SN_ERR_NULL_ARGUMENT;
    size_t codes_need, scales_need;
    const int rc = cache_need(*cache, &codes_need, &scales_need);
    if (rc != SN_OK) return rc;
    size_t row_count, moved, head_columns, end;
    if (!product(cache->batch, rows->time, &row_count) || !product(cache->kv_heads, cache->head_dim, &head_columns) ||
        !product(row_count, head_columns, &moved) || !sum(rows->position, rows->time, &end))
        return SN_ERR_OVERFLOW;
    if (positions == nullptr && end > cache->capacity) return SN_ERR_SHAPE;
    size_t packed_need = 0;
    if (append) {
        size_t key_end, value_end;
        if (!product(row_count, rows->width, &packed_need) || !sum(rows->key_column, head_columns, &key_end) ||
            !sum(rows->value_column, head_columns, &value_end))
            return SN_ERR_OVERFLOW;
        if (key_end > rows->width || value_end > rows->width) return SN_ERR_SHAPE;
        if (packed_len < packed_need) return SN_ERR_LENGTH_MISMATCH;
    } else if (keys_len < moved || values_len < moved) {
        return SN_ERR_LENGTH_MISMATCH;
    }
    if (positions != nullptr && positions_len < cache->batch) return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    const Bytes buffers[4] = {{k_codes, k_codes_len, codes_need},
                              {k_scales, k_scales_len, scales_need},
                              {v_codes, v_codes_len, codes_need},
                              {v_scales, v_scales_len, scales_need}};
    const int checked = check_buffers(buffers);
    if (checked != SN_OK) return checked;
    if (moved == 0) return SN_OK;
    if (append ? packed == nullptr : keys == nullptr || values == nullptr) return SN_ERR_NULL_ARGUMENT;
    const size_t positions_bytes = cache->batch * sizeof(uint32_t);
    if (append) {
        for (int i = 0; i < 4; ++i) {
            if (overlaps(buffers[i].data, buffers[i].need, packed, packed_need * sizeof(float)) ||
                overlaps(buffers[i].data, buffers[i].need, positions, positions_bytes))
                return SN_ERR_ALIASING;
            for (int j = 0; j < i; ++j)
                if (overlaps(buffers[i].data, buffers[i].need, buffers[j].data, buffers[j].need))
                    return SN_ERR_ALIASING;
        }
    } else {
        const size_t bytes = moved * sizeof(float);
        if (overlaps(keys, bytes, values, bytes) || overlaps(keys, bytes, positions, positions_bytes) ||
            overlaps(values, bytes, positions, positions_bytes))
            return SN_ERR_ALIASING;
        for (const Bytes& b : buffers)
            if (overlaps(keys, bytes, b.data, b.need) || overlaps(values, bytes, b.data, b.need))
                return SN_ERR_ALIASING;
    }
    CacheRowsArgs args;
    args.packed = packed;
    args.keys = keys;
    args.values = values;
    args.positions = positions;
    args.k_codes = const_cast<uint8_t*>(k_codes);
    args.k_scales = const_cast<uint8_t*>(k_scales);
    args.v_codes = const_cast<uint8_t*>(v_codes);
    args.v_scales = const_cast<uint8_t*>(v_scales);
    args.batch = int64_t(cache->batch);
    args.kv_heads = int64_t(cache->kv_heads);
    args.capacity = int64_t(cache->capacity);
    args.head_dim = int64_t(cache->head_dim);
    args.time = int64_t(rows->time);
    args.position = int64_t(rows->position);
    args.width = int64_t(rows->width);
    args.key_column = int64_t(rows->key_column);
    args.value_column = int64_t(rows->value_column);
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = append ? launch_cache_append(args, ctx->stream) : launch_cache_read(args, ctx->stream);
    return status(err);
}

// Floats from the first to past the last of [sequence][head][row] rows of `head_dim`, or false.
bool strided_need(const size_t (&counts)[3], const size_t (&strides)[3], size_t head_dim, size_t* need) {
    *need = head_dim;
    for (int i = 0; i < 3; ++i) {
        size_t span;
        if (!product(counts[i] - 1, strides[i], &span) || !sum(*need, span, need)) return false;
    }
    return true;
}

// Whether the strides nest, each at least what the smaller ones span, so that no two of those rows share an element.
bool nested(const size_t (&counts)[3], const size_t (&strides)[3], size_t head_dim) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return strides[i] < strides[j]; });
    size_t span = head_dim;
    for (int i : order) {
        if (counts[i] <= 1) continue;
        if (strides[i] < span) return false;
        span += (counts[i] - 1) * strides[i];
    }
    return true;
}

}  // namespace

extern "C" {

int sn_alloc_bytes(sn_context* ctx, size_t count, uint8_t** out) {
    if (ctx == nullptr || out == nullptr) return SN_ERR_NULL_ARGUMENT;
    *out = nullptr;
    if (count >= kLimit) return SN_ERR_OVERFLOW;
    float* p = nullptr;
    const int rc = sn_alloc_zeroed(ctx, (count + 3) / 4, &p);
    *out = reinterpret_cast<uint8_t*>(p);
    return rc;
}

int sn_upload_bytes(sn_context* ctx, const uint8_t* host, size_t count, uint8_t** out) {
    if (ctx == nullptr || out == nullptr || (host == nullptr && count > 0)) return SN_ERR_NULL_ARGUMENT;
    *out = nullptr;
    if (count >= kLimit) return SN_ERR_OVERFLOW;
    if (count == 0) return SN_OK;
    hipError_t err = hipSetDevice(ctx->device);
    void* p = nullptr;
    if (err == hipSuccess) err = hipMalloc(&p, count);
    if (err == hipSuccess) err = hipMemcpyAsync(p, host, count, hipMemcpyHostToDevice, ctx->stream);
    if (err == hipSuccess) err = hipStreamSynchronize(ctx->stream);
    if (err != hipSuccess) {
        if (p != nullptr) (void)hipFree(p);
        return status(err);
    }
    *out = static_cast<uint8_t*>(p);
    return SN_OK;
}

int sn_download_bytes(sn_context* ctx, const uint8_t* device, size_t count, uint8_t* host) {
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (count == 0) return SN_OK;
    if (device == nullptr || host == nullptr) return SN_ERR_NULL_ARGUMENT;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = hipMemcpyAsync(host, device, count, hipMemcpyDeviceToHost, ctx->stream);
    if (err == hipSuccess) err = hipStreamSynchronize(ctx->stream);
    return status(err);
}

int sn_free_bytes(sn_context* ctx, uint8_t* buffer) { return sn_free(ctx, reinterpret_cast<float*>(buffer)); }

int sn_fp4_sizes(size_t rows, size_t inner, size_t* codes_bytes, size_t* scales_bytes) {
    if (codes_bytes == nullptr || scales_bytes == nullptr) return SN_ERR_NULL_ARGUMENT;
    *codes_bytes = *scales_bytes = 0;
    const size_t blocks = inner / SN_FP4_BLOCK + (inner % SN_FP4_BLOCK != 0);
    size_t scales, codes;
    if (!product(rows, blocks, &scales) || !product(scales, SN_FP4_BLOCK / 2, &codes)) return SN_ERR_OVERFLOW;
    *codes_bytes = codes;
    *scales_bytes = scales;
    return SN_OK;
}

int sn_quantize_fp4(sn_context* ctx, size_t cols, size_t inner, uint32_t storage, const float* source,
                    size_t source_len, uint8_t* codes, size_t codes_len, uint8_t* scales, size_t scales_len) {
    return weight_call(ctx, true, cols, inner, storage, source, source_len, codes, codes_len, scales, scales_len);
}

int sn_dequantize_fp4(sn_context* ctx, size_t cols, size_t inner, uint32_t storage, const uint8_t* codes,
                      size_t codes_len, const uint8_t* scales, size_t scales_len, float* output, size_t output_len) {
    return weight_call(ctx, false, cols, inner, storage, output, output_len, codes, codes_len, scales, scales_len);
}

int sn_matmul_fp4(sn_context* ctx, const sn_matmul_spec* spec, const float* left, size_t left_len,
                  const uint8_t* codes, size_t codes_len, const uint8_t* scales, size_t scales_len,
                  const float* bias, size_t bias_len, float* output, size_t output_len) {
    // The right operand's elements are counted as sn_matmul counts them, its bytes below.
    const int rc = sn_matmul_validate(spec, left_len, SIZE_MAX, output_len);
    if (rc != SN_OK) return rc;
    if (spec->left_storage != SN_ROW_MAJOR || spec->right_storage != SN_TRANSPOSED || spec->batch_count != 1 ||
        spec->mask != SN_MASK_NONE)
        return SN_ERR_UNSUPPORTED;
    size_t codes_need, scales_need;
    if (sn_fp4_sizes(spec->cols, spec->inner, &codes_need, &scales_need) != SN_OK || spec->inner >= kMaxInner ||
        spec->cols >= kMaxCols)
        return SN_ERR_OVERFLOW;
    if (codes_len < codes_need || scales_len < scales_need) return SN_ERR_RIGHT_TOO_SMALL;
    if (bias != nullptr && bias_len != spec->cols) return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (spec->rows == 0 || spec->cols == 0) return SN_OK;
    const size_t left_bytes = spec->rows * spec->inner * sizeof(float);
    const size_t output_bytes = spec->rows * spec->cols * sizeof(float);
    if (output == nullptr || (spec->inner > 0 && (left == nullptr || codes == nullptr || scales == nullptr)))
        return SN_ERR_NULL_ARGUMENT;
    if (!aligned16(codes)) return SN_ERR_UNSUPPORTED;
    if (overlaps(output, output_bytes, left, left_bytes) || overlaps(output, output_bytes, codes, codes_need) ||
        overlaps(output, output_bytes, scales, scales_need) ||
        overlaps(output, output_bytes, bias, bias_len * sizeof(float)))
        return SN_ERR_ALIASING;
    ProductArgs args;
    args.x = left;
    args.codes = codes;
    args.scales = scales;
    args.bias = bias;
    args.y = output;
    args.rows = int64_t(spec->rows);
    args.cols = int64_t(spec->cols);
    args.inner = int64_t(spec->inner);
    args.blocks = blocks_of(args.inner);
    args.scale = spec->scale;
    args.accumulate = spec->write == SN_ACCUMULATE;
    args.bf16 = sn::kernel_for(ctx->kernel, spec->precision) == SN_KERNEL_MFMA_BF16;
    args.workspace = ctx->env.workspace;
    args.workspace_bytes = ctx->env.workspace_bytes;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = launch_product(args, ctx->stream);
    return status(err);
}

int sn_fp4_cache_append(sn_context* ctx, const sn_fp4_cache_shape* cache, const sn_fp4_cache_rows* rows,
                        const float* packed, size_t packed_len, const uint32_t* positions, size_t positions_len,
                        uint8_t* k_codes, size_t k_codes_len, uint8_t* k_scales, size_t k_scales_len,
                        uint8_t* v_codes, size_t v_codes_len, uint8_t* v_scales, size_t v_scales_len) {
    return cache_rows_call(ctx, true, cache, rows, packed, packed_len, positions, positions_len, k_codes, k_codes_len,
                           k_scales, k_scales_len, v_codes, v_codes_len, v_scales, v_scales_len, nullptr, 0, nullptr,
                           0);
}

int sn_fp4_cache_read(sn_context* ctx, const sn_fp4_cache_shape* cache, const sn_fp4_cache_rows* rows,
                      const uint8_t* k_codes, size_t k_codes_len, const uint8_t* k_scales, size_t k_scales_len,
                      const uint8_t* v_codes, size_t v_codes_len, const uint8_t* v_scales, size_t v_scales_len,
                      const uint32_t* positions, size_t positions_len, float* keys, size_t keys_len, float* values,
                      size_t values_len) {
    return cache_rows_call(ctx, false, cache, rows, nullptr, 0, positions, positions_len, k_codes, k_codes_len,
                           k_scales, k_scales_len, v_codes, v_codes_len, v_scales, v_scales_len, keys, keys_len,
                           values, values_len);
}

int sn_fp4_attention(sn_context* ctx, const sn_fp4_cache_shape* cache, const sn_fp4_attention_shape* shape,
                     const float* q, size_t q_len, const uint8_t* k_codes, size_t k_codes_len,
                     const uint8_t* k_scales, size_t k_scales_len, const uint8_t* v_codes, size_t v_codes_len,
                     const uint8_t* v_scales, size_t v_scales_len, const uint32_t* lengths, size_t lengths_len,
                     float* out, size_t out_len) {
    if (cache == nullptr || shape == nullptr) return SN_ERR_NULL_ARGUMENT;
    const sn_fp4_attention_shape& s = *shape;
    size_t codes_need, scales_need;
    const int rc = cache_need(*cache, &codes_need, &scales_need);
    if (rc != SN_OK) return rc;
    if (cache->kv_heads == 0 ? s.heads != 0 : s.heads % cache->kv_heads != 0) return SN_ERR_SHAPE;
    if (lengths == nullptr && s.keys > cache->capacity) return SN_ERR_SHAPE;
    size_t head_rows, all_rows;
    if (!product(s.heads, s.queries, &head_rows) || !product(cache->batch, head_rows, &all_rows) ||
        all_rows >= kMaxRows)
        return SN_ERR_OVERFLOW;
    const size_t counts[3] = {cache->batch, s.heads, s.queries};
    const size_t q_strides[3] = {s.q_sequence, s.q_head, s.q_row};
    const size_t out_strides[3] = {s.out_sequence, s.out_head, s.out_row};
    size_t q_need = 0, out_need = 0;
    if (all_rows > 0 && (!strided_need(counts, q_strides, cache->head_dim, &q_need) ||
                         !strided_need(counts, out_strides, cache->head_dim, &out_need)))
        return SN_ERR_OVERFLOW;
    if (q_len < q_need || out_len < out_need) return SN_ERR_LENGTH_MISMATCH;
    if (lengths != nullptr && lengths_len < cache->batch) return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    const Bytes buffers[4] = {{k_codes, k_codes_len, codes_need},
                              {k_scales, k_scales_len, scales_need},
                              {v_codes, v_codes_len, codes_need},
                              {v_scales, v_scales_len, scales_need}};
    const int checked = check_buffers(buffers);
    if (checked != SN_OK) return checked;
    if (all_rows == 0) return SN_OK;
    if (q == nullptr || out == nullptr) return SN_ERR_NULL_ARGUMENT;
    const size_t out_bytes = out_need * sizeof(float);
    if (!nested(counts, out_strides, cache->head_dim) || overlaps(out, out_bytes, q, q_need * sizeof(float)) ||
        overlaps(out, out_bytes, lengths, cache->batch * sizeof(uint32_t)))
        return SN_ERR_ALIASING;
    for (const Bytes& b : buffers)
        if (overlaps(out, out_bytes, b.data, b.need)) return SN_ERR_ALIASING;
    AttentionArgs args;
    args.q = q;
    args.k_codes = k_codes;
    args.k_scales = k_scales;
    args.v_codes = v_codes;
    args.v_scales = v_scales;
    args.lengths = lengths;
    args.out = out;
    args.batch = int64_t(cache->batch);
    args.heads = int64_t(s.heads);
    args.kv_heads = int64_t(cache->kv_heads);
    args.capacity = int64_t(cache->capacity);
    args.head_dim = int64_t(cache->head_dim);
    args.queries = int64_t(s.queries);
    args.keys = int64_t(s.keys);
    args.q_sequence = int64_t(s.q_sequence);
    args.q_head = int64_t(s.q_head);
    args.q_row = int64_t(s.q_row);
    args.out_sequence = int64_t(s.out_sequence);
    args.out_head = int64_t(s.out_head);
    args.out_row = int64_t(s.out_row);
    args.scale = s.scale;
    args.workspace = ctx->env.workspace;
    args.workspace_bytes = ctx->env.workspace_bytes;
    args.counters = ctx->env.counters;
    args.counter_count = ctx->env.counter_count;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = launch_attention(args, ctx->stream);
    return status(err);
}

}  // extern "C"
