/*
 * staleynet_fp4.h — serving with 4-bit weights and a 4-bit key/value cache:
 * part of libstaleynet_gemm.so, beside the fp32 entry points of
 * staleynet_gemm.h and in their manner (status codes, contexts, streams,
 * lengths checked on the host). None has a counterpart in the reference,
 * whose decode (crates/staleynet-model/src/decode.rs:64-161) reads fp32
 * weights and an fp32 cache; they are the 4-bit forms of sn_matmul /
 * sn_matmul_bias, sn_split_heads into a cache and sn_causal_attention.
 *
 * The format: 4-bit floats in blocks of 32 along a row (the OCP Microscaling
 * format with e2m1 elements and e8m0 scales). A code is sign (bit 3), two
 * exponent bits and a mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
 * negatives. Two codes to a byte, the lower index in the low half; a block's
 * 16 bytes are contiguous, a row's blocks follow each other, and the last is
 * padded with zeros where a row's length is no multiple of 32. Each block has
 * one scale byte s, a factor of 2^(s - 127), at [row][block] of a second
 * buffer. s = 0 .. 252; a block with s over 252 holds NaN in every place
 * (the format's own NaN is 255; 253 and 254 would pass fp32's range).
 * 4.25 bits a value.
 *
 * Rounding to it (sn_quantize_fp4, sn_fp4_cache_append): the block's factor is
 * the smallest power of two of which its largest magnitude is less than 7 (so
 * that rounding it to 6 is off by at most half a step), kept within 2^-127 ..
 * 2^125; values are rounded to the nearest code, ties to the even code, and
 * keep their sign (also of zero). A block of zeros has s = 0; one with an
 * infinity or NaN has s = 255 and codes 0.
 *
 * Limits, past which a call is SN_ERR_OVERFLOW: columns and inner length of a
 * matrix to quantize under 2^31; of a product, columns under 2^28 and inner
 * length under 2^25; a cache's batch * kv_heads under 2^21 and its capacity
 * under 2^30; batch * heads * queries of an attention call under 2^27.
 *
 * Buffers are bytes in device memory (sn_alloc_bytes, sn_upload_bytes, or any
 * other). Code buffers are 16-byte aligned (SN_ERR_UNSUPPORTED otherwise).
 * The calls on them are asynchronous on the context's stream, allocate nothing
 * and may be captured into a graph; those that make, copy and free them are as
 * their fp32 forms.
 */
#ifndef STALEYNET_FP4_H
#define STALEYNET_FP4_H

#include "staleynet_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Values of one block. */
#define SN_FP4_BLOCK 32u

/* ---- byte buffers ---------------------------------------------------------- */
/* As sn_alloc_zeroed, sn_upload, sn_download and sn_free, for bytes. */
int sn_alloc_bytes(sn_context *context, size_t count, uint8_t **out);
int sn_upload_bytes(sn_context *context, const uint8_t *host, size_t count, uint8_t **out);
int sn_download_bytes(sn_context *context, const uint8_t *device, size_t count, uint8_t *host);
int sn_free_bytes(sn_context *context, uint8_t *buffer);

/* Bytes of the codes and of the scales of `rows` rows of `inner` values:
 * rows * ceil(inner / 32) * 16 and rows * ceil(inner / 32). SN_ERR_OVERFLOW
 * where they do not fit. */
int sn_fp4_sizes(size_t rows, size_t inner, size_t *codes_bytes, size_t *scales_bytes);

/* ---- weights ---------------------------------------------------------------- */
/* A product's right operand [inner, cols], stored as `storage` says
 * (SN_ROW_MAJOR: element (k, c) at k * cols + c, as Linear keeps its weight;
 * SN_TRANSPOSED: at c * inner + k), rounded to 4 bits: one row of the format per
 * column c, its `inner` values in order. source_len counts floats
 * (SN_ERR_RIGHT_TOO_SMALL), the others bytes (SN_ERR_OUTPUT_TOO_SMALL). */
int sn_quantize_fp4(sn_context *context, size_t cols, size_t inner, uint32_t storage, const float *source,
                    size_t source_len, uint8_t *codes, size_t codes_len, uint8_t *scales, size_t scales_len);
/* The values the codes stand for, as that operand (exact). */
int sn_dequantize_fp4(sn_context *context, size_t cols, size_t inner, uint32_t storage, const uint8_t *codes,
                      size_t codes_len, const uint8_t *scales, size_t scales_len, float *output, size_t output_len);

/* The product of sn_matmul with a 4-bit right operand, and the bias of
 * sn_matmul_bias (null: none):
 *   output = scale * left * W (+ output, SN_ACCUMULATE) (+ bias per column)
 * left [rows, inner] row-major fp32, W [inner, cols] as sn_quantize_fp4 leaves
 * it. The spec is sn_matmul's: left_storage SN_ROW_MAJOR, right_storage
 * SN_TRANSPOSED (each column's values are contiguous), batch_count 1, no mask
 * (SN_ERR_UNSUPPORTED otherwise). The left operand's fp32 values are used in
 * full, subnormals too, as the exact sum of three bf16 values and of what those leave of
 * values under 2^-110 (SN_PRECISION_F32, and the
 * default with every context kernel but SN_KERNEL_MFMA_BF16), or rounded to
 * bf16 (SN_PRECISION_BF16, or that kernel); products are exact and summed in
 * fp32. Infinities and NaN follow IEEE arithmetic. Deterministic; a row's bits
 * do not depend on the values of the other rows. Lengths and codes as
 * sn_matmul_bias; codes or scales too short is SN_ERR_RIGHT_TOO_SMALL. Products
 * of more than 16 rows (32 rounded to bf16) whose output is too small to fill the GPU slice the inner
 * dimension, with partial sums in the context's workspace (so calls on one
 * context must not overlap); with a smaller workspace they slice less, or not. */
int sn_matmul_fp4(sn_context *context, const sn_matmul_spec *spec, const float *left, size_t left_len,
                  const uint8_t *codes, size_t codes_len, const uint8_t *scales, size_t scales_len,
                  const float *bias, size_t bias_len, float *output, size_t output_len);

/* ---- the key/value cache --------------------------------------------------- */
/* A cache of keys and values: per buffer [batch][kv_heads][capacity] rows of
 * head_dim values (32, 64 or 128; SN_ERR_UNSUPPORTED otherwise), that is
 * head_dim / 2 bytes of codes and head_dim / 32 of scales a row. */
typedef struct sn_fp4_cache_shape {
    size_t batch;
    size_t kv_heads;
    size_t capacity;
    size_t head_dim;
} sn_fp4_cache_shape;

/* `time` consecutive positions of each sequence, from positions[sequence] on
 * (device memory) where an array is given, else from `position` on; and where
 * the packed rows [batch * time, width] hold them: head h of the keys at columns
 * key_column + h * head_dim .., of the values at value_column + h * head_dim. */
typedef struct sn_fp4_cache_rows {
    size_t time;
    size_t position;
    size_t width;
    size_t key_column;
    size_t value_column;
} sn_fp4_cache_rows;

/* sn_split_heads of the keys and of the values into a cache at an offset, in
 * one call and rounded to 4 bits. A position past the capacity is not written
 * where it comes from `positions`; with `position`, time + position over the
 * capacity is SN_ERR_SHAPE, as are heads that run past a packed row. Lengths in
 * elements of their buffer: packed rows, positions, codes or scales too short is
 * SN_ERR_LENGTH_MISMATCH. */
int sn_fp4_cache_append(sn_context *context, const sn_fp4_cache_shape *cache, const sn_fp4_cache_rows *rows,
                        const float *packed, size_t packed_len, const uint32_t *positions, size_t positions_len,
                        uint8_t *k_codes, size_t k_codes_len, uint8_t *k_scales, size_t k_scales_len,
                        uint8_t *v_codes, size_t v_codes_len, uint8_t *v_scales, size_t v_scales_len);

/* The values held at those positions: keys and values [batch][kv_heads][time]
 * [head_dim], exact (rows->width and the columns are not used). Places of
 * positions past the capacity are set to 0. */
int sn_fp4_cache_read(sn_context *context, const sn_fp4_cache_shape *cache, const sn_fp4_cache_rows *rows,
                      const uint8_t *k_codes, size_t k_codes_len, const uint8_t *k_scales, size_t k_scales_len,
                      const uint8_t *v_codes, size_t v_codes_len, const uint8_t *v_scales, size_t v_scales_len,
                      const uint32_t *positions, size_t positions_len, float *keys, size_t keys_len,
                      float *values, size_t values_len);

/* ---- attention over that cache ---------------------------------------------- */
/* `heads` query heads of every sequence, a multiple of the cache's kv_heads
 * (head h reads key/value head h / (heads / kv_heads); SN_ERR_SHAPE otherwise),
 * `queries` of each. Query t of head h of sequence b is the head_dim floats at b *
 * q_sequence + h * q_head + t * q_row, its output at b * out_sequence + h *
 * out_head + t * out_row: columns of packed rows (row = the width, head =
 * head_dim) or head-major matrices (head = queries * head_dim, row = head_dim).
 * Sequence b holds n = lengths[b] positions (device memory) where an array is
 * given, else `keys`, at most the capacity; its queries are the last of them:
 * query t sees positions 0 ..= n - queries + t. */
typedef struct sn_fp4_attention_shape {
    size_t heads;
    size_t queries;
    size_t keys;
    size_t q_sequence;
    size_t q_head;
    size_t q_row;
    size_t out_sequence;
    size_t out_head;
    size_t out_row;
    float scale;
} sn_fp4_attention_shape;

/* out = softmax(scale * q K^T) V per query over the positions it sees, the
 * 4-bit form of sn_causal_attention (decode step and prompt chunk alike). A
 * query that sees no position (a sequence of length 0; padding ahead of a
 * shorter prompt) gives zeros; one whose scores are all -inf gives NaN. Positions a query does not see do not enter its
 * result, whatever they hold (also NaN blocks). fp32 arithmetic as in
 * sn_matmul_fp4: q times scale log2 e is rounded to fp32, and that is used in full, subnormals
 * too. Values are summed with weights of up to 2^8, their sum divided by the weights' at the end: where the
 * number of positions times the largest |value| passes 2^119, sums may overflow to infinities and NaN. A weight
 * under 2^-118 of the query's largest may count as 0. lengths over the capacity count as the capacity; `keys` over
 * it is SN_ERR_SHAPE. Buffers too short for the strides are SN_ERR_LENGTH_MISMATCH; out
 * overlapping q, the cache or the lengths is SN_ERR_ALIASING, and so are out strides that do
 * not nest: sorted, each has to be at least what the smaller ones span (head_dim floats and the
 * steps by them; strides of counts of one are not used), so that no two outputs share memory.
 * Strides that interleave without sharing are refused as well. Long caches are split over
 * workgroups whose partial results go through the context's workspace and are merged in a fixed
 * order, so calls on one context must not overlap; with a smaller workspace they are split
 * less, or not. Deterministic. */
int sn_fp4_attention(sn_context *context, const sn_fp4_cache_shape *cache, const sn_fp4_attention_shape *shape,
                     const float *q, size_t q_len, const uint8_t *k_codes, size_t k_codes_len,
                     const uint8_t *k_scales, size_t k_scales_len, const uint8_t *v_codes, size_t v_codes_len,
                     const uint8_t *v_scales, size_t v_scales_len, const uint32_t *lengths, size_t lengths_len,
                     float *out, size_t out_len);

#ifdef __cplusplus
}
#endif

#endif /* STALEYNET_FP4_H */
