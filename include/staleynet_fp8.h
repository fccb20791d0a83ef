/*
 * staleynet_fp8.h — products of 8-bit operands: part of libstaleynet_gemm.so,
 * beside the fp32 entry points of staleynet_gemm.h and the 4-bit ones of
 * staleynet_fp4.h and in their manner. None has a counterpart in the reference;
 * they are the 8-bit forms of sn_matmul / sn_matmul_bias, for prompts and
 * decode steps as for the three products of a training step.
 *
 * The format: 8-bit floats in blocks of 128 along a row, each block with a
 * scale byte. A code is e4m3 of the OCP 8-bit formats: sign (bit 7), four
 * exponent bits of bias 7, three mantissa bits; no infinities, 0x7F and 0xFF
 * are NaN, the largest value is 448 and the smallest 2^-9. A row's codes are
 * contiguous, one byte each, and padded with zeros to a multiple of 128. Its
 * scale bytes follow each other at [row][block] of a second buffer, each row's
 * padded to a multiple of 4. A byte s is a factor of 2^(s - 127), s = 3 ..
 * 246: one under 3 stands for 3, and a block with one over 246 holds NaN in
 * every place. 8.06 bits a value.
 *
 * Rounding to it (sn_quantize_fp8, sn_rms_norm_fp8): the block's factor is the
 * smallest power of two of which its largest magnitude is at most 464 (which
 * rounds to 448, off by half a step), kept within 2^-124 .. 2^119; values are
 * rounded to the nearest code, ties to the even code, past 448 factors to 448,
 * and keep their sign (also of zero). A block of zeros has s = 3; one with an
 * infinity or NaN has s = 255 and codes 0.
 *
 * Limits, past which a call is SN_ERR_OVERFLOW: rows and inner length of a
 * matrix to quantize under 2^31; of a product, rows under 2^28, columns under
 * 2^24, inner length under 2^23, and tiles of 256 x 256 outputs under 2^24.
 *
 * Buffers are bytes in device memory (sn_alloc_bytes of staleynet_fp4.h, or any
 * other). Code buffers are 16-byte aligned and scale buffers 4-byte aligned
 * (SN_ERR_UNSUPPORTED otherwise). The calls are asynchronous on the context's
 * stream, allocate nothing and may be captured into a graph.
 */
#ifndef STALEYNET_FP8_H
#define STALEYNET_FP8_H

#include "staleynet_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Values of one block. */
#define SN_FP8_BLOCK 128u

/* Bytes of the codes and of the scales of `rows` rows of `inner` values:
 * with b = ceil(inner / 128), rows * b * 128 and rows * 4 * ceil(b / 4).
 * SN_ERR_OVERFLOW where they do not fit. */
int sn_fp8_sizes(size_t rows, size_t inner, size_t *codes_bytes, size_t *scales_bytes);

/* An operand as `rows` rows of the format with `inner` values each: element
 * (r, k) is at r * inner + k of the source (SN_ROW_MAJOR: activations before a
 * product), or at k * rows + r (SN_TRANSPOSED: the columns of a weight as
 * Linear keeps it, [inner, rows]; or both operands of a weight's gradient).
 * The padding is written too. source_len counts floats
 * (SN_ERR_RIGHT_TOO_SMALL), the others bytes (SN_ERR_OUTPUT_TOO_SMALL). */
int sn_quantize_fp8(sn_context *context, size_t rows, size_t inner, uint32_t storage, const float *source,
                    size_t source_len, uint8_t *codes, size_t codes_len, uint8_t *scales, size_t scales_len);
/* The values the codes stand for, stored as `storage` says (exact). */
int sn_dequantize_fp8(sn_context *context, size_t rows, size_t inner, uint32_t storage, const uint8_t *codes,
                      size_t codes_len, const uint8_t *scales, size_t scales_len, float *output, size_t output_len);

/* The product of sn_matmul with both operands in the format, and the bias of
 * sn_matmul_bias (null: none):
 *   output = scale * X W (+ output, SN_ACCUMULATE) (+ bias per column)
 * X [rows, inner] as `rows` rows of the format, W [inner, cols] as `cols` rows,
 * one per column. The spec is sn_matmul's: left_storage SN_ROW_MAJOR,
 * right_storage SN_TRANSPOSED (each column's values are contiguous),
 * batch_count 1, no mask (SN_ERR_UNSUPPORTED otherwise); its precision changes
 * nothing. Products of codes and factors are exact and summed in fp32.
 * Infinities and NaN follow IEEE arithmetic. Deterministic; a row's bits do not
 * depend on the values of the other rows. An operand's buffers too short are
 * SN_ERR_LEFT_TOO_SMALL or SN_ERR_RIGHT_TOO_SMALL, the rest as
 * sn_matmul_bias. Products whose output is too small to fill the GPU slice the
 * inner dimension, with partial sums in the context's workspace (so calls on
 * one context must not overlap); with a smaller workspace they slice less, or
 * not. */
int sn_matmul_fp8(sn_context *context, const sn_matmul_spec *spec, const uint8_t *left_codes, size_t left_codes_len,
                  const uint8_t *left_scales, size_t left_scales_len, const uint8_t *right_codes,
                  size_t right_codes_len, const uint8_t *right_scales, size_t right_scales_len, const float *bias,
                  size_t bias_len, float *output, size_t output_len);

#ifdef __cplusplus
}
#endif

#endif /* STALEYNET_FP8_H */
