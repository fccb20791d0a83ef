/*
 * staleynet_norm.h — the residual stream's addition and root-mean-square norm
 * ahead of each Linear, with an output in 32 or 8 bits, and its gradients: part
 * of libstaleynet_gemm.so, in the manner of staleynet_gemm.h. The reference
 * norms and adds in kernels of their own
 * (crates/staleynet-model/src/layers/block.rs:160-189); here a block's addition, the
 * norm after it and the rounding for an 8-bit product (staleynet_fp8.h) are
 * one pass over the row.
 *
 * For each row of `width` values:
 *   s = x + residual                       (rounded to fp32; s = x without one)
 *   i = 1 / sqrt(mean(s^2) + epsilon)
 *   y = weight * s * i                     (computed in 64 bits, rounded once)
 * NaN and infinities follow IEEE arithmetic, and stay in their row. Rows are
 * dense, [rows, width]. epsilon is at least 0 and finite (SN_ERR_UNSUPPORTED
 * otherwise). Nothing is written where rows or width is 0. Limits, past which a
 * call is SN_ERR_OVERFLOW: rows under 2^31, width under 2^25. Lengths count
 * elements of their buffer (too short: SN_ERR_LENGTH_MISMATCH). The calls are
 * asynchronous on the context's stream, allocate nothing, may be captured into a
 * graph, and are deterministic.
 */
#ifndef STALEYNET_NORM_H
#define STALEYNET_NORM_H

#include "staleynet_fp8.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct sn_rms_norm_shape {
    size_t rows;
    size_t width;
    float epsilon;
} sn_rms_norm_shape;

/* out = y. residual null: none. sum (s, for the next block's addition and the
 * backward) and inverse (i, one a row, rounded to fp32, for the backward) are
 * written where given. sum may be x or residual itself, the stream updated in
 * place; any other overlap of an output with an input or another output is
 * SN_ERR_ALIASING. */
int sn_rms_norm(sn_context *context, const sn_rms_norm_shape *shape, const float *x, size_t x_len,
                const float *residual, size_t residual_len, const float *weight, size_t weight_len, float *sum,
                size_t sum_len, float *out, size_t out_len, float *inverse, size_t inverse_len);

/* The same with y rounded to 8-bit rows, the left operand of sn_matmul_fp8:
 * the bits that sn_quantize_fp8 would give of sn_rms_norm's output. It leaves no
 * inverse: a step that goes back through the norm has it from sn_rms_norm. */
int sn_rms_norm_fp8(sn_context *context, const sn_rms_norm_shape *shape, const float *x, size_t x_len,
                    const float *residual, size_t residual_len, const float *weight, size_t weight_len, float *sum,
                    size_t sum_len, uint8_t *codes, size_t codes_len, uint8_t *scales, size_t scales_len);

/* The gradients, from s and i as the forward left them and the gradient d_out
 * of y, with g = weight * d_out and n = s * i:
 *   d_x = d_sum + i * (g - n * mean(g * n))
 *   d_weight += sum over rows of d_out * n
 * d_sum (null: none) is the gradient that reaches s past the norm, along the
 * residual stream; d_x is the gradient of x and of the residual alike. d_weight
 * null: only d_x. d_x may be d_sum itself; any other overlap is
 * SN_ERR_ALIASING. epsilon is not used. Partial sums of d_weight go through the
 * context's workspace (so calls on one context must not overlap); its bits
 * depend on the workspace's size. */
int sn_rms_norm_backward(sn_context *context, const sn_rms_norm_shape *shape, const float *sum, size_t sum_len,
                         const float *inverse, size_t inverse_len, const float *weight, size_t weight_len,
                         const float *d_out, size_t d_out_len, const float *d_sum, size_t d_sum_len, float *d_x,
                         size_t d_x_len, float *d_weight, size_t d_weight_len);

#ifdef __cplusplus
}
#endif

#endif /* STALEYNET_NORM_H */
