/*
 * staleynet_logprobs.h — log probabilities of given tokens, with the entropy
 * and the likeliest alternatives, and their gradient: part of
 * libstaleynet_gemm.so, in the manner of staleynet_gemm.h. They stand beside
 * sn_cross_entropy, for scoring answers and for losses of a policy's own
 * samples, and take all of a row's classifiers in one call (the reference's
 * codebook heads, crates/staleynet-model/src/training.rs:208-239, or one
 * vocabulary).
 *
 * For each row and head, over the head's classes c with logits x, their largest
 * m, and the scale a (an inverse temperature):
 *   z_c = a (x_c - m),  T = log(sum of e^(z_c)),  log p_c = z_c - T
 *   logprob = log p_token,  entropy = H = -sum of p_c log p_c
 * A logit of -inf has probability 0 and adds nothing to H, and so has one that
 * is further below m than fp32 reaches. A row of a head with a NaN or +inf, or
 * without a finite logit, gives NaN in all but the top tokens, an empty token's
 * log probability (0) and the places past the classes. Sums are fp32; T is
 * log(1 + the sum without the largest term), so that log probabilities and
 * entropies near 0 keep their digits.
 */
#ifndef STALEYNET_LOGPROBS_H
#define STALEYNET_LOGPROBS_H

#include "staleynet_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Logits [rows, cols]: head h owns the `classes` columns from column_offset + h *
 * classes on (SN_ERR_SHAPE where they run past a row; classes at least 1 where
 * there are heads). Token h of a row is at row * token_stride + token_offset + h.
 * top: alternatives to list, at most 32 (SN_ERR_UNSUPPORTED otherwise, as is a
 * scale that is not positive and finite). rows * heads is under 2^31, classes
 * under 2^30, rows * cols under 2^40 (SN_ERR_OVERFLOW). */
typedef struct sn_logprob_shape {
    size_t rows;
    size_t cols;
    size_t column_offset;
    size_t classes;
    size_t heads;
    size_t token_stride;
    size_t token_offset;
    size_t top;
    float scale;
} sn_logprob_shape;

#define SN_LOGPROBS_LARGEST_TOP 32u

/* The forward. tokens are device memory (sn_upload_tokens), or null with
 * logprobs null. An empty token (SN_EMPTY_TOKEN) has log probability 0; one that
 * is no class, NaN. Outputs, each null where it is not wanted: logprobs and
 * entropies [rows][heads]; stats [rows][heads][2], {m, T}, for the backward;
 * top_tokens and top_logprobs [rows][heads][top], the classes of the largest
 * logits in falling order, equal ones by class, NaN ahead of all; places past
 * the classes hold SN_EMPTY_TOKEN and -inf. Buffers too short are
 * SN_ERR_LENGTH_MISMATCH, outputs that overlap an input or each other
 * SN_ERR_ALIASING. Asynchronous on the context's stream, allocates nothing, may
 * be captured, deterministic. Few rows of many classes are split over
 * workgroups, with partial results in the context's workspace (so calls on one
 * context must not overlap); with a smaller workspace they are split less, or
 * not. */
int sn_token_logprobs(sn_context *context, const sn_logprob_shape *shape, const float *logits, size_t logits_len,
                      const uint32_t *tokens, size_t tokens_len, float *logprobs, size_t logprobs_len,
                      float *entropies, size_t entropies_len, float *stats, size_t stats_len, uint32_t *top_tokens,
                      size_t top_tokens_len, float *top_logprobs, size_t top_logprobs_len);

/* The gradient of the logits, from the forward's stats and the gradients of its
 * log probabilities and entropies [rows][heads] (either null: none; entropies,
 * the forward's, go with d_entropies):
 *   grad_c = a (d_logprob ([c = token] - p_c) - d_entropy p_c (log p_c + H))
 * written to the heads' columns of grad [rows, cols]; other columns are left
 * alone. An empty token has no d_logprob term, one that is no class no [c =
 * token] term. A place with no d_logprob term (an empty token, or no
 * d_logprobs) and no d_entropy, or one of 0, has gradient 0 whatever its
 * logits; else a head with a NaN or +inf, or without a finite logit, has NaN.
 * tokens may be null without d_logprobs. grad may be logits itself; any other
 * overlap is SN_ERR_ALIASING. `top` is not used. */
int sn_token_logprobs_backward(sn_context *context, const sn_logprob_shape *shape, const float *logits,
                               size_t logits_len, const uint32_t *tokens, size_t tokens_len, const float *stats,
                               size_t stats_len, const float *entropies, size_t entropies_len,
                               const float *d_logprobs, size_t d_logprobs_len, const float *d_entropies,
                               size_t d_entropies_len, float *grad, size_t grad_len);

#ifdef __cplusplus
}
#endif

#endif /* STALEYNET_LOGPROBS_H */
