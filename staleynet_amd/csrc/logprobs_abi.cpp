// The C ABI of the log probabilities (include/staleynet_logprobs.h): checks of
// the arguments, then the kernels of logprobs.hip on the context's stream.
#include "staleynet_logprobs.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "abi_checks.h"
#include "context_internal.h"
#include "logprobs_internal.h"

// The struct's layout is part of the ABI (x86-64 / aarch64 LP64).
static_assert(sizeof(sn_logprob_shape) == 72 && offsetof(sn_logprob_shape, top) == 56 &&
                  offsetof(sn_logprob_shape, scale) == 64,
              "sn_logprob_shape layout");

namespace {

using namespace sn::abi;

constexpr size_t kMaxHeads = size_t(1) << 31;    // over the rows
constexpr size_t kMaxClasses = size_t(1) << 30;
constexpr size_t kMaxLogits = size_t(1) << 40;   // of a call: the kernels count chunks of them in 32 bits

struct Needs {
    size_t logits, places, tokens;
};

int check_shape(const sn_logprob_shape* shape, bool tokens, Needs* need) {
    if (shape == nullptr) return SN_ERR_NULL_ARGUMENT;
    const sn_logprob_shape& s = *shape;
    size_t columns, end;
    if (!product(s.rows, s.cols, &need->logits) || !product(s.rows, s.heads, &need->places) ||
        need->logits >= kMaxLogits || need->places >= kMaxHeads || s.classes >= kMaxClasses ||
        !product(s.heads, s.classes, &columns) || !sum(columns, s.column_offset, &end))
        return SN_ERR_OVERFLOW;
    if (end > s.cols || (s.heads > 0 && s.classes == 0)) return SN_ERR_SHAPE;
    if (s.top > SN_LOGPROBS_LARGEST_TOP || !(s.scale > 0.f) || !std::isfinite(s.scale)) return SN_ERR_UNSUPPORTED;
    need->tokens = 0;
    if (tokens && need->places > 0) {
        size_t span;
        if (!product(s.rows - 1, s.token_stride, &span) || !sum(span, s.token_offset, &span) ||
            !sum(span, s.heads, &need->tokens))
            return SN_ERR_OVERFLOW;
    }
    return SN_OK;
}

}  // namespace

extern "C" {

int sn_token_logprobs(sn_context* ctx, const sn_logprob_shape* shape, const float* logits, size_t logits_len,
                      const uint32_t* tokens, size_t tokens_len, float* logprobs, size_t logprobs_len,
                      float* entropies, size_t entropies_len, float* stats, size_t stats_len, uint32_t* top_tokens,
                      size_t top_tokens_len, float* top_logprobs, size_t top_logprobs_len) {
    Needs need;
    const int rc = check_shape(shape, logprobs != nullptr, &need);
    if (rc != SN_OK) return rc;
    size_t listed;
    if (!product(need.places, shape->top, &listed)) return SN_ERR_OVERFLOW;
    if (logits_len < need.logits || (logprobs != nullptr && (tokens_len < need.tokens || logprobs_len < need.places)) ||
        (entropies != nullptr && entropies_len < need.places) || (stats != nullptr && stats_len / 2 < need.places) ||
        (top_tokens != nullptr && top_tokens_len < listed) || (top_logprobs != nullptr && top_logprobs_len < listed))
        return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (need.places == 0) return SN_OK;
    if (logits == nullptr || (logprobs != nullptr && tokens == nullptr)) return SN_ERR_NULL_ARGUMENT;
    const size_t places = need.places * sizeof(float);
    const Span inputs[] = {{logits, need.logits * sizeof(float)}, {tokens, need.tokens * sizeof(uint32_t)}};
    const Span outputs[] = {{logprobs, places},
                            {entropies, places},
                            {stats, 2 * places},
                            {top_tokens, listed * sizeof(uint32_t)},
                            {top_logprobs, listed * sizeof(float)}};
    if (any_overlap(inputs, outputs)) return SN_ERR_ALIASING;
    sn::LogprobArgs args;
    args.logits = logits;
    args.tokens = tokens;
    args.logprobs = logprobs;
    args.entropies = entropies;
    args.stats = stats;
    args.top_tokens = top_tokens;
    args.top_logprobs = top_logprobs;
    args.rows = int64_t(shape->rows);
    args.cols = int64_t(shape->cols);
    args.column_offset = int64_t(shape->column_offset);
    args.classes = int64_t(shape->classes);
    args.heads = int64_t(shape->heads);
    args.token_stride = int64_t(shape->token_stride);
    args.token_offset = int64_t(shape->token_offset);
    args.top = top_tokens != nullptr || top_logprobs != nullptr ? int32_t(shape->top) : 0;
    args.scale = shape->scale;
    args.workspace = ctx->env.workspace;
    args.workspace_bytes = ctx->env.workspace_bytes;
    args.cu_count = ctx->env.cu_count;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = sn::launch_token_logprobs(args, ctx->stream);
    return status(err);
}

int sn_token_logprobs_backward(sn_context* ctx, const sn_logprob_shape* shape, const float* logits,
                               size_t logits_len, const uint32_t* tokens, size_t tokens_len, const float* stats,
                               size_t stats_len, const float* entropies, size_t entropies_len,
                               const float* d_logprobs, size_t d_logprobs_len, const float* d_entropies,
                               size_t d_entropies_len, float* grad, size_t grad_len) {
    Needs need;
    const int rc = check_shape(shape, d_logprobs != nullptr, &need);
    if (rc != SN_OK) return rc;
    if (logits_len < need.logits || grad_len < need.logits || stats_len / 2 < need.places ||
        (d_logprobs != nullptr && (tokens_len < need.tokens || d_logprobs_len < need.places)) ||
        (d_entropies != nullptr && (d_entropies_len < need.places || entropies_len < need.places)))
        return SN_ERR_LENGTH_MISMATCH;
    if (ctx == nullptr) return SN_ERR_NULL_ARGUMENT;
    if (need.places == 0) return SN_OK;
    if (logits == nullptr || grad == nullptr || stats == nullptr || (d_logprobs != nullptr && tokens == nullptr) ||
        (d_entropies != nullptr && entropies == nullptr))
        return SN_ERR_NULL_ARGUMENT;
    const size_t places = need.places * sizeof(float);
    const Span inputs[] = {{logits == grad ? nullptr : logits, need.logits * sizeof(float)},
                           {tokens, need.tokens * sizeof(uint32_t)},
                           {stats, 2 * places},
                           {d_entropies != nullptr ? entropies : nullptr, places},
                           {d_logprobs, places},
                           {d_entropies, places}};
    const Span outputs[] = {{grad, need.logits * sizeof(float)}};
    if (any_overlap(inputs, outputs)) return SN_ERR_ALIASING;
    sn::LogprobBackwardArgs args;
    args.logits = logits;
    args.tokens = tokens;
    args.stats = stats;
    args.entropies = entropies;
    args.d_logprobs = d_logprobs;
    args.d_entropies = d_entropies;
    args.grad = grad;
    args.rows = int64_t(shape->rows);
    args.cols = int64_t(shape->cols);
    args.column_offset = int64_t(shape->column_offset);
    args.classes = int64_t(shape->classes);
    args.heads = int64_t(shape->heads);
    args.token_stride = int64_t(shape->token_stride);
    args.token_offset = int64_t(shape->token_offset);
    args.scale = shape->scale;
    hipError_t err = hipSetDevice(ctx->device);
    if (err == hipSuccess) err = sn::launch_token_logprobs_backward(args, ctx->stream);
    return status(err);
}

}  // extern "C"
