// Interface between the log-probability entry points (logprobs_abi.cpp) and their kernels (logprobs.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "staleynet_logprobs.h"

namespace sn {

struct LogprobArgs {
    const float* logits = nullptr;
    const uint32_t* tokens = nullptr;
    float* logprobs = nullptr;
    float* entropies = nullptr;
    float* stats = nullptr;
    uint32_t* top_tokens = nullptr;
    float* top_logprobs = nullptr;
    int64_t rows = 0, cols = 0, column_offset = 0, classes = 0, heads = 0;
    int64_t token_stride = 0, token_offset = 0;
    int32_t top = 0;  // 0 where neither list is wanted
    float scale = 1.f;
    float* workspace = nullptr;
    size_t workspace_bytes = 0;
    int cu_count = 256;
};
hipError_t launch_token_logprobs(const LogprobArgs& args, hipStream_t stream);

struct LogprobBackwardArgs {
    const float* logits = nullptr;
    const uint32_t* tokens = nullptr;
    const float* stats = nullptr;
    const float* entropies = nullptr;
    const float* d_logprobs = nullptr;
    const float* d_entropies = nullptr;
    float* grad = nullptr;
    int64_t rows = 0, cols = 0, column_offset = 0, classes = 0, heads = 0;
    int64_t token_stride = 0, token_offset = 0;
    float scale = 1.f;
};
hipError_t launch_token_logprobs_backward(const LogprobBackwardArgs& args, hipStream_t stream);

}  // namespace sn
