// Log probabilities of given tokens, entropies and the likeliest classes, and
// their gradient (staleynet_logprobs.h has the formulas).
//
// With m the largest logit, z = a (x - m) and rest = the sum of e^z without one
// term of the largest: T = log(1 + rest), logprob = z_token - T, H = T + W / (1 +
// rest), W = the sum of e^z (-z), all of whose terms are positive. e^z is 2^(z log2 e)
// on the transcendental unit (v_exp_f32, about 1 ulp); rounding z log2 e adds
// at most |z| 2^-24 to a term's relative error. Bound by memory: 4 bytes a logit
// forward, 8 backward.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "logprobs_internal.h"

namespace sn {
namespace {

constexpr uint32_t kEmptyToken = SN_EMPTY_TOKEN;
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float exp_of(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

// An order of logits as integers: NaN is the largest, -0 equals 0; 0 is below all.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.f);
    if (x != x) return 0xffffffffu;
    return bits ^ (uint32_t(int32_t(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// A class with its logit, ordered by the logit and then with the lower class ahead; all are above 0 and below ~0.
constexpr uint32_t kClassMask = 0x7fffffffu;
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t c) { return uint64_t(key_of(x)) << 32 | (kClassMask - c); }
__device__ __forceinline__ uint32_t class_of(uint64_t entry) { return kClassMask - uint32_t(entry); }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) v = v + __shfl_xor(v, step);
    return v;
}
__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const uint64_t other = uint64_t(__shfl_xor(static_cast<unsigned long long>(v), step));
        v = other > v ? other : v;
    }
    return v;
}

// One wave a row and head.
__global__ __launch_bounds__(64) void logprobs_kernel(LogprobArgs a) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x;
    const int64_t place = blockIdx.x, row = place / a.heads, head = place - row * a.heads;
    const float* x = a.logits + row * a.cols + a.column_offset + head * a.classes;
    float m = -INFINITY;
    bool nan = false;
    for (int64_t c = lane; c < a.classes; c += 64) {
        nan |= x[c] != x[c];
        m = fmaxf(m, x[c]);
    }
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) m = fmaxf(m, __shfl_xor(m, step));
    float rest = 0.f, weighted = 0.f, equal = 0.f;
    for (int64_t c = lane; c < a.classes; c += 64) {
        const float z = (x[c] - m) * a.scale, e = exp_of(z);
        rest += x[c] < m ? e : 0.f;
        equal += x[c] == m ? 1.f : 0.f;
        weighted += e > 0.f ? e * -z : 0.f;
    }
    rest = wave_sum(rest) + (wave_sum(equal) - 1.f);
    weighted = wave_sum(weighted);
    if (__any(nan) || !(fabsf(m) < INFINITY)) rest = m = NAN;
    const float log_total = log1pf(rest);
    if (lane == 0) {
        if (a.logprobs != nullptr) {
            const uint32_t token = a.tokens[row * a.token_stride + a.token_offset + head];
            float lp = 0.f;
            if (token != kEmptyToken) lp = token < uint64_t(a.classes) ? (x[token] - m) * a.scale - log_total : NAN;
            a.logprobs[place] = lp;
        }
        if (a.entropies != nullptr) a.entropies[place] = log_total + weighted / (1.f + rest);
        if (a.stats != nullptr) a.stats[2 * place] = m, a.stats[2 * place + 1] = log_total;
    }
    // The likeliest, one pass each: the largest of (key, lower class first) below the last.
    uint64_t last = ~uint64_t(0);
    for (int i = 0; i < a.top; ++i) {
        uint64_t best = 0;
        for (int64_t c = lane; c < a.classes; c += 64) {
            const uint64_t entry = entry_of(x[c], uint32_t(c));
            if (entry < last && entry > best) best = entry;
        }
        last = wave_largest(best);
        if (lane == 0) {
            const bool none = last == 0;
            if (a.top_tokens != nullptr) a.top_tokens[place * a.top + i] = none ? kEmptyToken : class_of(last);
            if (a.top_logprobs != nullptr)
                a.top_logprobs[place * a.top + i] =
                    none ? -INFINITY : (logit_of(uint32_t(last >> 32)) - m) * a.scale - log_total;
        }
    }
}

// One wave a row and head.
__global__ __launch_bounds__(64) void logprobs_backward_kernel(LogprobBackwardArgs a) {
#pragma clang fp contract(off)
    const int64_t place = blockIdx.x, row = place / a.heads, head = place - row * a.heads;
    const int64_t first = row * a.cols + a.column_offset + head * a.classes;
    const float *x = a.logits + first, m = a.stats[2 * place], log_total = a.stats[2 * place + 1];
    float d_logprob = 0.f, d_entropy = 0.f, entropy = 0.f;
    uint32_t token = kEmptyToken;
    if (a.d_logprobs != nullptr) {
        token = a.tokens[row * a.token_stride + a.token_offset + head];
        if (token != kEmptyToken) d_logprob = a.d_logprobs[place];
    }
    if (a.d_entropies != nullptr) d_entropy = a.d_entropies[place], entropy = a.entropies[place];
    for (int64_t c = threadIdx.x; c < a.classes; c += 64) {
        const float log_p = (x[c] - m) * a.scale - log_total, p = exp_of(log_p);
        const float one = uint64_t(c) == token ? d_logprob : 0.f;
        const float more = p > 0.f ? d_entropy * (log_p + entropy) : 0.f;
        a.grad[first + c] = (one - p * (d_logprob + more)) * a.scale;
    }
}

}  // namespace

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(logprobs_kernel, dim3(unsigned(a.rows * a.heads)), dim3(64), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_token_logprobs_backward(const LogprobBackwardArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(logprobs_backward_kernel, dim3(unsigned(a.rows * a.heads)), dim3(64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sn
