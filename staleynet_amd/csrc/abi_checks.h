// Checks of arguments that the entry points of fp8.cpp, norm_abi.cpp and
// logprobs_abi.cpp share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "staleynet_gemm.h"

namespace sn {
namespace abi {

// Sizes and offsets stay below this, so that byte offsets fit the kernels' signed arithmetic.
constexpr size_t kLimit = size_t(1) << 60;

inline int status(hipError_t err) { return err == hipSuccess ? SN_OK : int(err); }

// a * b or a + b, or false where it reaches the limit.
inline bool product(size_t a, size_t b, size_t* out) { return !__builtin_mul_overflow(a, b, out) && *out < kLimit; }
inline bool sum(size_t a, size_t b, size_t* out) { return !__builtin_add_overflow(a, b, out) && *out < kLimit; }

// A buffer a call reads or writes: `bytes` of it are used (0 or null: not given).
struct Span {
    const void* data;
    size_t bytes;
};
inline bool overlaps(const Span& a, const Span& b) {
    if (a.data == nullptr || b.data == nullptr || a.bytes == 0 || b.bytes == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.data), b0 = reinterpret_cast<uintptr_t>(b.data);
    return a0 < b0 + b.bytes && b0 < a0 + a.bytes;
}
// Whether an output meets an input or another output.
template <int INPUTS, int OUTPUTS>
bool any_overlap(const Span (&inputs)[INPUTS], const Span (&outputs)[OUTPUTS]) {
    for (int i = 0; i < OUTPUTS; ++i) {
        for (const Span& in : inputs)
            if (overlaps(outputs[i], in)) return true;
        for (int j = 0; j < i; ++j)
            if (overlaps(outputs[i], outputs[j])) return true;
    }
    return false;
}

template <int BYTES>
bool aligned(const void* p) {
    return (reinterpret_cast<uintptr_t>(p) & (BYTES - 1)) == 0;
}

}  // namespace abi
}  // namespace sn
