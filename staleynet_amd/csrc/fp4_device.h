// Device code the 4-bit kernels share: a block's factor, its codes as bf16
// fragments, and fp32 values as exact sums of three bf16 values.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fp4_internal.h"
#include "split_bf16.h"

namespace sn {
namespace fp4 {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Between a wave's writes of LDS and its other lanes' reads of them, and back: the hardware
// keeps the order of one wave's accesses, the fences the compiler's (no instruction comes of them).
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// The factor a scale byte stands for: 2^(s - 127), subnormal for 0, NaN past
// the largest. The conversions below read its exponent; a product code * factor
// is exact in bf16 and in fp32 over that whole range (checked for every code and
// byte), and NaN for a NaN factor.
__device__ __forceinline__ float factor_of(uint32_t s) {
    const uint32_t bits = max(s << 23, 0x00400000u);
    return __builtin_bit_cast(float, s > kLargestScale ? 0x7fc00000u : bits);
}

// Eight codes of a block (a 32-bit word, lowest first) as bf16: one
// v_cvt_scalef32_pk_bf16_fp4 a pair, half an instruction a value.
__device__ __forceinline__ bf16x8 fragment_of(uint32_t word, float factor) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const u32x4 w = {
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, factor, 0))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, factor, 1))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, factor, 2))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, factor, 3)))};
    return __builtin_bit_cast(bf16x8, w);
}

// An fp32 value as the exact sum of three bf16 values of its sign, each the
// leading 8 significant bits of what is left (cut off, not rounded: the largest
// float stays finite, and 24 = 8 + 8 + 8). Exact from 2^-110 on; below, rest_of has
// what they leave. An infinity or NaN leaves NaN after the first part, which one
// comparison a pair finds; then it is its own first part
// and the others are 0, so that products follow IEEE arithmetic.
__device__ __forceinline__ uint32_t upper_halves(float x0, float x1) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x1), __builtin_bit_cast(uint32_t, x0), 0x07060302u);
}
__device__ __forceinline__ float cut(float x, uint32_t upper) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & upper);
}
__device__ __forceinline__ float quiet(float x) {  // a NaN whose upper half is one
    return x != x ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) | 0x00400000u) : x;
}
// What the three parts leave of a value, times 2^100: 0 but for magnitudes under 2^-110, whose bits under 2^-133
// (bf16's smallest subnormal, at which the last cut ends) the third part cannot hold. There are at most 16 of
// them, down to 2^-149, so that two parts hold them once they are lifted. notice() gathers, from the value
// the third part is cut from, whether there are any: those bits are the lower half of its word, and 0 in every
// other value, which has at most 8 bits left there.
constexpr float kRestLift = 0x1p100f;
__device__ __forceinline__ float rest_of(float x, uint32_t upper) {
#pragma clang fp contract(off)
    const float x1 = x - cut(x, upper);
    const float a1 = x1 != x1 ? 0.f : x1;
    const float a2 = a1 - cut(a1, upper);
    return (a2 - cut(a2, upper)) * kRestLift;
}
__device__ __forceinline__ void notice(uint32_t& left, float third0, float third1) {
    left |= __builtin_bit_cast(uint32_t, third0) | __builtin_bit_cast(uint32_t, third1);
    asm("" : "+v"(left));  // one running value: values gathered first would take registers
}
__device__ __forceinline__ bool noticed(uint32_t left) { return (left & 0xffffu) != 0; }

__device__ __forceinline__ SplitVector split_vector_of(const u32x4 (&w)[kParts]) {
    SplitVector out;
#pragma unroll
    for (int q = 0; q < kParts; ++q) out.part[q] = __builtin_bit_cast(bf16x8, w[q]);
    return out;
}
// Finite values only.
__device__ __forceinline__ SplitVector split_finite(const float (&x)[8], uint32_t upper) {
#pragma clang fp contract(off)
    u32x4 w[kParts];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float a = x[2 * p], b = x[2 * p + 1];
        const float a1 = a - cut(a, upper), b1 = b - cut(b, upper);
        w[0][p] = upper_halves(a, b);
        w[1][p] = upper_halves(a1, b1);
        w[2][p] = upper_halves(a1 - cut(a1, upper), b1 - cut(b1, upper));
    }
    return split_vector_of(w);
}
__device__ __forceinline__ SplitVector split_exact(const float (&x)[8], uint32_t upper, uint32_t& left) {
#pragma clang fp contract(off)
    u32x4 w[kParts];
    bool odd = false;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float a = x[2 * p], b = x[2 * p + 1];
        const float a1 = a - cut(a, upper), b1 = b - cut(b, upper);
        odd |= __builtin_isunordered(a1, b1);
        w[0][p] = upper_halves(a, b);
        w[1][p] = upper_halves(a1, b1);
        const float a2 = a1 - cut(a1, upper), b2 = b1 - cut(b1, upper);
        notice(left, a2, b2);
        w[2][p] = upper_halves(a2, b2);
    }
    if (__any(odd)) {
        left = ~0u;  // NaN among them
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            float part[2][kParts];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = x[2 * p + e];
                const float a1 = a - cut(a, upper);
                part[e][0] = quiet(a);
                part[e][1] = a1 != a1 ? 0.f : a1;
                part[e][2] = part[e][1] - cut(part[e][1], upper);
            }
#pragma unroll
            for (int q = 0; q < kParts; ++q) w[q][p] = upper_halves(part[0][q], part[1][q]);
        }
    }
    return split_vector_of(w);
}

}  // namespace fp4
}  // namespace sn
