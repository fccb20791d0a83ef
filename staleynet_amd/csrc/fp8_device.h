// Device code the 8-bit kernels share: a block's factor, fp32 values to codes,
// codes to fp32 and to bf16 fragments.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fp8_internal.h"

namespace sn {
namespace fp8 {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// Rows start at any 4-byte address; wide loads and stores need no more.
typedef f32x4 f32x4_unaligned __attribute__((aligned(4)));

// The factor a scale byte stands for, 2^(s - 127), NaN past the largest. With s
// at least 3 every code times its factor is at least 2^-133, bf16's least
// subnormal: exact in bf16 and in fp32.
__device__ __forceinline__ float factor_of(uint32_t s) {
    return __builtin_bit_cast(float, s > kLargestScale ? 0x7fc00000u : max(s, kLeastScale) << 23);
}

// The block's scale byte from its largest magnitude's bits (as an integer, so
// that infinities and NaN are the largest). A magnitude m 2^x, m in [1, 2), is
// at most 464 2^e = 1.8125 2^(e + 8) from e = x - 8 on, or x - 7 where m is
// larger than 1.8125; e + 127 is the exponent field less 8 (or 7).
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
    if (magnitude >= 0x7f800000u) return 255;
    const int32_t s = int32_t(magnitude >> 23) - 8 + ((magnitude & 0x007fffffu) > 0x00680000u ? 1 : 0);
    return uint32_t(min(max(s, int32_t(kLeastScale)), int32_t(kLargestScale)));
}

__device__ __forceinline__ uint32_t magnitude_of(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Four values' codes, lowest first. v_cvt_scalef32_pk_fp8_f32 divides by the
// factor and rounds once, to nearest even, subnormals too; past 464 factors it would
// give NaN, which only the largest factor's blocks reach: held at 448 before.
__device__ __forceinline__ uint32_t codes_of(const float* v, float factor) {
    const float largest = 448.f * factor;
    s16x2 word = {0, 0};
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, __builtin_amdgcn_fmed3f(v[0], -largest, largest),
                                                    __builtin_amdgcn_fmed3f(v[1], -largest, largest), factor, false);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, __builtin_amdgcn_fmed3f(v[2], -largest, largest),
                                                    __builtin_amdgcn_fmed3f(v[3], -largest, largest), factor, true);
    return __builtin_bit_cast(uint32_t, word);
}

// The values of four codes.
__device__ __forceinline__ f32x4 values_of(uint32_t word, float factor) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, factor, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, factor, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}

// Eight codes (two words, lowest first) times their factor as bf16, exactly:
// one v_cvt_scalef32_pk_bf16_fp8 a pair.
__device__ __forceinline__ bf16x8 fragment_of(uint32_t low, uint32_t high, float factor) {
    const u32x4 w = {
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, factor, false))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, factor, true))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, factor, false))),
        __builtin_bit_cast(uint32_t, bf16x2(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, factor, true)))};
    return __builtin_bit_cast(bf16x8, w);
}

// A division of row counts, in 32 bits where they fit: a fifth of the other's instructions.
__device__ __forceinline__ void divide(int64_t e, int64_t by, bool narrow, int64_t& quotient, int64_t& rest) {
    if (narrow) {
        quotient = uint32_t(e) / uint32_t(by);
        rest = uint32_t(e) - uint32_t(quotient) * uint32_t(by);
    } else {
        quotient = e / by;
        rest = e - quotient * by;
    }
}

// Eight values of a row from its value k on, zeros past its end.
__device__ __forceinline__ void load8(const float* from, int64_t k, int64_t inner, float (&v)[8]) {
    if (k + 8 <= inner) {
        const f32x4 a = *reinterpret_cast<const f32x4_unaligned*>(from + k);
        const f32x4 b = *reinterpret_cast<const f32x4_unaligned*>(from + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < inner ? from[k + i] : 0.f;
    }
}
__device__ __forceinline__ void store8(float* to, int64_t k, int64_t inner, const float (&v)[8]) {
    if (k + 8 <= inner) {
        *reinterpret_cast<f32x4_unaligned*>(to + k) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_unaligned*>(to + k + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < inner) to[k + i] = v[i];
    }
}

// Eight values of a block, sixteen neighbouring lanes a block: this lane's two
// words of codes, and the block's scale byte. Every lane of the sixteen has to call it.
__device__ __forceinline__ u32x2 quantize8(const float (&v)[8], uint32_t& s) {
    uint32_t magnitude = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) magnitude = max(magnitude, magnitude_of(v[i]));
#pragma unroll
    for (int step = 1; step < 16; step <<= 1) magnitude = max(magnitude, uint32_t(__shfl_xor(int(magnitude), step)));
    s = scale_byte(magnitude);
    if (s > kLargestScale) return u32x2{0, 0};
    const float factor = factor_of(s);
    return u32x2{codes_of(&v[0], factor), codes_of(&v[4], factor)};
}

// Where the row's sixteenth-lane `sixteenth` of block b stores its results; the
// last block's first lane also fills the row's padding scale bytes.
__device__ __forceinline__ void store_block(uint8_t* row_codes, uint8_t* row_scales, int64_t b, int sixteenth,
                                            int64_t blocks, u32x2 words, uint32_t s) {
    *reinterpret_cast<u32x2*>(row_codes + b * kBlock + 8 * sixteenth) = words;
    if (sixteenth == 0) {
        row_scales[b] = uint8_t(s);
        if (b == blocks - 1)
            for (int64_t pad = blocks; pad < scale_stride(blocks); ++pad) row_scales[pad] = 0;
    }
}

}  // namespace fp8
}  // namespace sn
