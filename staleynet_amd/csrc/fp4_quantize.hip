// fp32 to 4-bit blocks and back (staleynet_fp4.h has the format): weights
// (sn_quantize_fp4, sn_dequantize_fp4) and rows of a key/value cache
// (sn_fp4_cache_append, sn_fp4_cache_read).
//
// For a block of 32 values with largest magnitude A = m 2^x, m in [0.5, 1): the
// factor is 2^e, e = x - 3 (which puts A in [4, 8) factors), or x - 2 where
// m >= 7/8; codes are the values times 2^-e rounded to nearest, ties to even.
// The scaling is by a power of two, so each step is exact but the one rounding,
// which v_cvt_scalef32_pk_fp4_f32 does (its result was compared at every tie, its
// neighbours, past the largest code and at -0).
//
// All are bound by memory: 4 bytes a value on the fp32 side against 0.53. Where the fp32 values of
// a block are contiguous four lanes take it, eight values each: 32-byte loads or stores, a word of
// codes a lane, so a wave's codes are 256 contiguous bytes; the maximum is exchanged over
// four lanes. 8192 x 28672 weights: 184 us (5.8 TB/s) to 4 bits, 199 back, transposed; 301 to 321 and 232 to 253
// with contiguous columns, where a wave writes 16 bytes each to 64 rows of codes (blocks taken in
// runs of 4, 8 or 16 by a thread, to fill those rows' lines sooner: 331 to 342).
// Cache rows: 4 x 2000 rows of 8 heads of 64, appended in 8.8 us and read in 10.8 (4.2 and 3.4 TB/s, traced); 16 single
// rows, 2.6 us each way.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kThreads = 256;

// The block's scale byte from its largest magnitude's bits (as an integer, so
// that infinities and NaN are the largest).
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
    if (magnitude == 0) return 0;
    if (magnitude >= 0x7f800000u) return 255;
    // A >= 2^-126: its exponent field is x + 126, and its fraction is at least 3/4
    // where m >= 7/8. Subnormals are under 2^-126, where the factor is at its least.
    const int32_t s = int32_t(magnitude >> 23) - 2 + ((magnitude & 0x007fffffu) >= 0x00600000u ? 1 : 0);
    return uint32_t(min(max(s, 0), int32_t(kLargestScale)));
}

// Eight values' codes, lowest first.
__device__ __forceinline__ uint32_t codes_of(const float* v, float factor) {
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], factor, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], factor, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], factor, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], factor, 3);
    return word;
}

// Eight values of a block, four neighbouring lanes a block: this lane's word of
// codes, and the block's scale byte. Every lane of the four has to call it.
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], uint32_t& s) {
    uint32_t magnitude = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) magnitude = max(magnitude, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    magnitude = max(magnitude, uint32_t(__shfl_xor(int(magnitude), 1)));
    magnitude = max(magnitude, uint32_t(__shfl_xor(int(magnitude), 2)));
    s = scale_byte(magnitude);
    return s > kLargestScale ? 0 : codes_of(v, factor_of(s));
}

__device__ __forceinline__ void dequantize8(uint32_t word, uint32_t s, float (&v)[8]) {
    const float factor = factor_of(s);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, factor, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, factor, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, factor, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, factor, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}

// Weights whose columns are contiguous (SN_ROW_MAJOR): a block a thread, so that a wave reads or
// writes 64 neighbouring columns at once.
__global__ __launch_bounds__(kThreads) void quantize_columns_kernel(WeightArgs a) {
    const int64_t blocks = blocks_of(a.inner);
    const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= a.cols) return;
    for (int64_t b = blockIdx.y; b < blocks; b += gridDim.y) {
        const float* from = a.source + b * kBlock * a.cols + c;
        float v[32];
        uint32_t magnitude = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            v[i] = b * kBlock + i < a.inner ? from[i * a.cols] : 0.f;
            magnitude = max(magnitude, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
        }
        const uint32_t s = scale_byte(magnitude);
        u32x4 words = {0, 0, 0, 0};
        if (s <= kLargestScale) {
#pragma unroll
            for (int w = 0; w < 4; ++w) words[w] = codes_of(&v[8 * w], factor_of(s));
        }
        *reinterpret_cast<u32x4*>(a.codes + (c * blocks + b) * kBlockBytes) = words;
        a.scales[c * blocks + b] = uint8_t(s);
    }
}
__global__ __launch_bounds__(kThreads) void dequantize_columns_kernel(WeightArgs a) {
    const int64_t blocks = blocks_of(a.inner);
    const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= a.cols) return;
    for (int64_t b = blockIdx.y; b < blocks; b += gridDim.y) {
        const u32x4 words = *reinterpret_cast<const u32x4*>(a.codes + (c * blocks + b) * kBlockBytes);
        const uint32_t s = a.scales[c * blocks + b];
        float* to = a.output + b * kBlock * a.cols + c;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float v[8];
            dequantize8(words[w], s, v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (b * kBlock + 8 * w + i < a.inner) to[(8 * w + i) * a.cols] = v[i];
        }
    }
}

// Weights whose inner dimension is contiguous (SN_TRANSPOSED): four lanes a block. Rows start at any
// 4-byte address; wide loads and stores need no more.
typedef f32x4 f32x4_unaligned __attribute__((aligned(4)));
__device__ __forceinline__ void eighth_of(int64_t e, int64_t per_row, bool narrow, int64_t& row, int64_t& at) {
    if (narrow) {  // the division of 32-bit numbers is a fifth of the other's instructions
        row = uint32_t(e) / uint32_t(per_row);
        at = uint32_t(e) - uint32_t(row) * uint32_t(per_row);
    } else {
        row = e / per_row;
        at = e - row * per_row;
    }
}
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(WeightArgs a) {
    const int64_t per_row = 4 * blocks_of(a.inner), total = a.cols * per_row;
    const int64_t stride = int64_t(gridDim.x) * kThreads;
    // total is a multiple of 4: the four lanes of a block leave the loop together.
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < total; e += stride) {
        int64_t c, eighth;
        eighth_of(e, per_row, total <= int64_t(UINT32_MAX), c, eighth);
        const int64_t k = 8 * eighth;
        const float* from = a.source + c * a.inner + k;
        float v[8];
        if (k + 8 <= a.inner) {
            const f32x4 lo = *reinterpret_cast<const f32x4_unaligned*>(from);
            const f32x4 hi = *reinterpret_cast<const f32x4_unaligned*>(from + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < a.inner ? from[i] : 0.f;
        }
        uint32_t s;
        const uint32_t word = quantize8(v, s);
        reinterpret_cast<uint32_t*>(a.codes)[e] = word;
        if ((e & 3) == 0) a.scales[e >> 2] = uint8_t(s);
    }
}
__global__ __launch_bounds__(kThreads) void dequantize_rows_kernel(WeightArgs a) {
    const int64_t per_row = 4 * blocks_of(a.inner), total = a.cols * per_row;
    const int64_t stride = int64_t(gridDim.x) * kThreads;
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < total; e += stride) {
        int64_t c, eighth;
        eighth_of(e, per_row, total <= int64_t(UINT32_MAX), c, eighth);
        const int64_t k = 8 * eighth;
        float v[8];
        dequantize8(reinterpret_cast<const uint32_t*>(a.codes)[e], a.scales[e >> 2], v);
        float* to = a.output + c * a.inner + k;
        if (k + 8 <= a.inner) {
            *reinterpret_cast<f32x4_unaligned*>(to) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_unaligned*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < a.inner) to[i] = v[i];
        }
    }
}

// A workgroup takes packed rows (sequence b, token t), its threads the row's eights of
// values: those of the keys, head by head, then of the values, so that neighbouring lanes
// have neighbouring columns.
struct CachePlace {
    bool values;
    int32_t h, eighth;
};
template <int H>
__device__ __forceinline__ CachePlace cache_place(int32_t item, int32_t kv_heads) {
    const int32_t half = kv_heads * (H / 8);
    CachePlace p;
    p.values = item >= half;
    item -= p.values ? half : 0;
    p.h = item / (H / 8);
    p.eighth = item % (H / 8);
    return p;
}
// The cache position of a packed row, or -1 past the capacity.
__device__ __forceinline__ int64_t position_of(const CacheRowsArgs& a, int64_t b, int64_t t) {
    const int64_t at = (a.positions != nullptr ? int64_t(a.positions[b]) : a.position) + t;
    return at < a.capacity ? at : -1;
}

template <int H, bool VECTOR>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheRowsArgs a) {
    const int32_t heads = int32_t(a.kv_heads), items = 2 * heads * (H / 8);  // under 2^26
    for (int64_t row = blockIdx.x; row < a.batch * a.time; row += gridDim.x) {
        const int64_t b = row / a.time, at = position_of(a, b, row % a.time);
        if (at < 0) continue;
        // items is a multiple of 4: the four lanes of a block leave the loop together.
        for (int32_t item = threadIdx.x; item < items; item += blockDim.x) {
            const CachePlace p = cache_place<H>(item, heads);
            const float* from =
                a.packed + row * a.width + (p.values ? a.value_column : a.key_column) + p.h * H + 8 * p.eighth;
            float v[8];
            if (VECTOR) {
                const f32x4 lo = reinterpret_cast<const f32x4*>(from)[0], hi = reinterpret_cast<const f32x4*>(from)[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = from[i];
            }
            uint32_t s;
            const uint32_t word = quantize8(v, s);
            const int64_t cache_row = (b * heads + p.h) * a.capacity + at;
            uint8_t* codes = p.values ? a.v_codes : a.k_codes;
            uint8_t* scales = p.values ? a.v_scales : a.k_scales;
            reinterpret_cast<uint32_t*>(codes)[cache_row * (H / 8) + p.eighth] = word;
            if ((p.eighth & 3) == 0) scales[cache_row * (H / 32) + p.eighth / 4] = uint8_t(s);
        }
    }
}

template <int H, bool VECTOR>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(CacheRowsArgs a) {
    const int32_t heads = int32_t(a.kv_heads), items = 2 * heads * (H / 8);
    for (int64_t row = blockIdx.x; row < a.batch * a.time; row += gridDim.x) {
        const int64_t b = row / a.time, t = row % a.time, at = position_of(a, b, t);
        for (int32_t item = threadIdx.x; item < items; item += blockDim.x) {
            const CachePlace p = cache_place<H>(item, heads);
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (at >= 0) {
                const int64_t cache_row = (b * heads + p.h) * a.capacity + at;
                const uint8_t* codes = p.values ? a.v_codes : a.k_codes;
                const uint8_t* scales = p.values ? a.v_scales : a.k_scales;
                dequantize8(reinterpret_cast<const uint32_t*>(codes)[cache_row * (H / 8) + p.eighth],
                            scales[cache_row * (H / 32) + p.eighth / 4], v);
            }
            float* to = (p.values ? a.values : a.keys) + ((b * heads + p.h) * a.time + t) * H + 8 * p.eighth;
            if (VECTOR) {
                reinterpret_cast<f32x4*>(to)[0] = f32x4{v[0], v[1], v[2], v[3]};
                reinterpret_cast<f32x4*>(to)[1] = f32x4{v[4], v[5], v[6], v[7]};
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) to[i] = v[i];
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Enough workgroups for every thread to have one item, at most 2^20 (the
// kernels loop over the rest).
unsigned grid_of(int64_t items) {
    const int64_t groups = (items + kThreads - 1) / kThreads;
    return unsigned(groups < (int64_t(1) << 20) ? groups : int64_t(1) << 20);
}

}  // namespace

hipError_t launch_weights(const WeightArgs& a, bool quantize, hipStream_t stream) {
    const int64_t blocks = blocks_of(a.inner);
    if (a.cols == 0 || blocks == 0) return hipSuccess;
    if (a.transposed) {
        hipLaunchKernelGGL((quantize ? quantize_rows_kernel : dequantize_rows_kernel), dim3(grid_of(a.cols * blocks * 4)),
                           dim3(kThreads), 0, stream, a);
    } else {
        const int64_t groups = (a.cols + kThreads - 1) / kThreads;
        const dim3 grid(unsigned(groups), unsigned(std::min<int64_t>(blocks, 65535)));
        hipLaunchKernelGGL((quantize ? quantize_columns_kernel : dequantize_columns_kernel), grid, dim3(kThreads), 0,
                           stream, a);
    }
    return hipGetLastError();
}

namespace {

// One workgroup a packed row, up to 2^20 of them (they loop over the rest).
template <int H>
hipError_t launch_rows(const CacheRowsArgs& a, bool append, bool vector, hipStream_t stream) {
    const int64_t rows = a.batch * a.time, items = 2 * a.kv_heads * (H / 8);
    if (rows == 0 || items == 0) return hipSuccess;
    const dim3 grid(unsigned(std::min<int64_t>(rows, int64_t(1) << 20)));
    const dim3 threads(unsigned(std::min<int64_t>(kThreads, (items + 63) / 64 * 64)));
    auto* const kernel = append ? (vector ? cache_append_kernel<H, true> : cache_append_kernel<H, false>)
                                : (vector ? cache_read_kernel<H, true> : cache_read_kernel<H, false>);
    hipLaunchKernelGGL(kernel, grid, threads, 0, stream, a);
    return hipGetLastError();
}
hipError_t launch_rows(const CacheRowsArgs& a, bool append, bool vector, hipStream_t stream) {
    switch (a.head_dim) {
        case 32: return launch_rows<32>(a, append, vector, stream);
        case 64: return launch_rows<64>(a, append, vector, stream);
        default: return launch_rows<128>(a, append, vector, stream);
    }
}

}  // namespace

hipError_t launch_cache_append(const CacheRowsArgs& a, hipStream_t stream) {
    const bool vector = aligned16(a.packed) && a.width % 4 == 0 && a.key_column % 4 == 0 && a.value_column % 4 == 0;
    return launch_rows(a, true, vector, stream);
}

hipError_t launch_cache_read(const CacheRowsArgs& a, hipStream_t stream) {
    return launch_rows(a, false, aligned16(a.keys) && aligned16(a.values), stream);
}

}  // namespace fp4
}  // namespace sn
