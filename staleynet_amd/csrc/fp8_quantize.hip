// fp32 operands to 8-bit blocks of 128 and back (staleynet_fp8.h has the format):
// sn_quantize_fp8 and sn_dequantize_fp8.
//
// For a block with largest magnitude A the factor is 2^e, the smallest of which
// A is at most 464; codes are the values times 2^-e rounded to e4m3, to nearest
// even. The scaling is by a power of two, so each step is exact but the one
// rounding. Both ways are bound by memory: 4 bytes a value on the fp32 side
// against 1.01. 1999 x 4001 take 8.3 us there and 9.3 back (from the last-level
// cache), 8192 x 4096 30 us back (5.6 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp8_device.h"
#include "fp8_internal.h"

namespace sn {
namespace fp8 {
namespace {

constexpr int kThreads = 256;

// Rows whose values are contiguous: sixteen lanes a block, eight values each.
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(OperandArgs a) {
    const int64_t blocks = blocks_of(a.inner), per_row = 16 * blocks, total = a.rows * per_row;
    const int64_t stride = int64_t(gridDim.x) * kThreads;
    // total is a multiple of 16: the lanes of a block leave the loop together.
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < total; e += stride) {
        int64_t row, at;
        divide(e, per_row, total <= int64_t(UINT32_MAX), row, at);
        float v[8];
        load8(a.source + row * a.inner, 8 * at, a.inner, v);
        uint32_t s;
        const u32x2 words = quantize8(v, s);
        store_block(a.codes + row * blocks * kBlock, a.scales + row * scale_stride(blocks), at / 16, int(at % 16), blocks,
                    words, s);
    }
}
__global__ __launch_bounds__(kThreads) void dequantize_rows_kernel(OperandArgs a) {
    const int64_t blocks = blocks_of(a.inner), per_row = 16 * blocks, total = a.rows * per_row;
    const int64_t stride = int64_t(gridDim.x) * kThreads;
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < total; e += stride) {
        int64_t row, at;
        divide(e, per_row, total <= int64_t(UINT32_MAX), row, at);
        if (8 * at >= a.inner) continue;
        const u32x2 words = *reinterpret_cast<const u32x2*>(a.codes + row * blocks * kBlock + 8 * at);
        const float factor = factor_of(a.scales[row * scale_stride(blocks) + at / 16]);
        const f32x4 low = values_of(words[0], factor), high = values_of(words[1], factor);
        const float v[8] = {low[0], low[1], low[2], low[3], high[0], high[1], high[2], high[3]};
        store8(a.output + row * a.inner, 8 * at, a.inner, v);
    }
}

// Columns of a row-major source, [inner, rows]: a workgroup takes a block of 64 neighbouring rows of the format, a wave 32
// of its 128 values of each, so that loads and stores on the fp32 side are 256 contiguous bytes a wave. The codes are turned
// in LDS, so that eight lanes store a row's 128 bytes (14336 x 4096 from the last-level cache: 51 us, 5.8 TB/s,
// against 77 where each lane stored its own 32; 78 from HBM, and as long with 512 bytes a wave).
constexpr int kTurned = 128 + 16;  // bytes of a row in LDS: 16 rows' chunks are in different banks
__global__ __launch_bounds__(kThreads) void quantize_columns_kernel(OperandArgs a) {
    __shared__ uint32_t largest[4][64];
    __shared__ __attribute__((aligned(16))) uint8_t turned[64 * kTurned];
    const int64_t blocks = blocks_of(a.inner), row_groups = (a.rows + 63) / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t group = blockIdx.x; group < row_groups; group += gridDim.x)
        for (int64_t b = blockIdx.y; b < blocks; b += gridDim.y) {
            const int64_t row0 = group * 64, row = row0 + lane;
            const int64_t k0 = b * kBlock + 32 * wave;
            const float* from = a.source + k0 * a.rows + row;
            float v[32];
            uint32_t magnitude = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = row < a.rows && k0 + i < a.inner ? from[i * a.rows] : 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) magnitude = max(magnitude, magnitude_of(v[i]));
            largest[wave][lane] = magnitude;
            __syncthreads();
            magnitude = max(max(largest[0][lane], largest[1][lane]), max(largest[2][lane], largest[3][lane]));
            const uint32_t s = scale_byte(magnitude);
            u32x4 words[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (s <= kLargestScale) {
#pragma unroll
                for (int w = 0; w < 8; ++w) words[w / 4][w % 4] = codes_of(&v[4 * w], factor_of(s));
            }
            u32x4* to = reinterpret_cast<u32x4*>(turned + lane * kTurned + 32 * wave);
            to[0] = words[0];
            to[1] = words[1];
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 32 * h + threadIdx.x / 8, chunk = threadIdx.x % 8;
                if (row0 + r < a.rows)
                    *reinterpret_cast<u32x4*>(a.codes + ((row0 + r) * blocks + b) * kBlock + 16 * chunk) =
                        *reinterpret_cast<const u32x4*>(turned + r * kTurned + 16 * chunk);
            }
            if (wave == 0 && row < a.rows) {
                uint8_t* scales = a.scales + row * scale_stride(blocks);
                scales[b] = uint8_t(s);
                if (b == blocks - 1)
                    for (int64_t pad = blocks; pad < scale_stride(blocks); ++pad) scales[pad] = 0;
            }
        }
}
__global__ __launch_bounds__(kThreads) void dequantize_columns_kernel(OperandArgs a) {
    const int64_t blocks = blocks_of(a.inner), row_groups = (a.rows + 63) / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t group = blockIdx.x; group < row_groups; group += gridDim.x)
        for (int64_t b = blockIdx.y; b < blocks; b += gridDim.y) {
            const int64_t row = group * 64 + lane, k0 = b * kBlock + 32 * wave;
            if (row >= a.rows || k0 >= a.inner) continue;
            const u32x4* from = reinterpret_cast<const u32x4*>(a.codes + (row * blocks + b) * kBlock + 32 * wave);
            const u32x4 words[2] = {from[0], from[1]};
            const float factor = factor_of(a.scales[row * scale_stride(blocks) + b]);
            float* to = a.output + k0 * a.rows + row;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const f32x4 v = values_of(words[w / 4][w % 4], factor);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 + 4 * w + i < a.inner) to[(4 * w + i) * a.rows] = v[i];
            }
        }
}

}  // namespace

hipError_t launch_operand(const OperandArgs& a, bool quantize, hipStream_t stream) {
    const int64_t blocks = blocks_of(a.inner);
    if (a.transposed) {
        const dim3 grid(unsigned(std::min<int64_t>((a.rows + 63) / 64, 1 << 20)), unsigned(std::min<int64_t>(blocks, 256)));
        if (quantize)
            hipLaunchKernelGGL(quantize_columns_kernel, grid, dim3(kThreads), 0, stream, a);
        else
            hipLaunchKernelGGL(dequantize_columns_kernel, grid, dim3(kThreads), 0, stream, a);
    } else {
        const int64_t groups = (a.rows * blocks * 16 + kThreads - 1) / kThreads;
        const dim3 grid(unsigned(std::min<int64_t>(groups, 1 << 20)));
        if (quantize)
            hipLaunchKernelGGL(quantize_rows_kernel, grid, dim3(kThreads), 0, stream, a);
        else
            hipLaunchKernelGGL(dequantize_rows_kernel, grid, dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace fp8
}  // namespace sn
