// Products of two 8-bit operands (sn_matmul_fp8; staleynet_fp8.h has the format):
//   y = scale * X W (+ y) (+ bias)
//
// A code times its block's factor is exact in bf16, and a product of two such
// values is exact in fp32, so fragments are codes converted in registers and
// multiplied by the bf16 matrix instructions, which sum in fp32. The 8-bit
// matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4 and the 16x16x32 forms)
// would run twice as fast, but were measured to align the products of
// neighbouring k to the largest of them and to cut off what lies 13 bits below: random codes
// come out up to 2^-12 of the largest product wrong, where fp32 sums are
// asked for.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp8_device.h"
#include "fp8_internal.h"

namespace sn {
namespace fp8 {
namespace {

// One wave a 32 x 32 tile of the output, operands read from memory as they are
// needed. Lane l holds row l % 16 of a 16-row fragment and bytes 32 (l / 16) .. + 31
// of a block; the four 32-deep steps of a block take eight of them each,
// for both operands the same.
__global__ __launch_bounds__(256) void product_kernel(ProductArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row0 = (int64_t(blockIdx.y) * 2 + wave / 2) * 32, col0 = (int64_t(blockIdx.x) * 2 + wave % 2) * 32;
    if (row0 >= a.rows || col0 >= a.cols) return;
    const int64_t stride = a.blocks * kBlock, scale_row = scale_stride(a.blocks);
    f32x4 acc[2][2] = {};
    // Rows and columns past the last read the last one's; their results are not stored.
    const uint8_t *x[2], *x_scales[2], *w[2], *w_scales[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t row = min(row0 + 16 * i + lane % 16, a.rows - 1), col = min(col0 + 16 * i + lane % 16, a.cols - 1);
        x[i] = a.x + row * stride + 32 * (lane / 16);
        w[i] = a.w + col * stride + 32 * (lane / 16);
        x_scales[i] = a.x_scales + row * scale_row;
        w_scales[i] = a.w_scales + col * scale_row;
    }
    for (int64_t b = 0; b < a.blocks; ++b) {
        u32x4 xc[2][2], wc[2][2];
        float xf[2], wf[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                xc[i][h] = *reinterpret_cast<const u32x4*>(x[i] + b * kBlock + 16 * h);
                wc[i][h] = *reinterpret_cast<const u32x4*>(w[i] + b * kBlock + 16 * h);
            }
            xf[i] = factor_of(x_scales[i][b]);
            wf[i] = factor_of(w_scales[i][b]);
        }
#pragma unroll
        for (int step = 0; step < 4; ++step) {
            bf16x8 xb[2], wb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xb[i] = fragment_of(xc[i][step / 2][2 * (step % 2)], xc[i][step / 2][2 * (step % 2) + 1], xf[i]);
                wb[i] = fragment_of(wc[i][step / 2][2 * (step % 2)], wc[i][step / 2][2 * (step % 2) + 1], wf[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[i], wb[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t row = row0 + 16 * i + 4 * (lane / 16) + r, col = col0 + 16 * j + lane % 16;
                if (row >= a.rows || col >= a.cols) continue;
                float v = a.scale * acc[i][j][r];
                if (a.accumulate) v = a.y[row * a.cols + col] + v;
                if (a.bias != nullptr) v = v + a.bias[col];
                a.y[row * a.cols + col] = v;
            }
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    const int64_t tiles_m = (a.rows + 63) / 64, tiles_n = (a.cols + 63) / 64;
    for (int64_t first = 0; first < tiles_m; first += 65535) {
        ProductArgs part = a;
        part.x += first * 64 * a.blocks * kBlock;
        part.x_scales += first * 64 * scale_stride(a.blocks);
        part.y += first * 64 * a.cols;
        part.rows = std::min<int64_t>(a.rows - first * 64, 65535 * 64);
        const dim3 grid{unsigned(tiles_n), unsigned((part.rows + 63) / 64)};
        hipLaunchKernelGGL(product_kernel, grid, dim3(256), 0, stream, part);
    }
    return hipGetLastError();
}

}  // namespace fp8
}  // namespace sn
