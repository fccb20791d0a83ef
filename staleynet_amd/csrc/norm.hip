// The residual addition with the root-mean-square norm, and its gradients
// (staleynet_norm.h has the formulas).
//
// Bound by memory: 12 to 16 bytes a value against a handful of operations. A row
// is read once and stays in registers; its sum of squares and y are formed in 64
// bits (their products of fp32 values are exact there, and the vector units run
// them at the fp32 rate), so that y is the correctly rounded one but for
// about one value in 10^8, and codes next to a border are the definition's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp8_device.h"
#include "fp8_internal.h"

namespace sn {
namespace {

using namespace fp8;

// One workgroup a row, three passes over it: the sum, y, and (8 bits) the
// block's codes. Any width.
template <bool EIGHT>
__global__ __launch_bounds__(256) void rms_norm_kernel(RmsNormArgs a) {
    __shared__ double partial[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t blocks = blocks_of(a.width);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* x = a.x + row * a.width;
        const float* residual = a.residual == nullptr ? nullptr : a.residual + row * a.width;
        auto load = [&](int64_t k, float(&v)[8]) {
            load8(x, k, a.width, v);
            if (residual != nullptr) {
                float r[8];
                load8(residual, k, a.width, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] + r[i];
            }
        };
        double squares = 0;
        for (int64_t k = 8 * threadIdx.x; k < a.width; k += 8 * 256) {
            float v[8];
            load(k, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += double(v[i]) * double(v[i]);
        }
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) squares += __shfl_xor(squares, step);
        if (lane == 0) partial[wave] = squares;
        __syncthreads();
        squares = (partial[0] + partial[1]) + (partial[2] + partial[3]);
        __syncthreads();
        const double inverse = 1.0 / sqrt(squares / double(a.width) + double(a.epsilon));
        if (a.inverse != nullptr && threadIdx.x == 0) a.inverse[row] = float(inverse);
        for (int64_t k = 8 * threadIdx.x; k < blocks * kBlock; k += 8 * 256) {
            float s[8], w[8], y[8];
            load(k, s);
            load8(a.weight, k, a.width, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = float(double(s[i]) * double(w[i]) * inverse);
            if (a.sum != nullptr) store8(a.sum + row * a.width, k, a.width, s);
            if constexpr (EIGHT) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = k + i < a.width ? y[i] : 0.f;
                uint32_t scale;
                const u32x2 words = quantize8(y, scale);
                store_block(a.codes + row * blocks * kBlock, a.scales + row * scale_stride(blocks), k / kBlock,
                            int(k / 8 % 16), blocks, words, scale);
            } else {
                store8(a.out + row * a.width, k, a.width, y);
            }
        }
    }
}

// d_x, one workgroup a row.
__global__ __launch_bounds__(256) void rms_norm_grad_kernel(RmsNormBackwardArgs a) {
    __shared__ float partial[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float inverse = a.inverse[row];
        const float *s = a.sum + row * a.width, *d_out = a.d_out + row * a.width;
        float dot = 0.f;
        for (int64_t k = threadIdx.x; k < a.width; k += 256) dot += d_out[k] * a.weight[k] * (s[k] * inverse);
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) dot += __shfl_xor(dot, step);
        if (lane == 0) partial[wave] = dot;
        __syncthreads();
        dot = ((partial[0] + partial[1]) + (partial[2] + partial[3])) / float(a.width);
        __syncthreads();
        for (int64_t k = threadIdx.x; k < a.width; k += 256) {
            const float n = s[k] * inverse, g = d_out[k] * a.weight[k];
            const float before = a.d_sum == nullptr ? 0.f : a.d_sum[row * a.width + k];
            a.d_x[row * a.width + k] = before + inverse * (g - n * dot);
        }
    }
}

// d_weight, one thread a column.
__global__ __launch_bounds__(256) void rms_norm_weight_grad_kernel(RmsNormBackwardArgs a) {
    const int64_t k = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (k >= a.width) return;
    float total = 0.f;
    for (int64_t row = 0; row < a.rows; ++row)
        total += a.d_out[row * a.width + k] * (a.sum[row * a.width + k] * a.inverse[row]);
    a.d_weight[k] += total;
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& a, hipStream_t stream) {
    const dim3 grid(unsigned(std::min<int64_t>(a.rows, 1 << 20)));
    if (a.codes != nullptr)
        hipLaunchKernelGGL(rms_norm_kernel<true>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(rms_norm_kernel<false>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_rms_norm_backward(const RmsNormBackwardArgs& a, hipStream_t stream) {
    if (a.d_weight != nullptr) {  // before d_x, which may be written over d_sum but over no input of this one
        hipLaunchKernelGGL(rms_norm_weight_grad_kernel, dim3(unsigned((a.width + 255) / 256)), dim3(256), 0, stream, a);
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    hipLaunchKernelGGL(rms_norm_grad_kernel, dim3(unsigned(std::min<int64_t>(a.rows, 1 << 20))), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sn
