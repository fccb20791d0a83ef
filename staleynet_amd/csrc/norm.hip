// The residual addition with the root-mean-square norm, and its gradients
// (staleynet_norm.h has the formulas).
//
// Bound by memory: 12 to 16 bytes a value against a handful of operations. 8192 x 4096 with a residual takes 97 us in fp32
// (5.5 TB/s) and 88 to 97 with an 8-bit output; its gradients, 8192 x 768, 21 us and 2 to 5 for d_weight's partial sums. A row
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

// Sum, inverse and y of eight values of row `row` from k on, and where they go: fp32 or 8-bit.
template <bool EIGHT>
__device__ __forceinline__ void store_results(const RmsNormArgs& a, int64_t row, int64_t k, const float (&s)[8],
                                              double inverse) {
    float w[8], y[8];
    load8(a.weight, k, a.width, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = float(double(s[i]) * double(w[i]) * inverse);
    if (a.sum != nullptr) store8(a.sum + row * a.width, k, a.width, s);
    if constexpr (EIGHT) {
        const int64_t blocks = blocks_of(a.width);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = k + i < a.width ? y[i] : 0.f;
        uint32_t scale;
        const u32x2 words = quantize8(y, scale);
        if (k < blocks * kBlock)
            store_block(a.codes + row * blocks * kBlock, a.scales + row * scale_stride(blocks), k / kBlock, int(k / 8 % 16),
                        blocks, words, scale);
    } else {
        store8(a.out + row * a.width, k, a.width, y);
    }
}
__device__ __forceinline__ void load_sum(const RmsNormArgs& a, int64_t row, int64_t k, float (&v)[8]) {
    load8(a.x + row * a.width, k, a.width, v);
    if (a.residual != nullptr) {
        float r[8];
        load8(a.residual + row * a.width, k, a.width, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] + r[i];
    }
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) v += __shfl_xor(v, step);
    return v;
}
__device__ __forceinline__ double inverse_of(const RmsNormArgs& a, double squares) {
    return 1.0 / sqrt(squares / double(a.width) + double(a.epsilon));
}

// THREADS threads a row, GROUP of a workgroup; VECTORS vectors of eight values a thread, held from the one read on.
template <int THREADS, int VECTORS, bool EIGHT>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void rms_norm_kernel(RmsNormArgs a) {
    constexpr int kGroup = THREADS > 256 ? THREADS : 256, kRows = kGroup / THREADS;
    __shared__ double partial[kGroup / 64];
    const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
    for (int64_t rows = blockIdx.x; rows * kRows < a.rows; rows += gridDim.x) {
        // Waves past the last row leave (they are rows of their own, and meet no barrier): the sum may be written over x, so
        // that no row is anyone else's to read.
        const int64_t row = rows * kRows + group;
        static_assert(kRows == 1 || THREADS == 64, "a wave that leaves skips the barriers");
        if (kRows > 1 && row >= a.rows) break;
        float s[VECTORS][8];
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) load_sum(a, row, 8 * (thread + THREADS * i), s[i]);
        double squares = 0;
#pragma unroll
        for (int i = 0; i < VECTORS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) squares += double(s[i][j]) * double(s[i][j]);
        squares = wave_sum(squares);
        if constexpr (THREADS > 64) {
            if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = squares;
            __syncthreads();
            squares = 0;
#pragma unroll
            for (int i = 0; i < THREADS / 64; ++i) squares += partial[group * (THREADS / 64) + i];
            __syncthreads();
        }
        const double inverse = inverse_of(a, squares);
        if (!EIGHT && a.inverse != nullptr && thread == 0) a.inverse[row] = float(inverse);
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) store_results<EIGHT>(a, row, 8 * (thread + THREADS * i), s[i], inverse);
    }
}

// Rows wider than a workgroup holds, read twice.
template <bool EIGHT>
__global__ __launch_bounds__(512) void rms_norm_wide_kernel(RmsNormArgs a) {
    __shared__ double partial[8];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        double squares = 0;
        for (int64_t k = 8 * threadIdx.x; k < a.width; k += 8 * 512) {
            float v[8];
            load_sum(a, row, k, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += double(v[i]) * double(v[i]);
        }
        squares = wave_sum(squares);
        if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = squares;
        __syncthreads();
        squares = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) squares += partial[i];
        __syncthreads();
        const double inverse = inverse_of(a, squares);
        if (!EIGHT && a.inverse != nullptr && threadIdx.x == 0) a.inverse[row] = float(inverse);
        for (int64_t k = 8 * threadIdx.x; k < blocks_of(a.width) * kBlock; k += 8 * 512) {
            float s[8];
            load_sum(a, row, k, s);
            store_results<EIGHT>(a, row, k, s, inverse);
        }
    }
}

// The gradients: THREADS threads a row, THREADS / 64 of a workgroup's waves; VECTORS vectors of eight values a thread, the
// same columns in every row it takes, so that d_weight's sums stay in its registers until the workgroup's are
// added up in LDS (in the order of its row groups) and left as its row of `partial`.
template <int THREADS, int VECTORS, bool WEIGHT>
__global__ __launch_bounds__(THREADS > 512 ? THREADS : 512) void rms_norm_grad_kernel(RmsNormBackwardArgs a,
                                                                                              float* partial) {
#pragma clang fp contract(off)
    constexpr int kGroup = THREADS > 512 ? THREADS : 512, kRows = kGroup / THREADS, kSpan = 8 * THREADS * VECTORS;
    __shared__ float dots[kGroup / 64];
    __shared__ __attribute__((aligned(16))) float sums[WEIGHT && kRows > 1 ? kSpan : 4];
    const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS, wave = threadIdx.x >> 6;
    // The weight is held too, but where 16 waves of two vectors leave no registers for it (128 a lane).
    constexpr bool kHeld = THREADS < 1024 || VECTORS == 1;
    float w[VECTORS][8], d_w[VECTORS][8];
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
        if (kHeld) load8(a.weight, 8 * (thread + THREADS * i), a.width, w[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) d_w[i][j] = 0.f;
    }
    const float by_width = 1.f / float(a.width);
    const int64_t groups = (a.rows + kRows - 1) / kRows;
    for (int64_t rows = blockIdx.x; rows < groups; rows += gridDim.x) {
        // The last group's rows past the end are the last row again, without its results; d_sum, which d_x may be written
        // over, is not theirs to read.
        const int64_t row = min(rows * kRows + group, a.rows - 1);
        const bool live = rows * kRows + group < a.rows;
        const float inverse = a.inverse[row];
        float n[VECTORS][8], g[VECTORS][8], before[VECTORS][8];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) {
            const int64_t k = 8 * (thread + THREADS * i);
            load8(a.sum + row * a.width, k, a.width, n[i]);
            load8(a.d_out + row * a.width, k, a.width, g[i]);
            if (a.d_sum != nullptr && live) load8(a.d_sum + row * a.width, k, a.width, before[i]);
        }
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) {
            if (!kHeld) load8(a.weight, 8 * (thread + THREADS * i), a.width, w[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                n[i][j] *= inverse;
                if (WEIGHT && live) d_w[i][j] += g[i][j] * n[i][j];
                g[i][j] *= w[i][j];
                dot += g[i][j] * n[i][j];
            }
        }
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) dot += __shfl_xor(dot, step);
        if constexpr (THREADS > 64) {
            if ((threadIdx.x & 63) == 0) dots[wave] = dot;
            __syncthreads();
            dot = 0.f;
#pragma unroll
            for (int i = 0; i < THREADS / 64; ++i) dot += dots[group * (THREADS / 64) + i];
            __syncthreads();
        }
        dot *= by_width;
        if (live) {
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                float d_x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    d_x[j] = (a.d_sum != nullptr ? before[i][j] : 0.f) + inverse * (g[i][j] - n[i][j] * dot);
                store8(a.d_x + row * a.width, 8 * (thread + THREADS * i), a.width, d_x);
            }
        }
    }
    if constexpr (WEIGHT) {
        if constexpr (kRows > 1) {
            for (int turn = 0; turn < kRows; ++turn) {
                if (group == turn) {
#pragma unroll
                    for (int i = 0; i < VECTORS; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            f32x4* at = reinterpret_cast<f32x4*>(&sums[8 * (thread + THREADS * i) + 4 * h]);
                            f32x4 v = turn == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : *at;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                v[j] += d_w[i][4 * h + j];
                                d_w[i][4 * h + j] = v[j];
                            }
                            *at = v;
                        }
                }
                __syncthreads();
            }
        }
        if (group == kRows - 1) {
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                const int64_t k = 8 * (thread + THREADS * i);
                if (partial != nullptr) {
                    store8(partial + int64_t(blockIdx.x) * a.width, k, a.width, d_w[i]);
                } else {  // the only workgroup
                    float before[8];
                    load8(a.d_weight, k, a.width, before);
#pragma unroll
                    for (int j = 0; j < 8; ++j) before[j] += d_w[i][j];
                    store8(a.d_weight, k, a.width, before);
                }
            }
        }
    }
}

// d_weight from `count` rows of partial sums: 64 columns a workgroup, each of its 16 waves every sixteenth row.
__global__ __launch_bounds__(1024) void rms_norm_weight_grad_kernel(const float* partial, int64_t count, int64_t width,
                                                                    float* d_weight) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t k = int64_t(blockIdx.x) * 64 + lane;
    float total = 0.f;
    if (k < width) {
#pragma unroll 8
        for (int64_t row = wave; row < count; row += 16) total += partial[row * width + k];
    }
    sums[wave][lane] = total;
    __syncthreads();
    if (wave == 0 && k < width) {
        total = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) total += sums[i][lane];
        d_weight[k] += total;
    }
}

// Rows wider than a workgroup holds: d_x, one workgroup a row, read twice.
__global__ __launch_bounds__(512) void rms_norm_wide_grad_kernel(RmsNormBackwardArgs a) {
    __shared__ float dots[8];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float inverse = a.inverse[row];
        const float *s = a.sum + row * a.width, *d_out = a.d_out + row * a.width;
        float dot = 0.f;
        for (int64_t k = 8 * threadIdx.x; k < a.width; k += 8 * 512) {
            float n[8], g[8], w[8];
            load8(s, k, a.width, n);
            load8(d_out, k, a.width, g);
            load8(a.weight, k, a.width, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) dot += g[j] * w[j] * (n[j] * inverse);
        }
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) dot += __shfl_xor(dot, step);
        if ((threadIdx.x & 63) == 0) dots[threadIdx.x >> 6] = dot;
        __syncthreads();
        dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) dot += dots[i];
        dot *= 1.f / float(a.width);
        __syncthreads();
        for (int64_t k = 8 * threadIdx.x; k < a.width; k += 8 * 512) {
            float n[8], g[8], w[8], d_x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            load8(s, k, a.width, n);
            load8(d_out, k, a.width, g);
            load8(a.weight, k, a.width, w);
            if (a.d_sum != nullptr) load8(a.d_sum + row * a.width, k, a.width, d_x);
#pragma unroll
            for (int j = 0; j < 8; ++j) d_x[j] += inverse * (g[j] * w[j] - n[j] * inverse * dot);
            store8(a.d_x + row * a.width, k, a.width, d_x);
        }
    }
}

// And their d_weight, or any width's where the workspace holds no partial sums: 64 columns a workgroup, each of its 16
// waves a sixteenth of the rows.
__global__ __launch_bounds__(1024) void rms_norm_direct_weight_grad_kernel(RmsNormBackwardArgs a) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t k = int64_t(blockIdx.x) * 64 + lane;
    float total = 0.f;
    if (k < a.width) {
#pragma unroll 4
        for (int64_t row = wave; row < a.rows; row += 16)
            total += a.d_out[row * a.width + k] * (a.sum[row * a.width + k] * a.inverse[row]);
    }
    sums[wave][lane] = total;
    __syncthreads();
    if (wave == 0 && k < a.width) {
        total = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) total += sums[i][lane];
        a.d_weight[k] += total;
    }
}

template <int THREADS, int VECTORS>
hipError_t launch_grad(const RmsNormBackwardArgs& a, hipStream_t stream) {
    constexpr int kGroup = THREADS > 512 ? THREADS : 512, kRows = kGroup / THREADS;
    const int64_t groups = (a.rows + kRows - 1) / kRows;
    // Workgroups to fill the GPU with waves, four a SIMD (two of a row each: 8192 x 768 22.7 us against 26.0 with four, whose
    // partial sums are twice as many), and no more partial sums than the workspace holds.
    int64_t grid = std::min<int64_t>(groups, (THREADS == 64 ? 512 : 1024) / kGroup * a.cu_count);
    const dim3 block(kGroup);
    if (a.d_weight == nullptr) {
        hipLaunchKernelGGL((rms_norm_grad_kernel<THREADS, VECTORS, false>), dim3(unsigned(grid)), block, 0, stream, a, nullptr);
        return hipGetLastError();
    }
    if (grid == 1) {
        hipLaunchKernelGGL((rms_norm_grad_kernel<THREADS, VECTORS, true>), dim3(1), block, 0, stream, a, nullptr);
        return hipGetLastError();
    }
    const int64_t held = int64_t(a.workspace_bytes) / (4 * a.width);
    const dim3 columns(unsigned((a.width + 63) / 64));
    if (held < std::min<int64_t>(grid, 64)) {  // too few to be worth it
        hipLaunchKernelGGL(rms_norm_direct_weight_grad_kernel, columns, dim3(1024), 0, stream, a);
        hipLaunchKernelGGL((rms_norm_grad_kernel<THREADS, VECTORS, false>), dim3(unsigned(grid)), block, 0, stream, a, nullptr);
        return hipGetLastError();
    }
    grid = std::min(grid, held);
    hipLaunchKernelGGL((rms_norm_grad_kernel<THREADS, VECTORS, true>), dim3(unsigned(grid)), block, 0, stream, a, a.workspace);
    hipLaunchKernelGGL(rms_norm_weight_grad_kernel, columns, dim3(1024), 0, stream, a.workspace, grid, a.width, a.d_weight);
    return hipGetLastError();
}

template <int THREADS, int VECTORS, bool EIGHT>
hipError_t launch_rows(const RmsNormArgs& a, hipStream_t stream) {
    constexpr int kGroup = THREADS > 256 ? THREADS : 256, kRows = kGroup / THREADS;
    const int64_t groups = std::min<int64_t>((a.rows + kRows - 1) / kRows, 1 << 20);
    hipLaunchKernelGGL((rms_norm_kernel<THREADS, VECTORS, EIGHT>), dim3(unsigned(groups)), dim3(kGroup), 0, stream, a);
    return hipGetLastError();
}
template <bool EIGHT>
hipError_t launch_forward(const RmsNormArgs& a, hipStream_t stream) {
    if (a.width <= 512) return launch_rows<64, 1, EIGHT>(a, stream);
    // A row a wave where there are rows for all of them: with few, four waves leave sooner (1 x 768: 3.3 us against 4.7).
    if (a.width <= 1024 && a.rows > 4 * a.cu_count) return launch_rows<64, 2, EIGHT>(a, stream);
    if (a.width <= 2048) return launch_rows<256, 1, EIGHT>(a, stream);
    if (a.width <= 4096) return launch_rows<512, 1, EIGHT>(a, stream);
    if (a.width <= 8192) return launch_rows<1024, 1, EIGHT>(a, stream);
    if (a.width <= 16384) return launch_rows<1024, 2, EIGHT>(a, stream);
    const dim3 grid(unsigned(std::min<int64_t>(a.rows, 1 << 20)));
    hipLaunchKernelGGL(rms_norm_wide_kernel<EIGHT>, grid, dim3(512), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& a, hipStream_t stream) {
    return a.codes != nullptr ? launch_forward<true>(a, stream) : launch_forward<false>(a, stream);
}

hipError_t launch_rms_norm_backward(const RmsNormBackwardArgs& a, hipStream_t stream) {
    if (a.width <= 512) return launch_grad<64, 1>(a, stream);
    if (a.width <= 1024) return launch_grad<64, 2>(a, stream);
    if (a.width <= 2048) return launch_grad<256, 1>(a, stream);
    if (a.width <= 4096) return launch_grad<512, 1>(a, stream);
    if (a.width <= 8192) return launch_grad<1024, 1>(a, stream);
    if (a.width <= 16384) return launch_grad<1024, 2>(a, stream);
    if (a.d_weight != nullptr)  // before d_x, which may be written over d_sum but over no input of this one
        hipLaunchKernelGGL(rms_norm_direct_weight_grad_kernel, dim3(unsigned((a.width + 63) / 64)), dim3(1024), 0, stream, a);
    hipLaunchKernelGGL(rms_norm_wide_grad_kernel, dim3(unsigned(std::min<int64_t>(a.rows, 1 << 20))), dim3(512), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sn
