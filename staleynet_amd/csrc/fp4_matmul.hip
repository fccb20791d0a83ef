// Products with 4-bit weights: y = scale x W (+ y) (+ bias), x [rows, inner] fp32,
// W one row of 4-bit blocks per output column (staleynet_fp4.h).
//
// Mathematics: a code times its block's power of two is exact in bf16, and an
// fp32 value is the exact sum of three bf16 values (fp4_device.h), so x W is three
// bf16 products, each exact, summed in fp32 by the matrix cores: where fp32 times
// fp32 takes six (gemm_f32.h). A 16-byte load is one block of one column, and its
// 32 codes become matrix operands with 16 conversions, scale included; nothing is
// multiplied per group.
//
// Few rows: a wave takes 16 C columns and steps of 128 inner values (lane n, g: block g
// of the step for column n). The workgroup's waves take the steps in turn, and add their
// sums through LDS in wave order. The parts of all rows, 3 rows (bf16: 1) to each row of x, are
// the rows of T operands of 16: at most 5 rows need one matrix instruction for 512
// weights, 10 two, 16 three. The wave splits a step's x once, four values a lane, and
// passes the parts through LDS of its own. D = W x^T: a lane holds four consecutive
// columns of one part's sums. The codes and the x of the next step are on their way
// while this one's are used.
// More rows: 16 R rows to a wave, x split as it is used.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kStep = 128;        // inner values of a step: four blocks
constexpr int kMaxWaves = 8;

__device__ __forceinline__ bf16x8 rounded8(const float (&x)[8]) {
    const u32x4 w = {pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7])};
    return __builtin_bit_cast(bf16x8, w);
}

__device__ __forceinline__ void store_output(const ProductArgs& a, int64_t row, int64_t col, float sum) {
#pragma clang fp contract(off)
    float* y = a.y + row * a.cols + col;
    float out = a.scale * sum;
    if (a.accumulate) out = *y + out;
    if (a.bias != nullptr) out = out + a.bias[col];
    *y = out;
}

// A step's weights: per column tile the lane's block, 16 bytes of codes and the scale byte.
template <int C>
struct StepWeights {
    u32x4 w[C];
    uint32_t s[C];
};
template <int C>
__device__ __forceinline__ void load_weights(const ProductArgs& a, const int64_t (&block0)[C], int64_t block,
                                             StepWeights<C>& x) {
    // Past the row's last block: zeros (x is 0 there too).
    const bool ok = block < a.blocks;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t at = block0[c] + (ok ? block : 0);
        const u32x4 got = *reinterpret_cast<const u32x4*>(a.codes + at * kBlockBytes);
        const uint32_t byte = a.scales[at];
        x.w[c] = ok ? got : u32x4{0, 0, 0, 0};
        x.s[c] = ok ? byte : 127u;
    }
}

// Four values as PARTS parts, packed in pairs (split_exact has the arithmetic).
template <int PARTS>
__device__ __forceinline__ void split_four(const float (&x)[4], uint32_t upper, u32x2 (&w)[PARTS]) {
#pragma clang fp contract(off)
    if constexpr (PARTS == 1) {
        w[0] = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
    } else {
        float a[4], a1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = x[i];
            a1[i] = a[i] - cut(a[i], upper);
        }
        if (__any(__builtin_isunordered(a1[0], a1[1]) || __builtin_isunordered(a1[2], a1[3]))) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = quiet(a[i]);
                a1[i] = a1[i] != a1[i] ? 0.f : a1[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[0][i] = upper_halves(a[2 * i], a[2 * i + 1]);
            w[1][i] = upper_halves(a1[2 * i], a1[2 * i + 1]);
            w[2][i] = upper_halves(a1[2 * i] - cut(a1[2 * i], upper), a1[2 * i + 1] - cut(a1[2 * i + 1], upper));
        }
    }
}

// At most 16 T / PARTS rows. PARTS: 3, or 1 for x rounded to bf16.
template <int C, int T, int PARTS, bool VECTOR>
__global__ __launch_bounds__(64 * kMaxWaves) void few_rows_kernel(ProductArgs a) {
    // Parts [wave][PARTS rows][kStep + 8], then the waves' sums [wave][C][T][16 parts][16 columns].
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int PART_ROW = 2 * (kStep + 8);
    constexpr int PAIRS = (16 * T / PARTS + 1) / 2;  // of rows: 32 lanes load a row's step
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const int64_t col0 = int64_t(blockIdx.x) * (16 * C);
    const int rows = int(a.rows);
    const int64_t steps = (a.blocks + 3) / 4;
    int64_t block0[C];  // of this lane's columns; columns past the last read the last
#pragma unroll
    for (int c = 0; c < C; ++c) block0[c] = min(col0 + 16 * c + n, a.cols - 1) * a.blocks;

    f32x4 acc[C][T];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int o = 0; o < T; ++o) acc[c][o] = f32x4{0.f, 0.f, 0.f, 0.f};

    // x of a step: four values of rows 2 pair + half.
    float x[PAIRS][4];
    const int half = lane >> 5, quad = 4 * (lane & 31);
    auto load_x = [&](int64_t step) __attribute__((always_inline)) {
        const int64_t k = step * kStep + quad;
#pragma unroll
        for (int pair = 0; pair < PAIRS; ++pair) {
            if (2 * pair >= rows) break;
            const int row = 2 * pair + half;
            const float* from = a.x + row * a.inner + k;
            if (VECTOR) {
                const f32x4 v = row < rows && k < a.inner ? *reinterpret_cast<const f32x4*>(from) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) x[pair][e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[pair][e] = row < rows && k + e < a.inner ? from[e] : 0.f;
            }
        }
    };
    char* const parts = lds + wave * (PARTS * rows * PART_ROW);
    int part_read[T];  // lanes past the last part read the last; their sums are not used
#pragma unroll
    for (int o = 0; o < T; ++o) part_read[o] = min(16 * o + n, PARTS * rows - 1) * PART_ROW + g * (2 * kBlock);

    StepWeights<C> next;
    if (wave < steps) {
        load_weights<C>(a, block0, 4 * wave + g, next);
        load_x(wave);
    }
    for (int64_t step = wave; step < steps; step += waves) {
        const StepWeights<C> now = next;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int pair = 0; pair < PAIRS; ++pair) {
            if (2 * pair >= rows) break;
            u32x2 w[PARTS];
            split_four<PARTS>(x[pair], upper, w);
            const int row = 2 * pair + half;
            if (row < rows)
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    *reinterpret_cast<u32x2*>(parts + (q * rows + row) * PART_ROW + 2 * quad) = w[q];
        }
        __builtin_amdgcn_wave_barrier();
        if (step + waves < steps) {
            load_weights<C>(a, block0, 4 * (step + waves) + g, next);
            load_x(step + waves);
        }
        float factor[C];
#pragma unroll
        for (int c = 0; c < C; ++c) factor[c] = factor_of(now.s[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 xf[T];
#pragma unroll
            for (int o = 0; o < T; ++o) xf[o] = *reinterpret_cast<const bf16x8*>(parts + part_read[o] + 16 * i);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const bf16x8 wf = fragment_of(now.w[c][i], factor[c]);
#pragma unroll
                for (int o = 0; o < T; ++o)
                    acc[c][o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[o], acc[c][o], 0, 0, 0);
            }
        }
    }
    __syncthreads();  // the sums take the parts' place
    float* const sums = reinterpret_cast<float*>(lds);
    constexpr int WAVE_SUMS = C * T * 256;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int o = 0; o < T; ++o)
            *reinterpret_cast<f32x4*>(&sums[wave * WAVE_SUMS + (c * T + o) * 256 + n * 16 + 4 * g]) = acc[c][o];
    __syncthreads();
    for (int e = threadIdx.x; e < rows * 16 * C; e += blockDim.x) {
        const int row = e / (16 * C), c = e / 16 % C;
        const int64_t col = col0 + e % (16 * C);
        if (col >= a.cols) continue;
        const float* from = sums + c * (T * 256) + row * 16 + e % 16;
        float sum = 0.f;
        for (int w = 0; w < waves; ++w, from += WAVE_SUMS)
            sum += PARTS == 1 ? from[0] : from[0] + (from[16 * rows] + from[32 * rows]);
        store_output(a, row, col, sum);
    }
}

// Eight values of a row of x from k on, zeros past `inner`.
template <bool VECTOR>
__device__ __forceinline__ void load8(const float* row, int64_t k, int64_t inner, bool ok, float (&v)[8]) {
    if (VECTOR && ok && k + 8 <= inner) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(row + k), hi = *reinterpret_cast<const f32x4*>(row + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ok && k + i < inner ? row[k + i] : 0.f;
    }
}

// 16 R rows a workgroup.
template <int C, int R, int PARTS, bool VECTOR>
__global__ __launch_bounds__(64 * kMaxWaves) void rows_kernel(ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* const sums = reinterpret_cast<float*>(lds);  // [wave][C][R][16 rows][16 columns]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const int64_t col0 = int64_t(blockIdx.x) * (16 * C);
    const int64_t row0 = int64_t(blockIdx.y) * (16 * R);
    const int64_t rows = min(a.rows - row0, int64_t(16 * R));
    const int64_t steps = (a.blocks + 3) / 4;
    const float* xr[R];
    bool row_ok[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        row_ok[r] = 16 * r + n < rows;
        xr[r] = a.x + (row0 + (row_ok[r] ? 16 * r + n : 0)) * a.inner;
    }
    int64_t block0[C];
#pragma unroll
    for (int c = 0; c < C; ++c) block0[c] = min(col0 + 16 * c + n, a.cols - 1) * a.blocks;
    f32x4 acc[C][R];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    StepWeights<C> next;
    if (wave < steps) load_weights<C>(a, block0, 4 * wave + g, next);
    for (int64_t step = wave; step < steps; step += waves) {
        const StepWeights<C> now = next;
        if (step + waves < steps) load_weights<C>(a, block0, 4 * (step + waves) + g, next);
        float factor[C];
#pragma unroll
        for (int c = 0; c < C; ++c) factor[c] = factor_of(now.s[c]);
        const int64_t k = step * kStep + g * kBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 wf[C];
#pragma unroll
            for (int c = 0; c < C; ++c) wf[c] = fragment_of(now.w[c][i], factor[c]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v[8];
                load8<VECTOR>(xr[r], k + 8 * i, a.inner, row_ok[r], v);
                if (PARTS == 1) {
                    const bf16x8 xf = rounded8(v);
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        acc[c][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[c], xf, acc[c][r], 0, 0, 0);
                } else {
                    const SplitVector xf = split_exact(v, upper);
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int q = kParts - 1; q >= 0; --q)
                            acc[c][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[c], xf.part[q], acc[c][r], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r)
            *reinterpret_cast<f32x4*>(&sums[((wave * C + c) * R + r) * 256 + n * 16 + 4 * g]) = acc[c][r];
    __syncthreads();
    constexpr int tile_floats = C * R * 256;
    for (int e = threadIdx.x; e < tile_floats; e += blockDim.x) {
        const int64_t row = 16 * ((e >> 8) % R) + ((e >> 4) & 15), col = col0 + 16 * ((e >> 8) / R) + (e & 15);
        if (row >= rows || col >= a.cols) continue;
        float sum = 0.f;
        for (int w = 0; w < waves; ++w) sum += sums[w * tile_floats + e];
        store_output(a, row0 + row, col, sum);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int C, int T, int PARTS>
hipError_t few_rows(const ProductArgs& a, int waves, hipStream_t stream) {
    const bool vector = aligned16(a.x) && a.inner % 4 == 0;
    const dim3 grid(unsigned((a.cols + 16 * C - 1) / (16 * C)));
    const size_t lds = waves * std::max<size_t>(C * T * 256 * sizeof(float), PARTS * a.rows * 2 * (kStep + 8));
    hipLaunchKernelGGL((vector ? few_rows_kernel<C, T, PARTS, true> : few_rows_kernel<C, T, PARTS, false>), grid,
                       dim3(64 * waves), lds, stream, a);
    return hipGetLastError();
}

template <int C, int R, int PARTS>
hipError_t many_rows(const ProductArgs& a, int waves, hipStream_t stream) {
    const bool vector = aligned16(a.x) && a.inner % 4 == 0;
    const dim3 grid(unsigned((a.cols + 16 * C - 1) / (16 * C)), unsigned((a.rows + 16 * R - 1) / (16 * R)));
    const size_t lds = size_t(waves) * C * R * 256 * sizeof(float);
    hipLaunchKernelGGL((vector ? rows_kernel<C, R, PARTS, true> : rows_kernel<C, R, PARTS, false>), grid,
                       dim3(64 * waves), lds, stream, a);
    return hipGetLastError();
}

template <int T, int PARTS>
hipError_t few_rows_by_columns(const ProductArgs& a, int waves, hipStream_t stream) {
    const int64_t tiles = (a.cols + 15) / 16;
    if (tiles >= 3 * a.cu_count) return few_rows<4, T, PARTS>(a, waves, stream);
    if (4 * tiles >= 5 * a.cu_count) return few_rows<2, T, PARTS>(a, waves, stream);
    return few_rows<1, T, PARTS>(a, waves, stream);
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    if (a.rows == 0 || a.cols == 0) return hipSuccess;
    const int64_t steps = std::max<int64_t>(1, (a.blocks + 3) / 4);
    const int waves = int(std::min<int64_t>(8, steps));
    if (a.bf16 && a.rows <= 16) return few_rows_by_columns<1, 1>(a, waves, stream);
    if (!a.bf16 && a.rows <= 5) return few_rows_by_columns<1, 3>(a, waves, stream);
    if (!a.bf16 && a.rows <= 10) return few_rows_by_columns<2, 3>(a, waves, stream);
    if (!a.bf16 && a.rows <= 16) return few_rows_by_columns<3, 3>(a, waves, stream);
    const int many = int(std::min<int64_t>(4, steps));
    return a.bf16 ? many_rows<2, 4, 1>(a, many, stream) : many_rows<2, 4, 3>(a, many, stream);
}

}  // namespace fp4
}  // namespace sn
