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
// Few rows: a wave takes 16 C columns and steps of 128 inner values (lane n, g:
// block g of the step for column n). The workgroup's waves take the steps in turn,
// and add their sums through LDS in wave order. D = W x^T: a lane holds four
// consecutive columns of one row of y.
//   PACKED (at most 5 rows): the three parts of each row are rows of one operand, so
// one matrix instruction serves 512 weights; otherwise three do, for 16 rows at a
// time, R times.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kStep = 128;        // inner values of a step: four blocks
constexpr int kPackedRows = 5;    // 3 x 5 <= 16
constexpr int kMaxWaves = 16;

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

// One part (0, 1, 2) of eight values: `first` and `second` are the upper-half mask
// for the lanes that take the part after the first, after the second, else 0.
__device__ __forceinline__ bf16x8 one_part(const float (&x)[8], uint32_t first, uint32_t second) {
#pragma clang fp contract(off)
    float t[8];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x[i] - cut(x[i], first);
        t[i] = a - cut(a, second);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) odd |= __builtin_isunordered(t[i], t[i + 1]);
    if (__any(odd)) {  // infinities and NaN: their own first part, no others
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = t[i] != t[i] ? (first != 0 ? 0.f : quiet(t[i])) : t[i];
    }
    u32x4 w;
#pragma unroll
    for (int p = 0; p < 4; ++p) w[p] = upper_halves(t[2 * p], t[2 * p + 1]);
    return __builtin_bit_cast(bf16x8, w);
}

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

// PARTS: 3, or 1 for x rounded to bf16. PACKED: rows <= 5 and PARTS 3.
template <int C, int R, int PARTS, bool PACKED, bool VECTOR>
__global__ __launch_bounds__(64 * kMaxWaves) void few_rows_kernel(ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) float sums[];  // [wave][C][R][16 rows][16 columns]
    static_assert(!PACKED || (R == 1 && PARTS == 3), "packed parts share one operand");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const int64_t col0 = int64_t(blockIdx.x) * (16 * C);
    const int64_t row0 = int64_t(blockIdx.y) * (16 * R);
    const int64_t rows = min(a.rows - row0, int64_t(16 * R));
    const int64_t steps = (a.blocks + 3) / 4;

    // This lane's rows of x, and (packed) its part.
    const float* xr[R];
    bool row_ok[R];
    uint32_t first = 0, second = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        int64_t row = 16 * r + n;
        if (PACKED) {
            const int m = int(rows);
            const int part = n / m;
            row = n - part * m;
            row_ok[r] = part < 3;
            first = part > 0 ? upper : 0;
            second = part > 1 ? upper : 0;
        } else {
            row_ok[r] = row < rows;
        }
        xr[r] = a.x + (row0 + (row_ok[r] ? row : 0)) * a.inner;
    }
    int64_t block0[C];  // of this lane's columns; columns past the last read the last
#pragma unroll
    for (int c = 0; c < C; ++c) block0[c] = min(col0 + 16 * c + n, a.cols - 1) * a.blocks;

    f32x4 acc[C][R];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};

    u32x4 w[C];
    uint32_t s[C];
    auto load = [&](int64_t step) __attribute__((always_inline)) {
        const int64_t b = 4 * step + g;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            // Past the row's last block: zeros (x is 0 there too).
            const bool ok = b < a.blocks;
            const int64_t at = block0[c] + (ok ? b : 0);
            const u32x4 got = *reinterpret_cast<const u32x4*>(a.codes + at * kBlockBytes);
            const uint32_t byte = a.scales[at];
            w[c] = ok ? got : u32x4{0, 0, 0, 0};
            s[c] = ok ? byte : 127u;
        }
    };
    if (wave < steps) load(wave);
    for (int64_t step = wave; step < steps; step += waves) {
        u32x4 now[C];
        float factor[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            now[c] = w[c];
            factor[c] = factor_of(s[c]);
        }
        if (step + waves < steps) load(step + waves);
        const int64_t k = step * kStep + g * kBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 wf[C];
#pragma unroll
            for (int c = 0; c < C; ++c) wf[c] = fragment_of(now[c][i], factor[c]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v[8];
                load8<VECTOR>(xr[r], k + 8 * i, a.inner, row_ok[r], v);
                if (PACKED || PARTS == 1) {
                    const bf16x8 xf = PACKED ? one_part(v, first, second) : rounded8(v);
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        acc[c][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[c], xf, acc[c][r], 0, 0, 0);
                } else {
                    const SplitVector xf = split_exact(v, upper);
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int p = kParts - 1; p >= 0; --p)
                            acc[c][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[c], xf.part[p], acc[c][r], 0, 0, 0);
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
    const int tile_floats = C * R * 256;
    for (int e = threadIdx.x; e < tile_floats; e += blockDim.x) {
        const int col_in = e & 15, row_in = (e >> 4) & 15, r = (e >> 8) % R, c = (e >> 8) / R;
        const int64_t row = 16 * r + row_in, col = col0 + 16 * c + col_in;
        if (row >= rows || col >= a.cols) continue;
        float sum = 0.f;
        for (int w2 = 0; w2 < waves; ++w2) {
            const float* from = sums + w2 * tile_floats + e;
            sum += PACKED ? from[0] + (from[16 * rows] + from[32 * rows]) : from[0];
        }
        store_output(a, row0 + row, col, sum);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int C, int R, int PARTS, bool PACKED>
hipError_t few_rows(const ProductArgs& a, int waves, hipStream_t stream) {
    const bool vector = aligned16(a.x) && a.inner % 4 == 0;
    const dim3 grid(unsigned((a.cols + 16 * C - 1) / (16 * C)), unsigned((a.rows + 16 * R - 1) / (16 * R)));
    const size_t lds = size_t(waves) * C * R * 256 * sizeof(float);
    hipLaunchKernelGGL((vector ? few_rows_kernel<C, R, PARTS, PACKED, true>
                               : few_rows_kernel<C, R, PARTS, PACKED, false>),
                       grid, dim3(64 * waves), lds, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    if (a.rows == 0 || a.cols == 0) return hipSuccess;
    const int64_t steps = std::max<int64_t>(1, (a.blocks + 3) / 4);
    const int waves = int(std::min<int64_t>(8, steps));
    if (a.rows <= 16) {
        if (a.bf16) return few_rows<2, 1, 1, false>(a, waves, stream);
        if (a.rows <= kPackedRows) return few_rows<2, 1, 3, true>(a, waves, stream);
        return few_rows<2, 1, 3, false>(a, waves, stream);
    }
    const int many = int(std::min<int64_t>(4, steps));
    return a.bf16 ? few_rows<2, 4, 1, false>(a, many, stream) : few_rows<2, 4, 3, false>(a, many, stream);
}

}  // namespace fp4
}  // namespace sn
