// Products with 4-bit weights: y = scale x W (+ y) (+ bias), x [rows, inner] fp32,
// W one row of 4-bit blocks per output column (staleynet_fp4.h).
//
// Mathematics: a code times its block's power of two is exact in bf16, and an
// fp32 value is the exact sum of three bf16 values (fp4_device.h), so x W is three
// bf16 products, each exact, summed in fp32 by the matrix cores: where fp32 times
// fp32 takes six (gemm_f32.h). A 16-byte load is one block of one column, and its
// 32 codes become matrix operands with 16 conversions, scale included; nothing is
// multiplied per group. A workgroup whose x holds values under 2^-110, of which three parts may leave
// something, goes over its share a second time with that and adds the sums to its output. (Where none does, to look
// for them costs one OR a value: 1 x 8192 x 28672 29.6 us and 29.2 without, others under 1 %.)
//
// Few rows: a wave takes 16 C columns and a run of steps of 128 or 256 inner values (lane n, g:
// block g of the step for column n, or two); the workgroup's waves take consecutive runs, and add
// their sums through LDS in wave order. The parts of all rows, 3 rows (bf16: 1) to each row
// of x, are the rows of T operands of 16: at most 5 rows need one matrix instruction for
// 512 weights, 10 two, 16 three (bf16: 16 one, 32 two). The wave splits a step's x once, four values a lane, and
// passes the parts through LDS of its own. D = W x^T: a lane holds four consecutive
// columns of one part's sums. The codes and the x of the next step are on their way
// while this one's are used.
//   Scale bytes: a column's are 1 / 16 of its codes, and read byte by byte beside them they cost the
// address units as much as the codes do (1 x 8192 x 28672: 39 us, 28 without any; 31.5 so). So a
// lane reads 16 of one column at once, for the next steps, and the bytes
// pass through LDS.
//   What bounds it: W's bytes where there are many (1 x 8192 x 28672: 29.6 us, 125 MB at 4.2 TB/s), one
// launch where there are few (1 x 768 x 2304: 3.8 us), and at 16 rows (16 x 4096 x 14336: 15.4 to 16.1 us
// for 31 MB) the vector units, busy half the cycles with the split of x, which every workgroup does again.
// More rows: tiles staged in LDS, below.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"
#include "gemm_common.h"

namespace sn {
namespace fp4 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;        // inner values the matrix instructions take at once: four blocks
constexpr int kMaxWaves = 8;
constexpr int kScaleBytes = 1024;  // 16 of each lane

__device__ __forceinline__ void store_output(const ProductArgs& a, int64_t row, int64_t col, float sum) {
#pragma clang fp contract(off)
    float* y = a.y + row * a.cols + col;
    float out = a.scale * sum;
    if (a.accumulate) out = *y + out;
    if (a.bias != nullptr) out = out + a.bias[col];
    *y = out;
}
// A sum of what the parts of x left, to the output that theirs went to. A sum of 0 changes no bit.
__device__ __forceinline__ void add_rest(const ProductArgs& a, int64_t row, int64_t col, float sum) {
#pragma clang fp contract(off)
    if (sum != 0.f) a.y[row * a.cols + col] = a.y[row * a.cols + col] + a.scale * (sum * (1.f / kRestLift));
}

// How rows of x are read, four values from k (a multiple of 4) on, zeros where `ok` is not
// set or past `inner`. No branch, so that the loads of a step stay in flight: quads are whole
// (inner a multiple of 4), or the last ones are read from the row's end and shifted
// (rows start at any 4-byte address then; 16-byte loads need no more), or, under
// 4 values, one by one.
enum class Quads { kWhole, kShifted, kSingle };
template <Quads Q>
__device__ __forceinline__ f32x4 load4(const float* row, int64_t k, int64_t inner, bool ok) {
    typedef f32x4 f32x4_unaligned __attribute__((aligned(4)));
    const f32x4 zeros = {0.f, 0.f, 0.f, 0.f};
    f32x4 v = zeros;
    if constexpr (Q == Quads::kWhole) {
        v = ok && k < inner ? f32x4(*reinterpret_cast<const f32x4_unaligned*>(row + k)) : zeros;
    } else if constexpr (Q == Quads::kShifted) {
        const int64_t past = k + 4 - inner;  // values past the end, of these four
        const f32x4 got = *reinterpret_cast<const f32x4_unaligned*>(row + (past > 0 ? inner - 4 : k));
        const int shift = past <= 0 ? 0 : past >= 4 ? 4 : int(past);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = 0.f;
#pragma unroll
            for (int s = 0; s + e < 4; ++s) x = shift == s ? got[e + s] : x;
            v[e] = ok ? x : 0.f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ok && k + e < inner ? row[k + e] : 0.f;
    }
    return v;
}
Quads quads_of(int64_t inner) { return inner < 4 ? Quads::kSingle : inner % 4 == 0 ? Quads::kWhole : Quads::kShifted; }

// Four values as PARTS parts, packed in pairs (split_exact has the arithmetic), `left` noticing what three parts leave;
// or, where REST is set, that, lifted.
template <int PARTS, bool REST>
__device__ __forceinline__ void split_four(f32x4 x, uint32_t upper, u32x2 (&w)[PARTS], uint32_t& left) {
#pragma clang fp contract(off)
    if constexpr (PARTS == 1) {
        w[0] = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
    } else if constexpr (REST) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float a = rest_of(x[2 * i], upper), b = rest_of(x[2 * i + 1], upper);
            w[0][i] = upper_halves(a, b);
            w[1][i] = upper_halves(a - cut(a, upper), b - cut(b, upper));
            w[2][i] = 0;
        }
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
            const float a2 = a1[2 * i] - cut(a1[2 * i], upper), b2 = a1[2 * i + 1] - cut(a1[2 * i + 1], upper);
            notice(left, a2, b2);
            w[2][i] = upper_halves(a2, b2);
        }
    }
}

// Blocks of a column a lane takes in a step, as neighbours. Two make the four lanes of a column read 128 bytes of it,
// a cache line, at once; with one, the line is read for the first half and, where the codes in flight do not
// fit the caches, again for the other: 1 x 8192 x 28672 31.5 us, 29.3 with two (149 MB fetched for 125). With three
// operands, or fewer columns and so fewer codes in flight, the registers and the longer steps cost
// as much or more (16 x 4096 x 14336: 15.8 and 16.2 us; 1 x 4096 x 8192: 6.7 and 7.2).
constexpr int blocks_of_lane(int c, int t) { return c == 4 && t == 1 ? 2 : 1; }

// The columns' sums over the parts of x, to the output; or, where REST is set, over what those leave, added to it.
// At most 2 PAIRS rows, which PARTS (3, or 1 for x rounded to bf16) make at most 16 T. Returns whether the parts leave
// something in the workgroup.
template <int C, int T, int PAIRS, int PARTS, Quads Q, bool REST>
__device__ __forceinline__ bool few_rows_pass(const ProductArgs& a, char* lds, uint64_t& waves_left, int tid) {
    constexpr int J = blocks_of_lane(C, T);
    constexpr int STEP_BLOCKS = 4 * J;
    constexpr int PART_ROW = 2 * (kStep + 8);
    constexpr int SCALES = kScaleBytes;  // [four blocks of the run][column][block]
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int waves = blockDim.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const int64_t col0 = int64_t(blockIdx.x) * (16 * C);
    const int rows = int(a.rows);
    const int32_t blocks = int32_t(a.blocks), steps = (blocks + STEP_BLOCKS - 1) / STEP_BLOCKS;
    // The wave's run of steps.
    const int32_t each = (steps + waves - 1) / waves;
    const int32_t begin = wave * each, end = min(begin + each, steps);
    // The lane's columns, in blocks from the workgroup's first (32-bit byte offsets: inner < 2^25);
    // columns past the last read the last. Past a row's last block, where x is 0, the last
    // is read again.
    const int32_t last_col = int32_t(min(a.cols - col0, int64_t(16 * C))) - 1;
    uint32_t column[C];
#pragma unroll
    for (int c = 0; c < C; ++c) column[c] = uint32_t(min(16 * c + n, last_col)) * uint32_t(blocks);
    const uint8_t* const codes = a.codes + col0 * a.blocks * kBlockBytes;
    auto load = [&](int32_t step, u32x4 (&w)[J][C]) __attribute__((always_inline)) {
        const uint8_t* from = codes + int64_t(step) * (STEP_BLOCKS * kBlockBytes);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint32_t block = uint32_t(min(J * g + j, blocks - 1 - STEP_BLOCKS * step));
                w[j][c] = *reinterpret_cast<const u32x4*>(from + (column[c] + block) * uint32_t(kBlockBytes));
            }
    };
    // Scale bytes of RUN steps from `step` on: lane -> column lane % 16 C, 16 bytes of it. What
    // lies past the column's end is not used; past the buffer's, not read.
    constexpr int RUN = 16 / (C * J);
    const int scale_col = lane % (16 * C), scale_part = lane / (16 * C);
    const int64_t scale_row = (col0 + min(scale_col, last_col)) * a.blocks + 16 * scale_part;
    auto load_scales = [&](int32_t step) __attribute__((always_inline)) {
        typedef u32x4 u32x4_bytes __attribute__((aligned(1)));
        const int64_t at = scale_row + STEP_BLOCKS * step, total = a.cols * a.blocks;
        u32x4 s;
        if (at + 16 <= total) {
            s = *reinterpret_cast<const u32x4_bytes*>(a.scales + at);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) s[i] |= uint32_t(a.scales[min(at + 4 * i + b, total - 1)]) << (8 * b);
            }
        }
        return s;
    };

    // x of every Jth block of a step: four values of rows 2 pair + half, 32 lanes a row. Rows past the last are the
    // last again, written to its place.
    f32x4 x[PAIRS];
    const int half = lane >> 5, quad = 4 * (lane & 31);
    auto load_x = [&](int32_t step, int j) __attribute__((always_inline)) {
        const int64_t k = int64_t(step) * (STEP_BLOCKS * kBlock) + J * (quad & ~31) + 32 * j + (quad & 31);
#pragma unroll
        for (int pair = 0; pair < PAIRS; ++pair)
            x[pair] = load4<Q>(a.x + min(2 * pair + half, rows - 1) * a.inner, k, a.inner, true);
    };
    char* const wave_lds = lds + wave * (SCALES + PARTS * rows * PART_ROW);
    char* const parts = wave_lds + SCALES;
    int part_read[T];  // lanes past the last part read the last; their sums are not used
#pragma unroll
    for (int o = 0; o < T; ++o) part_read[o] = min(16 * o + n, PARTS * rows - 1) * PART_ROW + g * (2 * kBlock);

    f32x4 acc[C][T];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int o = 0; o < T; ++o) acc[c][o] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t left = 0;
    u32x4 next[J][C], next_scales;
    if (begin < end) {
        next_scales = load_scales(begin);
        load_x(begin, 0);
        load(begin, next);
    }
    for (int32_t step = begin; step < end; ++step) {
        const int32_t in_run = (step - begin) % RUN;
        if (in_run == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint32_t*>(wave_lds + ((4 * scale_part + i) * (16 * C) + scale_col) * 4) = next_scales[i];
            if (step + RUN < end) next_scales = load_scales(step + RUN);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            wave_lds_order();
#pragma unroll
            for (int pair = 0; pair < PAIRS; ++pair) {
                u32x2 split[PARTS];
                split_four<PARTS, REST>(x[pair], upper, split, left);
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    *reinterpret_cast<u32x2*>(parts + (q * rows + min(2 * pair + half, rows - 1)) * PART_ROW + 2 * quad) =
                        split[q];
            }
            wave_lds_order();
            u32x4 now[C];
#pragma unroll
            for (int c = 0; c < C; ++c) now[c] = next[j][c];
            if (j + 1 < J) {
                load_x(step, j + 1);
            } else if (step + 1 < end) {
                load_x(step + 1, 0);  // first: the next step splits x while its codes may be on their way
                load(step + 1, next);
            }
            float factor[C];
            const int32_t block = min(J * g + j, blocks - 1 - STEP_BLOCKS * step);
#pragma unroll
            for (int c = 0; c < C; ++c)
                factor[c] = factor_of(uint8_t(
                    wave_lds[((J * in_run + block / 4) * (16 * C) + 16 * c + n) * 4 + block % 4]));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x8 xf[T];
#pragma unroll
                for (int o = 0; o < T; ++o) xf[o] = *reinterpret_cast<const bf16x8*>(parts + part_read[o] + 16 * i);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const bf16x8 wf = fragment_of(now[c][i], factor[c]);
#pragma unroll
                    for (int o = 0; o < T; ++o)
                        acc[c][o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[o], acc[c][o], 0, 0, 0);
                }
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
    constexpr bool NOTICES = PARTS == 3 && !REST;
    if (NOTICES) {
        const bool any = __any(noticed(left));
        if (lane == 0) reinterpret_cast<uint8_t*>(&waves_left)[wave] = any;
    }
    __syncthreads();
    const uint64_t any_left = NOTICES ? waves_left & (~uint64_t(0) >> (64 - 8 * waves)) : 0;
    for (int e = tid; e < rows * 16 * C; e += blockDim.x) {
        const int row = e / (16 * C), c = e / 16 % C;
        const int64_t col = col0 + e % (16 * C);
        if (col >= a.cols) continue;
        const float* from = sums + c * (T * 256) + row * 16 + e % 16;
        float sum = 0.f;
        for (int w = 0; w < waves; ++w, from += WAVE_SUMS)
            sum += PARTS == 1 ? from[0] : from[0] + (from[16 * rows] + from[32 * rows]);
        if constexpr (REST)
            add_rest(a, row, col, sum);
        else
            store_output(a, row, col, sum);
    }
    return any_left != 0;
}

template <int C, int T, int PAIRS, int PARTS, Quads Q>
__global__ __launch_bounds__(64 * kMaxWaves) void few_rows_kernel(ProductArgs a) {
    // Scales and parts [wave][PARTS rows][kStep + 8], then the waves' sums [wave][C][T][16 parts][16 columns].
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ uint64_t waves_left;  // a byte a wave: whether the parts of its x leave something
    static_assert(kMaxWaves == 8, "a byte a wave");
    int tid = threadIdx.x;
    const bool any = few_rows_pass<C, T, PAIRS, PARTS, Q, false>(a, lds, waves_left, tid);
    if constexpr (PARTS == 3) {
        if (!any) return;     // of the workgroup
        __syncthreads();      // the parts take the sums' place
        asm("" : "+v"(tid));  // addresses worked out again, not kept in registers through the first pass
        few_rows_pass<C, T, PAIRS, PARTS, Q, true>(a, lds, waves_left, tid);
    }
}

// Many rows: tiles of 32 RT WR rows x 32 CT WC columns, WR x WC waves. x is split as it is
// staged in LDS, 64 inner values at a time, in two stages: while the matrix cores work
// on one, the next is split and written, and the one after is on its way in registers. A
// lane's 16 bytes of codes are a block of one column: 64 inner values of 32 columns a
// load. D = x W: a lane holds one column. Inner value 8 i + j of half h of a stage is
// element j of operand i of lanes h (as the block's words hold the codes).
//   2048 x 4096 x 4096 with fp32 inputs: 181 to 196 us, 350 to 380 TFLOP/s of products (1050 to 1140 of bf16 ones, matrix cores busy half the
// cycles; 130 us without any load, 150 without x's, and 175 to 177 with the next stage's split spread between the
// matrix instructions, which costs one part a tenth).
template <int RT, int CT, int WR, int WC, int PARTS, int SUBS>
struct TileShape {
    static constexpr int THREADS = 64 * WR * WC;
    static constexpr int ROWS = 32 * RT * WR, COLS = 32 * CT * WC;
    static constexpr int K = 64 * SUBS;     // of a stage
    static constexpr int ROW = 2 * K + 16;  // bytes of a staged row: 8 rows' reads on distinct banks
    static constexpr int PART = ROWS * ROW, STAGE = PARTS * PART;
    static constexpr int QUADS = ROWS * K / 4 / THREADS;  // of x a thread
    static_assert(QUADS * THREADS * 4 == ROWS * K, "whole quads");
};

// Slices of the inner dimension, `stages` stages each; with more than one the sums go to
// `sums` [slice][rows][cols], and another kernel adds them.
struct TileLaunch {
    int32_t tiles_m, tiles_n, slices, stages;
    float* sums;
};

// As few_rows_pass.
template <int RT, int CT, int WR, int WC, int PARTS, int SUBS, Quads Q, bool REST>
__device__ __forceinline__ void tile_pass(const ProductArgs& a, const TileLaunch& launch, char* stages,
                                          uint32_t* waves_left, int tid) {
    using S = TileShape<RT, CT, WR, WC, PARTS, SUBS>;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const uint32_t upper = upper_half_mask();
    int unused, slice, tile_m, tile_n;
    gemm::tile_coordinates(blockIdx.x, gridDim.x, launch.tiles_m, launch.tiles_n, launch.slices, unused, slice, tile_m,
                           tile_n);
    const int64_t row0 = int64_t(tile_m) * S::ROWS, col0 = int64_t(tile_n) * S::COLS;
    const int64_t wave_col = col0 + wave % WC * (32 * CT);
    const int wave_row = wave / WC * (32 * RT);
    // The slice's stages.
    const int32_t begin = slice * launch.stages;
    const int32_t end = min(begin + launch.stages, int32_t((a.blocks + 2 * SUBS - 1) / (2 * SUBS)));

    // x: QUADS of four values a thread, 16 SUBS threads to a row's stage.
    const int quad = 4 * (tid % (16 * SUBS)), first_row = tid / (16 * SUBS);
    constexpr int APART = S::THREADS / (16 * SUBS);
    f32x4 x[S::QUADS];
    auto load_x = [&](int32_t stage) __attribute__((always_inline)) {
        const int64_t k = int64_t(stage) * S::K + quad;
#pragma unroll
        for (int u = 0; u < S::QUADS; ++u) {
            const int64_t row = row0 + first_row + u * APART;
            x[u] = load4<Q>(a.x + (row < a.rows ? row : 0) * a.inner, k, a.inner, row < a.rows);
        }
    };
    uint32_t left = 0;
    auto store_x = [&](char* stage) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < S::QUADS; ++u) {
            u32x2 w[PARTS];
            split_four<PARTS, REST>(x[u], upper, w, left);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
                *reinterpret_cast<u32x2*>(stage + q * S::PART + (first_row + u * APART) * S::ROW + 2 * quad) = w[q];
        }
    };
    const int32_t blocks = int32_t(a.blocks);
    const int32_t last_col = int32_t(min(a.cols - col0, int64_t(S::COLS))) - 1;
    uint32_t column[CT];  // as in few_rows_kernel
#pragma unroll
    for (int c = 0; c < CT; ++c)
        column[c] = uint32_t(min(wave % WC * (32 * CT) + 32 * c + n, last_col)) * uint32_t(blocks);
    const uint8_t* const codes = a.codes + col0 * a.blocks * kBlockBytes;
    const uint8_t* const scales = a.scales + col0 * a.blocks;
    struct Weights {
        u32x4 w[SUBS][CT];
        uint32_t s[SUBS][CT];
    };
    auto load = [&](int32_t stage, Weights& x) __attribute__((always_inline)) {
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            const int32_t first = min(2 * (SUBS * stage + sub), blocks - 1);  // past the last in a partial stage
            const uint32_t block = uint32_t(min(h, blocks - 1 - first));
            const uint8_t* const from = codes + first * kBlockBytes;
            const uint8_t* const bytes = scales + first;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                x.w[sub][c] = *reinterpret_cast<const u32x4*>(from + (column[c] + block) * uint32_t(kBlockBytes));
                x.s[sub][c] = bytes[column[c] + block];
            }
        }
    };

    f32x16 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[r][c][e] = 0.f;

    Weights next;
    if (begin < end) {
        load(begin, next);
        load_x(begin);
        store_x(stages);
        if (begin + 1 < end) load_x(begin + 1);
    }
    __syncthreads();
    for (int32_t s = begin; s < end; ++s) {
        const Weights now = next;
        if (s + 1 < end) {
            load(s + 1, next);
            store_x(stages + (s + 1 - begin) % 2 * S::STAGE);
        }
        if (s + 2 < end) load_x(s + 2);
        const char* const from = stages + (s - begin) % 2 * S::STAGE + (wave_row + n) * S::ROW + 64 * h;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            float factor[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) factor[c] = factor_of(now.s[sub][c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x8 wf[CT];
#pragma unroll
                for (int c = 0; c < CT; ++c) wf[c] = fragment_of(now.w[sub][c][i], factor[c]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int q = PARTS - 1; q >= 0; --q) {
                        const bf16x8 xf = *reinterpret_cast<const bf16x8*>(from + q * S::PART + 32 * r * S::ROW +
                                                                           128 * sub + 16 * i);
#pragma unroll
                        for (int c = 0; c < CT; ++c)
                            acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xf, wf[c], acc[r][c], 0, 0, 0);
                    }
            }
        }
        __syncthreads();
    }
    if (PARTS == 3 && !REST) {
        const bool any = __any(noticed(left));
        if (lane == 0) waves_left[wave] = any;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int64_t col = wave_col + 32 * c + n;
        if (col >= a.cols) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int64_t row = row0 + wave_row + 32 * r + 8 * (e / 4) + 4 * h + e % 4;
                if (row >= a.rows) continue;
                float* const sum = &launch.sums[(slice * a.rows + row) * a.cols + col];
                if (REST && launch.slices > 1)
                    *sum = *sum + acc[r][c][e] * (1.f / kRestLift);
                else if (REST)
                    add_rest(a, row, col, acc[r][c][e]);
                else if (launch.slices > 1)
                    *sum = acc[r][c][e];
                else
                    store_output(a, row, col, acc[r][c][e]);
            }
    }
}

template <int RT, int CT, int WR, int WC, int PARTS, int SUBS, Quads Q>
__global__ __launch_bounds__(64 * WR * WC) void tile_kernel(ProductArgs a, TileLaunch launch) {
    __shared__ __attribute__((aligned(16))) char stages[2 * TileShape<RT, CT, WR, WC, PARTS, SUBS>::STAGE];
    __shared__ uint32_t waves_left[WR * WC];
    int tid = threadIdx.x;
    tile_pass<RT, CT, WR, WC, PARTS, SUBS, Q, false>(a, launch, stages, waves_left, tid);
    if constexpr (PARTS == 3) {
        __syncthreads();
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < WR * WC; ++w) any |= waves_left[w];
        if (any == 0) return;
        asm("" : "+v"(tid));
        tile_pass<RT, CT, WR, WC, PARTS, SUBS, Q, true>(a, launch, stages, waves_left, tid);
    }
}

// The slices' sums, added in slice order.
__global__ __launch_bounds__(256) void slice_sums_kernel(ProductArgs a, TileLaunch launch) {
    const int64_t total = a.rows * a.cols;
    for (int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x; e < total; e += int64_t(gridDim.x) * 256) {
        float sum = 0.f;
        for (int s = 0; s < launch.slices; ++s) sum += launch.sums[s * total + e];
        store_output(a, e / a.cols, e % a.cols, sum);
    }
}

template <int C, int T, int PAIRS, int PARTS>
hipError_t few_rows(const ProductArgs& a, hipStream_t stream) {
    const int64_t steps = (a.blocks + 4 * blocks_of_lane(C, T) - 1) / (4 * blocks_of_lane(C, T));
    const int waves = int(std::min<int64_t>(kMaxWaves, steps));
    const dim3 grid(unsigned((a.cols + 16 * C - 1) / (16 * C)));
    const size_t lds =
        waves * std::max<size_t>(C * T * 256 * sizeof(float), kScaleBytes + PARTS * a.rows * 2 * (kStep + 8));
    hipLaunchKernelGGL((quads_of(a.inner) == Quads::kWhole ? few_rows_kernel<C, T, PAIRS, PARTS, Quads::kWhole>
                                                           : few_rows_kernel<C, T, PAIRS, PARTS, Quads::kShifted>),
                       grid, dim3(64 * waves), lds, stream, a);
    return hipGetLastError();
}

template <int RT, int CT, int WR, int WC, int PARTS, int SUBS>
hipError_t tiles(ProductArgs a, int64_t wanted, hipStream_t stream) {
    using S = TileShape<RT, CT, WR, WC, PARTS, SUBS>;
    const int64_t tiles_n = (a.cols + S::COLS - 1) / S::COLS;
    const int64_t stages = (a.blocks + 2 * SUBS - 1) / (2 * SUBS);
    // As many rows a launch as its grid (under 2^32 threads) holds.
    const int64_t most = std::max<int64_t>(1, ((int64_t(1) << 32) - 1) / S::THREADS / tiles_n) * S::ROWS;
    const ProductArgs all = a;
    for (int64_t row = 0; row < all.rows; row += most) {
        a.rows = std::min(most, all.rows - row);
        a.x = all.x + row * all.inner;
        a.y = all.y + row * all.cols;
        TileLaunch launch;
        launch.tiles_m = int32_t((a.rows + S::ROWS - 1) / S::ROWS);
        launch.tiles_n = int32_t(tiles_n);
        const int64_t tiles = launch.tiles_m * tiles_n;
        const int64_t bytes = a.rows * a.cols * int64_t(sizeof(float));
        const int64_t room = a.workspace != nullptr ? int64_t(a.workspace_bytes) / bytes : 0;
        int64_t slices = std::min({wanted / tiles, stages * SUBS / 4, room});
        slices = std::max<int64_t>(1, slices);
        launch.stages = int32_t((stages + slices - 1) / slices);
        launch.slices = int32_t(std::max<int64_t>(1, (stages + launch.stages - 1) / std::max(1, launch.stages)));
        launch.sums = static_cast<float*>(a.workspace);
        auto* const kernel = quads_of(a.inner) == Quads::kWhole     ? tile_kernel<RT, CT, WR, WC, PARTS, SUBS, Quads::kWhole>
                             : quads_of(a.inner) == Quads::kShifted ? tile_kernel<RT, CT, WR, WC, PARTS, SUBS, Quads::kShifted>
                                                                    : tile_kernel<RT, CT, WR, WC, PARTS, SUBS, Quads::kSingle>;
        hipLaunchKernelGGL(kernel, dim3(unsigned(tiles * launch.slices)),
                           dim3(S::THREADS), 0, stream, a, launch);
        hipError_t err = hipGetLastError();
        if (err == hipSuccess && launch.slices > 1) {
            const int64_t groups = std::min<int64_t>((a.rows * a.cols + 255) / 256, int64_t(1) << 20);
            hipLaunchKernelGGL(slice_sums_kernel, dim3(unsigned(groups)), dim3(256), 0, stream, a, launch);
            err = hipGetLastError();
        }
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

// Tiles of 32 x 128 (27 KB of LDS, five workgroups a CU) hide their stages' latency best where
// there are few of them, and the inner dimension is sliced until they fill the CUs twice.
// Three parts: tiles of 128 x 256 (one a CU; 181 us at 2048 x 4096 x 4096 against 233) where the CUs' last
// round is full enough to keep that quarter: 2000 x 4096 x 4100 would be 346 us of them, 245 of small ones.
// One part: 64 x 128 where they fill the CUs twice (2000 x 4096 x 4100: 134 us, 187 of small ones and 222 of
// 128 x 256; 777 x 1001 x 1537, of which there are 169: 23 us against 15). Stages of 128 inner values there, whose
// three parts LDS has no room for (64: 141 and 19 us).
template <int PARTS>
hipError_t many_rows(const ProductArgs& a, hipStream_t stream) {
    const int64_t cus = a.cu_count;
    const auto up = [](int64_t x, int64_t unit) { return (x + unit - 1) / unit; };
    if constexpr (PARTS == 3) {
        const int64_t rounds = up(up(a.rows, 128) * up(a.cols, 256), cus);
        if (rounds * cus * (128 * 256) * 4 <= up(a.rows, 32) * 32 * up(a.cols, 128) * 128 * 5)
            return tiles<2, 2, 2, 4, PARTS, 1>(a, 0, stream);
    } else {
        if (up(a.rows, 64) * up(a.cols, 128) >= 2 * cus) return tiles<2, 1, 1, 4, PARTS, 2>(a, 0, stream);
    }
    return tiles<1, 1, 1, 4, PARTS, PARTS == 1 ? 2 : 1>(a, 2 * cus, stream);
}

// C = 4 tiles of 16 columns a wave use x's parts four times, but want 4 x as many columns: of 4096
// inner values, with 1 row and with 16, C = 1, 2 and 4 take
//   4096 columns:   5.3,  6.0,  7.6 us and 10.1, 10.8, 14.2 us
//   6144 columns:   7.0,  6.2,  7.7        18.4, 10.9, 14.3
//   12288 columns:  9.0,  9.3,  9.2        27.3, 20.5, 15.3
template <int T, int PAIRS, int PARTS>
hipError_t few_rows_by_columns(const ProductArgs& a, hipStream_t stream) {
    const int64_t tiles = (a.cols + 15) / 16;
    if (tiles >= 3 * a.cu_count) return few_rows<4, T, PAIRS, PARTS>(a, stream);
    if (4 * tiles >= 5 * a.cu_count) return few_rows<2, T, PAIRS, PARTS>(a, stream);
    return few_rows<1, T, PAIRS, PARTS>(a, stream);
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    if (a.rows == 0 || a.cols == 0) return hipSuccess;
    if (a.rows <= (a.bf16 ? 32 : 16) && a.inner >= 4) {
        // As few operands and loads of x as hold the rows (4096 x 8192: 2 rows 6.7 us, as 16 would be 11.3; one
        // rounded to bf16 6.1, and 7.4). 24 rows in bf16: 9.8 us at 4096 x 4096 and 14.8 at 4096 x 14336, where tiles take
        // 15.9 and 19.3; in fp32 they would be five operands or six, 18.6 and 47.7, tiles 17.4 and 25.1.
        if (a.bf16)
            return a.rows <= 2    ? few_rows_by_columns<1, 1, 1>(a, stream)
                   : a.rows <= 16 ? few_rows_by_columns<1, 8, 1>(a, stream)
                                  : few_rows_by_columns<2, 16, 1>(a, stream);
        return a.rows <= 2    ? few_rows_by_columns<1, 1, 3>(a, stream)
               : a.rows <= 5  ? few_rows_by_columns<1, 3, 3>(a, stream)
               : a.rows <= 10 ? few_rows_by_columns<2, 5, 3>(a, stream)
                              : few_rows_by_columns<3, 8, 3>(a, stream);
    }
    return a.bf16 ? many_rows<1>(a, stream) : many_rows<3>(a, stream);
}

}  // namespace fp4
}  // namespace sn
