// Products of two 8-bit operands (sn_matmul_fp8; staleynet_fp8.h has the format):
//   y = scale * X W (+ y) (+ bias)
// (sizes below are rows x inner dimension x columns)
//
// A code times its block's factor is exact in bf16, and a product of two such
// values is exact in fp32, so fragments are codes converted in registers and
// multiplied by the bf16 matrix instructions, which sum in fp32. The 8-bit
// matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4 and the 16x16x32 forms)
// would run twice as fast, but were measured to align the products of eight
// neighbouring k to the largest of them and to cut off what lies more than 13
// bits below: sums of 128 products of random codes come out up to 2^-11.2 of the
// largest product wrong (the bf16 instructions' 2^-19.9), where fp32 sums are
// asked for.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "fp8_device.h"
#include "fp8_internal.h"

namespace sn {
namespace fp8 {
namespace {

// An output value from its sum.
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t place, int64_t col, float sum) {
    float v = a.scale * sum;
    if (a.accumulate) v = a.y[place] + v;
    if (a.bias != nullptr) v = v + a.bias[col];
    a.y[place] = v;
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_pointer;

// Values of a tile's step along the inner dimension: half a block.
constexpr int kStep = 64;

// Waits until at most PENDING of this wave's vector-memory instructions are
// outstanding (vmcnt; expcnt and lgkmcnt left at their maxima).
template <int PENDING>
__device__ __forceinline__ void wait_loads() {
    static_assert(PENDING >= 0 && PENDING < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (PENDING & 15) | ((PENDING >> 4) << 14));
}
// A barrier that leaves the loads of later steps in flight (a fence would wait for them); this wave's reads of LDS are done.
__device__ __forceinline__ void stage_barrier() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); vmcnt and expcnt left at their maxima
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Few rows: bound by reading the weights once. A workgroup takes 16 C columns, its W waves the blocks of the inner
// dimension in turn, each with LDS of its own for two blocks; their sums are added up in the end, in the order of
// the waves. The columns are the left operand of the matrix instructions, up to 16 R rows of x the right one. Lane l
// holds row (or column) l % 16 of a fragment and bytes 32 (l / 16) .. + 31 of a block; the four 32-deep instructions of
// a block take eight of them each, for both operands the same. Loading them so from memory would have each lane of a
// load in another line than its neighbours, 64 lookups an instruction; through LDS eight lanes load a line together
// (16 x 14336 x 4096, weights
// from HBM: 14.9 us, 3.9 TB/s, against 20.4).
template <int R, int C, int W>
__device__ __forceinline__ void multiply_few(const ProductArgs& a, int slices) {
    constexpr int F = C + R, kPerWave = F * 16 * int(kBlock), kLoads = 2 * F;  // of eight rows each, a block
    // An array a stage, named by constants, so that the compiler knows which stage a read of LDS may depend on.
    __shared__ __attribute__((aligned(16))) uint8_t stage0[W * kPerWave], stage1[W * kPerWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint8_t* const stages[2] = {stage0 + wave * kPerWave, stage1 + wave * kPerWave};
    const int group = int(blockIdx.x) / slices, slice = int(blockIdx.x) - group * slices;
    const int64_t col0 = int64_t(group) * (16 * C);
    const int blocks = int(a.blocks), stride = W * slices, first = slice * W + wave;
    const uint32_t row_bytes = uint32_t(a.blocks * kBlock);
    const int64_t scale_row = scale_stride(a.blocks);
    // Columns and rows past the last are the last again; their results are not stored.
    const int last_col = int(min(int64_t(16 * C), a.cols - col0)) - 1, last_row = int(a.rows) - 1;
    const uint8_t* w = a.w + col0 * row_bytes;
    uint32_t from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = 8 * i + lane / 8;
        from[i] = uint32_t(i < 2 * C ? min(r, last_col) : min(r - 16 * C, last_row)) * row_bytes +
                  16 * ((lane % 8) ^ ((r >> 1) & 7));  // the chunk that slot l % 8 of the row holds
    }
    // A block's loads; of one past the last, of no bytes, which keeps the count of loads, and so the waits, fixed.
    auto load = [&](uint8_t* stage, int b) {
        const int bytes = __builtin_amdgcn_readfirstlane((b - blocks) >> 31);  // all, or none
        const __amdgpu_buffer_rsrc_t left = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(w), 0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t right = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.x), 0, bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(i < 2 * C ? left : right, (lds_pointer)(stage + 1024 * i), 16, from[i],
                                                     int(kBlock) * min(b, blocks), 0, 0);
    };
    // The scale bytes of four of this wave's blocks, from b on: lane l's are row (or column) l % 16's of block l / 16 of them.
    const uint8_t* scales[F];
#pragma unroll
    for (int i = 0; i < F; ++i)
        scales[i] = i < C ? a.w_scales + (col0 + min(16 * i + lane % 16, last_col)) * scale_row
                          : a.x_scales + min(16 * (i - C) + lane % 16, last_row) * scale_row;
    uint32_t next[F];
    auto load_scales = [&](int b) {
        const int at = min(b + stride * (lane / 16), blocks - 1);
#pragma unroll
        for (int i = 0; i < F; ++i) next[i] = scales[i][at];
    };
    // The 16 rows of a read are in different banks.
    const int at = lane % 16 * int(kBlock) + 16 * ((lane / 16 * 2) ^ (lane % 16 >> 1));
    f32x4 acc[C][R];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < R; ++i) acc[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (first < blocks) {
        load_scales(first);
        load(stages[0], first);
        load(stages[1], first + stride);
        for (int b0 = first; b0 < blocks; b0 += 4 * stride) {
            float factors[F];
#pragma unroll
            for (int i = 0; i < F; ++i) factors[i] = factor_of(next[i]);
            load_scales(b0 + 4 * stride);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int b = b0 + u * stride;
                if (b >= blocks) break;
                uint8_t* const stage = stages[u % 2];
                wait_loads<kLoads>();  // all but the other stage's
                asm volatile("" ::: "memory");
                u32x4 chunk[F][2];
#pragma unroll
                for (int i = 0; i < F; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        chunk[i][h] = *reinterpret_cast<const u32x4*>(stage + 16 * int(kBlock) * i + (at ^ (16 * h)));
                float factor[F];
#pragma unroll
                for (int i = 0; i < F; ++i) factor[i] = __shfl(factors[i], lane % 16 + 16 * u);
                __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is read
                asm volatile("" ::: "memory");
                load(stage, b + 2 * stride);
#pragma unroll
                for (int step = 0; step < 4; ++step) {
                    const int h = step / 2, q = 2 * (step % 2);
                    bf16x8 f[F];
#pragma unroll
                    for (int i = 0; i < F; ++i) f[i] = fragment_of(chunk[i][h][q], chunk[i][h][q + 1], factor[i]);
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[c], f[C + i], acc[c][i], 0, 0, 0);
                }
            }
        }
        wait_loads<0>();
        asm volatile("" ::: "memory");
    }
    // The waves' sums, [wave][C][R][64][4], each in its part of the first stage.
    constexpr int kWaveFloats = kPerWave / 4;
    static_assert(kWaveFloats >= 256 * C * R, "a wave's sums fit its part of a stage");
    float* const sums = reinterpret_cast<float*>(stage0);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < R; ++i)
            *reinterpret_cast<f32x4*>(&sums[wave * kWaveFloats + ((c * R + i) * 64 + lane) * 4]) = acc[c][i];
    __syncthreads();
    // A value is column 4 (l / 16) + r of its 16 and row l % 16 of its 16: consecutive threads take a row's columns.
    constexpr int kCols = 16 * C;
    for (int e = threadIdx.x; e < R * 16 * kCols; e += 64 * W) {
        const int row = e / kCols, in_group = e % kCols, c = in_group / 16, i = row / 16;
        const int64_t col = col0 + in_group;
        if (row >= a.rows || col >= a.cols) continue;
        const int from_lane = ((c * R + i) * 64 + in_group % 16 / 4 * 16 + row % 16) * 4 + in_group % 4;
        float total = 0.f;
#pragma unroll 4
        for (int v = 0; v < W; ++v) total += sums[v * kWaveFloats + from_lane];
        if (slices > 1)
            a.workspace[(int64_t(slice) * a.rows + row) * a.cols + col] = total;
        else
            finish(a, row * a.cols + col, col, total);
    }
}

template <int R, int C, int W>
__global__ __launch_bounds__(64 * W) void few_rows_kernel(ProductArgs a, int slices) {
    multiply_few<R, C, W>(a, slices);
}

// Block id -> slice and tile. Consecutive ids land on different XCDs, each with an L2 of its own: ids are regrouped so
// that an XCD takes a contiguous range, and tiles are walked in bands of 8 tile rows.
__device__ __forceinline__ void tile_of(int id, int count, int tiles_m, int tiles_n, int& slice, int& tile_m, int& tile_n) {
    constexpr int kXcds = 8, kBand = 8;
    const int xcd = id % kXcds, per = count / kXcds, more = count % kXcds;
    const int linear = (xcd < more ? xcd * (per + 1) : more * (per + 1) + (xcd - more) * per) + id / kXcds;
    slice = linear / (tiles_m * tiles_n);
    const int in_slice = linear - slice * (tiles_m * tiles_n);
    const int band = in_slice / (kBand * tiles_n), first = band * kBand, height = min(kBand, tiles_m - first);
    const int within = in_slice - first * tiles_n;
    // The divisions leave vector registers; what is the same in all lanes is kept in scalar ones.
    slice = __builtin_amdgcn_readfirstlane(slice);
    tile_n = __builtin_amdgcn_readfirstlane(within / height);
    tile_m = __builtin_amdgcn_readfirstlane(first + within - tile_n * height);
}

// Where a tile's 64-byte row pieces are in LDS: the 16-byte chunk c of row r is in slot c ^ swizzle(r), so that the 16
// rows a fragment read takes at once are in different banks.
__device__ __forceinline__ int swizzle(int row) { return (row >> 2) & 3; }

// Many rows: a BM x BN tile of the output a workgroup of four waves, each a quarter of it in 32 x 32 blocks.
//
// Bound by the matrix cores, and at large sizes by the power they draw: 6001 x 4096 x 14336 takes 554 to 589 us by the
// card (1196 to 1272 TFLOP/s; the library's bf16 product of the same shape 590), 8192 x 8192 x 8192 807 us (1362). A wave
// of the 256 x 256 tile converts 32 pairs a lane for sixteen matrix instructions of 32 cycles, one of the 128 x 256 tile 24
// for eight; it takes all 512 registers of a lane, and 16 of its 256 sums pass through scratch memory between the last
// product and the stores. A step of 64 along the inner dimension is four units of one 32x32x16 instruction a block; while a unit is multiplied the
// next one's codes are converted and the chunk after that is read from LDS. The one barrier of a step is in its middle:
// there every wave has read all of the step's stage, which takes the loads of STAGES steps ahead, and every wave's loads of
// the next stage have landed.
template <int BM, int BN, int STAGES, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void multiply_tile(const ProductArgs& a, int tiles_m, int tiles_n, int blocks_per_slice) {
    constexpr int kWaves = WAVES_M * WAVES_N, FM = BM / (32 * WAVES_M), FN = BN / (32 * WAVES_N), F = FM + FN;
    constexpr int kLoads = (BM + BN) / (16 * kWaves);  // of 16 rows each, a wave
    constexpr int kBytes = (BM + BN) * kStep;  // of a stage
    static_assert(BM % (16 * kWaves) == 0 && BN % (16 * kWaves) == 0, "a load is of rows or of columns");
    static_assert(STAGES >= 3 && STAGES <= 6 && STAGES != 5, "steps in rounds of an even number of stages");
    // An array a stage, named by constants, so that the compiler knows which stage a read of LDS may depend on.
    __shared__ __attribute__((aligned(16))) uint8_t stage0[kBytes], stage1[kBytes], stage2[kBytes];
    __shared__ __attribute__((aligned(16))) uint8_t stage3[STAGES > 3 ? kBytes : 16], stage4[STAGES > 4 ? kBytes : 16],
        stage5[STAGES > 4 ? kBytes : 16];
    uint8_t* const stages[6] = {stage0, stage1, stage2, stage3, stage4, stage5};
    const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int slice, tile_m, tile_n;
    tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, slice, tile_m, tile_n);
    const int64_t m0 = int64_t(tile_m) * BM, n0 = int64_t(tile_n) * BN;
    const int block0 = slice * blocks_per_slice, blocks = min(blocks_per_slice, int(a.blocks) - block0);
    const uint32_t stride = uint32_t(a.blocks * kBlock);
    const int64_t scale_row = scale_stride(a.blocks);

    // Load i of a wave brings rows 16 (kWaves i + wave) .. + 15 of the tile's rows, then columns: lane l the chunk that slot l %
    // 4 of row l / 4 holds. Rows past the last are the last again.
    const uint8_t* x = a.x + m0 * stride + block0 * kBlock;
    const uint8_t* w = a.w + n0 * stride + block0 * kBlock;
    const int last_m = int(min(int64_t(BM), a.rows - m0)) - 1, last_n = int(min(int64_t(BN), a.cols - n0)) - 1;
    uint32_t from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int r = 16 * (kWaves * i + wave) + lane / 4, chunk = (lane & 3) ^ swizzle(r);
        const int source = r < BM ? min(r, last_m) : min(r - BM, last_n);
        from[i] = uint32_t(source) * stride + 16 * chunk;
    }
    const int steps = 2 * blocks;
    // Loads FIRST to LAST of a step. Steps past the last load nothing (a buffer of no bytes), which keeps the count of
    // loads, and so the waits, fixed.
    auto load = [&](uint8_t* stage, int step, auto first, auto last) {
        const int bytes = __builtin_amdgcn_readfirstlane((step - steps) >> 31);  // all, or none
        const __amdgpu_buffer_rsrc_t left = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(x), 0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t right = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(w), 0, bytes, 0x00020000);
#pragma unroll
        for (int i = decltype(first)::value; i < decltype(last)::value; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(16 * kWaves * i < BM ? left : right,
                                                     (lds_pointer)(stage + (kWaves * i + wave) * 16 * kStep), 16, from[i],
                                                     kStep * step, 0, 0);
    };
    using L0 = std::integral_constant<int, 0>;
    using L1 = std::integral_constant<int, (kLoads + 3) / 4>;
    using L2 = std::integral_constant<int, (kLoads + 1) / 2>;
    using L3 = std::integral_constant<int, kLoads - kLoads / 4>;
    using L4 = std::integral_constant<int, kLoads>;

    // This wave's fragments: 32 of the tile's rows each (the swizzle is the same 32 rows on), and their scale bytes.
    const int wave_m = wave / WAVES_N * (32 * FM), wave_n = wave % WAVES_N * (32 * FN);
    const int at_m = (wave_m + row) * kStep + 16 * ((2 * half) ^ swizzle(row));
    const int at_n = (BM + wave_n + row) * kStep + 16 * ((2 * half) ^ swizzle(row));
    uint32_t scales[F];
#pragma unroll
    for (int i = 0; i < F; ++i)
        scales[i] = uint32_t(i < FM ? min(wave_m + 32 * i + row, last_m) : min(wave_n + 32 * (i - FM) + row, last_n)) *
                    uint32_t(scale_row);
    const __amdgpu_buffer_rsrc_t x_scales =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.x_scales + m0 * scale_row + block0), 0, -1, 0x00020000);
    const __amdgpu_buffer_rsrc_t w_scales =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.w_scales + n0 * scale_row + block0), 0, -1, 0x00020000);
    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    float factor[F];
    uint32_t next_scale[F];
    u32x4 chunk0[F], chunk1[F];  // 16 consecutive values of a lane, of two units: a step's first and its second half's
    bf16x8 even[F], odd[F];      // the fragments of units 0 and 2, and of 1 and 3
    auto read = [&](const uint8_t* stage, int q, u32x4(&chunk)[F]) {
#pragma unroll
        for (int i = 0; i < F; ++i)
            chunk[i] = *reinterpret_cast<const u32x4*>(
                stage + (i < FM ? (at_m ^ (16 * q)) + 32 * kStep * i : (at_n ^ (16 * q)) + 32 * kStep * (i - FM)));
    };
    auto convert = [&](const u32x4(&chunk)[F], int h, bf16x8(&f)[F]) {
#pragma unroll
        for (int i = 0; i < F; ++i) f[i] = fragment_of(chunk[i][2 * h], chunk[i][2 * h + 1], factor[i]);
    };
    auto multiply = [&](const bf16x8(&f)[F]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i], f[FM + j], acc[i][j], 0, 0, 0);
    };
    auto load_scales = [&](int block) {
        const int at = __builtin_amdgcn_readfirstlane(min(block, blocks - 1));
#pragma unroll
        for (int i = 0; i < F; ++i)
            next_scale[i] = __builtin_amdgcn_raw_buffer_load_b8(i < FM ? x_scales : w_scales, scales[i], at, 0);
    };
    auto take_scales = [&] {
#pragma unroll
        for (int i = 0; i < F; ++i) factor[i] = factor_of(next_scale[i]);
    };
    // Spreads a unit's conversions, LDS reads and loads over its matrix instructions.
    auto interleave = [&](auto reads, auto loads) {
        constexpr int kProducts = FM * FN, kLoaded = decltype(loads)::value;
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (4 * F + kProducts - 1) / kProducts, 0);
            if (decltype(reads)::value && i < F) __builtin_amdgcn_sched_group_barrier(0x100, (F + kProducts - 1) / kProducts, 0);
            if (i < kLoaded) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    // Step t, on stage t % STAGES = S. Entered with unit 0 converted and chunk 0 read. SECOND: of a block.
    auto step = [&](auto at, auto second, int t) {
        constexpr int S = decltype(at)::value;
        uint8_t *const stage = stages[S], *const next = stages[(S + 1) % STAGES], *const last = stages[(S + STAGES - 1) % STAGES];
        __builtin_amdgcn_sched_barrier(0);
        load(last, t + STAGES - 1, L2{}, L3{});
        read(stage, 1, chunk1);
        convert(chunk0, 1, odd);
        multiply(even);
        interleave(Yes{}, std::integral_constant<int, L3::value - L2::value>{});
        load(last, t + STAGES - 1, L3{}, L4{});
        convert(chunk1, 0, even);
        multiply(odd);
        interleave(No{}, std::integral_constant<int, L4::value - L3::value>{});
        wait_loads<kLoads * (STAGES - 2)>();
        stage_barrier();
        convert(chunk1, 1, odd);
        if constexpr (decltype(second)::value) {  // what is converted from here on is the next block's
            take_scales();
            load_scales((t >> 1) + 2);
        }
        load(stage, t + STAGES, L0{}, L1{});
        read(next, 0, chunk0);
        multiply(even);
        interleave(Yes{}, L1{});
        load(stage, t + STAGES, L1{}, L2{});
        convert(chunk0, 0, even);
        multiply(odd);
        interleave(No{}, std::integral_constant<int, L2::value - L1::value>{});
    };
    constexpr int kRound = STAGES % 2 == 0 ? STAGES : 2 * STAGES;  // an even number of steps that ends on the last stage
    // The blocks (of two steps) of a round, all of them or the `left` first.
    auto round = [&](int t, auto whole, int left) {
        auto block = [&](auto pair) {
            constexpr int P = 2 * decltype(pair)::value;
            if constexpr (P < kRound) {
                if (decltype(whole)::value || P < left) {
                    step(std::integral_constant<int, P % STAGES>{}, No{}, t + P);
                    step(std::integral_constant<int, (P + 1) % STAGES>{}, Yes{}, t + P + 1);
                }
            }
        };
        block(std::integral_constant<int, 0>{});
        block(std::integral_constant<int, 1>{});
        block(std::integral_constant<int, 2>{});
    };
    if (blocks > 0) {
        load_scales(0);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load(stages[i], i, L0{}, L4{});
        load(stages[STAGES - 1], STAGES - 1, L0{}, L2{});
        wait_loads<kLoads * (STAGES - 2) + L2::value>();
        take_scales();
        load_scales(1);
        stage_barrier();
        read(stage0, 0, chunk0);
        convert(chunk0, 0, even);
        int t = 0;
        for (; t + kRound <= steps; t += kRound) round(t, Yes{}, 0);
        round(t, No{}, steps - t);
        wait_loads<0>();
    }
    // Outputs of the smaller tiles pass the caches by (nt), which leaves operands in them: 200 x 768 x 16384 10.1 us against 11.5,
    // 2048 x 768 x 2304 15.0 against 16.5; with the larger ones 4096 x 4096 x 4096 took 118.5 against 114.9. Slices' sums too, to
    // no difference: 100 x 8192 x 8192 30.7 against 30.8, 512 x 14336 x 4096 71.3 to 72.2 against 71.3 to 72.6.
    constexpr int kStreamed = BM * BN <= 128 * 128 ? 2 : 0;
    // A buffer of each 32 rows' outputs (or of the slice's sums), of less than 2^31 bytes: places past the last row are out
    // of its range, and so is 2^31 with any row's offset, for columns past the last; such stores do nothing. A lane's
    // sixteen values of a block are rows 8 (r / 4) + 4 half + r % 4 of one column.
    const bool partial = gridDim.x > unsigned(tiles_m * tiles_n);
    float* y = partial ? a.workspace + int64_t(slice) * a.rows * a.cols : a.y;
    const uint32_t pitch = uint32_t(a.cols) * 4;
    uint32_t place[FN];
    float bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int64_t col = n0 + wave_n + 32 * j + row;
        place[j] = col < a.cols ? uint32_t(4 * half) * pitch + uint32_t(col) * 4 : 0x80000000u;
        bias[j] = a.bias != nullptr && !partial && col < a.cols ? a.bias[col] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t first = m0 + wave_m + 32 * i;
        const int64_t held = min(max(a.rows - first, int64_t(0)), int64_t(32));
        const __amdgpu_buffer_rsrc_t out =
            __builtin_amdgcn_make_buffer_rsrc(y + first * a.cols, 0, int(uint32_t(held) * pitch), 0x00020000);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            float before[16];
            if (a.accumulate && !partial) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    before[r] = __builtin_bit_cast(
                        float, __builtin_amdgcn_raw_buffer_load_b32(out, place[j], (8 * (r / 4) + r % 4) * pitch, 0));
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float v = acc[i][j][r];
                if (!partial) {
                    v = a.scale * v;
                    if (a.accumulate) v = before[r] + v;
                    if (a.bias != nullptr) v = v + bias[j];
                }
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), out, place[j],
                                                      (8 * (r / 4) + r % 4) * pitch, kStreamed);
            }
        }
    }
}

// Waves a SIMD: one of the largest tiles, whose sums take half of its registers or more, two of the next.
template <int BM, int BN, int STAGES, int WAVES_M, int WAVES_N>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N)
    __attribute__((amdgpu_waves_per_eu(BM * BN > 32768 ? 1 : BM * BN > 8192 ? 2 : 3))) void tile_kernel(
    ProductArgs a, int tiles_m, int tiles_n, int blocks_per_slice) {
    multiply_tile<BM, BN, STAGES, WAVES_M, WAVES_N>(a, tiles_m, tiles_n, blocks_per_slice);
}

// The slices' sums, in order.
__global__ __launch_bounds__(256) void slices_kernel(ProductArgs a, int slices) {
    const int64_t count = a.rows * a.cols;
    for (int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x; e < count; e += int64_t(gridDim.x) * 256) {
        float total = 0.f;
        for (int s = 0; s < slices; s += 8) {  // eight in flight
            float part[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) part[u] = s + u < slices ? a.workspace[(s + u) * count + e] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) total += part[u];
        }
        finish(a, e, e % a.cols, total);
    }
}
hipError_t launch_slices(const ProductArgs& a, int slices, hipStream_t stream) {
    const int64_t groups = std::min<int64_t>((a.rows * a.cols + 255) / 256, 16 * a.cu_count);
    hipLaunchKernelGGL(slices_kernel, dim3(unsigned(groups)), dim3(256), 0, stream, a, slices);
    return hipGetLastError();
}
// At most as many as the workspace holds sums of.
int64_t held_slices(const ProductArgs& a, int64_t slices) {
    return std::max<int64_t>(1, std::min<int64_t>(slices, int64_t(a.workspace_bytes / sizeof(float)) / (a.rows * a.cols)));
}

template <int BM, int BN, int STAGES>
hipError_t launch_tiles(const ProductArgs& a, int64_t slices, hipStream_t stream) {
    const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN;
    const int64_t per_slice = (a.blocks + slices - 1) / slices;
    slices = a.blocks == 0 ? 1 : (a.blocks + per_slice - 1) / per_slice;
    hipLaunchKernelGGL((tile_kernel<BM, BN, STAGES, 2, 2>), dim3(unsigned(tiles_m * tiles_n * slices)), dim3(256), 0, stream, a,
                       int(tiles_m), int(tiles_n), int(per_slice));
    const hipError_t err = hipGetLastError();
    return err != hipSuccess || slices == 1 ? err : launch_slices(a, int(slices), stream);
}

// Tiles and slices of the inner dimension by their time in us: a CU takes `block` for a block of a tile, whether it has
// one tile or several at once, and writes outputs at 20 KB a us; the slices' second kernel takes 3.5 and 1.5 more per
// million sums. The larger a tile, the fewer conversions and reads of LDS for each product, and the more its edges and last round
// waste. The times are of 8192 x 8192 x 8192 and 6001 x 14336 x 4096, where the tiles took, in this order:
//   817, 887, 918, 1069, 1389, 1736 us and 626, 563, 591, 711, 921, 1104 us,
// and for the two smallest of 100 x 8192 x 8192 and 65 x 4096 x 14336, where a CU has one of them (34.4 and 27.8 us).
struct Tile {
    int rows, cols;
    double block;
};
constexpr Tile kTiles[] = {{kLargestTile, kLargestTile, 3.00}, {192, 256, 2.42}, {128, 256, 1.70},
                           {128, 128, 0.99}, {64, 128, 0.75},  {64, 64, 0.475}};
void choose_tile(const ProductArgs& a, int& tile, int64_t& slices) {
    double least = 0;
    tile = -1;
    for (int i = 0; i < int(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
        const Tile& t = kTiles[i];
        const int64_t tiles = ((a.rows + t.rows - 1) / t.rows) * ((a.cols + t.cols - 1) / t.cols);
        if (tiles >= kMaxTiles) continue;  // never the largest
        const int64_t most = held_slices(a, std::min<int64_t>({2 * int64_t(a.cu_count) / tiles, a.blocks / 2, 32}));
        for (int64_t n = 1; n <= most; ++n) {
            const int64_t rounds = (tiles * n + a.cu_count - 1) / a.cu_count, blocks = (a.blocks + n - 1) / n;
            double cost = double(rounds) * (double(blocks) * t.block + double(t.rows * t.cols) * 4 / 20e3);
            if (n > 1) cost += 3.5 + 1.5e-6 * double(n * a.rows * a.cols);
            if (tile < 0 || cost < least) least = cost, tile = i, slices = n;
        }
    }
}

template <int R, int C, int W>
hipError_t launch_few_rows(const ProductArgs& a, hipStream_t stream) {
    const int64_t groups = (a.cols + 16 * C - 1) / (16 * C);
    // Slices of the inner dimension where column groups are few: a workgroup takes about 62 KB of operands in a us, the
    // second kernel 3 us (16 x 28672 x 768: 11.2 us in five slices, 22.1 in one).
    int64_t slices = 1;
    const double whole = double(16 * (R + C) * a.blocks * kBlock) / 62e3;
    double least = whole;
    const int64_t most = held_slices(a, std::min<int64_t>({a.cu_count / groups, a.blocks / W, 32}));
    for (int64_t n = 2; n <= most; ++n)
        if (whole / double(n) + 3 < least) least = whole / double(n) + 3, slices = n;
    hipLaunchKernelGGL((few_rows_kernel<R, C, W>), dim3(unsigned(groups * slices)), dim3(64 * W), 0, stream, a, int(slices));
    const hipError_t err = hipGetLastError();
    return err != hipSuccess || slices == 1 ? err : launch_slices(a, int(slices), stream);
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    // Few rows. Workgroups of 16 columns while every CU has at most one; beyond, more columns or fewer waves each, so that
    // the CUs hold all or most of them at once. Alternatives measured in us, rows x inner dimension x columns:
    //   16 x 14336 x 4224: <1, 2, 8> 20.9, <1, 1, 4> 23.3, <1, 1, 8> 24.5; 16 x 4096 x 14336: <1, 4, 4> 12.7, <1, 1, 4> 15.4;
    //   32 x 8192 x 28672: <2, 4, 3> 42.5, <2, 2, 4> 57.2, tiles 50.8; 32 x 4096 x 8192: <2, 2, 4> 8.9, tiles 12.3.
    // Forms that are next to each other in the rule, weights from HBM:
    //   16 x 4096 x 8192: <1, 2, 8> 10.4, <1, 1, 4> 11.3, <1, 4, 4> 12.3; 16 x 4096 x 12000: <1, 2, 8> 17.1, <1, 1, 4> 14.6, <1, 4, 4> 13.8;
    //   32 x 4096 x 4096: <2, 1, 12> 9.1, <2, 2, 4> 9.8, <2, 1, 8> 8.7; 32 x 14336 x 4096: <2, 1, 12> 19.6 to 21.1,
    //   <2, 2, 4> 19.2, <2, 1, 8> 19.5;
    //   64 x 8192 x 8192: <4, 1, 8> 33.6, <4, 2, 6> 26.6, <4, 2, 3> 26.1; 64 x 14336 x 4096: <4, 1, 8> 27.3, <4, 2, 6> 25.9;
    //   40 x 4096 x 4096: <4, 1, 8> 10.7, <4, 2, 6> 14.1; 64 x 8192 x 16000: <4, 2, 6> 49.1, <4, 2, 3> 43.
    // 33 to 64 rows for weights that come from HBM: 40 x 4096 x 4096 10.7, tiles 12.4; 64 x 4096 x 16384 24.7, tiles 28.1 (20.6 and
    // 20.0 from the last-level cache); 64 x 8192 x 16000 43, tiles 53.6 (40.5 and 36.7). The tiles lead where the inner dimension
    // is long and columns few: 64 x 8192 x 8192 26.6, tiles 25.4; 64 x 14336 x 4096 27.4, tiles 23.2.
    // Many columns of a short inner dimension are left to the tiles: 16 x 768 x 50304 13.2, tiles 10.9.
    const int64_t cu = a.cu_count, cols = a.cols;
    const bool few = a.rows <= 32 ? a.blocks > 8 || cols <= 64 * cu : a.rows <= 64 && cols <= 64 * cu;
    if (few) {
        if (a.rows <= 16) {
            if (cols <= 16 * cu) return launch_few_rows<1, 1, 8>(a, stream);
            if (cols <= 24 * cu) return launch_few_rows<1, 2, 8>(a, stream);
            return cols < 48 * cu ? launch_few_rows<1, 1, 4>(a, stream) : launch_few_rows<1, 4, 4>(a, stream);
        }
        if (a.rows <= 32) {
            if (cols <= 16 * cu) return launch_few_rows<2, 1, 12>(a, stream);
            return cols <= 64 * cu ? launch_few_rows<2, 2, 4>(a, stream) : launch_few_rows<2, 4, 3>(a, stream);
        }
        if (cols <= 16 * cu) return launch_few_rows<4, 1, 8>(a, stream);
        return cols <= 32 * cu ? launch_few_rows<4, 2, 6>(a, stream) : launch_few_rows<4, 2, 3>(a, stream);
    }
    int tile;
    int64_t slices;
    choose_tile(a, tile, slices);
    switch (tile) {
        case 0: return launch_tiles<256, 256, 3>(a, slices, stream);
        case 1: return launch_tiles<192, 256, 3>(a, slices, stream);
        case 2: return launch_tiles<128, 256, 3>(a, slices, stream);
        case 3: return launch_tiles<128, 128, 3>(a, slices, stream);
        case 4: return launch_tiles<64, 128, 3>(a, slices, stream);
        default: return launch_tiles<64, 64, 6>(a, slices, stream);
    }
}

}  // namespace fp8
}  // namespace sn
