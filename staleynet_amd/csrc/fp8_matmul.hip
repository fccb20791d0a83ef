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
#include <type_traits>

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
// Bound by the matrix cores, with the conversions beside them: a wave converts 24 pairs a lane for eight matrix instructions
// of 32 cycles. A step of 64 along the inner dimension is four units of one 32x32x16 instruction a block; while a
// unit is multiplied the next one's codes are converted and the chunk after that is read from LDS. The one barrier of a
// step is in its middle: there every wave has read all of the step's stage, which takes the loads of three steps
// ahead, and every wave's loads of the next stage have landed.
template <int BM, int BN, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void multiply_tile(const ProductArgs& a, int tiles_m, int tiles_n, int blocks_per_slice) {
    constexpr int kWaves = WAVES_M * WAVES_N, FM = BM / (32 * WAVES_M), FN = BN / (32 * WAVES_N), F = FM + FN;
    constexpr int kLoads = (BM + BN) / (16 * kWaves);  // of 16 rows each, a wave
    static_assert(BM % (16 * kWaves) == 0 && BN % (16 * kWaves) == 0, "a load is of rows or of columns");
    __shared__ __attribute__((aligned(16))) uint8_t stage0[(BM + BN) * kStep], stage1[(BM + BN) * kStep],
        stage2[(BM + BN) * kStep];
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
        const int bytes = -max(0, min(1, steps - step));  // all, or none
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
    const uint8_t* x_scales = a.x_scales + m0 * scale_row + block0;
    const uint8_t* w_scales = a.w_scales + n0 * scale_row + block0;
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
#pragma unroll
        for (int i = 0; i < F; ++i) next_scale[i] = ((i < FM ? x_scales : w_scales) + min(block, blocks - 1))[scales[i]];
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
    // Step t on its stage; `next` is the next step's, `before` the last's. Entered with unit 0 converted and chunk 0 read.
    auto step = [&](uint8_t* stage, const uint8_t* next, uint8_t* before, int t, auto second) {
        __builtin_amdgcn_sched_barrier(0);
        load(before, t + 2, L2{}, L3{});
        read(stage, 1, chunk1);
        convert(chunk0, 1, odd);
        multiply(even);
        interleave(Yes{}, std::integral_constant<int, L3::value - L2::value>{});
        load(before, t + 2, L3{}, L4{});
        convert(chunk1, 0, even);
        multiply(odd);
        interleave(No{}, std::integral_constant<int, L4::value - L3::value>{});
        wait_loads<kLoads>();
        stage_barrier();
        convert(chunk1, 1, odd);
        if constexpr (decltype(second)::value) {  // of a block: what is converted from here on is the next one's
            take_scales();
            load_scales((t >> 1) + 2);
        }
        load(stage, t + 3, L0{}, L1{});
        read(next, 0, chunk0);
        multiply(even);
        interleave(Yes{}, L1{});
        load(stage, t + 3, L1{}, L2{});
        convert(chunk0, 0, even);
        multiply(odd);
        interleave(No{}, std::integral_constant<int, L2::value - L1::value>{});
    };
    if (blocks > 0) {
        load_scales(0);
        load(stage0, 0, L0{}, L4{});
        load(stage1, 1, L0{}, L4{});
        load(stage2, 2, L0{}, L2{});
        take_scales();
        load_scales(1);
        wait_loads<0>();
        stage_barrier();
        read(stage0, 0, chunk0);
        convert(chunk0, 0, even);
        int t = 0;
        for (; t + 6 <= steps; t += 6) {
            step(stage0, stage1, stage2, t, No{});
            step(stage1, stage2, stage0, t + 1, Yes{});
            step(stage2, stage0, stage1, t + 2, No{});
            step(stage0, stage1, stage2, t + 3, Yes{});
            step(stage1, stage2, stage0, t + 4, No{});
            step(stage2, stage0, stage1, t + 5, Yes{});
        }
        if (t < steps) {  // two or four more
            step(stage0, stage1, stage2, t, No{});
            step(stage1, stage2, stage0, t + 1, Yes{});
            if (t + 2 < steps) {
                step(stage2, stage0, stage1, t + 2, No{});
                step(stage0, stage1, stage2, t + 3, Yes{});
            }
        }
        wait_loads<0>();
    }
    // A buffer of each 32 rows' outputs (or of the slice's sums): places past the last row or column are out of its
    // range, which stores nothing. A lane's sixteen values of a block are rows 8 (r / 4) + 4 half + r % 4 of one column.
    const bool partial = gridDim.x > unsigned(tiles_m * tiles_n);
    float* y = partial ? a.workspace + int64_t(slice) * a.rows * a.cols : a.y;
    const uint32_t pitch = uint32_t(a.cols) * 4;
    uint32_t place[FN];
    float bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int64_t col = n0 + wave_n + 32 * j + row;
        place[j] = col < a.cols ? uint32_t(4 * half) * pitch + uint32_t(col) * 4 : 0xffffffffu;
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
                                                      (8 * (r / 4) + r % 4) * pitch, 0);
            }
        }
    }
}

template <int BM, int BN, int WAVES_M, int WAVES_N>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_kernel(
    ProductArgs a, int tiles_m, int tiles_n, int blocks_per_slice) {
    multiply_tile<BM, BN, WAVES_M, WAVES_N>(a, tiles_m, tiles_n, blocks_per_slice);
}

// The slices' sums, in order.
__global__ __launch_bounds__(256) void slices_kernel(ProductArgs a, int slices) {
    const int64_t count = a.rows * a.cols;
    for (int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x; e < count; e += int64_t(gridDim.x) * 256) {
        float total = 0.f;
        for (int s = 0; s < slices; ++s) total += a.workspace[s * count + e];
        float v = a.scale * total;
        if (a.accumulate) v = a.y[e] + v;
        if (a.bias != nullptr) v = v + a.bias[e % a.cols];
        a.y[e] = v;
    }
}

template <int BM, int BN, int WAVES_M, int WAVES_N>
hipError_t launch_tiles(const ProductArgs& a, hipStream_t stream) {
    const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN, tiles = tiles_m * tiles_n;
    // Slices of the inner dimension until there are two workgroups a CU, of eight blocks at least.
    int64_t slices = std::min<int64_t>({2 * a.cu_count / tiles, a.blocks / 8, 32});
    slices = std::min<int64_t>(slices, int64_t(a.workspace_bytes / sizeof(float)) / (a.rows * a.cols));
    slices = std::max<int64_t>(slices, 1);
    const int64_t per_slice = (a.blocks + slices - 1) / slices;
    slices = a.blocks == 0 ? 1 : (a.blocks + per_slice - 1) / per_slice;
    hipLaunchKernelGGL((tile_kernel<BM, BN, WAVES_M, WAVES_N>), dim3(unsigned(tiles * slices)), dim3(64 * WAVES_M * WAVES_N), 0, stream, a, int(tiles_m),
                       int(tiles_n), int(per_slice));
    if (slices > 1) {
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
        const int64_t groups = std::min<int64_t>((a.rows * a.cols + 255) / 256, 16 * a.cu_count);
        hipLaunchKernelGGL(slices_kernel, dim3(unsigned(groups)), dim3(256), 0, stream, a, int(slices));
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
    if (a.rows > 64) {
        if (a.rows > 512) return launch_tiles<128, 256, 2, 2>(a, stream);
        return launch_tiles<64, 128, 2, 2>(a, stream);
    }
    const int64_t tiles_m = (a.rows + 63) / 64, tiles_n = (a.cols + 63) / 64;
    hipLaunchKernelGGL(product_kernel, dim3(unsigned(tiles_n), unsigned(tiles_m)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace fp8
}  // namespace sn
