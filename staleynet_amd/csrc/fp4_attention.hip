// Causal attention over a key/value cache in 4 bits (staleynet_fp4.h): out =
// softmax(scale q K^T) V per query, grouped heads, sequences of their own lengths.
//
// The queries that share a key/value head, (time, head of its group) pairs in that
// order, are rows; a wave takes 16 of them and walks over the keys 32 at a time,
// one pass with the running maximum m and sum l of the softmax (in powers of two: q
// carries scale log2 e).
//  * S^T = K q^T: keys are the rows of the matrix instruction's result, queries its
//    columns, so lane (n, g) holds for query n the scores of keys 4 g .. + 3 of each
//    16. K's codes are converted from the loaded words as they are (lane (n, g):
//    quarter g of key n); q, split exactly in three bf16 parts (fp4_device.h), stays
//    in registers.
//  * The softmax is per lane but for the maximum over the four lanes of a query.
//  * O^T += V^T P^T: a lane's eight probabilities, split, are the right operand as
//    they are, the operand's inner index being keys 4 g .. + 3 of the first 16 and
//    then of the second. V's codes become bf16 rows in LDS (a region of the wave's
//    own, no barrier) and are read back transposed in that order.
// Every product is exact; sums, maxima and probabilities are fp32.
//
// Waves: where a key/value head has few queries, a workgroup's waves share 16 rows and
// take every n-th 32 keys, their m, l and O merged through LDS in wave order; with
// many rows each wave takes 16 rows of its own. Long caches are also split over
// workgroups, whose O, m and l go through the workspace to a second kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kRows = 16;   // queries of a wave
constexpr int kKeys = 32;   // keys of a step
constexpr int kMaxWaves = 8;
constexpr int kMaxSplits = 512;

struct KernelArgs {
    AttentionArgs a;
    float q_scale;         // scale log2 e
    int32_t group;         // query heads of a key/value head
    int32_t row_tiles;     // of a key/value head
    int32_t waves_a_tile;  // 1, or all waves of the workgroup
    int32_t splits;        // workgroups of a tile's keys
    int32_t keys_a_split;  // a multiple of kKeys
    // splits > 1: O [item][split][16][head_dim] and then {m, l} [item][split][16].
    float* partial_o;
    float* partial_ml;
};

// Keys sequence b holds.
__device__ __forceinline__ int64_t held_by(const AttentionArgs& a, int64_t b) {
    const int64_t n = a.lengths != nullptr ? int64_t(a.lengths[b]) : a.keys;
    return min(n, a.capacity);
}

// LDS of one wave: 32 rows of V in bf16, 32 bytes more than their length apart (the
// four rows a transposing load's 16 lanes read, and the eight a write phase fills, lie
// on distinct banks); afterwards its O [16][h + 4], m and l.
template <int H>
struct WaveStage {
    static constexpr int ROW = 2 * H + 32;
    static constexpr int O_ROW = H + 4;
    static constexpr int O_BYTES = (kRows * O_ROW + 2 * kRows) * 4;
    static constexpr int BYTES = kKeys * ROW > O_BYTES ? kKeys * ROW : O_BYTES;
};

// Four rows x 16 columns of 16-bit values per 16 lanes, transposed: lane 4 i + s
// points at columns 4 s .. + 3 of row i, lane c receives column c of rows 0 .. 3.
__device__ __forceinline__ bf16x8 transposed(const char* first, const char* second) {
    typedef short four __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) four* lds_four;
    const four a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four)first);
    const four b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_four)second);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

template <int H>
__global__ __launch_bounds__(64 * kMaxWaves) void attention_kernel(KernelArgs p) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    constexpr int NF = H / 32;     // fragments of 32 over the head dim: words of a lane's quarter
    constexpr int TILES = H / 16;  // 16-column tiles of O
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();

    // Workgroup -> (split, key/value head, row tile), the last rows (which see the
    // most keys) first; neighbours are key/value heads, so that one XCD's workgroups
    // read few of them.
    const int64_t kv_all = a.batch * a.kv_heads;
    int64_t index = blockIdx.x;
    const int64_t kv = index % kv_all;
    index /= kv_all;
    const int split = int(index % p.splits);
    index /= p.splits;
    const int tiles_a_group = waves / p.waves_a_tile;
    const int64_t tile_groups = (p.row_tiles + tiles_a_group - 1) / tiles_a_group;
    const int64_t tile = (tile_groups - 1 - index) * tiles_a_group + wave / p.waves_a_tile;
    const int turn = wave % p.waves_a_tile;
    const int64_t b = kv / a.kv_heads, kv_head = kv % a.kv_heads;

    const int64_t length = held_by(a, b);
    const int64_t rows_all = a.queries * p.group;
    const int64_t row = tile * kRows + n;
    const bool tile_ok = tile < p.row_tiles;
    const bool row_ok = row < rows_all;
    const int64_t row_used = min(row, rows_all - 1);
    const int64_t t = row_used / p.group;
    const int64_t head = kv_head * p.group + row_used % p.group;
    // The last key this lane's query sees, and the ends of what the wave's first and last queries see.
    const int64_t before = length - a.queries;
    const int64_t last = before + t;
    const int64_t all_see = before + min(tile * kRows, rows_all - 1) / p.group + 1;
    const int64_t some_see = before + min(tile * kRows + kRows - 1, rows_all - 1) / p.group + 1;
    const int64_t split_first = int64_t(split) * p.keys_a_split;
    const int64_t end = tile_ok ? min(some_see, p.splits > 1 ? split_first + p.keys_a_split : some_see) : 0;

    const int64_t cache_row = kv * a.capacity;
    const uint8_t* k_codes = a.k_codes + cache_row * (H / 2) + g * (H / 8);
    const uint8_t* v_codes = a.v_codes + cache_row * (H / 2) + g * (H / 8);
    const uint8_t* k_scales = a.k_scales + cache_row * (H / 32) + g * (H / 4) / 32;
    const uint8_t* v_scales = a.v_scales + cache_row * (H / 32) + g * (H / 4) / 32;

    struct Words {
        uint32_t k[2][NF], v[2][NF];
        uint32_t ks[2], vs[2];
    };
    auto load_words = [](const uint8_t* from, uint32_t (&w)[NF]) __attribute__((always_inline)) {
        if constexpr (NF == 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(from);
            w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
        } else if constexpr (NF == 2) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(from);
            w[0] = x[0], w[1] = x[1];
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(from);
        }
    };
    // Keys past the end read the last key (their scores and values are replaced).
    auto load = [&](int64_t key0, Words& x) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t key = min(key0 + 16 * u + n, end - 1);
            load_words(k_codes + key * (H / 2), x.k[u]);
            load_words(v_codes + key * (H / 2), x.v[u]);
            x.ks[u] = k_scales[key * (H / 32)];
            x.vs[u] = v_scales[key * (H / 32)];
        }
    };

    // q of this lane's query: fragment i holds head dims g H / 4 + 8 i .. + 7, as K's words do.
    SplitVector q[NF];
    {
        const float* from = a.q + b * a.q_sequence + head * a.q_head + t * a.q_row + g * (H / 4);
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = row_ok && tile_ok ? from[8 * i + e] * p.q_scale : 0.f;
            q[i] = split_exact(x, upper);
        }
    }

    float m = -INFINITY, l = 0.f;  // l: of this lane's keys
    f32x4 o[TILES];
#pragma unroll
    for (int d = 0; d < TILES; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    char* const stage = lds + wave * Stage::BYTES;
    char* const v_write = stage + n * Stage::ROW + g * (H / 2);
    const char* const v_read = stage + (4 * g + (n >> 2)) * Stage::ROW + 8 * (n & 3);

    Words next;
    int64_t key0 = split_first + int64_t(turn) * kKeys;
    const int64_t step = int64_t(p.waves_a_tile) * kKeys;
    if (key0 < end) load(key0, next);
    for (; key0 < end; key0 += step) {
        Words now = next;
        if (key0 + step < end) load(key0 + step, next);
        const bool masked = key0 + kKeys > all_see || key0 + kKeys > end;  // of the wave

        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            const float factor = factor_of(now.ks[u]);
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                const bf16x8 k = fragment_of(now.k[u][i], factor);
#pragma unroll
                for (int part = kParts - 1; part >= 0; --part)
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[i].part[part], s[u], 0, 0, 0);
            }
        }
        // Values a query does not see must not reach it through 0 x NaN: in a step at the
        // end of what some query sees, NaN blocks are taken out here and the queries
        // that see them given NaN below.
        uint64_t poison[2] = {0, 0};
        if (masked) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t key = key0 + 16 * u + n;
                const bool nan = now.vs[u] > kLargestScale;
                poison[u] = __ballot(nan && key < end);
                if (nan || key >= end) {
                    now.vs[u] = 127;
#pragma unroll
                    for (int i = 0; i < NF; ++i) now.v[u][i] = 0;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t k = key0 + 16 * u + 4 * g + r;
                    s[u][r] = k <= last && k < end ? s[u][r] : -INFINITY;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float factor = factor_of(now.vs[u]);
#pragma unroll
            for (int i = 0; i < NF; ++i)
                *reinterpret_cast<bf16x8*>(v_write + 16 * u * Stage::ROW + 16 * i) = fragment_of(now.v[u][i], factor);
        }

        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float m_new = fmaxf(m, top);
            const float alpha = m_new == -INFINITY ? 1.f : exp2_of(m - m_new);
            m = m_new;
            l = l * alpha;
#pragma unroll
            for (int d = 0; d < TILES; ++d) o[d] = o[d] * alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = exp2_of(s[e / 4][e % 4] - base);
            l = l + x[e];
        }
        const SplitVector pr = split_exact(x, upper);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const bf16x8 v = transposed(v_read + 32 * d, v_read + 16 * Stage::ROW + 32 * d);
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part)
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pr.part[part], o[d], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
        if (poison[0] | poison[1]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                for (uint64_t left = poison[u]; left != 0; left &= left - 1) {
                    const int at = __builtin_ctzll(left);
                    const bool seen = key0 + 16 * u + (at & 15) <= last;
                    const int dim = (at >> 4) * (H / 4);  // the lane's quarter
#pragma unroll
                    for (int d = 0; d < TILES; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int here = 16 * d + 4 * g + r;
                            if (seen && here >= dim && here < dim + H / 4) o[d][r] = NAN;
                        }
                }
        }
    }
    l = l + __shfl_xor(l, 16);
    l = l + __shfl_xor(l, 32);

    float* out = a.out + b * a.out_sequence + head * a.out_head + t * a.out_row;
    if (p.waves_a_tile == 1 && p.splits == 1) {
        if (!row_ok || !tile_ok) return;
        const float scale = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < TILES; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) out[16 * d + 4 * g + r] = l == 0.f ? 0.f : o[d][r] * scale;
        return;
    }

    // Merge the workgroup's waves. (waves_a_tile is all of them here.)
    float* mine = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int d = 0; d < TILES; ++d) *reinterpret_cast<f32x4*>(mine + n * Stage::O_ROW + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        mine[kRows * Stage::O_ROW + n] = m;
        mine[kRows * Stage::O_ROW + kRows + n] = l;
    }
    __syncthreads();
    const int64_t first_row = tile * kRows;
    const int rows = int(min(rows_all - first_row, int64_t(kRows)));
    const int64_t item = tile * kv_all + kv;
    for (int e = threadIdx.x; e < rows * H; e += blockDim.x) {
        const int r = e / H, h = e % H;
        float top = -INFINITY;
        for (int w = 0; w < waves; ++w) {
            const float* from = reinterpret_cast<const float*>(lds + w * Stage::BYTES);
            top = fmaxf(top, from[kRows * Stage::O_ROW + r]);
        }
        float total = 0.f, sum = 0.f;
        for (int w = 0; w < waves; ++w) {
            const float* from = reinterpret_cast<const float*>(lds + w * Stage::BYTES);
            const float mw = from[kRows * Stage::O_ROW + r];
            const float weight = top == -INFINITY ? 1.f : exp2_of(mw - top);
            total = total + weight * from[kRows * Stage::O_ROW + kRows + r];
            sum = sum + weight * from[r * Stage::O_ROW + h];
        }
        if (p.splits == 1) {
            const int64_t rt = (first_row + r) / p.group, rh = kv_head * p.group + (first_row + r) % p.group;
            a.out[b * a.out_sequence + rh * a.out_head + rt * a.out_row + h] = total == 0.f ? 0.f : sum * (1.f / total);
        } else {
            const int64_t record = (item * p.splits + split) * kRows + r;
            p.partial_o[record * H + h] = sum;
            if (h == 0) {
                p.partial_ml[2 * record] = top;
                p.partial_ml[2 * record + 1] = total;
            }
        }
    }
}

// One row's partial results, in split order.
template <int H>
__global__ __launch_bounds__(H) void merge_kernel(KernelArgs p) {
#pragma clang fp contract(off)
    const AttentionArgs& a = p.a;
    const int64_t kv_all = a.batch * a.kv_heads;
    const int64_t rows_all = a.queries * p.group;
    const int64_t kv = int64_t(blockIdx.x) % kv_all, row = int64_t(blockIdx.x) / kv_all;
    const int64_t b = kv / a.kv_heads, kv_head = kv % a.kv_heads;
    const int64_t t = row / p.group, head = kv_head * p.group + row % p.group;
    const int64_t item = row / kRows * kv_all + kv;
    const int h = threadIdx.x;
    // The splits that hold a key some row of the tile sees: the others hold nothing for it.
    const int64_t tile_last = min(row / kRows * kRows + kRows - 1, rows_all - 1);
    const int64_t end = held_by(a, b) - a.queries + tile_last / p.group + 1;
    const int used = end > 0 ? int(min(int64_t(p.splits), (end + p.keys_a_split - 1) / p.keys_a_split)) : 0;
    const float* ml = p.partial_ml + (item * p.splits * kRows + row % kRows) * 2;
    const float* o = p.partial_o + (item * p.splits * kRows + row % kRows) * H + h;
    float top = -INFINITY;
    for (int s = 0; s < used; ++s) top = fmaxf(top, ml[int64_t(s) * 2 * kRows]);
    float total = 0.f, sum = 0.f;
    for (int s = 0; s < used; ++s) {
        const float weight = top == -INFINITY ? 1.f : exp2_of(ml[int64_t(s) * 2 * kRows] - top);
        total = total + weight * ml[int64_t(s) * 2 * kRows + 1];
        sum = sum + weight * o[int64_t(s) * kRows * H];
    }
    a.out[b * a.out_sequence + head * a.out_head + t * a.out_row + h] = total == 0.f ? 0.f : sum * (1.f / total);
}

template <int H>
hipError_t launch(KernelArgs p, int waves, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    const int tiles_a_group = waves / p.waves_a_tile;
    const int64_t groups = (p.row_tiles + tiles_a_group - 1) / tiles_a_group;
    const int64_t grid = a.batch * a.kv_heads * p.splits * groups;
    const int64_t rows = a.batch * a.kv_heads * a.queries * p.group;
    if (grid > INT32_MAX || rows > INT32_MAX) return hipErrorInvalidValue;
    const size_t lds = size_t(waves) * WaveStage<H>::BYTES;
    hipLaunchKernelGGL(attention_kernel<H>, dim3(unsigned(grid)), dim3(64 * waves), lds, stream, p);
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && p.splits > 1) {
        hipLaunchKernelGGL(merge_kernel<H>, dim3(unsigned(rows)), dim3(H), 0, stream, p);
        err = hipGetLastError();
    }
    return err;
}

}  // namespace

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream) {
    KernelArgs p;
    p.a = a;
    p.q_scale = a.scale * 1.44269504088896340736f;
    p.group = int32_t(a.heads / a.kv_heads);
    const int64_t rows = a.queries * p.group;
    p.row_tiles = int32_t((rows + kRows - 1) / kRows);
    const int64_t items = a.batch * a.kv_heads * p.row_tiles;
    const int64_t longest = a.lengths != nullptr ? a.capacity : a.keys;
    int waves = 4;
    p.waves_a_tile = 4;
    p.splits = 1;
    p.keys_a_split = 0;
    p.partial_o = p.partial_ml = nullptr;
    if (items >= 4 * a.cu_count && p.row_tiles >= 4) {
        p.waves_a_tile = 1;
    } else if (longest > 512) {
        // Workgroups of at least 512 keys, eight a CU at most.
        const int64_t wanted = std::min<int64_t>({(longest + 511) / 512, std::max<int64_t>(1, 8 * a.cu_count / items),
                                                  int64_t(kMaxSplits)});
        const int64_t bytes = items * kRows * (a.head_dim + 2) * int64_t(sizeof(float));
        const int64_t fits = a.workspace != nullptr ? int64_t(a.workspace_bytes) / bytes : 0;
        const int64_t splits = std::min(wanted, fits);
        if (splits > 1) {
            p.keys_a_split = int32_t(((longest + splits - 1) / splits + kKeys - 1) / kKeys * kKeys);
            p.splits = int32_t((longest + p.keys_a_split - 1) / p.keys_a_split);
            p.partial_o = a.workspace;
            p.partial_ml = a.workspace + items * p.splits * kRows * a.head_dim;
        }
    }
    switch (a.head_dim) {
        case 32: return launch<32>(p, waves, stream);
        case 64: return launch<64>(p, waves, stream);
        default: return launch<128>(p, waves, stream);
    }
}

}  // namespace fp4
}  // namespace sn
