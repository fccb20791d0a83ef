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
//    quarter g of key n); q is split exactly in three bf16 parts (fp4_device.h).
//  * The softmax is per lane but for the maximum over the four lanes of a query.
//  * O^T += V^T P^T: a lane's eight probabilities, split, are the right operand as
//    they are, the operand's inner index being keys 4 g .. + 3 of the first 16 and
//    then of the second. V's codes become bf16 rows in LDS (a region of the wave's
//    own, no barrier) and are read back transposed in that order.
// Every product is exact; sums, maxima and probabilities are fp32.
//
// Two forms. With few rows to a key/value head (a decode step) a workgroup's waves share 16
// rows and take every fourth 32 keys, q's parts in LDS; the keys are split over
// workgroups (split_attention_kernel). With many (a prompt chunk) each wave has 16
// rows of its own and all their keys (row_attention_kernel).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fp4_device.h"
#include "fp4_internal.h"
#include "gemm_common.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kRows = 16;  // queries of a wave
constexpr int kKeys = 32;  // keys of a step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

struct KernelArgs {
    AttentionArgs a;
    float q_scale;          // scale log2 e
    int32_t group;          // query heads of a key/value head
    int32_t row_tiles;      // of a key/value head
    int32_t workgroups;     // about as many workgroups as share the keys (0: one to a row tile)
    int32_t least_keys;     // of a workgroup, a multiple of kKeys kWaves
    uint32_t* counters;     // one a row tile of every key/value head, zero between calls
    float* records;         // [workgroup][row][H + 4]: O, m, l
};

// Keys sequence b holds. Positions are under 2^30 (fp4.cpp), so that they and the end of a
// step past them are 32-bit integers.
__device__ __forceinline__ int32_t held_by(const AttentionArgs& a, int64_t b) {
    return int32_t(min(a.lengths != nullptr ? a.lengths[b] : uint32_t(a.keys), uint32_t(a.capacity)));
}

// LDS of one wave: 32 rows of V in bf16, 32 bytes more than their length apart (the
// four rows a transposing load's 16 lanes read, and the eight a write phase fills, lie
// on distinct banks); the split form leaves the wave's O [16][h + 4], m and l there.
template <int H>
struct WaveStage {
    static constexpr int ROW = 2 * H + 32;
    static constexpr int O_ROW = H + 4;
    static constexpr int O_BYTES = (kRows * O_ROW + 2 * kRows) * 4;
    static constexpr int BYTES = kKeys * ROW > O_BYTES ? kKeys * ROW : O_BYTES;
    static constexpr int MAX_SPLITS = kWaves * BYTES / (kRows * 4);  // workgroups whose weights fit the stages
    static constexpr int Q_BYTES = H / 32 * kParts * 64 * 16;  // q's fragments, [fragment][part][lane]
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

// The largest of the four lanes n, n + 16, n + 32, n + 48, by exchanging halves and then
// quarters of the wave. (The copy is hidden from the compiler, which takes the results of
// a swap of a value with itself to be equal.)
__device__ __forceinline__ float largest_of_four(float x) {
    uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
    asm("" : "+v"(b));
    const auto halves = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    x = fmaxf(__builtin_bit_cast(float, uint32_t(halves[0])), __builtin_bit_cast(float, uint32_t(halves[1])));
    a = b = __builtin_bit_cast(uint32_t, x);
    asm("" : "+v"(b));
    const auto quarters = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(quarters[0])), __builtin_bit_cast(float, uint32_t(quarters[1])));
}

// One wave's 16 rows (lane n's query is row tile * 16 + n of key/value head kv).
struct Rows {
    int64_t b, kv_head, head;
    int32_t t;
    int32_t last;      // the last key this lane's query sees
    int32_t all_see;   // the first key that some query does not see
    int32_t some_see;  // the first key that no query sees
    bool ok;
};
__device__ __forceinline__ Rows rows_of(const KernelArgs& p, int64_t b, int64_t kv_head, int32_t tile, int32_t length,
                                        int n) {
    Rows r;
    const uint32_t group = uint32_t(p.group), rows = uint32_t(p.a.queries) * group;  // under 2^31
    const uint32_t first = uint32_t(tile) * kRows, row = first + n;
    r.b = b;
    r.kv_head = kv_head;
    r.ok = row < rows;
    const uint32_t used = min(row, rows - 1);
    r.t = int32_t(used / group);
    r.head = kv_head * p.group + used % group;
    const int32_t before = length - int32_t(p.a.queries);
    r.last = before + r.t;
    r.all_see = before + int32_t(first / group) + 1;
    r.some_see = before + int32_t(min(first + kRows - 1, rows - 1) / group) + 1;
    return r;
}

// Fragment i of this lane's query, split: head dims g H / 4 + 8 i .. + 7, as K's words hold them.
template <int H>
__device__ __forceinline__ SplitVector query_fragment(const KernelArgs& p, const Rows& r, int g, int i,
                                                      uint32_t upper) {
    const float* from = p.a.q + r.b * p.a.q_sequence + r.head * p.a.q_head + r.t * p.a.q_row + g * (H / 4) + 8 * i;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = r.ok ? from[e] * p.q_scale : 0.f;
    return split_exact(x, upper);
}

// The running softmax of a wave's rows: m and the unscaled O of this lane's query (dims
// 16 d + 4 g + r), and l over this lane's keys.
template <int H>
struct Running {
    float m = -INFINITY, l = 0.f;
    f32x4 o[H / 16];
};

// Keys key0, key0 + step, .. before `end`, 32 at a time. q(i, part): the fragments of q.
template <int H, class Query>
__device__ __forceinline__ void walk(const KernelArgs& p, const Rows& r, int32_t key0, int32_t step, int32_t end,
                                     char* stage, int n, int g, uint32_t upper, Query&& q,
                                     Running<H>& run) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    constexpr int NF = H / 32;     // fragments of 32 over the head dim: words of a lane's quarter
    constexpr int TILES = H / 16;  // 16-column tiles of O
    const AttentionArgs& a = p.a;
#pragma unroll
    for (int d = 0; d < TILES; ++d) run.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (key0 >= end) return;

    // The step's rows from a base the wave shares, and the lane's offsets from it.
    const int64_t cache_row = (r.b * a.kv_heads + r.kv_head) * a.capacity;
    const uint8_t* k_codes = a.k_codes + (cache_row + key0) * (H / 2);
    const uint8_t* v_codes = a.v_codes + (cache_row + key0) * (H / 2);
    const uint8_t* k_scales = a.k_scales + (cache_row + key0) * (H / 32);
    const uint8_t* v_scales = a.v_scales + (cache_row + key0) * (H / 32);
    const uint32_t code_at = g * (H / 8), scale_at = g * (H / 4) / 32;
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
    auto load = [&](int32_t first, Words& x) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t key = uint32_t(min(16 * u + n, end - 1 - first));
            load_words(k_codes + (key * (H / 2) + code_at), x.k[u]);
            load_words(v_codes + (key * (H / 2) + code_at), x.v[u]);
            x.ks[u] = k_scales[key * (H / 32) + scale_at];
            x.vs[u] = v_scales[key * (H / 32) + scale_at];
        }
        k_codes += int64_t(step) * (H / 2);
        v_codes += int64_t(step) * (H / 2);
        k_scales += int64_t(step) * (H / 32);
        v_scales += int64_t(step) * (H / 32);
    };
    char* const v_write = stage + n * Stage::ROW + g * (H / 2);
    const char* const v_read = stage + (4 * g + (n >> 2)) * Stage::ROW + 8 * (n & 3);

    Words next;
    load(key0, next);
    for (; key0 < end; key0 += step) {
        Words now = next;
        if (key0 + step < end) load(key0 + step, next);
        const bool masked = key0 + kKeys > r.all_see || key0 + kKeys > end;  // of the wave

        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float k_factor[2] = {factor_of(now.ks[0]), factor_of(now.ks[1])};
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const bf16x8 k0 = fragment_of(now.k[0][i], k_factor[0]), k1 = fragment_of(now.k[1][i], k_factor[1]);
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part) {
                const bf16x8 x = q(i, part);
                s[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, x, s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, x, s[1], 0, 0, 0);
            }
        }
        // Values a query does not see must not reach it through 0 x NaN: in a step at the
        // end of what some query sees, NaN blocks are taken out here and the queries
        // that see them given NaN below.
        uint64_t poison[2] = {0, 0};
        if (masked) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int32_t key = key0 + 16 * u + n;
                const bool nan = now.vs[u] > kLargestScale;
                poison[u] = __ballot(nan && key < end);
                if (nan || key >= end) {
                    now.vs[u] = 127;
#pragma unroll
                    for (int i = 0; i < NF; ++i) now.v[u][i] = 0;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t k = key0 + 16 * u + 4 * g + e;
                    s[u][e] = k <= r.last && k < end ? s[u][e] : -INFINITY;
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

        const float top = largest_of_four(fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                                fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))));
        if (__any(top > run.m)) {
            const float m_new = fmaxf(run.m, top);
            const float alpha = m_new == -INFINITY ? 1.f : exp2_of(run.m - m_new);
            run.m = m_new;
            run.l = run.l * alpha;
#pragma unroll
            for (int d = 0; d < TILES; ++d) run.o[d] = run.o[d] * alpha;
        }
        const float base = run.m == -INFINITY ? 0.f : run.m;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = exp2_of(s[e / 4][e % 4] - base);
            run.l = run.l + x[e];
        }
        const SplitVector pr = split_exact(x, upper);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const bf16x8 v = transposed(v_read + 32 * d, v_read + 16 * Stage::ROW + 32 * d);
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part)
                run.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pr.part[part], run.o[d], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
        if (poison[0] | poison[1]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                for (uint64_t left = poison[u]; left != 0; left &= left - 1) {
                    const int at = __builtin_ctzll(left);
                    const bool seen = key0 + 16 * u + (at & 15) <= r.last;
                    const int dim = (at >> 4) * (H / 4);  // the lane's quarter
#pragma unroll
                    for (int d = 0; d < TILES; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int here = 16 * d + 4 * g + e;
                            if (seen && here >= dim && here < dim + H / 4) run.o[d][e] = NAN;
                        }
                }
        }
    }
}

// A workgroup's share of the keys, from the lengths as the device has them: sequence
// b's n keys go to max(1, ceil(n / share)) workgroups for each of its row tiles, where
// share makes them about p.workgroups in all; then consecutive workgroups take
// consecutive shares of a tile, tiles of a sequence, sequences.
struct Share {
    int32_t b, length, keys;  // keys: that a workgroup takes
    int32_t tile;             // of the sequence: kv_head * row_tiles + row tile
    int32_t split, splits;
    int32_t first;            // the tile's first workgroup
    bool ok;
};
__device__ __forceinline__ Share share_of(const KernelArgs& p, int32_t most_splits, int lane) {
    const AttentionArgs& a = p.a;
    const int32_t tiles = int32_t(a.kv_heads) * p.row_tiles;  // of a sequence
    constexpr int32_t kUnit = kKeys * kWaves;
    const int32_t index = int32_t(blockIdx.x);
    Share s = {};
    s.splits = 1;
    if (p.workgroups == 0) {
        s.b = index / tiles;
        s.length = held_by(a, s.b);
        s.tile = index % tiles;
        s.first = index;
        s.ok = true;
        return s;
    }
    int64_t total = 0;
    int32_t longest = 0;
    for (int64_t b0 = 0; b0 < a.batch; b0 += 64) {
        const int32_t n = b0 + lane < a.batch ? held_by(a, b0 + lane) : 0;
        int64_t sum = n;
        int32_t most = n;
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) {
            sum += __shfl_xor(sum, step);
            most = max(most, __shfl_xor(most, step));
        }
        total += sum;
        longest = max(longest, most);
    }
    const int64_t even = (total * tiles + p.workgroups - 1) / p.workgroups;
    const int64_t share = min(max(even, int64_t((longest + most_splits - 1) / most_splits)), int64_t(longest));
    s.keys = __builtin_amdgcn_readfirstlane(max(p.least_keys, int32_t((share + kUnit - 1) / kUnit) * kUnit));
    int32_t before = 0;  // workgroups of the sequences so far
    for (int64_t b0 = 0; b0 < a.batch; b0 += 64) {
        const bool here = b0 + lane < a.batch;
        const int32_t n = here ? held_by(a, b0 + lane) : 0;
        const int32_t splits = here ? max(1, (n + s.keys - 1) / s.keys) : 0;
        int32_t sum = splits * tiles;  // inclusive over the lanes
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            const int32_t other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        const int32_t start = before + sum - splits * tiles;
        const uint64_t mine = __ballot(index >= start && index < start + splits * tiles);
        if (mine != 0) {
            const int from = __builtin_ctzll(mine);
            s.b = int32_t(b0) + from;
            s.length = __builtin_amdgcn_readlane(n, from);
            s.splits = __builtin_amdgcn_readlane(splits, from);
            const int32_t at = index - __builtin_amdgcn_readlane(start, from);
            s.tile = at / s.splits;
            s.split = at % s.splits;
            s.first = index - s.split;
            s.ok = true;
            return s;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return s;
}

// A decode step: the workgroup's waves share 16 rows and take every fourth 32 keys of
// its share; their m, l and O are merged through LDS in wave order, and those of a
// tile's workgroups by the last of them to arrive, in the workgroups' order (records
// and counter as in attention.hip's decode form: device-coherent stores, completed
// before the counter is raised).
template <int H>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(3, 3)))
void split_attention_kernel(KernelArgs p) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    constexpr int RECORD = H + 4;
    __shared__ __attribute__((aligned(16))) char stages[kWaves * Stage::BYTES];
    __shared__ __attribute__((aligned(16))) char q_lds[Stage::Q_BYTES];
    __shared__ uint32_t arrived_last;
    const AttentionArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const Share share = share_of(p, Stage::MAX_SPLITS, lane);
    if (!share.ok) return;
    const int32_t tile = share.tile % p.row_tiles;
    const Rows r = rows_of(p, share.b, share.tile / p.row_tiles, tile, share.length, n);

    // q's fragments, one a wave at a time.
    for (int i = wave; i < H / 32; i += kWaves) {
        const SplitVector x = query_fragment<H>(p, r, g, i, upper);
#pragma unroll
        for (int part = 0; part < kParts; ++part)
            *reinterpret_cast<bf16x8*>(q_lds + ((i * kParts + part) * 64 + lane) * 16) = x.part[part];
    }
    __syncthreads();
    const int32_t key_first = share.split * share.keys;
    const int32_t end = min(r.some_see, share.splits > 1 ? key_first + share.keys : r.some_see);
    char* const stage = stages + wave * Stage::BYTES;
    Running<H> run;
    walk<H>(p, r, key_first + wave * kKeys, kKeys * kWaves, end, stage, n, g, upper,
            [&](int i, int part) __attribute__((always_inline)) {
                return *reinterpret_cast<const bf16x8*>(q_lds + ((i * kParts + part) * 64 + lane) * 16);
            },
            run);
    run.l = run.l + __shfl_xor(run.l, 16);
    run.l = run.l + __shfl_xor(run.l, 32);

    float* mine = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int d = 0; d < H / 16; ++d) *reinterpret_cast<f32x4*>(mine + n * Stage::O_ROW + 16 * d + 4 * g) = run.o[d];
    if (g == 0) {
        mine[kRows * Stage::O_ROW + n] = run.m;
        mine[kRows * Stage::O_ROW + kRows + n] = run.l;
    }
    __syncthreads();
    const uint32_t first_row = uint32_t(tile) * kRows;
    const int rows = int(min(uint32_t(a.queries) * uint32_t(p.group) - first_row, uint32_t(kRows)));
    auto out_of = [&](int row) __attribute__((always_inline)) {
        const uint32_t at = first_row + row;
        return a.out + r.b * a.out_sequence + (r.kv_head * p.group + at % uint32_t(p.group)) * a.out_head +
               int64_t(at / uint32_t(p.group)) * a.out_row;
    };
    const __amdgpu_buffer_rsrc_t records = gemm::buffer_of(p.records + int64_t(share.first) * kRows * RECORD);
    for (int e = tid; e < rows * (H / 4); e += kThreads) {
        const int row = e / (H / 4), piece = e % (H / 4);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            top = fmaxf(top, reinterpret_cast<const float*>(stages + w * Stage::BYTES)[kRows * Stage::O_ROW + row]);
        float total = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float* from = reinterpret_cast<const float*>(stages + w * Stage::BYTES);
            const float weight = top == -INFINITY ? 1.f : exp2_of(from[kRows * Stage::O_ROW + row] - top);
            total = total + weight * from[kRows * Stage::O_ROW + kRows + row];
            sum = sum + weight * *reinterpret_cast<const f32x4*>(from + row * Stage::O_ROW + 4 * piece);
        }
        if (share.splits == 1) {
            const float inverse = 1.f / total;
            float* to = out_of(row) + 4 * piece;
#pragma unroll
            for (int c = 0; c < 4; ++c) to[c] = total == 0.f ? 0.f : sum[c] * inverse;
        } else {
            const int32_t at = (share.split * kRows + row) * RECORD;
            gemm::buffer_store4_coherent(records, (at + 4 * piece) * 4, sum);
            if (piece == 0) gemm::buffer_store4_coherent(records, (at + H) * 4, f32x4{top, total, 0.f, 0.f});
        }
    }
    if (share.splits == 1) return;
    __builtin_amdgcn_s_waitcnt(0);  // this thread's record is complete device-wide
    __syncthreads();
    uint32_t* const counter = p.counters + int64_t(share.b) * a.kv_heads * p.row_tiles + share.tile;
    if (tid == 0)
        arrived_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                       uint32_t(share.splits - 1);
    __syncthreads();
    if (!arrived_last) return;

    // Weights of the workgroups' records: 2^(m - the largest m), and the sums l so weighted.
    float* const weights = reinterpret_cast<float*>(stages);  // [row][split]
    float* const sums = reinterpret_cast<float*>(q_lds);      // [row]
    const int splits = share.splits;
    // 16 lanes a row.
    for (int row = tid / 16; row < rows; row += kThreads / 16) {
        float top = -INFINITY;
        for (int s = tid % 16; s < splits; s += 16) {
            const f32x4 ml = gemm::buffer_load4_coherent(records, ((s * kRows + row) * RECORD + H) * 4);
            weights[row * splits + s] = ml[0];
            top = fmaxf(top, ml[0]);
        }
#pragma unroll
        for (int step = 8; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor(top, step));
        float total = 0.f;
        for (int s = tid % 16; s < splits; s += 16) {
            const f32x4 ml = gemm::buffer_load4_coherent(records, ((s * kRows + row) * RECORD + H) * 4);
            const float weight = top == -INFINITY ? 1.f : exp2_of(ml[0] - top);
            weights[row * splits + s] = weight;
            total = total + weight * ml[1];
        }
#pragma unroll
        for (int step = 8; step > 0; step >>= 1) total = total + __shfl_xor(total, step);
        if (tid % 16 == 0) sums[row] = total;
    }
    __syncthreads();
    for (int e = tid; e < rows * (H / 4); e += kThreads) {
        const int row = e / (H / 4), piece = e % (H / 4);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        constexpr int kBatch = 8;
        for (int s0 = 0; s0 < splits; s0 += kBatch) {
            f32x4 part[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                part[u] = gemm::buffer_load4_coherent(
                    records, s0 + u < splits ? (((s0 + u) * kRows + row) * RECORD + 4 * piece) * 4 : gemm::kOutOfRange);
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (s0 + u < splits) sum = sum + weights[row * splits + s0 + u] * part[u];
        }
        const float total = sums[row], inverse = 1.f / total;
        float* to = out_of(row) + 4 * piece;
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = total == 0.f ? 0.f : sum[c] * inverse;
    }
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A prompt chunk: each wave has 16 rows of its own and walks over all their keys.
template <int H>
__global__ __launch_bounds__(kThreads) void row_attention_kernel(KernelArgs p) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    __shared__ __attribute__((aligned(16))) char stages[kWaves * Stage::BYTES];
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    // The last rows, which see the most keys, first; neighbouring workgroups are
    // key/value heads, so that one XCD's read few of them.
    const uint32_t kv_all = uint32_t(a.batch * a.kv_heads), kv = blockIdx.x % kv_all;
    const int32_t groups = (p.row_tiles + kWaves - 1) / kWaves;
    const int32_t tile = (groups - 1 - int32_t(blockIdx.x / kv_all)) * kWaves + wave;
    if (tile >= p.row_tiles) return;  // the kernel has no barrier
    const uint32_t b = kv / uint32_t(a.kv_heads);
    const Rows r = rows_of(p, b, kv % uint32_t(a.kv_heads), tile, held_by(a, b), n);
    SplitVector q[H / 32];
#pragma unroll
    for (int i = 0; i < H / 32; ++i) q[i] = query_fragment<H>(p, r, g, i, upper);
    Running<H> run;
    walk<H>(p, r, 0, kKeys, r.some_see, stages + wave * Stage::BYTES, n, g, upper,
            [&](int i, int part) __attribute__((always_inline)) { return q[i].part[part]; }, run);
    run.l = run.l + __shfl_xor(run.l, 16);
    run.l = run.l + __shfl_xor(run.l, 32);
    if (!r.ok) return;
    float* out = a.out + r.b * a.out_sequence + r.head * a.out_head + int64_t(r.t) * a.out_row;
    const float inverse = 1.f / run.l;
#pragma unroll
    for (int d = 0; d < H / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[16 * d + 4 * g + e] = run.l == 0.f ? 0.f : run.o[d][e] * inverse;
}

template <int H>
hipError_t launch(const AttentionArgs& a, KernelArgs p, hipStream_t stream) {
    const int64_t tiles = a.batch * a.kv_heads * p.row_tiles;
    const int64_t longest = a.lengths != nullptr ? a.capacity : a.keys;
    if (tiles >= 4 * a.cu_count && p.row_tiles >= kWaves) {
        const int64_t grid = a.batch * a.kv_heads * ((p.row_tiles + kWaves - 1) / kWaves);
        if (grid > INT32_MAX) return hipErrorInvalidValue;
        hipLaunchKernelGGL(row_attention_kernel<H>, dim3(unsigned(grid)), dim3(kThreads), 0, stream, p);
        return hipGetLastError();
    }
    // Three workgroups a CU are resident (registers and LDS); the keys go to about as many.
    const int64_t resident = 3 * int64_t(a.cu_count);
    const int64_t record_bytes = kRows * (H + 4) * int64_t(sizeof(float));
    const int64_t room = a.workspace != nullptr ? int64_t(a.workspace_bytes) / record_bytes : 0;
    const int64_t wanted = std::min(resident, room - tiles);
    p.least_keys = kKeys * kWaves;
    int64_t grid = tiles;
    if (wanted > 0 && tiles < resident && size_t(tiles) <= a.counter_count && longest > p.least_keys) {
        // At most `wanted` shares that are full and one a tile that is not.
        p.workgroups = int32_t(wanted);
        grid = std::min(wanted + tiles, tiles * ((longest + p.least_keys - 1) / p.least_keys));
    }
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(split_attention_kernel<H>, dim3(unsigned(grid)), dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream) {
    KernelArgs p;
    p.a = a;
    p.q_scale = a.scale * 1.44269504088896340736f;
    p.group = int32_t(a.heads / a.kv_heads);
    p.row_tiles = int32_t((a.queries * p.group + kRows - 1) / kRows);
    p.workgroups = 0;
    p.least_keys = 0;
    p.counters = a.counters;
    p.records = a.workspace;
    switch (a.head_dim) {
        case 32: return launch<32>(a, p, stream);
        case 64: return launch<64>(a, p, stream);
        default: return launch<128>(a, p, stream);
    }
}

}  // namespace fp4
}  // namespace sn
