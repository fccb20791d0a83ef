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
//    quarter g of key n); q is split exactly in three bf16 parts (fp4_device.h; what they leave of
//    values under 2^-110 is a product more, by workgroups that have such values).
//  * The softmax is per lane but for the maximum over the four lanes of a query.
//  * O^T += V^T P^T: a lane's eight probabilities, split, are the right operand as
//    they are, the operand's inner index being keys 4 g .. + 3 of the first 16 and
//    then of the second. V's codes become bf16 rows in LDS (a region of the wave's
//    own, no barrier) and are read back transposed in that order.
// Every product is exact; sums, maxima and probabilities are fp32.
//
// A workgroup's waves share 16 rows and take the steps in turn, q's parts in LDS. (Waves with
// rows of their own, each walking over all keys, left two waves a SIMD in step with the
// longest sequence: 292 us for two 1000-query chunks against up to 6001 positions, 197 so.)
// Where there are few rows (a decode step) workgroups share a tile's keys as well.
//   What bounds it: 64 heads on 8 of 131071 keys, 143 MB, 37 to 41 us (3.5 to 3.9 TB/s); 16 sequences of up to 8192 keys, 12.6 us,
// and 12 heads on 701 keys, 8.2 us: one launch and a chain of loads, steps and the merge. Chunks of 1000
// queries against 6001 keys: 195 to 210 us, 0.8 to 0.9 PFLOP/s of bf16 products, where conversions, exponentials, splits and LDS
// each take about as long as the matrix cores, which are busy 42 % of the cycles.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "fp4_device.h"
#include "fp4_internal.h"
#include "gemm_common.h"

namespace sn {
namespace fp4 {
namespace {

constexpr int kRows = 16;  // queries of a wave
constexpr int kKeys = 32;  // keys of a step
constexpr int kSplitWaves = 8;  // of a workgroup where several share a tile's keys
constexpr int kTileWaves = 4;   // of one that has a tile to itself, where tiles fill the CUs

struct KernelArgs {
    AttentionArgs a;
    float q_scale;          // scale log2 e
    int32_t group;          // query heads of a key/value head
    int32_t row_tiles;      // of a key/value head
    int32_t workgroups;     // that share the keys, but for one more a tile (0: one to a tile)
    int32_t least_keys;     // of a workgroup's share, a multiple of kKeys kSplitWaves
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
    const uint32_t group = uint32_t(p.group), rows = uint32_t(p.a.queries) * group;  // under 2^27
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

// Fragment i of this lane's query, split: head dims g H / 4 + 8 i .. + 7, as K's words hold them. `left` notices what the
// parts leave of them; query_rest has that, lifted, as two parts.
template <int H>
__device__ __forceinline__ void query_values(const KernelArgs& p, const Rows& r, int g, int i, float (&x)[8]) {
    const float* from = p.a.q + r.b * p.a.q_sequence + r.head * p.a.q_head + r.t * p.a.q_row + g * (H / 4) + 8 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = r.ok ? from[e] * p.q_scale : 0.f;
}
template <int H>
__device__ __forceinline__ SplitVector query_fragment(const KernelArgs& p, const Rows& r, int g, int i,
                                                      uint32_t upper, uint32_t& left) {
    float x[8];
    query_values<H>(p, r, g, i, x);
    return split_exact(x, upper, left);
}
template <int H>
__device__ __forceinline__ SplitVector query_rest(const KernelArgs& p, const Rows& r, int g, int i, uint32_t upper) {
    float x[8];
    query_values<H>(p, r, g, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = rest_of(x[e], upper);
    return split_finite(x, upper);
}

// The running softmax of a wave's rows: m and the unscaled O of this lane's query (dims
// 16 d + 4 g + r), and l over this lane's keys.
template <int H>
struct Running {
    float m = -INFINITY, l = 0.f;
    f32x4 o[H / 16];
};

// Keys key0, key0 + step, .. before `end`, 32 at a time. q(i, part): the fragments of q.
// The scores of the next step are formed beside the softmax and O of this one, so that the
// matrix cores and the vector units have work of their own; codes are loaded two steps
// (K) and one (V) ahead. m is raised only where a score passes it by 8 (numerators up to
// 2^8 are as exact), which after a few steps is never: O is hardly rescaled.
// ready() makes them usable, while the first codes are on their way, and tells whether they leave something of q; then
// each step's scores are corrected by a product with that, from codes loaded again.
template <int H, class Ready, class Query>
__device__ __forceinline__ void walk(const KernelArgs& p, const Rows& r, int32_t key0, int32_t step, int32_t end,
                                     char* stage, int n, int g, uint32_t upper, Ready&& ready, Query&& q,
                                     Running<H>& run) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    constexpr int NF = H / 32;     // fragments of 32 over the head dim: words of a lane's quarter
    constexpr int TILES = H / 16;  // 16-column tiles of O
    const AttentionArgs& a = p.a;
#pragma unroll
    for (int d = 0; d < TILES; ++d) run.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The step's rows from a base the wave shares, and the lane's offsets from it.
    const int64_t cache_row = (r.b * a.kv_heads + r.kv_head) * a.capacity;
    const uint32_t code_at = g * (H / 8), scale_at = g * (H / 4) / 32;
    struct Words {
        uint32_t w[2][NF];
        uint32_t s[2];
    };
    // The 32 keys from `first` on (a step's, so `first` is under `end`); keys past the end
    // read the last key (their scores and values are replaced).
    auto load = [&](const uint8_t* codes, const uint8_t* scales, int32_t first, Words& x)
                    __attribute__((always_inline)) {
        codes += (cache_row + first) * (H / 2);
        scales += (cache_row + first) * (H / 32);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t key = uint32_t(min(16 * u + n, end - 1 - first));
            const uint8_t* from = codes + (key * (H / 2) + code_at);
            if constexpr (NF == 4) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(from);
                x.w[u][0] = v[0], x.w[u][1] = v[1], x.w[u][2] = v[2], x.w[u][3] = v[3];
            } else if constexpr (NF == 2) {
                const u32x2 v = *reinterpret_cast<const u32x2*>(from);
                x.w[u][0] = v[0], x.w[u][1] = v[1];
            } else {
                x.w[u][0] = *reinterpret_cast<const uint32_t*>(from);
            }
            x.s[u] = scales[key * (H / 32) + scale_at];
        }
    };
    struct Scores {
        f32x4 s[2];
    };
    // Two chains of sums a tile (the first parts, and the others), so that they overlap.
    auto scores = [&](const Words& k) __attribute__((always_inline)) {
        f32x4 most[2], rest[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) most[u] = rest[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float factor[2] = {factor_of(k.s[0]), factor_of(k.s[1])};
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            bf16x8 f[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) f[u] = fragment_of(k.w[u][i], factor[u]);
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part) {
                const bf16x8 x = q(i, part);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    f32x4& to = part == 0 ? most[u] : rest[u];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[u], x, to, 0, 0, 0);
                }
            }
        }
        Scores out;
#pragma unroll
        for (int u = 0; u < 2; ++u) out.s[u] = most[u] + rest[u];
        return out;
    };
    char* const v_write = stage + n * Stage::ROW + g * (H / 2);
    const char* const v_read = stage + (4 * g + (n >> 2)) * Stage::ROW + 8 * (n & 3);

    Words k_next, v_next;
    if (key0 < end) {
        load(a.k_codes, a.k_scales, key0, k_next);
        load(a.v_codes, a.v_scales, key0, v_next);
    }
    const bool left = ready();
    if (key0 >= end) return;
    Scores s_next = scores(k_next);
    load(a.k_codes, a.k_scales, min(key0 + step, end - 1), k_next);
    for (; key0 < end; key0 += step) {
        Scores s = s_next;
        Words v = v_next;
        if (left) {
            Words k;
            load(a.k_codes, a.k_scales, key0, k);
            f32x4 rest[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                const SplitVector x = query_rest<H>(p, r, g, i, upper);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int part = 1; part >= 0; --part)
                        rest[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fragment_of(k.w[u][i], factor_of(k.s[u])),
                                                                          x.part[part], rest[u], 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) s.s[u] = s.s[u] + rest[u] * (1.f / kRestLift);
        }
        // What queries do not see is replaced: -inf for its scores, 0 for its values, since
        // 0 x NaN would reach them. NaN blocks of keys that some queries see are taken out as
        // well, and those queries given NaN below.
        uint64_t poison[2] = {0, 0};
        if (key0 + kKeys > r.all_see || key0 + kKeys > end) {  // of the wave
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int32_t key = key0 + 16 * u + n;
                const bool nan = v.s[u] > kLargestScale;
                poison[u] = __ballot(nan && key < end);
                if (nan || key >= end) {
                    v.s[u] = 127;
#pragma unroll
                    for (int i = 0; i < NF; ++i) v.w[u][i] = 0;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t k = key0 + 16 * u + 4 * g + e;
                    s.s[u][e] = k <= r.last && k < end ? s.s[u][e] : -INFINITY;
                }
            }
        }
        const float top = largest_of_four(fmaxf(fmaxf(fmaxf(s.s[0][0], s.s[0][1]), fmaxf(s.s[0][2], s.s[0][3])),
                                                fmaxf(fmaxf(s.s[1][0], s.s[1][1]), fmaxf(s.s[1][2], s.s[1][3]))));
        if (__any(top > run.m + 8.f)) {
            const float m_new = fmaxf(run.m, top);
            const float alpha = m_new == -INFINITY ? 1.f : exp2_of(run.m - m_new);
            run.m = m_new;
            run.l = run.l * alpha;
#pragma unroll
            for (int d = 0; d < TILES; ++d) run.o[d] = run.o[d] * alpha;
        }
        // Past the last step these are the last key again, and not used: no branch divides the
        // matrix instructions from the vector ones.
        load(a.v_codes, a.v_scales, min(key0 + step, end - 1), v_next);
        s_next = scores(k_next);
        load(a.k_codes, a.k_scales, min(key0 + 2 * step, end - 1), k_next);

#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float factor = factor_of(v.s[u]);
#pragma unroll
            for (int i = 0; i < NF; ++i)
                *reinterpret_cast<bf16x8*>(v_write + 16 * u * Stage::ROW + 16 * i) = fragment_of(v.w[u][i], factor);
        }
        const float base = run.m == -INFINITY ? 0.f : run.m;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = exp2_of(s.s[e / 4][e % 4] - base);
        // The step's sum first: one by one, a lane's sum of equal weights would end at 2^24 of them.
        run.l = run.l + (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
        const SplitVector pr = split_finite(x, upper);  // a NaN reaches the result through l
        wave_lds_order();
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const bf16x8 f = transposed(v_read + 32 * d, v_read + 16 * Stage::ROW + 32 * d);
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part)
                run.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pr.part[part], run.o[d], 0, 0, 0);
        }
        wave_lds_order();
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

// Sums over lanes 0 .. this one (neighbours within rows of 16, then rows: data-parallel
// moves, no LDS).
__device__ __forceinline__ uint32_t sums_up_to_lane(uint32_t x) {
    auto move = [](auto control, auto rows, uint32_t v) __attribute__((always_inline)) {
        return uint32_t(
            __builtin_amdgcn_update_dpp(0, int(v), decltype(control)::value, decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    x += move(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}, x);  // from the lane before
    x += move(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}, x);  // two before
    x += move(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}, x);
    x += move(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}, x);
    x += move(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}, x);  // lane 15 to row 1, 47 to row 3
    x += move(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}, x);  // lane 31 to rows 2 and 3
    return x;
}

// A workgroup's share of the keys, from the lengths as the device has them. Sequence b's
// n keys go to ceil(n / share) workgroups for each of its row tiles, or to one where n
// is at most two least shares (merging two records costs what they save: 300 keys 7.2 us
// in one, 8.7 in two; 701 8.8 and 8.6). share is an even share of all keys, raised by
// eighths until the workgroups that have over half a share number at most p.workgroups,
// so that none of them waits for another to end (80 tiles of 4000 keys on 256
// workgroups: 33 us with 320 shares, 21 with 240). Consecutive workgroups take consecutive
// shares of a tile, tiles of a sequence, sequences.
struct Share {
    int32_t b, length, keys;  // keys: that a workgroup takes
    int32_t tile;             // of the sequence: kv_head * row_tiles + row tile
    int32_t split, splits;
    int32_t first;            // the tile's first workgroup
    bool ok;
};
__device__ __forceinline__ Share share_of(const KernelArgs& p, int lane) {
    const AttentionArgs& a = p.a;
    const int32_t tiles = int32_t(a.kv_heads) * p.row_tiles;  // of a sequence
    constexpr int32_t kUnit = kKeys * kSplitWaves;
    const int32_t index = int32_t(blockIdx.x);
    Share s = {};
    s.splits = 1;
    if (p.workgroups == 0) {
        // The last rows, which see the most keys, first; a head's next rows go to the next XCD, so
        // that each has rows of long and of short sequences (one XCD a head: 289 us for two
        // chunks of different lengths, 197 so).
        const int32_t heads = int32_t(a.batch * a.kv_heads), head = (index % heads + index / heads) % heads;
        s.b = head / int32_t(a.kv_heads);
        s.length = held_by(a, s.b);
        s.tile = head % int32_t(a.kv_heads) * p.row_tiles + (p.row_tiles - 1 - index / heads);
        s.first = index;
        s.ok = true;
        return s;
    }
    const int32_t batch = int32_t(a.batch);  // under p.workgroups
    auto held = [&](int32_t b) __attribute__((always_inline)) { return b < batch ? held_by(a, b) : 0; };
    const int32_t n0 = held(lane);
    // The sum over the sequences of f(keys held).
    auto sum_over = [&](auto f) __attribute__((always_inline)) {
        if (batch == 1) return int64_t(uint32_t(__builtin_amdgcn_readfirstlane(f(n0))));
        int64_t sum = 0;
        for (int32_t b0 = 0; b0 < batch; b0 += 64) {
            const int32_t n = b0 == 0 ? n0 : held(b0 + lane);
            sum += uint32_t(__builtin_amdgcn_readlane(sums_up_to_lane(b0 + lane < batch ? f(n) : 0), 63));
        }
        return sum;
    };
    const int64_t even = sum_over([](int32_t n) { return n / kKeys; }) * tiles / p.workgroups * kKeys;
    int32_t keys = max(p.least_keys, int32_t((min(even, a.capacity) + kUnit - 1) / kUnit) * kUnit);
    auto splits_of = [&](int32_t n) __attribute__((always_inline)) {
        return n <= 2 * p.least_keys ? 1 : (n - 1) / keys + 1;  // n + keys may pass 2^31
    };
    auto filled = [&](int32_t n) __attribute__((always_inline)) { return n > keys / 2 ? splits_of(n) : 0; };
    while (keys < a.capacity && sum_over(filled) * tiles > p.workgroups)
        keys = min(int32_t(a.capacity) + kUnit, (keys + keys / 8 + kUnit - 1) / kUnit * kUnit);
    s.keys = __builtin_amdgcn_readfirstlane(keys);
    int32_t before = 0;  // workgroups of the sequences so far
    for (int32_t b0 = 0; b0 < batch; b0 += 64) {
        const int32_t n = b0 == 0 ? n0 : held(b0 + lane);
        const int32_t splits = b0 + lane < batch ? splits_of(n) : 0;
        const int32_t sum = int32_t(sums_up_to_lane(splits * tiles));
        const int32_t start = before + sum - splits * tiles;
        const uint64_t mine = __ballot(index >= start && index < start + splits * tiles);
        if (mine != 0) {
            const int from = __builtin_ctzll(mine);
            s.b = b0 + from;
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

// 16 rows: the waves' m, l and O are merged through LDS in wave order, and, where
// workgroups share the tile's keys, those of the workgroups by the last of them to
// arrive, in the workgroups' order (records and counter as in attention.hip's decode
// form: device-coherent stores, completed before the counter is raised).
template <int H, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void attention_kernel(KernelArgs p) {
#pragma clang fp contract(off)
    using Stage = WaveStage<H>;
    constexpr int RECORD = H + 4;
    constexpr int PIECES = H / 4;
    __shared__ __attribute__((aligned(16))) char stages[W * Stage::BYTES];
    __shared__ __attribute__((aligned(16))) char q_lds[Stage::Q_BYTES];
    __shared__ uint32_t arrived_last;
    __shared__ uint32_t fragments_left;  // a byte each: whether its parts leave something of q
    const AttentionArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const uint32_t upper = upper_half_mask();
    const Share share = share_of(p, lane);
    if (!share.ok) return;
    const int32_t tile = share.tile % p.row_tiles;
    const Rows r = rows_of(p, share.b, share.tile / p.row_tiles, tile, share.length, n);
    const int32_t key_first = share.split * share.keys;
    const int32_t end = min(r.some_see, share.splits > 1 ? key_first + share.keys : r.some_see);
    char* const stage = stages + wave * Stage::BYTES;
    Running<H> run;
    walk<H>(p, r, key_first + wave * kKeys, kKeys * W, end, stage, n, g, upper,
            [&]() __attribute__((always_inline)) {  // q's fragments, one a wave
                static_assert(H / 32 <= W, "a wave has at most one");
                if (wave < H / 32) {
                    uint32_t left = 0;
                    const SplitVector x = query_fragment<H>(p, r, g, wave, upper, left);
                    const bool any = __any(noticed(left));
                    if (lane == 0) reinterpret_cast<uint8_t*>(&fragments_left)[wave] = any;
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        *reinterpret_cast<bf16x8*>(q_lds + ((wave * kParts + part) * 64 + lane) * 16) = x.part[part];
                }
                __syncthreads();
                return (__builtin_amdgcn_readfirstlane(fragments_left) & (~0u >> (32 - H / 4))) != 0;
            },
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
    const int units = rows * PIECES;  // of four floats of a row, at most 512
    auto store = [&](int unit, float total, f32x4 sum) __attribute__((always_inline)) {
        const uint32_t at = first_row + uint32_t(unit / PIECES);
        float* to = a.out + r.b * a.out_sequence + (r.kv_head * p.group + at % uint32_t(p.group)) * a.out_head +
                    int64_t(at / uint32_t(p.group)) * a.out_row + 4 * (unit % PIECES);
        const float inverse = 1.f / total;
        // No term: nothing is seen, or every score is -inf, of which there is no softmax.
        const float nothing = share.length - int32_t(a.queries) + int32_t(at / uint32_t(p.group)) < 0 ? 0.f : NAN;
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = total == 0.f ? nothing : sum[c] * inverse;
    };
    const __amdgpu_buffer_rsrc_t records = gemm::buffer_of(p.records + int64_t(share.first) * kRows * RECORD);
    for (int unit = tid; unit < units; unit += 64 * W) {
        const int row = unit / PIECES, piece = unit % PIECES;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w)
            top = fmaxf(top, reinterpret_cast<const float*>(stages + w * Stage::BYTES)[kRows * Stage::O_ROW + row]);
        float total = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float* from = reinterpret_cast<const float*>(stages + w * Stage::BYTES);
            const float weight = top == -INFINITY ? 1.f : exp2_of(from[kRows * Stage::O_ROW + row] - top);
            total = total + weight * from[kRows * Stage::O_ROW + kRows + row];
            sum = sum + weight * *reinterpret_cast<const f32x4*>(from + row * Stage::O_ROW + 4 * piece);
        }
        if (share.splits == 1) {
            store(unit, total, sum);
        } else {
            const int32_t at = (share.split * kRows + row) * RECORD;
            gemm::buffer_store4_coherent(records, (at + 4 * piece) * 4, sum);
            if (piece == 0) gemm::buffer_store4_coherent(records, (at + H) * 4, f32x4{top, total, 0.f, 0.f});
        }
    }
    if (W != kSplitWaves || share.splits == 1) return;
    static_assert(W != kSplitWaves || kRows * PIECES <= 64 * W, "a thread has at most one unit below");
    __builtin_amdgcn_s_waitcnt(0);  // this thread's record is complete device-wide
    __syncthreads();
    uint32_t* const counter = p.counters + int64_t(share.b) * a.kv_heads * p.row_tiles + share.tile;
    if (tid == 0)
        arrived_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                       uint32_t(share.splits - 1);
    __syncthreads();
    if (!arrived_last) return;

    // Threads of group j fold records j, j + groups, .. of their unit, eight in flight, and
    // group 0 the groups' results, in that order.
    constexpr int kBatch = 8;
    const int groups = min(64 * W / units, (share.splits + kBatch - 1) / kBatch);
    const int group = tid / units, unit = tid % units;
    float m = -INFINITY, l = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (group < groups) {
        const int32_t row_at = unit / PIECES * RECORD, piece_at = 4 * (unit % PIECES);
        for (int s0 = group; s0 < share.splits; s0 += kBatch * groups) {
            f32x4 ml[kBatch], part[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int s = s0 + u * groups;
                const int32_t at = s * kRows * RECORD + row_at;
                ml[u] = gemm::buffer_load4_coherent(records, s < share.splits ? (at + H) * 4 : gemm::kOutOfRange);
                part[u] =
                    gemm::buffer_load4_coherent(records, s < share.splits ? (at + piece_at) * 4 : gemm::kOutOfRange);
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (s0 + u * groups >= share.splits) ml[u][0] = -INFINITY;  // read as zeros: weight 0
                top = fmaxf(top, ml[u][0]);
            }
            const float base = top == -INFINITY ? 0.f : top, kept = exp2_of(m - base);
            m = top;
            l = l * kept;
            sum = sum * kept;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const float weight = exp2_of(ml[u][0] - base);
                l = l + weight * ml[u][1];
                sum = sum + weight * part[u];
            }
        }
    }
    if (groups == 1) {
        if (group == 0) store(unit, l, sum);
        if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    // (Every thread is past its last read of the stages: two barriers ago.)
    float* const folded = reinterpret_cast<float*>(stages);  // [group][unit]: O, m, l
    static_assert(64 * W * 24 <= W * Stage::BYTES, "the groups' results fit the stages");
    if (group < groups) {
        float* to = folded + 6 * tid;
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = sum[c];
        to[4] = m;
        to[5] = l;
    }
    __syncthreads();
    if (group == 0) {
        float top = m;
        for (int j = 1; j < groups; ++j) top = fmaxf(top, folded[6 * (j * units + unit) + 4]);
        const float base = top == -INFINITY ? 0.f : top, kept = exp2_of(m - base);
        l = l * kept;
        sum = sum * kept;
        for (int j = 1; j < groups; ++j) {
            const float* from = folded + 6 * (j * units + unit);
            const float weight = exp2_of(from[4] - base);
            l = l + weight * from[5];
            sum = sum + weight * f32x4{from[0], from[1], from[2], from[3]};
        }
        store(unit, l, sum);
    }
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int H>
hipError_t launch(const AttentionArgs& a, KernelArgs p, hipStream_t stream) {
    const int64_t tiles = a.batch * a.kv_heads * p.row_tiles;
    const int64_t longest = a.lengths != nullptr ? a.capacity : a.keys;
    // Workgroups of eight waves that a CU has room for (LDS at h = 128, registers else).
    const int64_t resident = (H == 128 ? 1 : 2) * int64_t(a.cu_count);
    const int64_t record_bytes = kRows * (H + 4) * int64_t(sizeof(float));
    const int64_t room = a.workspace != nullptr ? int64_t(a.workspace_bytes) / record_bytes : 0;
    const int64_t wanted = std::min(resident, room - tiles);
    p.least_keys = kKeys * kSplitWaves;
    int64_t grid = tiles;
    if (wanted > tiles && size_t(tiles) <= a.counter_count && longest > 2 * p.least_keys) {
        // Besides the shares over half full, which are at most `wanted`, one a tile.
        p.workgroups = int32_t(wanted);
        grid = std::min(wanted + tiles, tiles * ((longest + p.least_keys - 1) / p.least_keys));
    }
    // Tiles that fill the CUs by themselves need no eight waves each: of 3000 keys with h = 128, 400 tiles
    // take 45.4 us of eight waves and 41.2 of four, 1600 tiles 147 and 125. (Fewer tiles are
    // shared where the workspace allows it, else each has what one workgroup can give; 48 of 300 keys: 6.8
    // either way.)
    if (tiles > resident)
        hipLaunchKernelGGL((attention_kernel<H, kTileWaves>), dim3(unsigned(grid)), dim3(64 * kTileWaves), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_kernel<H, kSplitWaves>), dim3(unsigned(grid)), dim3(64 * kSplitWaves), 0, stream, p);
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
