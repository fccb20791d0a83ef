// Log probabilities of given tokens, entropies and the likeliest classes, and
// their gradient (staleynet_logprobs.h has the formulas).
//
// With m the largest logit, z = a (x - m) and rest = the sum of e^z without one
// term of the largest: T = log(1 + rest), logprob = z_token - T, H = T + W / (1 +
// rest), W = the sum of e^z (-z), all of whose terms are positive. e^z is 2^(z log2 e)
// on the transcendental unit (v_exp_f32, about 1 ulp); the factor a log2 e and its
// product with x - m add at most 2^-23 |z| to a term's relative error.
//
// Bound by memory: 4 bytes a logit forward, 8 backward. A wave holds up to 2048
// classes of a row's head in registers, so a logit is read once: their maximum,
// then the sums, then the likeliest. Longer rows are chunks of 2048 whose {m,
// rest, W} are merged, and where rows are few the chunks go to several waves,
// whose parts a second kernel merges in order (joining them in the first, by the
// last wave to arrive, took as long: 25.6 us against 24.9, 128 x 131072 with 20
// listed).
//
// The likeliest k of a chunk: the k-th largest of the 64 lanes' maxima, found by
// bisection over ballots, is a bound that at least k values reach and few
// others do; those are gathered in LDS and each finds its rank by comparing
// with all. Where too many reach it (many equal values) they are taken one by
// one instead.
//
// 128 x 131072 (67 MB): 13.0 us (5.2 TB/s) and 4 for the merge; 18.5 and 7.5 with
// 20 listed, three quarters of the vector units' cycles. 4096 x 16 x 1024: 48.5 us
// (5.5 TB/s), 69 with 5 listed; its gradient 94 us (5.7 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "logprobs_internal.h"

namespace sn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_unaligned __attribute__((aligned(4)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;          // of a workgroup, each on its own
constexpr int kChunk = 2048;       // classes a wave holds
constexpr int kLargestTop = SN_LOGPROBS_LARGEST_TOP;
constexpr int kCandidates = 96;    // gathered at once
constexpr int kListed = kCandidates + kLargestTop;
constexpr uint32_t kEmptyToken = SN_EMPTY_TOKEN;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// An order of logits as integers: NaN is the largest, -0 equals 0; 0 is below all.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.f);
    return x != x ? 0xffffffffu : bits ^ (uint32_t(int32_t(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t kLeastKey = 0x007fffffu;  // of -inf
// A class with its logit, ordered by the logit and then with the lower class ahead; all are above 0 and below ~0.
constexpr uint32_t kClassMask = 0x7fffffffu;
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t c) { return uint64_t(key) << 32 | (kClassMask - c); }
__device__ __forceinline__ uint32_t class_of(uint64_t entry) { return kClassMask - uint32_t(entry); }

// Reductions over a wave by lane moves within the vector unit (DPP: 1, 2, 4 and 8 lanes within a row of 16, then the
// rows' last lanes to the next rows): lane 63 has the result, which a scalar register takes. A move's lanes without a
// source keep `rest`.
template <int CONTROL, int ROWS>
__device__ __forceinline__ float moved(float v, float rest) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, rest), __builtin_bit_cast(int, v),
                                                                 CONTROL, ROWS, 0xf, false));
}
template <class Op>
__device__ __forceinline__ float wave_reduce(float v, float rest, Op op) {
    v = op(v, moved<0x111, 0xf>(v, rest));
    v = op(v, moved<0x112, 0xf>(v, rest));
    v = op(v, moved<0x114, 0xf>(v, rest));
    v = op(v, moved<0x118, 0xf>(v, rest));
    v = op(v, moved<0x142, 0xa>(v, rest));
    v = op(v, moved<0x143, 0xc>(v, rest));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const uint64_t other = uint64_t(__shfl_xor(static_cast<unsigned long long>(v), step));
        v = other > v ? other : v;
    }
    return v;
}
// Between a wave's writes of LDS and its other lanes' reads of them, and back: the hardware
// keeps the order of one wave's accesses, the fences the compiler's.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// a log2 e, finite: at 0 differences it gives 0.
__device__ __forceinline__ float factor_of(float scale) { return fminf(scale * kLog2e, FLT_MAX); }
// The largest logit of some classes, the sum of the others' e^z and W over them, in units of log2 e.
struct Sums {
    float m, rest, weighted;
};
// Those of both. A part without a finite logit has m = -inf and rest = 0, or NaN.
__device__ __forceinline__ Sums merged(Sums a, Sums b, float factor) {
    if (b.m > a.m) {
        const Sums t = a;
        a = b;
        b = t;
    }
    if (b.m == -INFINITY) {
        a.rest += b.rest;
        return a;
    }
    const float away = (a.m - b.m) * factor, e = __builtin_amdgcn_exp2f(-away);
    a.rest += e * (1.f + b.rest);
    a.weighted += e > 0.f ? e * (b.weighted + (1.f + b.rest) * away) : 0.f;
    return a;
}

// The `top` largest of `count` entries, at most kListed, made(0) .. made(count - 1) from the list, sorted to the list's
// start: each lane's entries, two at most, find their ranks. Returns how many there are.
template <class Made>
__device__ __forceinline__ int rank_entries(uint64_t* list, int count, int top, Made made) {
    const int lane = threadIdx.x & 63;
    const uint64_t first = lane < count ? made(lane) : 0, second = lane + 64 < count ? made(lane + 64) : 0;
    wave_lds_order();
    list[lane] = first;
    if (count > 64) list[lane + 64] = second;
    wave_lds_order();
    int rank1 = 0, rank2 = 0;
#pragma unroll 4
    for (int i = 0; i < count; i += 2) {  // the list read two at once by all lanes, with zeros behind the last
        const u64x2 others = *reinterpret_cast<const u64x2*>(&list[i]);
        rank1 += (others[0] > first) + (others[1] > first);
        if (count > 64) rank2 += (others[0] > second) + (others[1] > second);
    }
    wave_lds_order();
    if (lane < count && rank1 < top) list[rank1] = first;
    if (lane + 64 < count && rank2 < top) list[rank2] = second;
    wave_lds_order();
    return min(count, top);
}
static_assert(kListed == 128, "two entries a lane");

// The `top` largest entries of a chunk's values and of the `held` sorted ones in list[0 .. held), sorted, to list[0 .. top);
// returns how many there are. Lane l's value i is of class chunk + 4 (l + 64 (i / 4)) + i % 4, in memory at x[class], none
// from `end` on; `largest` is the lane's largest, NaN aside, and `nan` says, the same in all lanes, whether there is one.
// Where `top` are held, a value has to be above the last of them (its class is higher). The list has room for kListed
// entries.
template <int N>
__device__ __forceinline__ int select_top(const float (&value)[N], const float* x, uint32_t chunk, uint32_t end, float largest,
                                          bool nan, int top, uint64_t* list, int held) {
    const int lane = threadIdx.x & 63;
    const auto class_at = [&](int i) { return chunk + 4 * (lane + 64 * (i / 4)) + i % 4; };
    // Keys from `bound` on are candidates. At first what is above the held ones, or any (-inf's key is the least).
    uint32_t bound = held == top ? uint32_t(__builtin_amdgcn_readfirstlane(int(list[top - 1] >> 32))) : kLeastKey - 1;
    if (bound == 0xffffffffu) return held;  // as many NaN
    ++bound;
    int count = held;
    if (!nan) {
        const uint32_t key = key_of(largest);
        if (!__any(key >= bound)) return held;
        // The `top`-th largest of the lanes' maxima, to 16 bits: `top` values reach it, and few more. Not needed where
        // few lanes have anything above the held ones.
        uint32_t reached = 0;
        const auto bisect = [&](uint32_t bit) {
            if (__popcll(__ballot(key >= (reached | bit))) >= top) reached |= bit;
        };
        if (__popcll(__ballot(key >= bound)) > kLargestTop / 2) {
#pragma unroll
            for (int b = 31; b >= 16; --b) bisect(1u << b);
            bound = max(bound, reached);
        }
        const auto gather = [&](float v, uint32_t c, float least) {
            const bool candidate = v >= least && c < end;
            const uint64_t mask = __ballot(candidate);
            const int at = count + __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
            if (candidate && at < kListed)  // made an entry below, once for all
                list[at] = uint64_t(__builtin_bit_cast(uint32_t, v)) << 32 | c;
            count += __popcll(mask);
        };
        const float least = logit_of(bound);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (__ballot(value[i] >= least) != 0) gather(value[i], class_at(i), least);
        // Too many within 2^-7 of the bound: to all its bits, from memory.
        if (count > kListed) {
            reached = 0;
#pragma nounroll
            for (int b = 31; b >= 0; --b) bisect(1u << b);
            bound = max(bound, reached);
            count = held;
#pragma nounroll
            for (int i = 0; i < N; ++i) {
                const uint32_t c = class_at(i);
                gather(c < end ? x[c] : -INFINITY, c, logit_of(bound));
            }
        }
        wave_lds_order();
    }
    if (nan || count > kListed) {
        // One by one: the largest below the last, of the lanes' values and of the list's first `held`.
        const uint64_t own = lane < held ? list[lane] : 0;
        uint64_t mine = 0, last = ~uint64_t(0);
        wave_lds_order();
        int found = 0;
        for (; found < top; ++found) {
            uint64_t best = own < last ? own : 0;
#pragma nounroll
            for (int i = 0; i < N; ++i) {
                const uint32_t c = class_at(i), key = c < end ? key_of(x[c]) : 0;
                const uint64_t entry = key >= bound ? entry_of(key, c) : 0;
                if (entry < last && entry > best) best = entry;
            }
            last = wave_largest(best);
            if (last == 0) break;
            if (lane == found) mine = last;
        }
        if (lane < found) list[lane] = mine;
        wave_lds_order();
        return found;
    }
    return rank_entries(list, count, top, [&](int at) {
        const uint64_t found = list[at];
        return at < held ? found : entry_of(key_of(__builtin_bit_cast(float, uint32_t(found >> 32))), uint32_t(found));
    });
}

// Where a place's head starts in the logits and its token in the tokens.
struct Place {
    int64_t logits, token;
};
template <class Args>
__device__ __forceinline__ Place place_of(const Args& a, uint32_t place) {
    uint32_t row = place, head = 0;
    if (a.heads > 1) {
        row = place / uint32_t(a.heads);
        head = place - row * uint32_t(a.heads);
    }
    return Place{row * a.cols + a.column_offset + head * a.classes, row * a.token_stride + a.token_offset + head};
}

// The given token and its logit (NaN where it is no class), read ahead of what is computed meanwhile.
struct Given {
    uint32_t token;
    float logit;
};
__device__ __forceinline__ Given given_of(const LogprobArgs& a, const Place& at) {
    Given g = {kEmptyToken, NAN};
    if (a.logprobs == nullptr) return g;
    g.token = a.tokens[at.token];
    if (g.token < uint64_t(a.classes)) g.logit = a.logits[at.logits + g.token];
    return g;
}

// A place's results: from its sums and its list.
__device__ __forceinline__ void finish(const LogprobArgs& a, uint32_t place, const Given& given, Sums s, const uint64_t* list,
                                       int found) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63;
    if (!(fabsf(s.m) < INFINITY) || s.rest != s.rest) s.m = s.rest = NAN;
    const float log_total = log1pf(s.rest);
    if (lane == 0) {
        if (a.logprobs != nullptr)
            a.logprobs[place] = given.token == kEmptyToken ? 0.f : (given.logit - s.m) * a.scale - log_total;
        if (a.entropies != nullptr) a.entropies[place] = log_total + s.weighted * kLn2 / (1.f + s.rest);
        if (a.stats != nullptr) a.stats[2 * int64_t(place)] = s.m, a.stats[2 * int64_t(place) + 1] = log_total;
    }
    if (lane < a.top) {
        const bool none = lane >= found;
        const uint64_t entry = none ? 0 : list[lane];
        if (a.top_tokens != nullptr) a.top_tokens[int64_t(place) * a.top + lane] = none ? kEmptyToken : class_of(entry);
        if (a.top_logprobs != nullptr)
            a.top_logprobs[int64_t(place) * a.top + lane] =
                none ? -INFINITY : (logit_of(uint32_t(entry >> 32)) - s.m) * a.scale - log_total;
    }
}

// What the parts leave in the workspace: their sums, [place][part] of four floats, then their lists, [place][part][top].
__host__ __device__ constexpr int64_t part_bytes(int top) { return 16 + 8 * int64_t(top); }
__device__ __forceinline__ uint64_t* lists_of(const LogprobArgs& a, int64_t parts) {
    return reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(a.workspace) + 16 * parts);
}

// VECTORS vectors of four classes a lane; a wave an item: part `item % parts` of place `item / parts`, the chunks from
// part * chunks_per_part on.
template <int VECTORS, bool TOP>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(4))) void logprobs_kernel(
    LogprobArgs a, uint32_t items, int parts, int chunks_per_part) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? kWaves : 1][TOP ? kListed : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint64_t* list = lists[TOP ? wave : 0];
    for (uint32_t item = blockIdx.x * kWaves + wave; item < items; item += gridDim.x * kWaves) {
        const uint32_t place = parts == 1 ? item : item / uint32_t(parts);
        const int part = int(item - place * uint32_t(parts));
        const Place at = place_of(a, place);
        const float* x = a.logits + at.logits;
        const Given given = parts == 1 ? given_of(a, at) : Given{};
        const int64_t begin = int64_t(part) * chunks_per_part * (256 * VECTORS);
        const int64_t end = min(begin + int64_t(chunks_per_part) * (256 * VECTORS), a.classes);
        const float factor = factor_of(a.scale);
        Sums total = {-INFINITY, 0.f, 0.f};
        int found = 0;
        for (int64_t chunk = begin; chunk < end; chunk += 256 * VECTORS) {
            float v[4 * VECTORS];
            const bool whole = chunk + 256 * VECTORS <= end;
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                const int64_t c = chunk + 4 * (lane + 64 * i);
                if (whole || c + 4 <= end) {
                    const f32x4 loaded = *reinterpret_cast<const f32x4_unaligned*>(x + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[4 * i + j] = loaded[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[4 * i + j] = c + j < end ? x[c + j] : -INFINITY;
                }
            }
            Sums s = {-INFINITY, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4 * VECTORS; ++i) s.m = fmaxf(s.m, v[i]);
            const float largest = s.m;
            s.m = wave_max(s.m);
            // A NaN is no maximum, but its term makes `rest` NaN. Equal ones to the maximum count 1 each, without one of them.
            int others = 0;  // over the wave
#pragma unroll
            for (int i = 0; i < 4 * VECTORS; ++i) {
                const float z = (v[i] - s.m) * factor, e = __builtin_amdgcn_exp2f(z);
                const bool other = !(v[i] == s.m);
                s.rest += other ? e : 0.f;
                others += __popcll(__ballot(other));
                s.weighted = fmaf(-e, fmaxf(z, -FLT_MAX), s.weighted);  // 0 of z = -inf, and of a NaN what `rest` makes up for
            }
            s.rest = wave_sum(s.rest);
            if (s.m != -INFINITY) s.rest += float(256 * VECTORS - 1 - others);
            s.weighted = wave_sum(s.weighted);
            total = merged(total, s, factor);
            if constexpr (TOP)
                found = select_top(v, x, uint32_t(chunk), uint32_t(end), largest, __any(s.rest != s.rest), a.top, list, found);
        }
        if (parts == 1) {
            finish(a, place, given, total, list, found);
        } else {
            if (lane == 0) reinterpret_cast<f32x4*>(a.workspace)[item] = f32x4{total.m, total.rest, total.weighted, 0.f};
            if (TOP && lane < a.top) lists_of(a, items)[int64_t(item) * a.top + lane] = lane < found ? list[lane] : 0;
        }
    }
}

// The likeliest of `parts` sorted lists of `top` entries, 0 behind their last: to list[0 .. top), sorted; returns how many
// there are. A lane a part, 64 at a time: the `top`-th largest of their firsts (or where these are few, of their first
// eight) is a bound that few others reach.
__device__ __forceinline__ int merge_lists(const uint64_t* entries, int parts, int top, uint64_t* list) {
    const int lane = threadIdx.x & 63;
    int found = 0;
    for (int group = 0; group < parts; group += 64) {
        const uint64_t* own = entries + int64_t(group + lane) * top;
        const int size = group + lane < parts ? top : 0;
        constexpr int kAhead = 8;
        uint64_t ahead[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) ahead[j] = j < size ? own[j] : 0;
        const bool few = min(parts - group, 64) < 2 * top;
        const uint64_t above = found == top ? list[top - 1] + 1 : 1;
        uint64_t bound;
        int count;
        const auto gather = [&](uint64_t entry) {
            const uint64_t mask = __ballot(entry >= bound);
            const int at = count + __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
            if (entry >= bound && at < kListed) list[at] = entry;
            count += __popcll(mask);
            return mask != 0;
        };
        for (int low = 16; low >= 0; low -= 16) {  // to 16 bits, or if that leaves too many, to all
            uint32_t reached = 0;
#pragma nounroll
            for (int b = 31; b >= low; --b) {
                const uint32_t tried = reached | 1u << b;
                int reaching = __popcll(__ballot(uint32_t(ahead[0] >> 32) >= tried));
                if (few) {
#pragma unroll
                    for (int j = 1; j < kAhead; ++j) reaching += __popcll(__ballot(uint32_t(ahead[j] >> 32) >= tried));
                }
                if (reaching >= top) reached = tried;
            }
            bound = max(above, uint64_t(reached) << 32);
            count = found;
            bool more = true;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) more = gather(ahead[j]);
            for (int j = kAhead; j < top && more && count <= kListed; ++j) more = gather(j < size ? own[j] : 0);
            if (count <= kListed) break;
        }
        wave_lds_order();
        if (count <= kListed) {
            found = rank_entries(list, count, top, [&](int at) { return list[at]; });
            continue;
        }
        // Many equal ones: one by one, the largest of the held ones and of the parts' next.
        uint64_t held = lane < found ? list[lane] : 0, next = ahead[0], mine = 0;
        wave_lds_order();
        int taken = 0, j = 0;
        for (; taken < top; ++taken) {
            const uint64_t best = wave_largest(max(held, next));
            if (best == 0) break;
            if (lane == taken) mine = best;
            if (held == best) held = 0;
            if (next == best) next = ++j < size ? own[j] : 0;
        }
        if (lane < taken) list[lane] = mine;
        wave_lds_order();
        found = taken;
    }
    return found;
}

// A wave a place: its parts merged, in order.
template <bool TOP>
__global__ __launch_bounds__(64 * kWaves) void merge_kernel(LogprobArgs a, uint32_t places, int parts) {
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? kWaves : 1][TOP ? kListed : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t place = blockIdx.x * kWaves + wave; place < places; place += gridDim.x * kWaves) {
        const f32x4* in = reinterpret_cast<const f32x4*>(a.workspace) + int64_t(place) * parts;
        const Given given = given_of(a, place_of(a, place));
        const float factor = factor_of(a.scale);
        Sums total = {-INFINITY, 0.f, 0.f};
        for (int p = lane; p < parts; p += 64) {
            const f32x4 s = in[p];
            total = merged(total, Sums{s[0], s[1], s[2]}, factor);
        }
        int found = 0;
        if constexpr (TOP)
            found = merge_lists(lists_of(a, int64_t(places) * parts) + int64_t(place) * parts * a.top, parts, a.top, lists[wave]);
#pragma unroll
        for (int step = 1; step < 64; step <<= 1)
            total = merged(total, Sums{__shfl_xor(total.m, step), __shfl_xor(total.rest, step), __shfl_xor(total.weighted, step)},
                           factor);
        total = Sums{__shfl(total.m, 0), __shfl(total.rest, 0), __shfl(total.weighted, 0)};
        finish(a, place, given, total, lists[TOP ? wave : 0], found);
    }
}

// VECTORS vectors of four classes a lane, a wave an item: chunk `item % chunks` of place `item / chunks`.
template <int VECTORS>
__global__ __launch_bounds__(64 * kWaves) void logprobs_backward_kernel(LogprobBackwardArgs a, uint32_t items,
                                                                        uint32_t chunks) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t item = blockIdx.x * kWaves + wave; item < items; item += gridDim.x * kWaves) {
        const uint32_t place = chunks == 1 ? item : item / chunks;
        const int64_t chunk = int64_t(item - place * chunks) * (256 * VECTORS);
        const Place at = place_of(a, place);
        const int64_t first = at.logits;
        const float *x = a.logits + first, m = a.stats[2 * int64_t(place)], log_total = a.stats[2 * int64_t(place) + 1];
        float* grad = a.grad + first;
        float d_logprob = 0.f, d_entropy = 0.f, entropy = 0.f;
        uint32_t token = kEmptyToken;
        if (a.d_logprobs != nullptr) {
            token = a.tokens[at.token];
            if (token != kEmptyToken) d_logprob = a.d_logprobs[place];
        }
        if (a.d_entropies != nullptr) d_entropy = a.d_entropies[place], entropy = a.entropies[place];
        auto grad_of = [&](float logit, int64_t c) {
            const float log_p = (logit - m) * a.scale - log_total, p = __builtin_amdgcn_exp2f(log_p * kLog2e);
            const float one = uint64_t(c) == token ? d_logprob : 0.f;
            const float more = p > 0.f ? d_entropy * (log_p + entropy) : 0.f;
            return (one - p * (d_logprob + more)) * a.scale;
        };
        f32x4 v[VECTORS];
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) {
            const int64_t c = chunk + 4 * (lane + 64 * i);
            if (c + 4 <= a.classes) v[i] = *reinterpret_cast<const f32x4_unaligned*>(x + c);
        }
        // No term: zeros, also in a head whose p is NaN. (Ahead of the logits' loads the branch had them wait for the token's:
        // 333 x 50001 23.0 us against 21.4.)
        if (token == kEmptyToken && d_entropy == 0.f) {
            const int64_t end = min(chunk + 256 * VECTORS, a.classes);
            for (int64_t c = chunk + lane; c < end; c += 64) grad[c] = 0.f;
            continue;
        }
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) {
            const int64_t c = chunk + 4 * (lane + 64 * i);
            if (c + 4 <= a.classes) {
                f32x4 g;
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] = grad_of(v[i][j], c + j);
                *reinterpret_cast<f32x4_unaligned*>(grad + c) = g;
            } else {
                for (int64_t k = c; k < a.classes; ++k) grad[k] = grad_of(x[k], k);
            }
        }
    }
}

// Workgroups for that many waves' items, within the 2^32 threads of a launch; the kernels' waves loop over the rest.
// Items are counted in 32 bits, and so is the loop's step past them: places are less than 2^31, with parts only where they
// are few, and the backward's chunks of 1024 of the less than 2^40 logits are less than 2^30 besides one a place, of which
// there are less than 2^30 where a head has more than one.
unsigned groups_of(int64_t items) { return unsigned(std::min<int64_t>((items + kWaves - 1) / kWaves, 1 << 22)); }

template <int VECTORS>
void launch_forward(const LogprobArgs& a, int64_t items, int parts, int chunks_per_part, hipStream_t stream) {
    const dim3 grid(groups_of(items)), block(64 * kWaves);
    if (a.top > 0)
        hipLaunchKernelGGL((logprobs_kernel<VECTORS, true>), grid, block, 0, stream, a, uint32_t(items), parts, chunks_per_part);
    else
        hipLaunchKernelGGL((logprobs_kernel<VECTORS, false>), grid, block, 0, stream, a, uint32_t(items), parts, chunks_per_part);
}

}  // namespace

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
    const int64_t places = a.rows * a.heads;
    if (a.classes <= kChunk) {
        if (a.classes <= 256)
            launch_forward<1>(a, places, 1, 1, stream);
        else if (a.classes <= 512)
            launch_forward<2>(a, places, 1, 1, stream);
        else if (a.classes <= 1024)
            launch_forward<4>(a, places, 1, 1, stream);
        else
            launch_forward<8>(a, places, 1, 1, stream);
        return hipGetLastError();
    }
    // Parts: enough waves to fill the GPU (32 a CU), as many as the merge takes and the workspace holds.
    const int64_t chunks = (a.classes + kChunk - 1) / kChunk;
    int64_t parts = std::min(chunks, (32 * int64_t(a.cu_count) + places - 1) / places);
    parts = std::min<int64_t>(parts, a.top > 0 ? kChunk / a.top : kChunk);
    parts = std::min<int64_t>(parts, int64_t(a.workspace_bytes) / (places * part_bytes(a.top)));
    parts = std::max<int64_t>(parts, 1);
    const int64_t chunks_per_part = (chunks + parts - 1) / parts;
    parts = (chunks + chunks_per_part - 1) / chunks_per_part;
    launch_forward<8>(a, places * parts, int(parts), int(chunks_per_part), stream);
    if (parts > 1) {
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
        const dim3 grid(groups_of(places)), block(64 * kWaves);
        if (a.top > 0)
            hipLaunchKernelGGL(merge_kernel<true>, grid, block, 0, stream, a, uint32_t(places), int(parts));
        else
            hipLaunchKernelGGL(merge_kernel<false>, grid, block, 0, stream, a, uint32_t(places), int(parts));
    }
    return hipGetLastError();
}

hipError_t launch_token_logprobs_backward(const LogprobBackwardArgs& a, hipStream_t stream) {
    const int64_t places = a.rows * a.heads, chunks = (a.classes + 1023) / 1024;
    const dim3 block(64 * kWaves);
    if (a.classes <= 512)
        hipLaunchKernelGGL(logprobs_backward_kernel<2>, dim3(groups_of(places)), block, 0, stream, a, uint32_t(places), 1u);
    else
        hipLaunchKernelGGL(logprobs_backward_kernel<4>, dim3(groups_of(places * chunks)), block, 0, stream, a,
                           uint32_t(places * chunks), uint32_t(chunks));
    return hipGetLastError();
}

}  // namespace sn
