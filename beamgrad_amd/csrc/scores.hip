// SPDX-License-Identifier: MIT
//
// Log-probabilities of given tokens, entropies, the most likely tokens, and
// the logits' gradient (include/beamgrad_score.h).
//
// Mathematics. One pass over a row: each thread keeps the maximum m of its
// values, s = sum e^(x - m) and, for the entropy, t = sum (x - m) e^(x - m), all
// brought to a new maximum once for every 64 bytes that it reads; the threads' are
// joined at the end. log p = (x - m) - log s in this order (m and log s stay
// apart: their sum would lose the low bits of a likely token's log p), H = log s -
// t / s.
//
// The alternatives come out of the same pass: every thread's m is the maximum of
// its share of the row, so the least of the `top` largest of the threads' maxima (as
// many from each wavefront) is reached by at least `top` values, and what reaches it
// lies with the threads whose own maximum does: little more than `top` threads, whose shares (a few hundred values of a large
// vocabulary) are read again, from the cache. What they hold beside the alternatives
// is little where the large values lie anywhere (20 of 151936 at random: one or two). It is much
// where they lie together, so that some wavefront has none of them: logits that fall or rise
// with the token, a mask that leaves one stretch; where one wavefront has a short row and
// all its threads are wanted; and where values are equal in great number. Where more than kKept reach it,
// the threshold is raised: a pass over the row counts what reaches it in 1024 equal steps of the values'
// order, the step of the `top`-th largest is counted in its turn until few enough reach its low
// end (one pass, seldom two, at most four) or it is one value, whose first ones are taken. Where fewer than `top`
// reach the first threshold, all that are above -inf have, and the first ones at -inf follow.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "beamgrad_score.h"
#include "engine.hpp"
#include "paged.hpp"
#include "regions.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kThreads = 256;  // of a row's workgroup; short rows: one wavefront
constexpr int kManyThreads = 512;  // where rows are few
constexpr int kAtOnce = 4;     // 16-byte reads of a thread in flight
constexpr int kMaxTop = 64;
constexpr int kKept = 512;     // values beside the alternatives that a workgroup ranks
constexpr int kCounts = 1024;  // equal steps of values that are counted at once: 10 bits of
constexpr int kPasses = 4;     // 32, at most
constexpr int kMaxParts = 64;  // of a row
constexpr int64_t kCacheBytes = int64_t{200} << 20;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kFar = -1000.0f;  // e^kFar is 0 in 32 bits

struct Rows {
    const char* logits;
    int64_t outer, inner;  // strides in bytes
    Divider width;         // rows of an outer one
    int32_t V, top;
    const void* tokens;
    bool i64;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    int64_t* top_tokens;
    float4* stats;  // m, log s, H, unused

    __device__ const char* row(uint32_t r) const {
        const uint32_t o = width.quotient(r);
        return logits + o * outer + static_cast<int64_t>(r - o * width.d) * inner;
    }
    __device__ int token(uint32_t r) const {  // -1: none
        const int64_t t = i64 ? static_cast<const int64_t*>(tokens)[r] : static_cast<const int32_t*>(tokens)[r];
        return t >= 0 && t < V ? static_cast<int>(t) : -1;
    }
};

// A part's sums, in the workspace where rows are split.
struct Sums {
    float m, s, t, none;
};

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

template <class X>
__device__ __forceinline__ X uniform(X x) { return static_cast<X>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); }

// Values in the order of unsigned numbers, the two zeros as one (NaN does not come here).
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// A value and its place as one number: the larger value, of equal ones the
// lower place, is larger. 0 is below all of them.
__device__ __forceinline__ uint64_t key_of(float x, int place) {
    return static_cast<uint64_t>(order_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(place));
}
__device__ __forceinline__ int place_of(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }
__device__ __forceinline__ float value_of(uint64_t key) { return of_order(static_cast<uint32_t>(key >> 32)); }

template <class T>
constexpr int kEach = 16 / sizeof(T);

// 16 bytes of a row, or of its gradient. STREAM: past the caches, where the call's rows
// would not stay in them.
template <bool STREAM>
__device__ __forceinline__ u32x4 read16(const char* from) {
    const u32x4_any* const at = reinterpret_cast<const u32x4_any*>(from);
    return STREAM ? __builtin_nontemporal_load(at) : *at;
}
template <bool STREAM>
__device__ __forceinline__ void write16(char* to, u32x4 x) {
    u32x4_any* const at = reinterpret_cast<u32x4_any*>(to);
    if (STREAM)
        __builtin_nontemporal_store(x, at);
    else
        *at = x;
}

// The 16 bytes at place v of a row's end `V`: what lies past it is -inf.
template <class T>
__device__ __forceinline__ void values_at(const char* row, int v, int V, float* x) {
    const u32x4 raw = load16(row + static_cast<int64_t>(v) * sizeof(T), static_cast<int64_t>(V - v) * sizeof(T));
    T e[kEach<T>];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < kEach<T>; ++i) x[i] = v + i < V ? static_cast<float>(e[i]) : -__builtin_inff();
}

template <class T>
__device__ __forceinline__ float value_at(const char* row, int v) {
    return static_cast<float>(reinterpret_cast<const T*>(row)[v]);
}

template <bool ENTROPY>
__device__ __forceinline__ void take(Sums& a, const float* x, int n) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < n; ++i) m = fmaxf(m, x[i]);
    const float d0 = a.m - m, w = exp_of(d0);
    if (ENTROPY) a.t = w * __builtin_fmaf(a.s, fmaxf(d0, kFar), a.t);
    a.s *= w;
    a.m = m;
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const float d = x[i] - m, e = exp_of(d);
        a.s += e;
        if (ENTROPY) a.t = __builtin_fmaf(e, fmaxf(d, kFar), a.t);
    }
}

// A thread's share of [from, to) of a row: 16 bytes of every THREADS * 16.
template <class T, bool ENTROPY, int THREADS, bool STREAM>
__device__ __forceinline__ Sums sums_of(const char* row, int from, int to) {
    constexpr int E = kEach<T>;
    Sums a{-FLT_MAX, 0.0f, 0.0f, 0.0f};
    int64_t v = from + static_cast<int>(threadIdx.x) * E;
    constexpr int64_t step = THREADS * E;
    float x[kAtOnce * E];
    for (; v + (kAtOnce - 1) * step + E <= to; v += kAtOnce * step) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const u32x4 raw = read16<STREAM>(row + (v + i * step) * sizeof(T));
            T e[E];
            __builtin_memcpy(e, &raw, 16);
#pragma unroll
            for (int j = 0; j < E; ++j) x[i * E + j] = static_cast<float>(e[j]);
        }
        take<ENTROPY>(a, x, kAtOnce * E);
    }
    if (v < to) {  // the last round
        u32x4 raw[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (v + i * step + E <= to) raw[i] = read16<STREAM>(row + (v + i * step) * sizeof(T));
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t at = v + i * step;
            T e[E];
            __builtin_memcpy(e, &raw[i], 16);
            if (at < to && at + E > to) {
                values_at<T>(row, static_cast<int>(at), to, x + i * E);
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) x[i * E + j] = at < to ? static_cast<float>(e[j]) : -__builtin_inff();
            }
        }
        take<ENTROPY>(a, x, kAtOnce * E);
    }
    return a;
}

// Over a wavefront, of all lanes at once: lane i takes lane i - 1's, - 2's, - 4's and -
// 8's within its 16, then the last of each 16's; lane 63 has all.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float x, float none) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <class Op>
__device__ __forceinline__ float over_wave(float x, float none, Op op) {
    x = op(x, moved<0x111, 0xf>(x, none));
    x = op(x, moved<0x112, 0xf>(x, none));
    x = op(x, moved<0x114, 0xf>(x, none));
    x = op(x, moved<0x118, 0xf>(x, none));
    x = op(x, moved<0x142, 0xa>(x, none));
    x = op(x, moved<0x143, 0xc>(x, none));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float wave_max(float x) {
    return over_wave(x, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return over_wave(x, 0.0f, [](float a, float b) { return a + b; });
}

// To a maximum that is not lower.
__device__ __forceinline__ void raise(Sums& a, float m) {
    const float d = a.m - m, w = exp_of(d);
    a.t = w * __builtin_fmaf(a.s, fmaxf(d, kFar), a.t);
    a.s *= w;
    a.m = m;
}
__device__ __forceinline__ Sums joined_wave(Sums a) {
    raise(a, wave_max(a.m));
    return {a.m, wave_sum(a.s), wave_sum(a.t), 0.0f};
}

constexpr int kDumped = 64;  // threads whose values fit LDS

template <int THREADS, int VALUES = 1>
struct Shared {
    Sums waves[THREADS / 64];
    int flagged[THREADS], flags, kept, found[THREADS / 64];
    float floor[THREADS / 64];   // what reaches the least of them may be an alternative
    union {
        uint64_t keys[kKept + 8];
        uint32_t counts[kCounts];
    };
    uint32_t low, high;  // of what is counted
    int above;           // values over `high`
    float dump[VALUES > 1 ? kDumped * (VALUES + 1) : 1];
};

template <int THREADS, int VALUES>
__device__ __forceinline__ Sums joined_block(Sums a, Shared<THREADS, VALUES>& lds) {
    constexpr int WAVES = THREADS / 64;
    a = joined_wave(a);
    if (WAVES == 1) return a;
    if ((threadIdx.x & 63) == 0) lds.waves[threadIdx.x >> 6] = a;
    __syncthreads();
    Sums of[WAVES];
    float m = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        of[w] = lds.waves[w];
        m = fmaxf(m, of[w].m);
    }
    a = {m, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        raise(of[w], m);
        a.s += of[w].s;
        a.t += of[w].t;
    }
    return a;
}

// How many of n keys are larger; 8 at once (and MORE such reads, where registers are free), zeros behind them.
template <int MORE>
__device__ __forceinline__ int larger_of(const uint64_t* keys, int n, uint64_t key) {
    int above = 0;
#pragma unroll MORE
    for (int j = 0; j < n; j += 8) {
        uint64_t other[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) other[k] = keys[j + k];
#pragma unroll
        for (int k = 0; k < 8; ++k) above += other[k] > key;
    }
    return above;
}

// The `top` largest keys of [from, to), given the thread's maximum and that of all, in order to
// each(rank, key). `values`: what the thread read of it, where that is all of its share:
// those of few threads go through LDS, for all threads to look through.
// Fewer than `top` values: key 0 for the rest.
template <class T, int THREADS, int VALUES, class Each>
__device__ __forceinline__ void alternatives(const char* row, int from, int to, int top, float mine, float most, const float (&values)[VALUES],
                                             Shared<THREADS, VALUES>& lds, Each each) {
    constexpr int E = kEach<T>, WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) lds.flags = lds.kept = 0;
    // of each wavefront's maxima as many as make `top` together: the lowest of these. (Of
    // wavefronts that have no full round, none: theirs may be no values. Without any that has one,
    // all values are few enough.)
    const int full = min(WAVES, (to - from) / (64 * E)), wanted = full > 0 ? (top + full - 1) / full : 1;
    if (wanted <= 16) {
        float left = mine, largest = wave_max(mine);
        for (int n = __popcll(__ballot(left == largest)); n < wanted; n += __popcll(__ballot(left == largest))) {
            left = left == largest ? -__builtin_inff() : left;
            largest = wave_max(left);
        }
        if (lane == 0) lds.floor[tid >> 6] = largest;
    } else {
        int rank = 0;
#pragma unroll
        for (int j = 0; j < 64; ++j) {
            const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), j));
            rank += other > mine || (other == mine && j < lane);
        }
        if (rank == wanted - 1) lds.floor[tid >> 6] = mine;
    }
    __syncthreads();
    float floor = full > 0 ? lds.floor[0] : -FLT_MAX;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) floor = w < full ? fminf(floor, lds.floor[w]) : floor;
    const auto keep = [&](float x, int place) {
        if (place >= to || !(x >= floor)) return;
        const int at = atomicAdd(&lds.kept, 1);
        if (at < kKept) lds.keys[at] = key_of(x, place);
    };
    if (mine >= floor) {
        const int slot = atomicAdd(&lds.flags, 1);
        lds.flagged[slot] = tid;
        if constexpr (VALUES > 1)
            if (slot < kDumped)
#pragma unroll
                for (int i = 0; i < VALUES; ++i) lds.dump[slot * (VALUES + 1) + i] = values[i];
    }
    __syncthreads();
    const int flags = lds.flags;
    if (VALUES > 1 && flags <= kDumped) {
        for (int i = tid; i < flags * VALUES; i += THREADS) {
            const int of = i / VALUES, v = i - of * VALUES;
            keep(lds.dump[of * (VALUES + 1) + v], from + ((v / E) * THREADS + lds.flagged[of]) * E + v % E);
        }
    } else {
        const int shares = (to - from + THREADS * E - 1) / (THREADS * E), items = flags * shares;
        for (int i = tid; i < items; i += THREADS) {
            const int v = from + ((i % shares) * THREADS + lds.flagged[i / shares]) * E;
            if (v >= to) continue;
            float x[E];
            values_at<T>(row, v, to, x);
#pragma unroll
            for (int j = 0; j < E; ++j) keep(x[j], v + j);
        }
    }
    __syncthreads();
    const int all = min(top, to - from);
    int n = uniform(lds.kept);
    bool tied = false;  // those at the floor are not kept, and are more than are wanted
    constexpr int kFew = std::min(kKept, 4 * THREADS);  // that are ranked sooner than their number is brought down
    if (n > kFew) {
        // All values from the floor to the maximum are counted in equal steps, then those of
        // the step that the `top`-th largest lies in, until few reach its low end or it is one value.
        constexpr int kUnused = sizeof(T) == 4 ? 0 : std::is_same<T, _Float16>::value ? 13 : 16;  // low bits that T does not have
        const auto all_values = [&](auto use) {
            constexpr int kStep = THREADS * E;
            int v0 = from;
#pragma unroll 1
            for (; to - v0 >= kAtOnce * kStep; v0 += kAtOnce * kStep) {
                u32x4 raw[kAtOnce];
                const char* const at = row + static_cast<int64_t>(v0 + tid * E) * sizeof(T);
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) raw[i] = *reinterpret_cast<const u32x4_any*>(at + i * kStep * sizeof(T));
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    T e[E];
                    __builtin_memcpy(e, &raw[i], 16);
#pragma unroll
                    for (int j = 0; j < E; ++j) use(static_cast<float>(e[j]), v0 + i * kStep + tid * E + j);
                }
            }
#pragma unroll 1
            for (; v0 < to; v0 += kStep) {
                const int v = v0 + tid * E;
                float x[E];
                values_at<T>(row, min(v, to), to, x);
#pragma unroll
                for (int j = 0; j < E; ++j) use(x[j], min(v + j, to));
            }
        };
        uint32_t low = uniform(order_of(floor) >> kUnused), high = uniform(order_of(most) >> kUnused);
        int above = 0;
        for (int pass = 0;; ++pass) {
            tied = low == high || pass == kPasses;  // (the last pass leaves one value, unless the row is being written)
            if (tied) break;
            const int shift = max(0, 22 - __builtin_clz(high - low));
            __syncthreads();  // what is read of LDS before is read
#pragma unroll 1
            for (int i = tid; i < kCounts; i += THREADS) lds.counts[i] = 0;
            __syncthreads();
            all_values([&](float x, int place) {
                const uint32_t o = order_of(x) >> kUnused, step = (o - low) >> shift;
                const bool counts = place < to && o >= low && o <= high;
                // the first lane's step by one addition: many values may be in one
                const uint64_t which = __ballot(counts);
                if (which == 0) return;
                const int lead = __builtin_ctzll(which);
                const bool same = counts && step == static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(step), lead));
                const int together = __popcll(__ballot(same));
                if (counts && (!same || lane == lead)) atomicAdd(&lds.counts[step], same ? static_cast<uint32_t>(together) : 1u);
            });
            __syncthreads();
            if (tid < 64) {  // steps from the highest down, some of a lane
                constexpr int kOwn = kCounts / 64;
                uint32_t sum = 0;
#pragma unroll 4
                for (int i = 0; i < kOwn; ++i) sum += lds.counts[kCounts - 1 - (tid * kOwn + i)];
                uint32_t upto = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t y = __shfl_up(upto, d);
                    if (lane >= d) upto += y;
                }
                const uint32_t left = static_cast<uint32_t>(top - above);
                uint32_t before = upto - sum;
                if (before < left && upto >= left) {
                    int step = kCounts - 1 - tid * kOwn;
#pragma unroll 1
                    for (; before + lds.counts[step] < left; --step) before += lds.counts[step];
                    lds.low = low + (static_cast<uint32_t>(step) << shift);
                    lds.high = min(high, lds.low + ((1u << shift) - 1));
                    lds.above = above + static_cast<int>(before);
                    lds.kept = lds.above + static_cast<int>(lds.counts[step]);
                }
            }
            __syncthreads();
            low = uniform(lds.low), high = uniform(lds.high), above = uniform(lds.above);
            if (uniform(lds.kept) <= kFew) break;
        }
        floor = of_order(low << kUnused | (low >> (31 - kUnused) != 0 ? 0u : (1u << kUnused) - 1));  // a value of T
        __syncthreads();
        if (tid == 0) lds.kept = 0;
        __syncthreads();
        if (!tied || above > 0)
            all_values([&](float x, int place) {
                if (!tied || order_of(x) >> kUnused > low) keep(x, place);
            });
        __syncthreads();
        n = min(uniform(lds.kept), kKept);
    }
    if (tid < 8) lds.keys[n + tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
        const uint64_t key = lds.keys[i];
        const int above = larger_of<2>(lds.keys, n, key);
        if (above < top) each(above, key);
    }
    if (n < all && !tied && tid < 64) {  // of the first `all` places at most n are not at -inf
        const float x = tid < all ? value_at<T>(row, from + tid) : 0.0f;
        const uint64_t none = __ballot(x == -__builtin_inff());
        const int at = n + __popcll(none & ((uint64_t{1} << tid) - 1));
        if (x == -__builtin_inff() && at < all) each(at, key_of(x, from + tid));
    }
    if (tied) {
        // the first ones that equal the floor, round after round
        for (int64_t v0 = from; v0 < to && n < all; v0 += THREADS * E) {
            const int v = static_cast<int>(v0) + tid * E;
            float x[E];
            values_at<T>(row, min(v, to), to, x);
            unsigned hits = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) hits |= static_cast<unsigned>(v + j < to && x[j] == floor) << j;
            if (!__syncthreads_or(hits)) continue;
            const int here = __popc(hits);
            int upto = here;
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(upto, d);
                if (lane >= d) upto += y;
            }
            if (lane == 63) lds.found[tid >> 6] = upto;
            __syncthreads();
            int at = n + upto - here;
            for (int w = 0; w < WAVES; ++w) {
                if (w < tid >> 6) at += lds.found[w];
                n += uniform(lds.found[w]);
            }
            __syncthreads();
            for (; hits != 0 && at < all; hits &= hits - 1, ++at) each(at, key_of(floor, v + __builtin_ctz(hits)));
        }
    }
    for (int k = all + tid; k < top; k += THREADS) each(k, uint64_t{0});
}

struct Normal {
    float m, log_s, entropy;
    bool empty;  // nothing in the row is possible
    __device__ float logp(float x) const { return empty ? -__builtin_inff() : (x - m) - log_s; }
};

__device__ __forceinline__ Normal normal_of(const Sums& a) {
    const bool empty = a.s == 0.0f;
    const float log_s = logf(a.s);
    return {a.m, log_s, empty ? 0.0f : log_s - a.t / a.s, empty};
}

// What one thread writes of a row, whose token's logit is x.
__device__ __forceinline__ void write_row(const Rows& p, uint32_t r, float x, const Normal& n) {
    p.logprobs[r] = n.logp(x);
    if (p.entropy) p.entropy[r] = n.entropy;
    if (p.stats) p.stats[r] = float4{n.m, n.empty ? __builtin_inff() : n.log_s, n.entropy, 0.0f};
}

__device__ __forceinline__ void write_alternative(const Rows& p, uint32_t r, int rank, uint64_t key, const Normal& n) {
    const int64_t at = static_cast<int64_t>(r) * p.top + rank;
    p.top_logprobs[at] = n.logp(value_of(key));
    p.top_tokens[at] = place_of(key);
}

// A row of no token, or (`bad`) one that holds NaN or +inf: by all threads.
template <int THREADS>
__device__ __forceinline__ void write_none(const Rows& p, uint32_t r, bool bad) {
    const float nan = __builtin_nanf("");
    if (threadIdx.x == 0) {
        p.logprobs[r] = bad ? nan : 0.0f;
        if (p.entropy) p.entropy[r] = bad ? nan : 0.0f;
        if (p.stats) p.stats[r] = float4{nan, nan, nan, 0.0f};
    }
    for (int k = threadIdx.x; k < p.top; k += THREADS) {
        p.top_logprobs[static_cast<int64_t>(r) * p.top + k] = bad ? nan : -__builtin_inff();
        p.top_tokens[static_cast<int64_t>(r) * p.top + k] = -1;
    }
}

// A workgroup for a row; a wavefront for a row of two rounds of its reads. Bound by HBM
// where the rows fill the card several times: some 3080 of 4096 of 128256 in bfloat16 (the others have
// no token) in 129 us, 6.1 TB/s. Some hundred rows are two workgroups a CU, none of which has
// a round on its way while it computes another: 490 of 50257 in float16 13.9 us, 3.5 TB/s, with 4 alternatives 17.2, with
// the entropy too 17.9 (21 under a trace, among 170 rows without a token). Few rows: latency, 4 of 32000 in float32 with 5
// alternatives 7 us.
template <class T, bool ENTROPY, int THREADS, bool STREAM>
__global__ __launch_bounds__(THREADS) void score_rows(const Rows p) {
    __shared__ Shared<THREADS> lds;
    const uint32_t r = blockIdx.x;
    const int token = p.token(r);
    if (token < 0) return write_none<THREADS>(p, r, false);
    const char* const row = p.row(r);
    const float x = value_at<T>(row, token);
    const Sums mine = sums_of<T, ENTROPY, THREADS, STREAM>(row, 0, p.V);
    const Sums all = joined_block(mine, lds);
    if (!(all.s <= FLT_MAX)) return write_none<THREADS>(p, r, true);
    const Normal n = normal_of(all);
    if (threadIdx.x == 0) write_row(p, r, x, n);
    if (p.top > 0)
        alternatives<T>(row, 0, p.V, p.top, mine.m, all.m, {0.0f}, lds, [&](int rank, uint64_t key) { write_alternative(p, r, rank, key, n); });
}

// x: a part of `part` values of row y. Sums and alternatives go to the workspace.
// Bound by latency: the read, the wavefronts' maxima, the ranking. 32 rows of 151936 in
// bfloat16 with 20 alternatives 9.0 to 9.9 us (the bytes alone 1.9; a launch that does nothing 2 to 3).
// With ONE a part is one round of the workgroup's reads, which stay in registers: they
// begin while the token is still read, and are looked through for the alternatives.
template <class T, bool ENTROPY, bool ONE>
__global__ __launch_bounds__(kThreads) void score_parts(const Rows p, const int part, Sums* sums, uint64_t* keys) {
    constexpr int E = kEach<T>, VALUES = ONE ? kAtOnce * E : 1;
    __shared__ Shared<kThreads, VALUES> lds;
    const uint32_t r = blockIdx.y;
    const char* const row = p.row(r);
    const int from = blockIdx.x * part, to = min(p.V, from + part);
    float x[VALUES];
    Sums mine{-FLT_MAX, 0.0f, 0.0f, 0.0f};
    if constexpr (ONE) {
        u32x4 raw[kAtOnce];
        const int v0 = from + static_cast<int>(threadIdx.x) * E;
        const char* const at = row + static_cast<int64_t>(v0) * sizeof(T);
        constexpr int kStep = kThreads * E;
        if (to - from == VALUES * kThreads) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) raw[i] = *reinterpret_cast<const u32x4_any*>(at + i * kStep * sizeof(T));
        } else {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                raw[i] = v0 + i * kStep < to ? load16(at + i * kStep * sizeof(T), static_cast<int64_t>(to - v0 - i * kStep) * sizeof(T)) : u32x4{0, 0, 0, 0};
        }
        if (p.token(r) < 0) return;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            T e[E];
            __builtin_memcpy(e, &raw[i], 16);
#pragma unroll
            for (int j = 0; j < E; ++j) x[i * E + j] = v0 + i * kStep + j < to ? static_cast<float>(e[j]) : -__builtin_inff();
        }
        take<ENTROPY>(mine, x, VALUES);
    } else {
        if (p.token(r) < 0) return;
        mine = sums_of<T, ENTROPY, kThreads, false>(row, from, to);
    }
    const Sums all = joined_block(mine, lds);
    const int64_t at = static_cast<int64_t>(r) * gridDim.x + blockIdx.x;
    if (threadIdx.x == 0) sums[at] = all;
    if (p.top > 0 && all.s <= FLT_MAX)
        alternatives<T>(row, from, to, p.top, mine.m, all.m, x, lds, [&](int rank, uint64_t key) { keys[at * p.top + rank] = key; });
}

// A workgroup joins the parts of a row. The parts' alternatives are in order: of the
// j-th of each part but the last, j * (parts - 1) >= top, the lowest is reached by `top` of
// them, so what lies below it is none. (The last part may be short, and its j-th low.) Where
// the largest lie in a few parts, much reaches it; then the same is asked of the j-th of the
// ceil(top / j) parts in which it is largest, for j = 1, 2, 4 .. top, and the highest answer
// counts: of no j more than 1 / j of the keys pass. 32 rows of 19 parts: 5.0 us, of two dependent reads and the ranking.
template <class T>
__global__ __launch_bounds__(kThreads) void score_join(const Rows p, const int parts, const Sums* sums, const uint64_t* keys) {
    constexpr int kFirst = 4;  // keys of a thread that are read ahead
    __shared__ uint64_t kept[kMaxParts * kMaxTop + 8];
    __shared__ uint64_t lowest, floors[kThreads / 64];
    __shared__ int found;
    const uint32_t r = blockIdx.x;
    const int token = p.token(r), tid = threadIdx.x;
    const int64_t first = static_cast<int64_t>(r) * parts;
    Sums all = (tid & 63) < parts ? sums[first + (tid & 63)] : Sums{-FLT_MAX, 0.0f, 0.0f, 0.0f};
    const uint64_t* const mine = keys + first * p.top;
    const int n = parts * p.top, whole = parts - 1, j = (p.top + whole - 1) / whole - 1;
    uint64_t ahead[kFirst];
#pragma unroll
    for (int i = 0; i < kFirst; ++i) ahead[i] = i * kThreads + tid < n ? mine[i * kThreads + tid] : 0;
    uint64_t floor = p.top > 0 && tid < whole ? mine[tid * p.top + j] : ~uint64_t{0};
    if (token < 0) return write_none<kThreads>(p, r, false);
    const float x = value_at<T>(p.row(r), token);
    if (tid == 0) found = 0;
    all = joined_wave(all);
    if (!(all.s <= FLT_MAX)) return write_none<kThreads>(p, r, true);
    const Normal normal = normal_of(all);
    if (tid == 0) write_row(p, r, x, normal);
    if (p.top == 0) return;
    if (tid < 64) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint32_t lo = __shfl_xor(static_cast<uint32_t>(floor), d), hi = __shfl_xor(static_cast<uint32_t>(floor >> 32), d);
            const uint64_t other = static_cast<uint64_t>(hi) << 32 | lo;
            floor = other < floor ? other : floor;
        }
        if (tid == 0) lowest = floor;
    }
    __syncthreads();
    floor = lowest;
    const auto take = [&](uint64_t key) {
        if (key >= floor && key != 0) kept[atomicAdd(&found, 1)] = key;
    };
    const auto take_all = [&] {
#pragma unroll
        for (int i = 0; i < kFirst; ++i) take(ahead[i]);
        for (int i = kFirst * kThreads + tid; i < n; i += kThreads) take(mine[i]);
        __syncthreads();
    };
    take_all();
    int m = uniform(found);
    if (m > kKept) {
        __syncthreads();  // every wavefront has read how many there are
        const int lane = tid & 63, wave = tid >> 6;
        for (int i = wave; 1 << i < 2 * p.top; i += kThreads / 64) {
            const int each = min(1 << i, p.top), of = (p.top + each - 1) / each;
            if (of > parts) continue;
            const uint64_t key = lane < parts ? mine[lane * p.top + each - 1] : 0;
            const auto at = [&](int q) {
                const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(key), q), hi = __builtin_amdgcn_readlane(static_cast<int>(key >> 32), q);
                return static_cast<uint64_t>(hi) << 32 | lo;
            };
            int above = 0;
            for (int q = 0; q < parts; ++q) above += at(q) > key;
            const uint64_t which = __ballot(key != 0 && above == of - 1);
            if (which != 0) floor = max(floor, at(__builtin_ctzll(which)));
        }
        if (lane == 0) floors[wave] = floor;
        if (tid == 0) found = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) floor = max(floor, floors[w]);
        take_all();
        m = uniform(found);
    }
    if (tid < 8) kept[m + tid] = 0;
    __syncthreads();
    for (int i = tid; i < m; i += kThreads) {
        const int above = larger_of<4>(kept, m, kept[i]);
        if (above < p.top) write_alternative(p, r, above, kept[i], normal);
    }
}

// ---------------------------------------------------------------------------
// The gradient
// ---------------------------------------------------------------------------

struct Grads {
    const float* logprobs;
    const float* entropy;
    const float* top;
    char* logits;  // the gradient
};

// x: `part` values of row y (parts first: grid x = rows * parts). p_v comes
// from the row's m and log s. The token and the alternatives, whose own gradients
// come in addition, are written over by a thread for each: with g their sum at v,
// g (1 - p_v) - p_v (A - g + ...) has no cancellation where p_v is near 1.
// 32 KB of a row for a workgroup, so that long rows fill the card evenly. Bound by HBM:
// 4096 rows of 128256 in bfloat16, 3080 of them read, in 336 us, 5.5 TB/s; 660 of
// 50257 in float16 with the entropy in 21.8 us, 5.3 TB/s.
template <class T, bool ENTROPY, int THREADS, bool STREAM>
__global__ __launch_bounds__(THREADS) void score_backward(const Rows p, const Grads g, const Divider parts, const int part) {
    constexpr int E = kEach<T>;
    __shared__ int places[kMaxTop + 1];
    __shared__ float given[kMaxTop + 1];
    const uint32_t r = parts.quotient(blockIdx.x);
    const int from = static_cast<int>(blockIdx.x - r * parts.d) * part, to = min(p.V, from + part), tid = threadIdx.x;
    const int token = p.token(r);
    char* const out = g.logits + static_cast<int64_t>(r) * p.V * sizeof(T);
    const float4 stats = p.stats[r];
    const float m = stats.x, log_s = stats.y, H = stats.z;
    if (token < 0 || log_s == __builtin_inff()) {
        const u32x4 zero = {0, 0, 0, 0};
        for (int64_t v = from + tid * E; v < to; v += THREADS * E) {
            if (v + E <= to)
                write16<STREAM>(out + v * sizeof(T), zero);
            else
                store16(out + v * sizeof(T), zero, (to - v) * sizeof(T));
        }
        return;
    }
    const char* const row = p.row(r);
    const int top = g.top ? p.top : 0;
    const float given_token = g.logprobs ? g.logprobs[r] : 0.0f, gH = ENTROPY ? g.entropy[r] : 0.0f;
    float sum = given_token;
    for (int k = 0; k < top; ++k) sum += g.top[static_cast<int64_t>(r) * p.top + k];
    const auto rest = [&](float d, float by) { return ENTROPY ? __builtin_fmaf(gH, fmaxf(d, kFar) + H, by) : by; };
    for (int64_t v = from + tid * E; v < to; v += THREADS * E) {
        const bool whole = v + E <= to;
        float x[E];
        if (whole) {
            const u32x4 raw = read16<STREAM>(row + v * sizeof(T));
            T e[E];
            __builtin_memcpy(e, &raw, 16);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = static_cast<float>(e[i]);
        } else {
            values_at<T>(row, static_cast<int>(v), to, x);
        }
        T y[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = (x[i] - m) - log_s;
            y[i] = static_cast<T>(-exp_of(d) * rest(d, sum));
        }
        u32x4 raw;
        __builtin_memcpy(&raw, y, 16);
        if (whole)
            write16<STREAM>(out + v * sizeof(T), raw);
        else
            store16(out + v * sizeof(T), raw, (to - v) * sizeof(T));
    }
    for (int k = tid; k <= top; k += THREADS) {
        places[k] = k == 0 ? token : static_cast<int>(p.top_tokens[static_cast<int64_t>(r) * p.top + k - 1]);
        given[k] = k == 0 ? given_token : g.top[static_cast<int64_t>(r) * p.top + k - 1];
    }
    __threadfence_block();
    __syncthreads();
    for (int k = tid; k <= top; k += THREADS) {
        const int v = places[k];
        if (v < from || v >= to || (k > 0 && v == token)) continue;
        float by = given[k];
        if (k == 0)
            for (int i = 1; i <= top; ++i) by += places[i] == v ? given[i] : 0.0f;
        const float d = (value_at<T>(row, v) - m) - log_s;
        reinterpret_cast<T*>(out)[v] = static_cast<T>(__builtin_fmaf(by, -expm1f(d), -exp_of(d) * rest(d, sum - by)));
    }
}

// ---------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------

int element_size(int data_type) { return data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2; }

bool valid_sizes(const BeamgradTokenLogprobs* a) {
    return a && (a->data_type == DBS_CUDA_DTYPE_F32 || a->data_type == DBS_CUDA_DTYPE_F16 || a->data_type == DBS_CUDA_DTYPE_BF16) &&
           a->outer > 0 && a->inner > 0 && static_cast<int64_t>(a->outer) * a->inner < int64_t{1} << 24 && a->vocab > 0 &&
           a->vocab <= 1 << 30 && a->top >= 0 && a->top <= kMaxTop && a->top <= a->vocab && a->strides[0] >= 0 && a->strides[1] >= 0;
}

Region region_of(const void* at, int64_t bytes) { return {reinterpret_cast<uintptr_t>(at), {1, 1}, {0, 0}, bytes}; }
Region logits_of(const BeamgradTokenLogprobs& a) {
    const int size = element_size(a.data_type);
    return {reinterpret_cast<uintptr_t>(a.logits), {a.outer, a.inner}, {a.strides[0] * size, a.strides[1] * size}, static_cast<int64_t>(a.vocab) * size};
}

Rows rows_of(const BeamgradTokenLogprobs& a) {
    const int size = element_size(a.data_type);
    return {static_cast<const char*>(a.logits), a.strides[0] * size, a.strides[1] * size, Divider::of(static_cast<uint32_t>(a.inner)),
            a.vocab, a.top, a.tokens, a.tokens_i64 != 0, a.logprobs, a.entropy, a.top_logprobs, a.top_tokens, reinterpret_cast<float4*>(a.stats)};
}

// A row of up to two rounds of a wavefront is one's work.
bool is_short(int vocab, int size) { return static_cast<int64_t>(vocab) * size <= 2 * 64 * 16 * kAtOnce; }

// Few long rows are split, so that the card's 256 CUs have work, in parts of 16 KB at
// least (a round of a workgroup's reads); a second launch joins them. A workgroup to itself
// is the sooner done the shorter the rows and the more there are of them. bfloat16 without
// alternatives, us, split and whole: 16 rows of 32000 6.5, 6.3; of 50257 6.6, 7.2; 64 rows
// of 50257 8.1, 7.9; of 100000 9.3, 9.9; 130 of 100000 11.9, 10.2; 1000 of 100000 49.1, 39.6.
int parts_of(const BeamgradTokenLogprobs& a) {
    constexpr int64_t kWanted = 1024, kLeast = kThreads * 16 * kAtOnce;
    const int64_t rows = static_cast<int64_t>(a.outer) * a.inner, bytes = static_cast<int64_t>(a.vocab) * element_size(a.data_type);
    if (a.vocab <= 40000 || rows * 1000 >= a.vocab) return 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(kWanted + rows - 1) / rows, (bytes + kLeast - 1) / kLeast, kMaxParts})));
}

// Threads of a row's workgroup. Where the rows do not fill the card by themselves, 512 have
// more of a row on its way: 200 rows of 64000 in bfloat16 8.9 us, 10.0 with 256; 600 rows
// 20.7, 18.8.
int threads_of_row(int64_t rows, int vocab, int size) {
    if (is_short(vocab, size)) return 64;
    return rows < 400 && static_cast<int64_t>(vocab) * size > 32 * 1024 ? kManyThreads : kThreads;
}

// Values of a part: whole rounds of a workgroup's reads.
int part_values(int vocab, int parts, int size) {
    const int64_t round = kThreads * 16 / size, each = (vocab + parts - 1) / parts;
    return static_cast<int>(std::min<int64_t>((each + round - 1) / round * round, 1 << 30));
}

// Rows that the card's 256 MB of memory-side cache do not hold are read, and their
// gradient is written, past it: what a pass would leave there is gone before the next
// one asks for it. Forward and backward of bfloat16 rows of 32000, through the caches
// and past them, us: 131 MB of logits 68, 78; 192 MB 103, 109; 262 MB 157, 143; 790 MB
// of 128256: 504, 447.
bool is_stream(int64_t rows, int vocab, int size) { return rows * vocab * size > kCacheBytes; }

// launch(type, entropy, stream, threads)
template <class Launch>
void by_type(int data_type, bool entropy, bool stream, int threads, Launch launch) {
    const auto sized = [&](auto t, auto e, auto s) {
        if (threads == 64)
            launch(t, e, s, std::integral_constant<int, 64>{});
        else if (threads == kThreads)
            launch(t, e, s, std::integral_constant<int, kThreads>{});
        else
            launch(t, e, s, std::integral_constant<int, kManyThreads>{});
    };
    const auto streamed = [&](auto t, auto e) {
        if (stream)
            sized(t, e, std::true_type{});
        else
            sized(t, e, std::false_type{});
    };
    const auto typed = [&](auto t) {
        if (entropy)
            streamed(t, std::true_type{});
        else
            streamed(t, std::false_type{});
    };
    if (data_type == DBS_CUDA_DTYPE_F32)
        typed(float{});
    else if (data_type == DBS_CUDA_DTYPE_F16)
        typed(_Float16{});
    else
        typed(__bf16{});
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_token_logprobs_workspace_size(const BeamgradTokenLogprobs* args) {
    if (!valid_sizes(args)) return -1;
    const int64_t rows = static_cast<int64_t>(args->outer) * args->inner;
    const int parts = parts_of(*args);
    return parts == 1 ? 0 : rows * parts * static_cast<int64_t>(sizeof(Sums) + args->top * sizeof(uint64_t));
}

DBS_CUDA_EXPORT int beamgrad_token_logprobs(const BeamgradTokenLogprobs* args, void* workspace, int64_t workspace_bytes,
                                            void* stream_ptr) {
    if (!valid_sizes(args) || !args->logits || !args->tokens || !args->logprobs ||
        (args->top > 0 && (!args->top_logprobs || !args->top_tokens)))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int64_t rows = static_cast<int64_t>(args->outer) * args->inner;
    const int64_t bytes = beamgrad_token_logprobs_workspace_size(args);
    if (bytes > 0 && (!workspace || workspace_bytes < bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Rows p = rows_of(*args);
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const bool entropy = args->entropy != nullptr;  // its gradient needs it too
    int parts = parts_of(*args);
    const int size = element_size(args->data_type), part = part_values(p.V, parts, size);
    by_type(args->data_type, entropy, is_stream(rows, p.V, size), threads_of_row(rows, p.V, size), [&](auto t, auto with_entropy, auto streams, auto threads) {
        using T = decltype(t);
        constexpr bool kEntropy = decltype(with_entropy)::value;
        constexpr int kOfRow = decltype(threads)::value;
        if (parts == 1) {
            score_rows<T, kEntropy, kOfRow, decltype(streams)::value><<<static_cast<unsigned>(rows), kOfRow, 0, stream>>>(p);
            return;
        }
        parts = (p.V + part - 1) / part;
        Sums* const sums = static_cast<Sums*>(workspace);
        uint64_t* const keys = reinterpret_cast<uint64_t*>(sums + rows * parts);
        const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(rows));
        if (part <= kThreads * kAtOnce * kEach<T>)
            score_parts<T, kEntropy, true><<<grid, kThreads, 0, stream>>>(p, part, sums, keys);
        else
            score_parts<T, kEntropy, false><<<grid, kThreads, 0, stream>>>(p, part, sums, keys);
        score_join<T><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(p, parts, sums, keys);
    });
    return finish_call(stream, hipGetLastError());
}

DBS_CUDA_EXPORT int beamgrad_token_logprobs_backward(const BeamgradTokenLogprobs* args, const float* grad_logprobs,
                                                     const float* grad_entropy, const float* grad_top, void* grad_logits,
                                                     void* stream_ptr) {
    if (!valid_sizes(args) || !args->logits || !args->tokens || !args->stats || !grad_logits ||
        (grad_top && (args->top == 0 || !args->top_tokens)))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Rows p = rows_of(*args);
    const int64_t rows = static_cast<int64_t>(args->outer) * args->inner;
    const int size = element_size(args->data_type);
    // 32 KB of a row for a workgroup
    const int part = part_values(p.V, static_cast<int>(std::max<int64_t>(1, static_cast<int64_t>(p.V) * size / (32 * 1024))), size);
    const int64_t parts = (p.V + part - 1) / part;
    if (rows * parts >= int64_t{1} << 24 || !apart(region_of(grad_logits, rows * p.V * size), logits_of(*args)))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Grads g{grad_logprobs, grad_entropy, grad_top, static_cast<char*>(grad_logits)};
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    by_type(args->data_type, grad_entropy != nullptr, is_stream(rows, p.V, size), is_short(p.V, size) ? 64 : kThreads,
            [&](auto t, auto with_entropy, auto streams, auto threads) {
        constexpr int kOfPart = std::min(decltype(threads)::value, kThreads);
        score_backward<decltype(t), decltype(with_entropy)::value, kOfPart, decltype(streams)::value>
            <<<static_cast<unsigned>(rows * parts), kOfPart, 0, stream>>>(p, g, Divider::of(static_cast<uint32_t>(parts)), part);
    });
    return finish_call(stream, hipGetLastError());
}

}  // extern "C"
