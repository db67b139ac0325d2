// SPDX-License-Identifier: MIT
//
// A paged cache cut to its heaviest tokens (include/beamgrad_state.h).
//
// Two launches. evict_select, a workgroup for each row of weights: the key of the
// m-th largest weight digit by digit (counts of 11, 11 and 10 bits in LDS), then,
// in the tokens' order, which of them stay: a list of their places. evict_move: a
// token's new place is never behind its old one, so a workgroup that has some bytes
// of every token moves them in the tokens' order without a buffer; what it writes in a
// round was read in that round or before. Bound by HBM, which moves each kept byte
// twice.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "beamgrad_state.h"
#include "engine.hpp"
#include "paged.hpp"
#include "pools.hpp"
#include "regions.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kCutThreads = 512;
constexpr int kCutWaves = kCutThreads / 64;
constexpr int kDigits = 2048;
constexpr int kEach = 4;     // weights of a thread and round, one after the other
constexpr int kRound = kCutThreads * kEach;
constexpr int kHeld = 4;     // rounds whose weights stay in registers
constexpr int kAtOnce = 8;   // reads of a thread in flight
constexpr int kMoveThreads = 256;
constexpr int kLeastWidth = 4;  // columns of a workgroup
constexpr int kTokens = kMoveThreads / kLeastWidth * kAtOnce;  // of a round, at most
constexpr int kPoolsOfLaunch = 64;
constexpr int kSetsOfLaunch = 64;
constexpr int kMaxHeads = 1024;
constexpr int kMaxSequences = 65535;
constexpr int64_t kMaxRow = 2 << 20;  // bytes of a token in a pool: so that a launch holds its pieces

// Weights of a launch.
struct WeightSet {
    const float* from[kSetsOfLaunch];
    float* to[kSetsOfLaunch];
    int64_t sequence[kSetsOfLaunch], head[kSetsOfLaunch];  // strides
    int32_t first;  // number of the launch's first
};

struct Evict {
    Table t;
    const int32_t* budgets;
    int32_t budget, recent, first, heads;
    int64_t places;   // of a sequence
    int64_t listed;   // of a list
    int32_t* lists;   // [sets][S][heads][listed]
    int32_t* live;    // [S]: tokens that stay, -1: the sequence stays as it is
};

struct Cut {
    int n, keep, first, recent;  // tokens, those that stay; of these the first and last ones
};

__device__ __forceinline__ Cut cut_of(const Evict& p, int s) {
    const int n = p.t.span.length(p.t.lengths[s]);
    const int b = max(0, p.budgets ? p.budgets[s] : p.budget), r = min(p.recent, b);
    return {n, b, min(p.first, b - r), r};
}

// A weight in the order of unsigned numbers; NaN is the least.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, w + 0.0f);
    if (w != w) return 0;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Sums of the threads ahead, and of all.
__device__ __forceinline__ uint32_t ahead_of(uint32_t x, uint32_t* lds, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kCutWaves; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    return before + sum - x;
}

// kEach weights from token i on; 0 from `end` on.
__device__ __forceinline__ void weights_at(const float* from, int i, int end, float* x) {
    if (i + kEach <= end) {
        const u32x4 raw = *reinterpret_cast<const u32x4_any*>(from + i);
        __builtin_memcpy(x, &raw, sizeof(raw));
        return;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) x[j] = i + j < end ? from[i + j] : 0.0f;
}

// A row of weights [c.first, end), of which `want` stay: what stays, in order, to
// each(place, token, weight). HELD: their keys fit the registers of the workgroup, and are read once.
struct Choice {
    uint32_t counts[kDigits], sums[kCutWaves];
    uint32_t held_sums[kHeld][kCutWaves];
    uint32_t digit, rest;
    bool whole;  // all that have the digit stay
};

template <bool HELD, class Each>
__device__ __forceinline__ void choose(const float* from, int first, int end, int want, const float (&w)[kHeld * kEach], Choice& lds, Each each) {
    const int tid = threadIdx.x;
    // the want-th largest key, and how many that equal it stay
    uint32_t key = 0, mask = 0, left = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bits = pass == 2 ? 1023 : 2047;
        for (int i = tid; i < kDigits; i += kCutThreads) lds.counts[i] = 0;
        __syncthreads();
        const auto count = [&](uint32_t o) {
            if ((o & mask) == key) atomicAdd(&lds.counts[o >> shift & bits], 1u);
        };
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < kHeld * kEach; ++i)
                if (first + (i / kEach) * kRound + tid * kEach + i % kEach < end) count(order_of(w[i]));
        } else {
            for (int i0 = first + tid; i0 < end; i0 += kCutThreads * kAtOnce) {
                float x[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) x[j] = i0 + j * kCutThreads < end ? from[i0 + j * kCutThreads] : 0.0f;
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j)
                    if (i0 + j * kCutThreads < end) count(order_of(x[j]));
            }
        }
        __syncthreads();
        // digits from the largest down, some of a thread
        constexpr int kOwn = kDigits / kCutThreads;
        const int top = kDigits - 1 - kOwn * tid;
        uint32_t of[kOwn], sum = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) sum += of[i] = lds.counts[top - i];
        uint32_t total;
        uint32_t above = ahead_of(sum, lds.sums, total);
        if (above < left && above + sum >= left) {
            int i = 0;
            for (; above + of[i] < left; ++i) above += of[i];
            lds.digit = top - i;
            lds.rest = left - above;
            lds.whole = of[i] == left - above;
        }
        __syncthreads();
        key |= lds.digit << shift;
        mask |= bits << shift;
        left = lds.rest;
        const bool whole = lds.whole;
        __syncthreads();
        if (whole) break;  // the digits behind do not matter
    }
    // larger ones and the first `left` equal ones, in order; both counts in one number
    const auto tally = [&](int i, const float* x) {
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const uint32_t m = order_of(x[j]) & mask;
            if (i + j < end) n += m > key ? 1u : m == key ? 1u << 16 : 0u;
        }
        return n;
    };
    const auto emit = [&](int i, const float* x, uint32_t big, uint32_t same) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (i + j >= end) continue;
            const uint32_t m = order_of(x[j]) & mask;
            if (m > key || (m == key && same < left)) each(first + static_cast<int>(big + min(same, left)), i + j, x[j]);
            big += m > key;
            same += m == key;
        }
    };
    uint32_t larger = 0, equal = 0;
    if constexpr (HELD) {
        // all rounds' sums at once
        const int lane = tid & 63, wave = tid >> 6;
        uint32_t mine[kHeld], upto[kHeld];
#pragma unroll
        for (int r = 0; r < kHeld; ++r) upto[r] = mine[r] = tally(first + r * kRound + tid * kEach, w + r * kEach);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
#pragma unroll
            for (int r = 0; r < kHeld; ++r) {
                const uint32_t y = __shfl_up(upto[r], d);
                if (lane >= d) upto[r] += y;
            }
        if (lane == 63)
#pragma unroll
            for (int r = 0; r < kHeld; ++r) lds.held_sums[r][wave] = upto[r];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            uint32_t before = upto[r] - mine[r], total = 0;
#pragma unroll
            for (int v = 0; v < kCutWaves; ++v) {
                if (v < wave) before += lds.held_sums[r][v];
                total += lds.held_sums[r][v];
            }
            emit(first + r * kRound + tid * kEach, w + r * kEach, larger + (before & 0xffff), equal + (before >> 16));
            larger += total & 0xffff;
            equal += total >> 16;
        }
    } else {
        for (int i0 = first; i0 < end; i0 += kRound) {
            const int i = i0 + tid * kEach;
            float x[kEach];
            uint32_t total;
            weights_at(from, i, end, x);
            const uint32_t before = ahead_of(tally(i, x), lds.sums, total);
            emit(i, x, larger + (before & 0xffff), equal + (before >> 16));
            larger += total & 0xffff;
            equal += total >> 16;
        }
    }
}

// x: a sequence; y: a row of weights, the last: counts of pages, copied; z: a set.
// 1024 rows of 4500 to 8000 weights, of which 4096 stay, in 38 us (25 MB read and 49 written, 32 of
// weights and 17 of lists, 1.9 TB/s; the vector unit is busy for 42 % of it, the rest waits for the digits' counts); ten rows of
// 900 in 9 us, most of it dependent reads: lengths, pages, their counts. Equal weights, which one
// counter takes, cost up to 1.7 times as much: 64 rows of 30000 in a call of 70 us 117.
__global__ __launch_bounds__(kCutThreads) void evict_select(const Evict p, const WeightSet set) {
    __shared__ Choice lds;
    const int s = blockIdx.x, tid = threadIdx.x, head = blockIdx.y;
    if (head == p.heads) {
        if (blockIdx.z == 0 && set.first == 0)
            for (int64_t i = static_cast<int64_t>(s) * kCutThreads + tid; i < p.t.span.n_pages; i += static_cast<int64_t>(gridDim.x) * kCutThreads)
                p.t.refs_out[i] = p.t.refs[i];
        return;
    }
    const int number = set.first + static_cast<int>(blockIdx.z);
    const float* const from = set.from[blockIdx.z] + s * set.sequence[blockIdx.z] + head * set.head[blockIdx.z];
    const int64_t row = static_cast<int64_t>(s) * p.heads + head;
    float* const to = set.to[blockIdx.z] + row * p.places;
    const Cut c = cut_of(p, s);
    const int end = c.n - c.recent, want = c.keep - c.recent - c.first;
    const bool held = end - c.first <= kHeld * kRound;
    bool stays = c.n <= c.keep;
    float w[kHeld * kEach];
    if (!stays) {
        // read while the pages are looked through
#pragma unroll
        for (int r = 0; r < kHeld; ++r) weights_at(from, c.first + r * kRound + tid * kEach, held ? end : 0, w + r * kEach);
        // every token has a page, and those that are written are the sequence's alone
        const int pages = p.t.span.held(c.n), low = static_cast<int>(p.t.span.page.quotient(c.first)), high = p.t.span.held(c.keep);
        bool bad = false;
        for (int column = tid; column < pages; column += kCutThreads) {
            const int32_t page = p.t.pages[static_cast<int64_t>(s) * p.t.span.P + column];
            bad |= !p.t.span.is_page(page) || (column >= low && column < high && p.t.refs[page] != 1);
        }
        stays = __syncthreads_or(bad);
    }
    if (tid == 0 && head == 0 && number == 0) p.live[s] = stays ? -1 : c.keep;
    if (stays) {
        for (int64_t i = tid; i < p.places; i += kCutThreads) to[i] = from[i];
        return;
    }
    int32_t* const list = p.lists + (static_cast<int64_t>(number) * p.t.S * p.heads + row) * p.listed;
    for (int i = tid; i < c.first; i += kCutThreads) {
        list[i] = i;
        to[i] = from[i];
    }
    for (int i = tid; i < c.recent; i += kCutThreads) {
        list[c.keep - c.recent + i] = c.n - c.recent + i;
        to[c.keep - c.recent + i] = from[c.n - c.recent + i];
    }
    for (int64_t i = c.keep + tid; i < p.places; i += kCutThreads) to[i] = 0.0f;
    if (want == 0) return;
    const auto each = [&](int place, int token, float weight) {
        list[place] = token;
        to[place] = weight;
    };
    if (held)
        choose<true>(from, c.first, end, want, w, lds, each);
    else
        choose<false>(from, c.first, end, want, w, lds, each);
}

struct MoveSet {
    char* base[kPoolsOfLaunch];
    int32_t weights[kPoolsOfLaunch];  // number of the set of weights
    int64_t part, page_stride, token_stride;  // bytes of a head
    int32_t n, width, pieces;  // 16-byte columns of a workgroup, workgroups of a head
    Divider columns;           // width
};

// x: a sequence; y: some columns of a head, the last (with `table`): the table; z: a pool.
// 32 pools of 8 sequences of 4500 to 8000 tokens, each of 8 heads of 128 in bfloat16 keeping
// 4096: 894 us, 4.3 GB, 4.8 TB/s. Every token behind the first that goes is moved: one of 4097 that goes
// costs as much where it is the oldest, and next to nothing (the whole call 130 us) where it is the newest.
__global__ __launch_bounds__(kMoveThreads) void evict_move(const Evict p, const MoveSet set, const bool table) {
    const int s = blockIdx.x, tid = threadIdx.x;
    const int keep = p.live[s];
    if (table && blockIdx.y + 1 == gridDim.y) {
        if (blockIdx.z > 0) return;
        const int n = p.t.span.length(p.t.lengths[s]), held = keep < 0 ? p.t.span.P : p.t.span.held(keep);
        if (tid == 0) p.t.lengths_out[s] = keep < 0 ? n : keep;
        for (int column = tid; column < p.t.span.P; column += kMoveThreads) {
            const int64_t at = static_cast<int64_t>(s) * p.t.span.P + column;
            const int32_t page = p.t.pages[at];
            p.t.pages_out[at] = column < held ? page : -1;
            if (column >= held && p.t.span.is_page(page)) atomicAdd(&p.t.refs_out[page], -1);
        }
        return;
    }
    if (keep <= 0) return;
    // where the tokens of three rounds lie, and go: read, written, looked up
    __shared__ int64_t from[3][kTokens], to[3][kTokens];
    const int head = blockIdx.y / set.pieces, piece = blockIdx.y - head * set.pieces;
    const int token_of = set.columns.quotient(tid), column = tid - token_of * set.width;
    const int tokens = min(kMoveThreads / set.width, kMoveThreads / kLeastWidth), round = tokens * kAtOnce;
    const int64_t byte = (static_cast<int64_t>(piece) * set.width + column) * 16, left = set.part - byte;
    const bool mine = token_of < tokens && left > 0;
    const int64_t row = (static_cast<int64_t>(set.weights[blockIdx.z]) * p.t.S + s) * p.heads + head;
    const int32_t* const list = p.lists + row * p.listed;
    char* const base = set.base[blockIdx.z] + head * set.part + byte;
    const int32_t* const pages = p.t.pages + static_cast<int64_t>(s) * p.t.span.P;
    const auto place = [&](int token) {
        const int c = static_cast<int>(p.t.span.page.quotient(token));
        return pages[c] * set.page_stride + (token - c * static_cast<int>(p.t.span.page.d)) * set.token_stride;
    };
    const auto look_up = [&](int buffer, int64_t j0) {
        for (int i = tid; i < round; i += kMoveThreads) {
            const int64_t j = j0 + i;
            const int source = j < keep ? list[j] : -1;
            const bool moves = source >= 0 && source != j;
            from[buffer][i] = moves ? place(source) : -1;
            to[buffer][i] = moves ? place(static_cast<int>(j)) : -1;
        }
    };
    u32x4 x[2][kAtOnce];
    const auto read = [&](auto which, int buffer) {
        constexpr int w = decltype(which)::value;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t at = mine ? from[buffer][i * tokens + token_of] : -1;
            if (at >= 0) x[w][i] = load16(base + at, left);
        }
    };
    const auto write = [&](auto which, int buffer) {
        constexpr int w = decltype(which)::value;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t at = mine ? to[buffer][i * tokens + token_of] : -1;
            if (at >= 0) store16(base + at, x[w][i], left);
        }
    };
    look_up(0, 0);
    look_up(1, round);
    __syncthreads();
    read(std::integral_constant<int, 0>{}, 0);
    int buffer = 0;
    const auto step = [&](int64_t j0, auto which) {
        constexpr int w = decltype(which)::value;
        const int next = buffer == 2 ? 0 : buffer + 1, last = next == 2 ? 0 : next + 1;
        // all reads of the round are done before its writes; the next round's, of later tokens,
        // lie behind what these write
        __builtin_amdgcn_s_waitcnt(0x0070);
        __syncthreads();
        if (j0 + round < keep) read(std::integral_constant<int, 1 - w>{}, next);
        write(which, buffer);
        if (j0 + 2 * round < keep) look_up(last, j0 + 2 * round);
        buffer = next;
    };
    for (int64_t j0 = 0; j0 < keep; j0 += 2 * round) {
        step(j0, std::integral_constant<int, 0>{});
        if (j0 + round < keep) step(j0 + round, std::integral_constant<int, 1>{});
    }
}

// ---------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------

bool valid(const BeamgradPools* pools, const BeamgradEviction* a, int sequences, int table_pages) {
    if (!valid_pools(pools) || !a || a->reserved != 0 || pools->n < 1 || a->n_weights < 1 || pools->n % a->n_weights != 0 || a->heads < 1 ||
        a->heads > kMaxHeads || a->recent < 0 || a->first < 0 || sequences > kMaxSequences || !valid_span(sequences, table_pages, pools->n_pages, pools->page_tokens))
        return false;
    for (int i = 0; i < pools->n; ++i)
        if (pools->row_bytes[i] % a->heads != 0 || pools->row_bytes[i] > kMaxRow) return false;
    return true;
}

int64_t places_of(const BeamgradPools& pools, int table_pages) { return static_cast<int64_t>(table_pages) * pools.page_tokens; }
int64_t listed_of(const BeamgradPools& pools, const BeamgradEviction& a, int table_pages) {
    const int64_t places = places_of(pools, table_pages);
    return a.budgets ? places : std::max<int64_t>(1, std::min<int64_t>(places, a.budget));
}

// The pools and the new weights are written while the old weights are read.
bool lie_apart(const BeamgradPools& pools, const BeamgradEviction& a, int S, int64_t places) {
    const int64_t size = sizeof(float);
    const auto written = [&](int i) {
        if (i < pools.n)
            return Region{reinterpret_cast<uintptr_t>(pools.base[i]), {pools.n_pages, pools.page_tokens}, {pools.page_stride[i], pools.token_stride[i]}, pools.row_bytes[i]};
        return Region{reinterpret_cast<uintptr_t>(a.to_weights[i - pools.n]), {S, a.heads}, {a.heads * places * size, places * size}, places * size};
    };
    const auto read = [&](int i) {
        return Region{reinterpret_cast<uintptr_t>(a.weights[i]), {S, a.heads}, {a.weight_strides[2 * i] * size, a.weight_strides[2 * i + 1] * size}, places * size};
    };
    return all_apart(pools.n + a.n_weights, written, a.n_weights, read);
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_evict_tokens_workspace_size(const BeamgradPools* pools, const BeamgradEviction* args,
                                                             int sequences, int table_pages) {
    if (!valid(pools, args, sequences, table_pages)) return -1;
    const double lists = static_cast<double>(args->n_weights) * sequences * args->heads * static_cast<double>(listed_of(*pools, *args, table_pages));
    if (lists > 1.0e12) return -1;
    return static_cast<int64_t>(sizeof(int32_t)) *
           (sequences + static_cast<int64_t>(args->n_weights) * sequences * args->heads * listed_of(*pools, *args, table_pages));
}

DBS_CUDA_EXPORT int beamgrad_evict_tokens(const BeamgradPools* pools, const BeamgradEviction* args,
                                          const BeamgradTable* from, int sequences, int table_pages,
                                          const BeamgradTable* to, void* workspace, int64_t workspace_bytes, void* stream_ptr) try {
    const int64_t bytes = beamgrad_evict_tokens_workspace_size(pools, args, sequences, table_pages);
    if (bytes < 0 || !workspace || workspace_bytes < bytes || !valid_table(from) || !valid_table(to) || !args->weights ||
        !args->weight_strides || !args->to_weights || !tables_apart(*from, *to, sequences, table_pages, pools->n_pages))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const BeamgradEviction& a = *args;
    for (int i = 0; i < a.n_weights; ++i)
        if (!a.weights[i] || !a.to_weights[i] || a.weight_strides[2 * i] < 0 || a.weight_strides[2 * i + 1] < 0 ||
            a.weight_strides[2 * i] > int64_t{1} << 40 || a.weight_strides[2 * i + 1] > int64_t{1} << 40)
            return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int64_t places = places_of(*pools, table_pages);
    if (!lie_apart(*pools, a, sequences, places)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    Evict p{};
    p.t = table_of(*from, *to, sequences, table_pages, pools->n_pages, pools->page_tokens);
    p.budgets = a.budgets;
    p.budget = a.budget, p.recent = a.recent, p.first = a.first, p.heads = a.heads;
    p.places = places;
    p.listed = listed_of(*pools, a, table_pages);
    p.live = static_cast<int32_t*>(workspace);
    p.lists = p.live + sequences;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = hipSuccess;
    for (int first = 0; first < a.n_weights && e == hipSuccess; first += kSetsOfLaunch) {
        const int n = std::min(kSetsOfLaunch, a.n_weights - first);
        WeightSet set{};
        set.first = first;
        for (int i = 0; i < n; ++i) {
            set.from[i] = a.weights[first + i];
            set.to[i] = a.to_weights[first + i];
            set.sequence[i] = a.weight_strides[2 * (first + i)];
            set.head[i] = a.weight_strides[2 * (first + i) + 1];
        }
        evict_select<<<dim3(static_cast<unsigned>(sequences), static_cast<unsigned>(a.heads + 1), static_cast<unsigned>(n)), kCutThreads, 0, stream>>>(p, set);
        e = hipGetLastError();
    }
    // pools of one geometry together
    std::vector<bool> done(pools->n);
    bool table = true;
    for (int i = 0; i < pools->n && e == hipSuccess; ++i) {
        if (done[i]) continue;
        MoveSet set{};
        set.part = pools->row_bytes[i] / a.heads;
        set.page_stride = pools->page_stride[i];
        set.token_stride = pools->token_stride[i];
        for (int j = i; j < pools->n && set.n < kPoolsOfLaunch; ++j) {
            if (done[j] || pools->row_bytes[j] != pools->row_bytes[i] || pools->page_stride[j] != pools->page_stride[i] ||
                pools->token_stride[j] != pools->token_stride[i])
                continue;
            done[j] = true;
            set.base[set.n] = static_cast<char*>(pools->base[j]);
            set.weights[set.n] = j / (pools->n / a.n_weights);
            ++set.n;
        }
        // 128 bytes of a token for a workgroup (a line of the cache; with 256 the call of many
        // layers took 909 us, with 128 889); where those are few, 64
        const int64_t columns = (set.part + 15) / 16;
        int64_t width = std::min<int64_t>(columns, 8);
        while (width > kLeastWidth && static_cast<int64_t>(sequences) * set.n * a.heads * ((columns + width - 1) / width) < 1024) width /= 2;
        set.width = static_cast<int32_t>(width);
        set.columns = Divider::of(static_cast<uint32_t>(width));
        set.pieces = static_cast<int32_t>((columns + width - 1) / width);
        const int64_t y = static_cast<int64_t>(a.heads) * set.pieces + (table ? 1 : 0);
        evict_move<<<dim3(static_cast<unsigned>(sequences), static_cast<unsigned>(y), static_cast<unsigned>(set.n)), kMoveThreads, 0, stream>>>(p, set, table);
        e = hipGetLastError();
        table = false;
    }
    return finish_call(stream, e);
} catch (const std::bad_alloc&) {
    return DBS_CUDA_STATUS_OUT_OF_MEMORY;
}

}  // extern "C"
