// SPDX-License-Identifier: MIT
//
// The pages of a cache between the steps of a search
// (include/beamgrad_state.h): forking, extending, writing, keeping.
//
// The tables are small (some kilobytes) and the tokens that move are few, so a
// call is bound by its launches and by the chain of dependent reads in them:
// what needs all sequences and the free list at once (which sequence takes which
// free page) is one workgroup's work, in LDS and two scans; the copies, which
// are bound by HBM where they are large, are spread over (sequence, pool).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "beamgrad_state.h"
#include "engine.hpp"
#include "paged.hpp"
#include "regions.hpp"
#include "rows.hpp"
#include "torch_engine.hpp"

using namespace dbs_hip;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kPoolsOfLaunch = 64;  // whose addresses one launch's arguments hold

// Pools of one geometry.
struct PoolSet {
    char* base[kPoolsOfLaunch];
    const char* news[kPoolsOfLaunch];  // write_tokens
    int64_t news_seq[kPoolsOfLaunch], news_token[kPoolsOfLaunch];
    int64_t row_bytes, page_stride, token_stride;
    int32_t n;
};

struct Table {
    const int32_t* pages;
    const int32_t* lengths;
    const int32_t* refs;
    int32_t* pages_out;
    int32_t* lengths_out;
    int32_t* refs_out;
    PageSpan span;
    int32_t S;
};

__device__ __forceinline__ int page_at(const Table& t, int s, int column) {
    const int32_t entry = t.pages[static_cast<int64_t>(s) * t.span.P + column];
    return t.span.is_page(entry) ? entry : -1;
}

// Exclusive sum over a workgroup of kPlanThreads, and the total.
__device__ int block_rank(int x, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(sum, off);
        if (lane >= off) sum += y;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    return before + sum - x;
}

// The first `want` free pages in order, to list; how many there are. With
// `clone` the whole of refs is copied to it on the way.
__device__ int free_pages(const int32_t* refs, int n_pages, int want, int32_t* list, int32_t* clone, int* lds) {
    constexpr int kEach = 8;  // pages of a thread and round: their reads are in flight together
    int found = 0;
    for (int64_t at = 0; at < n_pages && (clone || found < want); at += kPlanThreads * kEach) {
        const int64_t mine = at + threadIdx.x * kEach;
        int held[kEach], n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) held[i] = mine + i < n_pages ? refs[mine + i] : 1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            n += held[i] <= 0;
            if (clone && mine + i < n_pages) clone[mine + i] = held[i];
        }
        int total;
        int rank = found + block_rank(n, lds, total);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (held[i] <= 0) {
                if (rank < want) list[rank] = static_cast<int32_t>(mine + i);
                ++rank;
            }
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------

// Per sequence: the first of those that continue it, how many do, how many of
// these copy its last page; of a sequence of the new table, its fresh page (-1:
// it needs none, -2: it holds nothing).
struct ForkPlan {
    int32_t* kids;
    int32_t* copies;
    int32_t* fresh;
};

// Workgroup 0 plans; the others copy refs. Dependent reads: 4.6 us for 4 sequences,
// 7 for 128 over 8500 pages.
__global__ __launch_bounds__(kPlanThreads) void fork_plan(const Table t, const void* parents, const bool i64,
                                                          const ForkPlan plan, int32_t* list) {
    if (blockIdx.x > 0) {
        const int64_t step = static_cast<int64_t>(gridDim.x - 1) * kPlanThreads;
        for (int64_t i = static_cast<int64_t>(blockIdx.x - 1) * kPlanThreads + threadIdx.x; i < t.span.n_pages; i += step)
            t.refs_out[i] = t.refs[i];
        return;
    }
    __shared__ int lds[kPlanThreads / 64];
    // the first sequence that continues each one, and their counts: in LDS where
    // there is a thread for each, else in memory (plan.fresh until the fresh pages
    // are known)
    __shared__ int32_t near[3][kPlanThreads];
    const bool small = t.S <= kPlanThreads;
    int32_t* const first = small ? near[0] : plan.fresh;
    int32_t* const kids = small ? near[1] : plan.kids;
    int32_t* const copies = small ? near[2] : plan.copies;
    for (int s = threadIdx.x; s < t.S; s += kPlanThreads) {
        first[s] = t.S;
        kids[s] = 0;
        copies[s] = 0;
    }
    __syncthreads();
    for (int s = threadIdx.x; s < t.S; s += kPlanThreads) {
        const int p = parent_of(parents, i64, s, t.S);
        if (p >= 0) atomicMin(&first[p], s);
    }
    __syncthreads();
    // a rank for every sequence that copies, kept where its fresh page will be
    int copying = 0;
    for (int s0 = 0; s0 < t.S; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        bool copy = false;
        int p = -1, n = 0;
        if (s < t.S) {
            p = parent_of(parents, i64, s, t.S);
            if (p >= 0) {
                n = t.span.length(t.lengths[p]);
                const int whole = static_cast<int>(t.span.page.quotient(n));
                copy = n > whole * static_cast<int>(t.span.page.d) && page_at(t, p, whole) >= 0 &&
                       __hip_atomic_load(&first[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != s;
            }
        }
        int total;
        const int rank = copying + block_rank(copy, lds, total);
        copying += total;
        if (s < t.S) {
            t.lengths_out[s] = n;
            list[t.S + s] = copy ? rank : -1;
        }
    }
    const int found = free_pages(t.refs, t.span.n_pages, copying, list, nullptr, lds);
    for (int s = threadIdx.x; s < t.S; s += kPlanThreads) {
        const int p = parent_of(parents, i64, s, t.S), rank = list[t.S + s];
        int fresh = -1;
        bool live = p >= 0;
        if (rank >= 0) {
            if (rank < found) {
                fresh = list[rank];
                atomicAdd(&copies[p], 1);
            } else {
                live = false;  // no page left for its tokens
                t.lengths_out[s] = 0;
            }
        }
        if (live) atomicAdd(&kids[p], 1);
        plan.fresh[s] = live ? fresh : -2;
    }
    if (!small) return;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < t.S) {
        plan.kids[threadIdx.x] = kids[threadIdx.x];
        plan.copies[threadIdx.x] = copies[threadIdx.x];
    }
}

// HBM where much moves: 62 pages of up to 15 tokens of 2 KB in 64 pools in 24 us,
// 5 TB/s.
// y = 0: row x of the new table, and what becomes of the pages of the old row
// x; y > 0: the last page's tokens of sequence x in pool y - 1.
__global__ __launch_bounds__(kCopyThreads) void fork_apply(const Table t, const void* parents, const bool i64,
                                                           const ForkPlan plan, const PoolSet pools, const bool table) {
    const int s = blockIdx.x;
    const int fresh = plan.fresh[s];
    const int p = fresh == -2 ? -1 : parent_of(parents, i64, s, t.S);
    if (table && blockIdx.y == 0) {
        const int P = t.span.P;
        int32_t* const row = t.pages_out + static_cast<int64_t>(s) * P;
        const int tail = p >= 0 ? static_cast<int>(t.span.page.quotient(t.span.length(t.lengths[p]))) : 0;
        const int32_t* const from = t.pages + static_cast<int64_t>(max(p, 0)) * P;
        for (int c = threadIdx.x; c < P; c += kCopyThreads)
            row[c] = p < 0 ? -1 : c == tail && fresh >= 0 ? fresh : from[c];
        if (fresh >= 0 && threadIdx.x == 0) atomicAdd(&t.refs_out[fresh], 1);
        // the old row: each page is held by those that continue it, but a last
        // page that is not full not by those that copied it
        const int more = plan.kids[s] - 1, copied = plan.copies[s];
        const int old_tail = copied ? static_cast<int>(t.span.page.quotient(t.span.length(t.lengths[s]))) : -1;
        if (more != 0 || copied)
            for (int c = threadIdx.x; c < P; c += kCopyThreads) {
                const int page = page_at(t, s, c), by = more - (c == old_tail ? copied : 0);
                if (page >= 0 && by != 0) atomicAdd(&t.refs_out[page], by);
            }
        return;
    }
    if (fresh < 0) return;
    const int n = t.span.length(t.lengths[p]);
    const int tail = static_cast<int>(t.span.page.quotient(n));
    const int page = page_at(t, p, tail);
    const int pool = blockIdx.y - (table ? 1 : 0);
    const char* const from = pools.base[pool] + page * pools.page_stride;
    char* const to = pools.base[pool] + fresh * pools.page_stride;
    int64_t rows = n - tail * static_cast<int64_t>(t.span.page.d), bytes = pools.row_bytes;
    if (pools.token_stride == bytes) {  // one run
        bytes *= rows;
        rows = 1;
    }
    for (int64_t r = 0; r < rows; ++r)
        for (int64_t c = threadIdx.x * 16; c < bytes; c += kCopyThreads * 16)
            store16(to + r * pools.token_stride + c, load16(from + r * pools.token_stride + c, bytes - c), bytes - c);
}

// ---------------------------------------------------------------------------
// extend
// ---------------------------------------------------------------------------

// Workgroup 0 takes the pages and writes the entries that may be new; the
// others copy the rest of the table. One workgroup's reads of refs and its scans:
// 4.8 us for 4 sequences, 6.8 for 128 over 8500 pages; it looks through the whole
// pool, 0.9 us more for every 1000 pages (65536: 63 us, a million: 960).
// A rank counts what the sequences before want, of those that find too few too: after
// one of these no later sequence finds a page.
__global__ __launch_bounds__(kPlanThreads) void extend_kernel(const Table t, const int32_t* counts, int32_t* list) {
    const int P = t.span.P;
    const auto wants = [&](int s, int& held, int& n) { // fresh pages
        n = t.span.length(t.lengths[s]);
        const int64_t more = static_cast<int64_t>(n) + max(counts[s], 0);
        held = t.span.held(n);
        if (more > static_cast<int64_t>(P) * t.span.page.d) return -1;  // more than the table holds
        return t.span.held(static_cast<int>(more)) - held;
    };
    if (blockIdx.x > 0) {
        const int64_t step = static_cast<int64_t>(gridDim.x - 1) * kPlanThreads, cells = static_cast<int64_t>(t.S) * P;
        for (int64_t i = static_cast<int64_t>(blockIdx.x - 1) * kPlanThreads + threadIdx.x; i < cells; i += step) {
            const int s = static_cast<int>(i / P), c = static_cast<int>(i - static_cast<int64_t>(s) * P);
            int held, n;
            const int fresh = wants(s, held, n);
            if (c < held || c >= held + fresh) t.pages_out[i] = t.pages[i];
        }
        return;
    }
    __shared__ int lds[kPlanThreads / 64];
    int wanted = 0;
    for (int s0 = 0; s0 < t.S; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        int held, n;
        int total;
        block_rank(s < t.S ? max(wants(s, held, n), 0) : 0, lds, total);
        wanted = min(wanted + total, t.span.n_pages);
    }
    const int found = free_pages(t.refs, t.span.n_pages, wanted, list, t.refs_out, lds);
    int before = 0;
    for (int s0 = 0; s0 < t.S; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        int held = 0, n = 0, total;
        const int fresh = s < t.S ? wants(s, held, n) : 0;
        const int rank = before + block_rank(max(fresh, 0), lds, total);
        before = min(before + total, t.span.n_pages);
        if (s >= t.S) continue;
        const bool ok = fresh >= 0 && (fresh == 0 || rank + fresh <= found);
        t.lengths_out[s] = ok ? n + max(counts[s], 0) : n;
        for (int i = 0; i < fresh; ++i) {
            const int64_t cell = static_cast<int64_t>(s) * P + held + i;
            t.pages_out[cell] = ok ? list[rank + i] : t.pages[cell];
            if (ok) t.refs_out[list[rank + i]] = 1;
        }
    }
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------

// A thread has 16 bytes of a token's row (x) in a pool (y), and finds the token's
// place itself: 8.8 us for 116 tokens of 2 KB in 64 pools, latency.
__global__ __launch_bounds__(kCopyThreads) void write_kernel(const PageSpan span, const int32_t* pages,
                                                             const int32_t* lengths, const int32_t* counts,
                                                             const int64_t tokens, const Divider width,
                                                             const Divider chunks, const PoolSet pools) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
    // a row of news has chunks.d chunks; the launch has fewer than 2^31 of them
    const uint32_t row = chunks.quotient(static_cast<uint32_t>(at));
    if (row >= tokens) return;
    const uint32_t s = width.quotient(row), i = row - s * width.d;
    const int n = span.length(lengths[s]);
    const int count = min(counts ? max(counts[s], 0) : static_cast<int>(width.d), min(static_cast<int>(width.d), n));
    if (static_cast<int>(i) >= count) return;
    const int token = n - count + static_cast<int>(i);
    const uint32_t column = span.page.quotient(token);
    const int32_t page = pages[static_cast<int64_t>(s) * span.P + column];
    if (!span.is_page(page)) return;
    const int64_t c = (at - static_cast<int64_t>(row) * chunks.d) * 16;
    const char* const from = pools.news[blockIdx.y] + s * pools.news_seq[blockIdx.y] + i * pools.news_token[blockIdx.y];
    char* const to = pools.base[blockIdx.y] + page * pools.page_stride + (token - column * span.page.d) * pools.token_stride;
    store16(to + c, load16(from + c, pools.row_bytes - c), pools.row_bytes - c);
}

// ---------------------------------------------------------------------------
// keep
// ---------------------------------------------------------------------------

struct Kept {
    int start, n; // the first drafted token, and how many of them stay
};

// By all threads of a workgroup; `lds` is one int.
__device__ Kept kept_of(const Table& t, const int32_t* drafted, const int32_t* keep, const int32_t* kept, int width, int s,
                        int* lds) {
    const int length = t.span.length(t.lengths[s]);
    const int draft = min(max(drafted[s], 0), length);
    const int n = min(max(kept[s], 0), min(width, draft));
    if (threadIdx.x == 0) *lds = n;
    __syncthreads();
    const int32_t* const row = keep + static_cast<int64_t>(s) * width;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int before = i > 0 ? row[i - 1] : -1;
        if (row[i] <= before || row[i] >= draft || before < -1) atomicMin(lds, i);
    }
    __syncthreads();
    return {length - draft, *lds};
}

// The kept tokens of sequence x in `each` pools from y * each on, and as the last y
// the counts of the pages, copied. Where the tokens lie is looked up once, by a
// thread for each; then a thread moves 16 bytes of every token: the numbers
// ascend, so a token's new place is read by no later one, and eight are read
// before they are written.
__global__ __launch_bounds__(kCopyThreads) void keep_move(const Table t, const int32_t* drafted, const int32_t* keep,
                                                          const int32_t* kept, const int width, const PoolSet pools,
                                                          const int each, const Divider chunks) {
    if (blockIdx.y + 1 == gridDim.y) {
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i < t.span.n_pages;
             i += static_cast<int64_t>(gridDim.x) * kCopyThreads)
            t.refs_out[i] = t.refs[i];
        return;
    }
    constexpr int kAtOnce = 8, kPlaces = 128;
    __shared__ int first_bad;
    __shared__ int64_t from[kPlaces], to[kPlaces];  // -1: the token stays, or has no page
    const int s = blockIdx.x;
    const Kept k = kept_of(t, drafted, keep, kept, width, s, &first_bad);
    const int32_t* const row = keep + static_cast<int64_t>(s) * width;
    const auto place = [&](int token) -> int64_t {
        const int column = static_cast<int>(t.span.page.quotient(token)), page = page_at(t, s, column);
        return page < 0 ? -1 : page * pools.page_stride + (token - column * static_cast<int64_t>(t.span.page.d)) * pools.token_stride;
    };
    const int pool0 = static_cast<int>(blockIdx.y) * each, items = min(each, pools.n - pool0) * static_cast<int>(chunks.d);
    for (int i0 = 0; i0 < k.n; i0 += kPlaces) {
        const int here = min(k.n - i0, kPlaces);
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < here) {
            const int i = i0 + threadIdx.x, node = row[i];
            const int64_t source = node != i ? place(k.start + node) : -1;
            from[threadIdx.x] = source;
            to[threadIdx.x] = source >= 0 ? place(k.start + i) : -1;
        }
        __syncthreads();
        for (int item = threadIdx.x; item < items; item += kCopyThreads) {
            const int pool = static_cast<int>(chunks.quotient(item)), c = (item - pool * static_cast<int>(chunks.d)) * 16;
            char* const base = pools.base[pool0 + pool] + c;
            const int64_t left = pools.row_bytes - c;
            for (int i1 = 0; i1 < here; i1 += kAtOnce) {
                u32x4 x[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (i1 + i < here && to[i1 + i] >= 0) x[i] = load16(base + from[i1 + i], left);
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (i1 + i < here && to[i1 + i] >= 0) store16(base + to[i1 + i], x[i], left);
            }
        }
    }
}

__global__ __launch_bounds__(kCopyThreads) void keep_table(const Table t, const int32_t* drafted, const int32_t* keep,
                                                           const int32_t* kept, const int width) {
    __shared__ int first_bad;
    const int s = blockIdx.x;
    const Kept k = kept_of(t, drafted, keep, kept, width, s, &first_bad);
    const int held = t.span.held(k.start + k.n);
    if (threadIdx.x == 0) t.lengths_out[s] = k.start + k.n;
    const int64_t row = static_cast<int64_t>(s) * t.span.P;
    for (int c = threadIdx.x; c < t.span.P; c += kCopyThreads) {
        if (c < held) {
            t.pages_out[row + c] = t.pages[row + c];
            continue;
        }
        const int page = page_at(t, s, c);
        t.pages_out[row + c] = -1;
        if (page >= 0) atomicAdd(&t.refs_out[page], -1);
    }
}

// One launch, as torch's own conversion (which keeps the low words) takes.
__global__ __launch_bounds__(kCopyThreads) void narrow_kernel(const int64_t* from, int32_t* to, const int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x;
    if (i < n) to[i] = static_cast<int32_t>(min(max(from[i], static_cast<int64_t>(INT32_MIN)), static_cast<int64_t>(INT32_MAX)));
}

// ---------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------

// Tables of up to 2^30 entries: what all sequences want together is summed, and
// becomes places in a list, in 31 bits.
bool valid_span(int sequences, int table_pages, int n_pages, int page_tokens) {
    return sequences > 0 && table_pages > 0 && n_pages > 0 && page_tokens > 0 &&
           static_cast<int64_t>(sequences) * table_pages <= int64_t{1} << 30 &&
           (static_cast<int64_t>(table_pages) + 1) * page_tokens <= INT32_MAX - 65536;
}

bool valid_pools(const BeamgradPools* p) {
    if (!p || p->n < 0 || p->reserved != 0) return false;
    if (p->n > 0 && (!p->base || !p->row_bytes || !p->page_stride || !p->token_stride)) return false;
    for (int i = 0; i < p->n; ++i)
        if (!p->base[i] || p->row_bytes[i] <= 0 || p->page_stride[i] < 0 || p->token_stride[i] < 0) return false;
    return true;
}

// A pool, or a token of one, that lies where another does would be moved twice, and
// in no order; what is read meanwhile must not change.
bool lie_apart(const BeamgradPools& p, const void* const* news, const int64_t* news_strides, int sequences, int tokens) {
    const auto pool = [&](int i) {
        return Region{reinterpret_cast<uintptr_t>(p.base[i]), {p.n_pages, p.page_tokens}, {p.page_stride[i], p.token_stride[i]}, p.row_bytes[i]};
    };
    const auto rows = [&](int i) {
        return Region{reinterpret_cast<uintptr_t>(news[i]), {sequences, tokens}, {news_strides[2 * i], news_strides[2 * i + 1]}, p.row_bytes[i]};
    };
    return all_apart(p.n, pool, news ? p.n : 0, rows);
}

bool valid_table(const BeamgradTable* t) { return t && t->pages && t->lengths && t->refs; }

// The new table is written while the old one is read: none of its parts may lie in
// it, or in each other.
bool tables_apart(const BeamgradTable& from, const BeamgradTable& to, int S, int P, int n_pages) {
    const int32_t* const parts[6] = {to.pages, to.lengths, to.refs, from.pages, from.lengths, from.refs};
    const int64_t size[3] = {static_cast<int64_t>(S) * P, S, n_pages};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 6; ++j) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(parts[i]), b = reinterpret_cast<uintptr_t>(parts[j]);
            if (a < b + size[j % 3] * sizeof(int32_t) && b < a + size[i] * sizeof(int32_t)) return false;
        }
    return true;
}

Table table_of(const BeamgradTable& from, const BeamgradTable& to, int S, int P, int n_pages, int page_tokens) {
    return {from.pages, from.lengths, from.refs, to.pages, to.lengths, to.refs,
            {Divider::of(static_cast<uint32_t>(page_tokens)), n_pages, P}, S};
}

// The pools in sets of one geometry, as many as a launch's arguments hold;
// `each` launches a set. Without pools it is called once, with an empty set.
template <class Each>
hipError_t over_pools(const BeamgradPools& p, const void* const* news, const int64_t* news_strides, Each each) {
    const auto alike = [&](int i, int j) {
        return p.row_bytes[j] == p.row_bytes[i] && p.page_stride[j] == p.page_stride[i] &&
               p.token_stride[j] == p.token_stride[i];
    };
    bool first = true;
    for (int i = 0; i < p.n; ++i) {
        bool seen = false;
        for (int j = 0; j < i && !seen; ++j) seen = alike(i, j);
        PoolSet set{};
        set.row_bytes = p.row_bytes[i];
        set.page_stride = p.page_stride[i];
        set.token_stride = p.token_stride[i];
        for (int j = i; j < p.n && !seen; ++j) {
            if (alike(i, j)) {
                set.base[set.n] = static_cast<char*>(p.base[j]);
                if (news) {
                    set.news[set.n] = static_cast<const char*>(news[j]);
                    set.news_seq[set.n] = news_strides[2 * j];
                    set.news_token[set.n] = news_strides[2 * j + 1];
                }
                ++set.n;
            }
            if (set.n == kPoolsOfLaunch || (j + 1 == p.n && set.n > 0)) {
                const hipError_t e = each(set, first);
                if (e != hipSuccess) return e;
                first = false;
                set.n = 0;
            }
        }
    }
    return first ? each(PoolSet{}, true) : hipSuccess;
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_fork_pages_workspace_size(int sequences) {
    return sequences > 0 ? 5 * static_cast<int64_t>(sequences) * static_cast<int64_t>(sizeof(int32_t)) : -1;
}

DBS_CUDA_EXPORT int beamgrad_fork_pages(const BeamgradPools* pools, const BeamgradTable* from, const void* parents,
                                        int parents_i64, int sequences, int table_pages, const BeamgradTable* to,
                                        void* workspace, int64_t workspace_bytes, void* stream_ptr) {
    if (!valid_pools(pools) || !valid_table(from) || !valid_table(to) || !parents || !workspace ||
        !valid_span(sequences, table_pages, pools->n_pages, pools->page_tokens) ||
        workspace_bytes < beamgrad_fork_pages_workspace_size(sequences) ||
        !tables_apart(*from, *to, sequences, table_pages, pools->n_pages) || !lie_apart(*pools, nullptr, nullptr, 0, 0))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Table t = table_of(*from, *to, sequences, table_pages, pools->n_pages, pools->page_tokens);
    int32_t* const ws = static_cast<int32_t*>(workspace);
    const ForkPlan plan{ws, ws + sequences, ws + 2 * static_cast<int64_t>(sequences)};
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const unsigned clones = static_cast<unsigned>(std::min<int64_t>(64, (pools->n_pages + 4 * kPlanThreads - 1) / (4 * kPlanThreads)));
    fork_plan<<<1 + clones, kPlanThreads, 0, stream>>>(t, parents, parents_i64 != 0, plan,
                                                       ws + 3 * static_cast<int64_t>(sequences));
    hipError_t e = hipGetLastError();
    if (e == hipSuccess)
        e = over_pools(*pools, nullptr, nullptr, [&](const PoolSet& set, bool first) {
            fork_apply<<<dim3(static_cast<unsigned>(sequences), static_cast<unsigned>(set.n + (first ? 1 : 0))),
                         kCopyThreads, 0, stream>>>(t, parents, parents_i64 != 0, plan, set, first);
            return hipGetLastError();
        });
    return finish_call(stream, e);
}

DBS_CUDA_EXPORT int64_t beamgrad_extend_pages_workspace_size(int n_pages) {
    return n_pages > 0 ? static_cast<int64_t>(n_pages) * static_cast<int64_t>(sizeof(int32_t)) : -1;
}

DBS_CUDA_EXPORT int beamgrad_extend_pages(const BeamgradTable* from, const int32_t* counts, int sequences,
                                          int table_pages, int n_pages, int page_tokens, const BeamgradTable* to,
                                          void* workspace, int64_t workspace_bytes, void* stream_ptr) {
    if (!valid_table(from) || !valid_table(to) || !counts || !workspace ||
        !valid_span(sequences, table_pages, n_pages, page_tokens) ||
        workspace_bytes < beamgrad_extend_pages_workspace_size(n_pages) || !tables_apart(*from, *to, sequences, table_pages, n_pages))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Table t = table_of(*from, *to, sequences, table_pages, n_pages, page_tokens);
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const int64_t cells = static_cast<int64_t>(sequences) * table_pages;
    const unsigned clones = static_cast<unsigned>(std::min<int64_t>(256, (cells + 4 * kPlanThreads - 1) / (4 * kPlanThreads)));
    extend_kernel<<<1 + clones, kPlanThreads, 0, stream>>>(t, counts, static_cast<int32_t*>(workspace));
    return finish_call(stream, hipGetLastError());
}

DBS_CUDA_EXPORT int beamgrad_write_tokens(const BeamgradPools* pools, const void* const* news,
                                          const int64_t* news_strides, const int32_t* pages, const int32_t* lengths,
                                          const int32_t* counts, int sequences, int table_pages, int tokens,
                                          void* stream_ptr) {
    if (!valid_pools(pools) || !pages || !lengths || (pools->n > 0 && (!news || !news_strides)) || tokens <= 0 ||
        !valid_span(sequences, table_pages, pools->n_pages, pools->page_tokens))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int64_t rows = static_cast<int64_t>(sequences) * tokens;
    for (int i = 0; i < pools->n; ++i)
        if (!news[i] || news_strides[2 * i] < 0 || news_strides[2 * i + 1] < 0 ||
            static_cast<double>(rows) * static_cast<double>(pools->row_bytes[i] / 16 + 1) > 2.0e9)
            return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!lie_apart(*pools, news, news_strides, sequences, tokens)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const PageSpan span{Divider::of(static_cast<uint32_t>(pools->page_tokens)), pools->n_pages, table_pages};
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const hipError_t e = over_pools(*pools, news, news_strides, [&](const PoolSet& set, bool) {
        if (set.n == 0) return hipSuccess;
        const int64_t chunks = (set.row_bytes + 15) / 16;
        write_kernel<<<dim3(static_cast<unsigned>((rows * chunks + kCopyThreads - 1) / kCopyThreads), static_cast<unsigned>(set.n)),
                       kCopyThreads, 0, stream>>>(span, pages, lengths, counts, rows, Divider::of(static_cast<uint32_t>(tokens)),
                                                  Divider::of(static_cast<uint32_t>(chunks)), set);
        return hipGetLastError();
    });
    return finish_call(stream, e);
}

DBS_CUDA_EXPORT int beamgrad_keep_tokens(const BeamgradPools* pools, const BeamgradTable* from, const int32_t* drafted,
                                         const int32_t* keep, const int32_t* kept, int sequences, int table_pages,
                                         int width, const BeamgradTable* to, void* stream_ptr) {
    if (!valid_pools(pools) || !valid_table(from) || !valid_table(to) || !drafted || !kept || width < 0 ||
        (width > 0 && !keep) || !valid_span(sequences, table_pages, pools->n_pages, pools->page_tokens) ||
        !tables_apart(*from, *to, sequences, table_pages, pools->n_pages) || !lie_apart(*pools, nullptr, nullptr, 0, 0))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Table t = table_of(*from, *to, sequences, table_pages, pools->n_pages, pools->page_tokens);
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = over_pools(*pools, nullptr, nullptr, [&](const PoolSet& set, bool first) {
        // a workgroup takes several pools while that leaves many workgroups
        const int64_t chunks = std::max<int64_t>((set.row_bytes + 15) / 16, 1);
        int each = 1;
        while (each < set.n && each * chunks < 2 * kCopyThreads && static_cast<int64_t>(sequences) * set.n > 1024 * each) each *= 2;
        const int rounds = set.n > 0 ? (set.n + each - 1) / each : 0;
        (void)first;  // every launch copies the counts: to the same values
        const unsigned y = static_cast<unsigned>(rounds + 1);
        keep_move<<<dim3(static_cast<unsigned>(sequences), y), kCopyThreads, 0, stream>>>(
            t, drafted, keep, kept, width, set, each, Divider::of(static_cast<uint32_t>(chunks)));
        return hipGetLastError();
    });
    if (e == hipSuccess) {
        keep_table<<<static_cast<unsigned>(sequences), kCopyThreads, 0, stream>>>(t, drafted, keep, kept, width);
        e = hipGetLastError();
    }
    return finish_call(stream, e);
}

DBS_CUDA_EXPORT int beamgrad_narrow_indices(const int64_t* from, int32_t* to, int64_t n, void* stream_ptr) {
    if (n < 0 || n > INT32_MAX || (n > 0 && (!from || !to))) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    if (n > 0) narrow_kernel<<<static_cast<unsigned>((n + kCopyThreads - 1) / kCopyThreads), kCopyThreads, 0, stream>>>(from, to, n);
    return finish_call(stream, n > 0 ? hipGetLastError() : hipSuccess);
}

}  // extern "C"
