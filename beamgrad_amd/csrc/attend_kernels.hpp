// SPDX-License-Identifier: MIT
//
// Attention over a paged cache (include/beamgrad_state.h says what it
// computes): the kernel that reads the cache, and its launch.
//
// Work. An item is a tile of query rows of one cache head against a range of
// keys: rows are (token, head of the group of G that share the cache's head),
// of one sequence, or of all beams of an example against the pages they share.
// The items of a call, cut along their keys into units of KW keys, lie in one
// line; each workgroup takes an equal stretch of it, whatever the lengths
// (they are on the device, so the host cannot plan with them). An item that lies
// whole in a stretch is finished there; of another, each piece leaves its sums
// and attend_join puts them together.
//
// Mathematics. With S^T = K Q^T by 16 x 16 matrix instructions, a lane holds
// four keys of one query, so the softmax's running maximum m and total l of a
// query lie in lanes and never meet LDS, and the four keys are what the same
// lane has to give to O^T = V^T P^T: P stays in its registers. V's columns come
// from LDS by transposing reads (float32: by plain ones). m is raised only when
// a tile's maximum passes it by 2^8: sums stay below 2^8 times their number in
// float32, and most tiles need no rescaling of the sums. P is rounded to the
// operands' 16 bits for the matrix instruction (float32 inputs: not at all). In
// float16 all of a row's values are held times 2^7 (and m raised at 2^7), so that the
// largest lies between 2^7 and 2^14, a quarter of the type's range: many that are
// small beside one large, 2^-21 of it, keep all of their bits, and what is lost is 2^-32
// of it a key. The
// result is divided by the sum of the rounded values, in 32 bits, by one more
// matrix instruction with a row of ones: vector instructions are what bounds a
// tile of many rows, and a weighted mean of rounded weights has no error where the
// values are equal. The log-sum that a caller asks for is the unrounded values'.
//
// What bounds it, on one MI355X: few rows, the reads (two sequences of 90000 to
// 131000 tokens, 8 cache heads of 128, bfloat16: 946 MB in 170 us, 5.6 TB/s); many
// rows, the latency of a tile's steps with two workgroups a CU, whose registers are
// full (4 prompts' ends of 1000 tokens over 1500 to 4500, 32 heads of 64: 113 GFLOP
// in 223 us under the profiler, 209 a call with the join without it; vector
// instructions issued in 55 % of the time, matrix ones busy in 28); short caches, the
// chain of dependent reads (700 tokens: 10 us, of which launch and lengths 3).
#pragma once

#include <type_traits>

#include "attend.hpp"
#include "dbs_cuda.h"
#include "matrix.hpp"

// of a lambda: its captures and arrays stay in registers
#define BEAMGRAD_INLINE __attribute__((always_inline))

namespace dbs_hip {
namespace attend {

typedef short i16x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) char global_char;

// Sizes of a kernel.
template <int DTYPE, int DP, int SHAPE>
struct Dims {
    static constexpr bool k32 = DTYPE == DBS_CUDA_DTYPE_F32;
    static constexpr int kSize = k32 ? 4 : 2;
    static constexpr int kRows = attend_rows(SHAPE);
    // Blocks of 16 rows of a wavefront, and how the four lie: queries and sums of
    // two blocks of wide float32 heads do not fit the registers, and its matrix
    // instructions are so long that one block keeps them busy (300 asking tokens, 2000
    // cached, heads of 256: 160 us, 541 with two blocks). 16-bit heads of 256: tiles up
    // to 64 rows likewise (16 sequences of 4000 to 8000, 60 rows: 220 us, 547 with two).
    static constexpr int kRowBlocks = SHAPE == kRows16 || attend_thin(DTYPE, DP) || (DP == 256 && SHAPE <= kRows64) ? 1 : 2;
    static constexpr int kRowWaves = kRows / (16 * kRowBlocks);
    static_assert(kRowWaves == 1 || kRowWaves == 2 || kRowWaves == 4);
    static constexpr int kKeyWaves = 4 / kRowWaves;
    // Keys of a wavefront's tile: 32 fill the 16-bit matrix instruction's depth
    // for P V, 16 the float32 one's. A tile shared by four wavefronts is twice
    // as long, for half the barriers, where two tiles' scores fit the registers
    // beside the sums: trees at width 128 take 98 us with 64 keys and 88 with 32.
    static constexpr int kKeys = SHAPE == kRows128 ? (k32 ? 32 : DP <= 64 ? 64 : 32) : (k32 ? 16 : 32);
    static constexpr int kKeyBlocks = kKeys / 16;
    // The softmax's values are held times 2^kLift.
    static constexpr float kLift = DTYPE == DBS_CUDA_DTYPE_F16 ? 7.0f : 0.0f;
    static constexpr int kChunks = DP * kSize / 16;  // 16-byte chunks of a row
    static constexpr int kRowBytes = kChunks * 16;
    static constexpr int kSteps = kChunks / 4;  // matrix steps of a key block's scores
    static constexpr int kDimBlocks = DP / 16;
    static constexpr int kRegion = kKeys * kRowBytes;  // of keys or values of a wavefront's tile
    static constexpr int kLoads = kKeys * kChunks / 64 / kRowWaves;  // 16-byte loads a lane makes of a region
    // Chunk c of row r lies at c ^ (r & kSwizzle): reads of one chunk of many
    // rows meet different banks.
    static constexpr int kSwizzle = kChunks % 16 == 0 ? 15 : 7;
    // Tiles shared by wavefronts have two places: one is filled while the other
    // is used. A wavefront's own tile has one: the CU's other wavefronts use theirs
    // meanwhile.
    static constexpr int kPlaces = kRowWaves > 1 ? 2 : 1;
    static constexpr int kTile = 2 * kKeyWaves * kRegion;  // keys and values
    static constexpr int kAccs = kDimBlocks * kRowBlocks;
    static constexpr int kMerge = kKeyWaves > 1 ? kAccs * 4 * 64 * 16 : 0;
    static constexpr int kLds = kPlaces * kTile > kMerge ? kPlaces * kTile : kMerge;
    static constexpr int kTokens = kRows;  // of a tile of rows, at most
    // Beginning and ending a piece takes some 5 us: as long as four rounds of four
    // small tiles, or one or two large ones.
    static constexpr int kPieceCost = kRowWaves == 4 ? 2 : 4 * kKeyWaves;
    static constexpr int kSlot = kRows * (DP + 3);  // floats of a partial result
    // workgroups of a CU: what its 160 KB of LDS hold
    static constexpr int kOther = kTokens * (kAttendMaxTree / 8) + 2 * kAttendMaxTree + 12 * kKeyWaves * kRows + 20 * kAttendSequences + 64;
    static constexpr int kFit = 160 * 1024 / (kLds + kOther);
    // and its registers: sums, two tiles' scores and the queries of a wide head take
    // more than half of a SIMD's
    static constexpr int kResident = kFit >= 2 && (kRowWaves == 1 || kChunks <= 16) ? 2 : 1;
};

// The place of a piece's partial result. Without shared pages a workgroup
// leaves at most two: of the item it starts in the middle of, and of the item
// it does not finish. With them every piece leaves one: workgroup + item grows
// from piece to piece along the line, so no two have the same.
__device__ __forceinline__ int64_t slot_of(const AttendParams& p, int workgroup, int item, bool starts) {
    return p.shared ? workgroup + item : 2 * workgroup + (starts ? 1 : 0);
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
    const int lo = __shfl(static_cast<int>(x), lane), hi = __shfl(static_cast<int>(x >> 32), lane);
    return static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) | static_cast<uint32_t>(lo));
}

// The kernel's arguments, read again: what a phase of the kernel needs of them
// is not held in scalar registers over the others, where the loop over the keys
// has none to spare.
__device__ __forceinline__ const AttendParams& arguments() {
    auto at = (const __attribute__((address_space(4))) AttendParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const AttendParams*)at;
}

// x, of which the compiler knows nothing: what is computed from it stays where it
// is used, in the branches that are rarely taken, and takes no registers elsewhere.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Waits for loads and LDS operations, which the compiler knows of and moves no
// access of memory over.
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_all() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The maximum over the four lanes that hold a query: lanes 32 apart, then 16.
__device__ __forceinline__ float quad_max(float x) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x);
    const auto half = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t low = half[0], high = half[1];
    x = fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
    const uint32_t both = __builtin_bit_cast(uint32_t, x);
    const auto row = __builtin_amdgcn_permlane16_swap(both, both, false, false);
    const uint32_t even = row[0], odd = row[1];
    return fmaxf(__builtin_bit_cast(float, even), __builtin_bit_cast(float, odd));
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The sum over the lanes up to each one.
__device__ __forceinline__ int wave_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return x;
}

// ---------------------------------------------------------------------------
// Sequences and their units
// ---------------------------------------------------------------------------

struct Sequence {
    int length, count; // cached tokens, the last `count` of which ask
    __device__ __forceinline__ int prefix() const { return length - count; }
};

__device__ __forceinline__ Sequence sequence(const AttendParams& p, int s) {
    const int length = p.span.length(p.lengths[s]);
    int count = p.counts ? p.counts[s] : p.N;
    count = min(max(count, 0), min(p.N, length));
    return {length, count};
}

// The keys that row tile `tile` of a sequence has to read end here: all of
// them with a tree; in a chain, those up to its last token's.
template <int ROWS>
__device__ __forceinline__ int key_end(const AttendParams& p, const Sequence& s, int tile) {
    if (p.parents) return s.length;
    return s.prefix() + min(s.count, static_cast<int>(p.G.quotient((tile + 1) * ROWS - 1)) + 1);
}

__device__ __forceinline__ int row_tiles(const AttendParams& p, const Sequence& s, int rows) {
    return (s.count * static_cast<int>(p.G.d) + rows - 1) / rows;
}

// What a workgroup knows of the call's sequences.
struct Board {
    int length[kAttendSequences], count[kAttendSequences];
    int first[kAttendSequences];   // a cache head's elements of the line ahead of the sequence's (and its group's shared ones)
    int shared[kAttendSequences];  // of a group: tokens in pages that its beams share
    int leader[kAttendSequences];  // of a group: a live sequence
    int sum[4], items[4], largest[4];
};

struct Totals {
    int line, items, largest;  // of a cache head: units, items; the largest item's units
};

// The line's elements ahead of each sequence, from those of each (thread s:
// sequence s); returns a cache head's.
__device__ __forceinline__ int set_line(Board& b, int elements) {
    const int upto = wave_upto(elements), wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) b.sum[wave] = upto;
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += b.sum[w];
        total += b.sum[w];
    }
    b.first[threadIdx.x] = before + upto - elements;
    __syncthreads();
    return uniform(total);
}

// Fills the board. Sequence s is thread s's.
template <int ROWS>
__device__ __forceinline__ Totals fill_board(const AttendParams& p, Board& b, int unit_log) {
    const int s = threadIdx.x, unit = 1 << unit_log;
    Sequence me{0, 0};
    if (s < p.S) me = sequence(p, s);
    b.length[s] = me.length;
    b.count[s] = me.count;
    int units = 0, from = 0, items = 0, largest = 0;
    if (p.shared) {
        const int group = s / p.K, groups = p.S / p.K;
        const int want = s < groups ? p.shared[s] : 0;
        b.shared[s] = INT32_MAX;
        b.leader[s] = INT32_MAX;
        __syncthreads();
        if (me.count > 0) {
            atomicMin(&b.shared[group], me.prefix());
            atomicMin(&b.leader[group], s);
        }
        __syncthreads();
        if (s < groups) {
            const int n = b.leader[s] == INT32_MAX ? 0 : min(max(want, 0), b.shared[s]);
            b.shared[s] = static_cast<int>(p.span.page.quotient(n) * p.span.page.d);
        }
        __syncthreads();
        if (s < p.S) from = b.shared[group];
        if (s < p.S && s == group * p.K && from > 0) {
            largest = (from + unit - 1) >> unit_log;
            items = p.shared_tiles;
            units = items * largest;
        }
    }
    if (me.count > 0) {
        const int tiles = row_tiles(p, me, ROWS);
        items += tiles;
        largest = max(largest, (me.length - from + unit - 1) >> unit_log);
        if (p.parents || tiles == 1)
            units += tiles * ((me.length - from + unit - 1) >> unit_log);
        else
            for (int t = 0; t < tiles; ++t) units += (key_end<ROWS>(p, me, t) - from + unit - 1) >> unit_log;
    }
    items = wave_upto(items);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) largest = max(largest, __shfl_xor(largest, d));
    if ((s & 63) == 63) {
        b.items[s >> 6] = items;
        b.largest[s >> 6] = largest;
    }
    Totals total{set_line(b, units), 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        total.items += b.items[w];
        total.largest = max(total.largest, b.largest[w]);
    }
    return {total.line, uniform(total.items), uniform(total.largest)};
}

// The line in pieces of up to `each` units of one item, in place of units.
template <int ROWS>
__device__ __forceinline__ int pieces_board(const AttendParams& p, Board& b, int unit_log, int each) {
    const int s = threadIdx.x, unit = 1 << unit_log;
    const Sequence me{b.length[s], b.count[s]};
    int pieces = 0, from = 0;
    if (p.shared && s < p.S) {
        from = b.shared[s / p.K];
        if (s % p.K == 0) pieces = p.shared_tiles * ((((from + unit - 1) >> unit_log) + each - 1) / each);
    }
    if (me.count > 0) {
        const int tiles = row_tiles(p, me, ROWS);
        if (p.parents || tiles == 1)
            pieces += tiles * ((((me.length - from + unit - 1) >> unit_log) + each - 1) / each);
        else
            for (int t = 0; t < tiles; ++t) pieces += (((key_end<ROWS>(p, me, t) - from + unit - 1) >> unit_log) + each - 1) / each;
    }
    return set_line(b, pieces);
}

// ---------------------------------------------------------------------------
// The kernel
// ---------------------------------------------------------------------------

// A piece of an item: rows of `tile`, keys [key0, end).
struct Piece {
    int seq;    // whose pages are read
    int head;   // of the cache
    int tile;
    int key0, end;
    int item;
    bool shared;  // the rows are those of all beams of the group
    bool starts;  // it holds the item's first key
    bool whole;   // the rows' whole result
    Sequence own; // of seq
};

template <int DTYPE, int DP, int SHAPE>
__global__ __launch_bounds__(kAttendThreads, (Dims<DTYPE, DP, SHAPE>::kResident)) void attend_kernel(const AttendParams) {
    using E = Elem<DTYPE>;
    using T = typename E::T;
    using Frag = typename E::Frag;
    using Quad = typename E::Quad;
    using X = Dims<DTYPE, DP, SHAPE>;
    constexpr int RB = X::kRowBlocks, KB = X::kKeyBlocks, KEYS = X::kKeys, DB = X::kDimBlocks, ROWS = X::kRows;
    constexpr int WK = X::kKeyWaves, WR = X::kRowWaves;
    constexpr float kInf = __builtin_inff();

    __shared__ __attribute__((aligned(1024))) char lds[X::kLds];
    __shared__ float stats[3][WK][ROWS];
    __shared__ uint32_t sees[X::kTokens * (kAttendMaxTree / 32)];
    __shared__ int16_t up[kAttendMaxTree];
    __shared__ Board board;
    __shared__ int odd;  // the piece's rows have to be computed again

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int quad = lane >> 4, col = lane & 15;
    const int wr = wave % WR, wk = wave / WR;

    const AttendParams& p0 = arguments();
    // this workgroup's stretch of the units
    constexpr int kKeyLog = KEYS == 64 ? 6 : KEYS == 32 ? 5 : 4;
    const int unit_log = kKeyLog + p0.unit_shift, unit = 1 << unit_log;
    const Totals board_totals = fill_board<ROWS>(p0, board, unit_log);
    const int items = board_totals.items * p0.Hkv;
    int head_line = board_totals.line, total = head_line * p0.Hkv;
    int each = (total + p0.grid - 1) / p0.grid;
    each = (max(each, 1) + WK - 1) / WK * WK;
    // Many items, none of them larger than a stretch: a workgroup for each whole
    // one, no pieces to join, and the hardware hands them out as workgroups end.
    const bool whole_items = WR > 1 && !p0.shared && items >= 2 * p0.grid && board_totals.largest <= each;
    // Or each item is cut by itself, so that no workgroup has pieces of two: a piece
    // costs as much as kPieceCost units beside its own, but these cuts are longer.
    // With `each` of either form there are at most grid pieces: an item has at most
    // units / each + 1, or at most `cuts`.
    bool by_pieces = false;
    if (!whole_items && items <= p0.grid && items > 0) {
        const int cuts = p0.grid / items;
        int longer = (board_totals.largest + cuts - 1) / cuts;
        if (items < p0.grid) longer = min(longer, (total + p0.grid - items - 1) / (p0.grid - items));
        longer = (max(longer, 1) + WK - 1) / WK * WK;
        by_pieces = longer - each <= X::kPieceCost || static_cast<int64_t>(longer - each) * total <= static_cast<int64_t>(X::kPieceCost) * each * items;
        if (by_pieces) {
            each = longer;
            head_line = pieces_board<ROWS>(p0, board, unit_log, each);
            total = head_line * p0.Hkv;
        }
    }
    const int stretch = by_pieces ? 1 : each;
    int mine, at, stop;
    Piece chosen;
    if (whole_items) {
        // The items with the most keys first, so that the last to end are short; the
        // heads of a sequence's tile lie side by side, on as many XCDs as there are
        // heads up to eight, and a head's tiles find its keys there.
        const int entries = p0.S * p0.own_tiles;
        const int rank = static_cast<int>(blockIdx.x) / p0.Hkv;
        chosen.head = static_cast<int>(blockIdx.x) - rank * p0.Hkv;
        if (rank >= entries) return;
        int entry = rank;
        if (entries <= kAttendThreads) {
            // sorted: a thread counts the entries ahead of its own
            const int mine_seq = threadIdx.x / p0.own_tiles, mine_tile = threadIdx.x - mine_seq * p0.own_tiles;
            int keys = -1;
            if (static_cast<int>(threadIdx.x) < entries) {
                const Sequence q{board.length[mine_seq], board.count[mine_seq]};
                keys = mine_tile < row_tiles(p0, q, ROWS) ? key_end<ROWS>(p0, q, mine_tile) : 0;
            }
            int* const sorted = reinterpret_cast<int*>(lds);
            sorted[threadIdx.x] = keys;
            __syncthreads();
            int ahead = 0;
            for (int i = 0; i < entries; ++i) ahead += sorted[i] > keys || (sorted[i] == keys && i < static_cast<int>(threadIdx.x));
            __syncthreads();
            if (keys >= 0) sorted[ahead] = threadIdx.x;
            __syncthreads();
            entry = uniform(sorted[rank]);
        } else {
            entry = entries - 1 - rank;  // the last tiles have the most
        }
        if (entries <= kAttendThreads) {
            chosen.seq = entry / p0.own_tiles;
            chosen.tile = entry - chosen.seq * p0.own_tiles;
        } else {
            chosen.tile = entry / p0.S;
            chosen.seq = entry - chosen.tile * p0.S;
        }
        chosen.own = {uniform(board.length[chosen.seq]), uniform(board.count[chosen.seq])};
        if (chosen.tile >= row_tiles(p0, chosen.own, ROWS)) return;
        mine = 0, at = 0, stop = 1;
    } else {
        // neighbours share keys, so they lie on one XCD: workgroups go round the
        // eight of them
        const int busy = (total + stretch - 1) / stretch, per_xcd = (busy + 7) / 8;
        mine = static_cast<int>(blockIdx.x & 7) * per_xcd + static_cast<int>(blockIdx.x >> 3);
        if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || mine >= busy) return;
        at = mine * stretch;
        stop = min(at + stretch, total);
    }

    while (at < stop) {
        const AttendParams& p1 = arguments();
        // the item at `at`, and the piece of it in the stretch
        Piece w;
        int group = 0;
        if (whole_items) {
            w = chosen;
            w.key0 = 0;
            w.end = key_end<ROWS>(p1, w.own, w.tile);
            w.item = w.head * p1.head_items + w.seq * p1.own_tiles + w.tile;
            w.shared = false;
            w.starts = w.whole = true;
            if (threadIdx.x == 0) p1.info[w.item] = make_int4(0, 0, 0, 0);
            at = stop;
        } else {
            w.head = at / head_line;
            int off = at - w.head * head_line;  // in the head, then in the sequence, then in the item
            int seq = -1;
            for (int s0 = 0; s0 < p1.S; s0 += 64) {
                const bool ahead = s0 + lane < p1.S && board.first[s0 + lane] <= off;
                seq += __popcll(__ballot(ahead));
            }
            off -= uniform(board.first[seq]);
            group = p1.shared ? seq / p1.K : seq;
            const int from = p1.shared ? uniform(board.shared[group]) : 0;
            // elements of the line that so many units are
            const auto elements = [&](int units) { return by_pieces ? (units + each - 1) / each : units; };
            int units = (from + unit - 1) >> unit_log, end = from, length = elements(units);
            int place_in_head = group * (p1.shared_tiles + p1.K * p1.own_tiles);
            w.shared = p1.shared && seq == group * p1.K && off < p1.shared_tiles * length;
            if (w.shared) {
                w.tile = off / length;
                off -= w.tile * length;
                w.seq = uniform(board.leader[group]);
                w.own = {uniform(board.length[w.seq]), uniform(board.count[w.seq])};
                w.key0 = 0;
                place_in_head += w.tile;
            } else {
                if (p1.shared && seq == group * p1.K) off -= p1.shared_tiles * length;
                w.seq = seq;
                w.own = {uniform(board.length[seq]), uniform(board.count[seq])};
                w.key0 = from;
                if (p1.parents || row_tiles(p1, w.own, ROWS) == 1) {
                    end = w.own.length;
                    units = (end - from + unit - 1) >> unit_log;
                    length = elements(units);
                    w.tile = off / length;
                    off -= w.tile * length;
                } else {
                    // tiles of rows that read ever more keys: a lane for each
                    for (w.tile = 0;; w.tile += 64) {
                        const int t = w.tile + lane;
                        const int mine_end = key_end<ROWS>(p1, w.own, t);
                        const int mine_units = t < p1.own_tiles ? (mine_end - from + unit - 1) >> unit_log : 0;
                        const int n = elements(mine_units), upto = wave_upto(n);
                        const uint64_t past = __ballot(upto > off);
                        if (past) {
                            const int first = __builtin_ctzll(past);
                            w.tile += first;
                            units = __shfl(mine_units, first);
                            length = __shfl(n, first);
                            off -= __shfl(upto, first) - length;
                            end = __shfl(mine_end, first);
                            break;
                        }
                        off -= __shfl(upto, 63);
                    }
                }
                place_in_head += p1.shared_tiles + (seq - group * p1.K) * p1.own_tiles + w.tile;
            }
            off = uniform(off);
            units = uniform(units);
            length = uniform(length);
            end = uniform(end);
            w.tile = uniform(w.tile);
            w.item = uniform(w.head * p1.head_items + place_in_head);
            w.starts = off == 0;
            int first_unit = off, n_units, last;
            if (by_pieces) {
                first_unit = off * each;
                n_units = min(each, units - first_unit);
                last = mine - off + length - 1;
                w.whole = length == 1 && from == 0;
                at = stop;
            } else {
                const int start = at - off, until = min(start + units, stop);
                n_units = until - at;
                last = (start + units - 1) / each;
                w.whole = w.starts && until == start + units && from == 0;
                at = until;
            }
            w.key0 += first_unit << unit_log;
            w.end = min(end, w.key0 + (n_units << unit_log));
            if (w.starts && threadIdx.x == 0) p1.info[w.item] = make_int4(mine, last, from > 0, 0);
        }

        // ---- the piece's rows ----
        const AttendParams& p = arguments();
        const int prefix = w.own.prefix();
        int token[RB];     // of the sequence's asking tokens
        int64_t place[RB]; // of the row in out and lse, in rows; -1: no such row
        Frag q[RB][X::kSteps];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            int r = w.tile * ROWS + (wr * RB + rb) * 16 + col;
            int seq = w.seq, count = w.own.count;
            if (w.shared) {
                const int beam = static_cast<int>(p.beam_rows.quotient(r));
                r -= beam * static_cast<int>(p.beam_rows.d);
                seq = group * p.K + beam;
                count = beam < p.K ? board.count[seq] : 0;
            }
            const int G = static_cast<int>(p.G.d), n = static_cast<int>(p.G.quotient(r)), h = w.head * G + (r - n * G);
            token[rb] = n;
            const bool row = n < count;
            place[rb] = row ? (static_cast<int64_t>(seq) * p.N + n) * p.H + h : -1;
            const char* at_q = static_cast<const char*>(p.q) + (row ? seq * p.qs + n * p.qn + h * p.qh : 0);
#pragma unroll
            for (int i = 0; i < X::kSteps; ++i) {
                const int byte = (i * 4 + quad) * 16;
                q[rb][i] = row && byte < p.D * X::kSize ? *reinterpret_cast<const Frag*>(at_q + byte) : Frag{};
            }
        }
        // keys before this are seen by every row of the tile
        int masked_from = INT32_MAX;
        const int first_token = static_cast<int>(p.G.quotient(w.tile * ROWS));
        if (!w.shared) masked_from = prefix + (p.parents ? 0 : first_token + 1);
        if (masked_from >= w.end) masked_from = INT32_MAX;  // as of a single token
        const int words = (p.N + 31) >> 5;
        if (p.parents && masked_from != INT32_MAX) {
            // which drafted tokens each token of the tile sees, as bits
            __syncthreads();
            for (int i = threadIdx.x; i < p.N; i += kAttendThreads)
                up[i] = static_cast<int16_t>(min(max(p.parents[static_cast<int64_t>(w.seq) * p.N + i], -1), p.N));
            __syncthreads();
            for (int i = threadIdx.x; i < X::kTokens; i += kAttendThreads) {
                uint32_t* bits = sees + i * words;
                for (int j = 0; j < words; ++j) bits[j] = 0;
                for (int n = first_token + i; n >= 0 && n < p.N;) {
                    bits[n >> 5] |= 1u << (n & 31);
                    const int parent = up[n];
                    n = parent < n ? parent : -1;
                }
            }
            __syncthreads();
        }

        // ---- over the keys ----
        const char* const k_head = static_cast<const char*>(p.k) + w.head * p.kh;
        const char* const v_head = static_cast<const char*>(p.v) + w.head * p.vh;
        const int32_t* const row_pages = p.pages + static_cast<int64_t>(w.seq) * p.span.P;
        const int chunks = p.D * X::kSize / 16;

        const float scale = p.scale;
        f32x4 o[DB][RB];
        float m[RB], l[RB], limit[RB], shift[RB];
        f32x4 sum_l[RB];  // 16-bit types: the sum of the rounded values, once for every row
        const bool with_lse = p.lse != nullptr;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m[rb] = limit[rb] = -kInf;
            shift[rb] = 0.0f;
            l[rb] = 0.0f;
            sum_l[rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db][rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const float slack = p.slack;

        // The page-table entry of token first + lane of a tile, read well before
        // it is needed; then the place that it gives, -1 without a page.
        int32_t entry = -1;
        uint32_t in_page = 0;
        const auto look_up = [&](int first) BEAMGRAD_INLINE {
            const uint32_t token = first + lane, page = p.span.page.quotient(token);
            in_page = token - page * p.span.page.d;
            entry = -1;
            if (lane < KEYS && first + lane < w.end) entry = row_pages[page];
        };
        const bool alike = p.kp == p.vp && p.kt == p.vt;  // the usual: one offset serves both
        const auto locate = [&](int64_t& k_at, int64_t& v_at) BEAMGRAD_INLINE {
            const bool there = p.span.is_page(entry);
            const auto offset = [&](uint32_t page16, uint32_t token16) BEAMGRAD_INLINE {
                const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(entry)) * page16 + static_cast<uint64_t>(in_page) * token16;
                return there ? static_cast<int64_t>(at << 4) : -1;
            };
            k_at = offset(p.kp16, p.kt16);
            v_at = k_at;
            if (!alike) v_at = offset(p.vp16, p.vt16);
            return __ballot(there);
        };
        // this wavefront's share of a tile, from memory straight into LDS
        constexpr uint64_t kFull = ~uint64_t{0} >> (64 - KEYS);
        const auto fill = [&](bool values, char* region, const char* head, int64_t mine_at, uint64_t there) BEAMGRAD_INLINE {
            if (there == kFull) {
#pragma unroll
                for (int i = 0; i < X::kLoads; ++i) {
                    const int block = i * WR + wr;  // of 64 chunks
                    const int c = block * 64 + lane, row = c / X::kChunks, chunk = (c % X::kChunks) ^ (row & X::kSwizzle);
                    const char* const from = head + shfl64(mine_at, row) + chunk * 16;
                    if (chunks == X::kChunks || chunk < chunks)
                        __builtin_amdgcn_global_load_lds((global_char*)from, (lds_char*)(region + block * 1024), 16, 0, 0);
                }
                return;
            }
            // What no token fills must not be a NaN or an infinity, as a value (as a
            // key it is masked). All these stores come before the loads: between
            // them each would wait for the loads ahead of it.
            const int lane_here = opaque(lane);
            if (values) {
#pragma unroll
                for (int i = 0; i < X::kLoads; ++i) {
                    const int c = (i * WR + wr) * 64 + lane_here;
                    if (!((there >> (c / X::kChunks)) & 1)) *reinterpret_cast<f32x4*>(region + c * 16) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
#pragma unroll
            for (int i = 0; i < X::kLoads; ++i) {
                const int block = i * WR + wr;
                const int c = block * 64 + lane_here, row = c / X::kChunks, chunk = (c % X::kChunks) ^ (row & X::kSwizzle);
                const int64_t row_at = shfl64(mine_at, row);
                if (row_at >= 0 && chunk < chunks)
                    __builtin_amdgcn_global_load_lds((global_char*)(head + row_at + chunk * 16), (lds_char*)(region + block * 1024), 16, 0, 0);
            }
        };
        const auto region = [&](int place, int value) { return lds + place * X::kTile + (value * WK + wk) * X::kRegion; };

        // scores: s[kb][rb][i] of key 16 kb + 4 quad + i and row col of block rb
        const auto score = [&](const char* k_lds, f32x4 (&s)[KB][RB]) BEAMGRAD_INLINE {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) s[kb][rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const int row = kb * 16 + col;
#pragma unroll
                for (int i = 0; i < X::kSteps; ++i) {
                    const Frag a = *reinterpret_cast<const Frag*>(k_lds + row * X::kRowBytes +
                                                                  ((i * 4 + quad) ^ (row & X::kSwizzle)) * 16);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) s[kb][rb] = E::mma(a, q[rb][i], s[kb][rb]);
                }
            }
        };
        // Softmax of a tile's scores and the product with its values.
        const auto absorb = [&](int first, uint64_t there, const char* v_lds, f32x4 (&s)[KB][RB]) BEAMGRAD_INLINE {
            const bool hides = first + KEYS > masked_from;
            if (hides || there != kFull) {
                // A value that is no number or infinite, of a token that some rows of
                // the tile do not see, would reach them as 0 * inf: the join computes
                // these rows again, one by one.
                if (hides) {
                    bool none = false;
                    for (int c = opaque(lane); c < KEYS * X::kChunks; c += 64) {
                        const Frag x = *reinterpret_cast<const Frag*>(v_lds + c * 16);
#pragma unroll
                        for (int e = 0; e < 16 / X::kSize; ++e)
                            none |= first + c / X::kChunks >= masked_from && !(__builtin_fabsf(static_cast<float>(x[e])) < kInf);
                    }
                    if (none) odd = 1;
                }
                const int q4 = opaque(quad * 4);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    // the lane's four keys of the block: without a page, or hidden
                    const uint32_t page = static_cast<uint32_t>(there >> (kb * 16 + q4));
                    const int drafted = first + kb * 16 + q4 - prefix;
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        uint32_t seen = 15;
                        if (hides) {
                            if (p.parents) {
                                // four bits of the token's row from `drafted` on, those
                                // before the first drafted token set
                                const int in = max(drafted, 0), at = min(in >> 5, words - 1), row = min(token[rb] - first_token, X::kTokens - 1) * words;
                                const uint64_t two = sees[row + at] | static_cast<uint64_t>(at + 1 < words ? sees[row + at + 1] : 0) << 32;
                                const uint32_t bits = in < p.N ? static_cast<uint32_t>(two >> (in & 31)) : 0;
                                seen = drafted >= 0 ? bits : drafted <= -4 ? 15 : bits << -drafted | ((1u << -drafted) - 1);
                            } else {
                                const int n = token[rb] - drafted + 1;  // of them are seen
                                seen = n >= 4 ? 15 : n <= 0 ? 0 : (1u << n) - 1;
                            }
                        }
                        seen &= page;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][rb][i] = (seen >> i) & 1 ? s[kb][rb][i] : -kInf;
                    }
                }
            }
            // the maximum, raised where the tile's passes it by 2^8
            float top[RB];
            bool raise = false;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                top[rb] = s[0][rb][0];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[rb] = fmaxf(top[rb], s[kb][rb][i]);
                top[rb] = quad_max(top[rb]);
                raise |= top[rb] > limit[rb];
            }
            if (__any(raise)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    if (!(top[rb] > limit[rb])) top[rb] = m[rb];
                    // nothing seen yet: the sums are zero
                    const float by = m[rb] == -kInf || m[rb] == top[rb] ? 1.0f : __builtin_amdgcn_exp2f((m[rb] - top[rb]) * scale);
                    m[rb] = top[rb];
                    limit[rb] = top[rb] + slack;
                    shift[rb] = top[rb] == -kInf ? 0.0f : __builtin_fmaf(-top[rb], scale, X::kLift);
                    l[rb] *= by;
                    sum_l[rb] *= by;
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db][rb] *= by;
                }
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[kb][rb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][rb][i], scale, shift[rb]));
            }
            if constexpr (X::k32) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = kb * 16 + quad * 4 + i;
#pragma unroll
                        for (int db = 0; db < DB; ++db) {
                            const float a = *reinterpret_cast<const float*>(
                                v_lds + row * X::kRowBytes + ((db * 4 + (col >> 2)) ^ (row & X::kSwizzle)) * 16 + (col & 3) * 4);
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb)
                                o[db][rb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[kb][rb][i], o[db][rb], 0, 0, 0);
                        }
                    }
            } else {
                const Frag ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
                for (int pair = 0; pair < KB / 2; ++pair) {
                    Frag pr[RB];
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const Quad lo = __builtin_convertvector(s[2 * pair][rb], Quad);
                        const Quad hi = __builtin_convertvector(s[2 * pair + 1][rb], Quad);
                        pr[rb] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                        sum_l[rb] = E::mma(ones, pr[rb], sum_l[rb]);
                    }
                    // lane 4 j + c of a quad reads half a chunk of row j of four,
                    // and gets column `col` of the sixteen
                    const int row = pair * 32 + quad * 4 + (col >> 2), half = (col & 3) >> 1, byte = (col & 1) * 8;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        i16x4 part[2];
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int r = row + 16 * t;
                            part[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) i16x4*)(v_lds + r * X::kRowBytes +
                                                                          ((db * 2 + half) ^ (r & X::kSwizzle)) * 16 + byte));
                        }
                        const Frag a = __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) o[db][rb] = E::mma(a, pr[rb], o[db][rb]);
                    }
                }
            }
            if (X::k32 || with_lse) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
                        l[rb] += (s[kb][rb][0] + s[kb][rb][1]) + (s[kb][rb][2] + s[kb][rb][3]);
            }
        };
        const int rounds = (w.end - w.key0 + WK * KEYS - 1) / (WK * KEYS), mine_first = w.key0 + wk * KEYS;
        constexpr int kNext = WK * KEYS;
        look_up(mine_first);
        __syncthreads();  // the last piece's tiles are done with
        if (threadIdx.x == 0) odd = 0;
        if (chunks == X::kChunks) __syncthreads();
        if (chunks < X::kChunks) {
            // the columns past the width are zeros in every tile
            for (int i = threadIdx.x; i < X::kPlaces * X::kTile / 16; i += kAttendThreads)
                reinterpret_cast<f32x4*>(lds)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            __syncthreads();
        }
        if constexpr (X::kPlaces == 2) {
            // Tile t has place t & 1. While a tile's softmax keeps the vector
            // instructions busy, the matrix instructions have the next one's scores:
            // keys come two tiles ahead, values one.
            f32x4 s[2][KB][RB];
            int64_t k_at, v_at, v_next;
            uint64_t there = locate(k_at, v_at), there_next = 0;
            look_up(mine_first + kNext);
            fill(true, region(0, 1), v_head, v_at, there);
            fill(false, region(0, 0), k_head, k_at, there);
            if (rounds > 1) {
                there_next = locate(k_at, v_next);
                look_up(mine_first + 2 * kNext);
                fill(false, region(1, 0), k_head, k_at, there_next);
            }
            wait_all();
            barrier();
            score(region(0, 0), s[0]);
            const auto step = [&]<int PLACE>(std::integral_constant<int, PLACE>, int round) BEAMGRAD_INLINE {
                const int first = mine_first + round * kNext;
                // keys of the next tile and values of this one have come, for all
                // wavefronts, and all have done with what the next ones overwrite
                wait_all();
                barrier();
                uint64_t there_after = 0;
                if (round + 1 < rounds) fill(true, region(PLACE ^ 1, 1), v_head, v_next, there_next);
                if (round + 2 < rounds) {
                    there_after = locate(k_at, v_next);
                    look_up(first + 3 * kNext);
                    fill(false, region(PLACE, 0), k_head, k_at, there_after);
                }
                if (round + 1 < rounds) score(region(PLACE ^ 1, 0), s[PLACE ^ 1]);
                absorb(first, there, region(PLACE, 1), s[PLACE]);
                there = there_next;
                there_next = there_after;
            };
            for (int round = 0; round < rounds; round += 2) {
                step(std::integral_constant<int, 0>{}, round);
                if (round + 1 < rounds) step(std::integral_constant<int, 1>{}, round + 1);
            }
        } else {
            for (int first = mine_first; first < w.end; first += kNext) {  // no barriers
                int64_t k_at, v_at;
                const uint64_t there = locate(k_at, v_at);
                look_up(first + kNext);
                wait_lds();
                fill(true, region(0, 1), v_head, v_at, there);
                fill(false, region(0, 0), k_head, k_at, there);
                wait_all();
                f32x4 s[KB][RB];
                score(region(0, 0), s);
                absorb(first, there, region(0, 1), s);
            }
        }

        // ---- the piece's result ----
        const AttendParams& p2 = arguments();
        __syncthreads();
        const bool again = odd != 0;
        float sum[RB];  // what the result is divided by; l is the log-sum's
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            l[rb] += __shfl_xor(l[rb], 16);
            l[rb] += __shfl_xor(l[rb], 32);
            sum[rb] = X::k32 ? l[rb] : sum_l[rb][0];
        }
        if constexpr (WK > 1) {
            // the wavefronts along the keys: rescaled to their common maximum
            // and summed through LDS, each wavefront a share of the sums
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                if (quad == 0) {
                    stats[0][wk][(wr * RB + rb) * 16 + col] = m[rb];
                    stats[1][wk][(wr * RB + rb) * 16 + col] = l[rb];
                    stats[2][wk][(wr * RB + rb) * 16 + col] = sum[rb];
                }
            __syncthreads();
            f32x4* const sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int r = (wr * RB + rb) * 16 + col;
                float top = -kInf, all_l = 0.0f, all = 0.0f;
#pragma unroll
                for (int i = 0; i < WK; ++i) top = fmaxf(top, stats[0][i][r]);
                const auto weight = [&](float x) { return x == -kInf ? 0.0f : __builtin_amdgcn_exp2f((x - top) * p2.scale); };
#pragma unroll
                for (int i = 0; i < WK; ++i) {
                    const float by = weight(stats[0][i][r]);
                    all_l = __builtin_fmaf(by, stats[1][i][r], all_l);
                    all = __builtin_fmaf(by, stats[2][i][r], all);
                }
                const float by = weight(m[rb]);
#pragma unroll
                for (int db = 0; db < DB; ++db) sums[(wave * X::kAccs + db * RB + rb) * 64 + lane] = o[db][rb] * by;
                m[rb] = top;
                l[rb] = all_l;
                sum[rb] = all;
            }
            __syncthreads();
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                if (db % WK != wk) continue;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < WK; ++i) x += sums[((i * WR + wr) * X::kAccs + db * RB + rb) * 64 + lane];
                    o[db][rb] = x;
                }
            }
        }
        if (w.whole && again && threadIdx.x == 0) p2.info[w.item].w = 1;
        float* const part = p2.partial + slot_of(p2, mine, w.item, w.starts) * X::kSlot;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            if (place[rb] < 0) continue;
            const int r = (wr * RB + rb) * 16 + col;
            if (w.whole) {
                const float by = sum[rb] > 0.0f || sum[rb] != sum[rb] ? 1.0f / sum[rb] : 0.0f;
                T* const out = static_cast<T*>(p2.out) + place[rb] * p2.D;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (db % WK != wk) continue;
                    const int d = db * 16 + quad * 4;
                    if (d < p2.D) *reinterpret_cast<Quad*>(out + d) = __builtin_convertvector(o[db][rb] * by, Quad);
                }
                if (p2.lse && wk == 0 && quad == 0)
                    p2.lse[place[rb]] = l[rb] > 0.0f || l[rb] != l[rb]
                                           ? (m[rb] * p2.scale + (__builtin_amdgcn_logf(l[rb]) - X::kLift)) * 0.693147180559945309f
                                           : -kInf;
            } else {
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (db % WK != wk) continue;
                    *reinterpret_cast<f32x4*>(part + r * DP + db * 16 + quad * 4) = o[db][rb];
                }
                if (wk == 0 && quad == 0) {
                    part[ROWS * DP + r] = again ? __builtin_nanf("") : m[rb];
                    part[ROWS * DP + ROWS + r] = sum[rb];
                    part[ROWS * DP + 2 * ROWS + r] = l[rb];
                }
            }
        }
    }
}

// One row by a workgroup, key by key, as the formula has it: for rows that the
// matrix instructions would spoil.
template <int DTYPE>
__device__ __forceinline__ void plain_row(const AttendParams& p, int seq, const Sequence& s, int n, int head, int h, float* weights,
                                       float* lds) {
    using T = typename Elem<DTYPE>::T;
    constexpr float kInf = __builtin_inff();
    const int64_t place = (static_cast<int64_t>(seq) * p.N + n) * p.H + h;
    const T* const q = reinterpret_cast<const T*>(static_cast<const char*>(p.q) + seq * p.qs + n * p.qn + h * p.qh);
    const int32_t* const pages = p.pages + static_cast<int64_t>(seq) * p.span.P;
    const auto reduce = [&](float x, bool max) {
        __syncthreads();
        lds[threadIdx.x] = x;
        __syncthreads();
        float all = lds[0];
        for (int i = 1; i < kAttendThreads; ++i) all = max ? fmaxf(all, lds[i]) : all + lds[i];
        return all;
    };
    float top = -kInf, total = 0.0f, sum = 0.0f;
    for (int first = 0; first < s.length; first += kAttendThreads) {
        const int t = first + static_cast<int>(threadIdx.x), drafted = t - s.prefix();
        const uint32_t page = p.span.page.quotient(t);
        bool seen = t < s.length && p.span.is_page(pages[min(static_cast<int>(page), p.span.P - 1)]);
        if (seen && drafted >= 0) {
            int at = n;
            if (p.parents)
                while (at > drafted) {
                    const int parent = p.parents[static_cast<int64_t>(seq) * p.N + at];
                    at = parent < at ? parent : -1;
                }
            seen = p.parents ? at == drafted : drafted <= n;
        }
        float score = -kInf;
        if (seen) {
            const int64_t at = pages[page] * p.kp + (t - page * p.span.page.d) * p.kt + head * p.kh;
            const T* const k = reinterpret_cast<const T*>(static_cast<const char*>(p.k) + at);
            score = 0.0f;
            for (int d = 0; d < p.D; ++d) score = __builtin_fmaf(static_cast<float>(q[d]), static_cast<float>(k[d]), score);
        }
        const float next = fmaxf(top, reduce(score, true));
        const float by = top == next || top == -kInf ? 1.0f : __builtin_amdgcn_exp2f((top - next) * p.scale);
        const float weight = !seen || score == -kInf ? 0.0f : __builtin_amdgcn_exp2f((score - next) * p.scale);
        top = next;
        total = total * by + reduce(weight, false);
        sum *= by;
        weights[threadIdx.x] = seen ? weight : -1.0f;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < p.D)
            for (int i = 0; i < min(s.length - first, kAttendThreads); ++i) {
                if (weights[i] == -1.0f) continue;
                const uint32_t column = p.span.page.quotient(first + i);
                const int64_t at = pages[column] * p.vp + (first + i - column * p.span.page.d) * p.vt + head * p.vh;
                const T* const v = reinterpret_cast<const T*>(static_cast<const char*>(p.v) + at);
                sum = __builtin_fmaf(weights[i], static_cast<float>(v[threadIdx.x]), sum);
            }
        __syncthreads();
    }
    const bool any = total > 0.0f || total != total;
    if (static_cast<int>(threadIdx.x) < p.D) static_cast<T*>(p.out)[place * p.D + threadIdx.x] = static_cast<T>(any ? sum / total : 0.0f);
    if (p.lse && threadIdx.x == 0)
        p.lse[place] = any ? (top * p.scale + __builtin_amdgcn_logf(total)) * 0.693147180559945309f : -kInf;
}

// The rows of an item of a sequence (x) whose results lie in pieces, y of as many
// as a workgroup takes at once: a thread has four columns of a row, and where rows
// are few, several threads share the pieces of one. All reads of eight pieces are in
// flight together: their places follow from the item's first and last workgroup. A
// row that asks nothing gets 0 and -inf. Takes 4 us for a few pieces of 32 rows, 9
// for 33 pieces of each of 64 rows.
// Rows of which a piece's maximum is no number are computed again, as are those of
// an item that says so.
template <int DTYPE, int DP, int SHAPE>
__global__ __launch_bounds__(kAttendThreads) void attend_join(const AttendParams p) {
    using E = Elem<DTYPE>;
    using T = typename E::T;
    using Quad = typename E::Quad;
    using X = Dims<DTYPE, DP, SHAPE>;
    constexpr int ROWS = X::kRows, PER_ROW = DP / 4, SLOTS = kAttendThreads / PER_ROW, AT_ONCE = 8;
    constexpr float kInf = __builtin_inff();
    __shared__ f32x4 sums[kAttendThreads];
    __shared__ float tops[kAttendThreads], totals[kAttendThreads], totals_l[kAttendThreads];
    __shared__ int again;

    const int G = static_cast<int>(p.G.d);
    int x = blockIdx.x;
    const int tile = x % p.own_tiles;
    x /= p.own_tiles;
    const int head = x % p.Hkv, seq = x / p.Hkv;
    const int group = seq / p.K, beam = seq - group * p.K;
    const int group_items = head * p.head_items + group * (p.shared_tiles + p.K * p.own_tiles);
    const int own_item = group_items + p.shared_tiles + beam * p.own_tiles + tile;
    const Sequence s = sequence(p, seq);
    const int tile_rows = min(ROWS, p.N * G - tile * ROWS), live = min(tile_rows, s.count * G - tile * ROWS);
    int4 own = make_int4(0, 0, 0, 0);
    if (live > 0) own = p.info[own_item];
    const bool whole = own.x == own.y && !own.z;
    if (whole && !own.w && live == tile_rows) return;
    if (threadIdx.x == 0) again = own.w;
    __syncthreads();

    // threads of a row side by side, then the rows, then the shares of the pieces
    int shares = 1;
    while (2 * shares * tile_rows <= SLOTS) shares *= 2;
    const int rows_at_once = SLOTS / shares;
    const int slot = threadIdx.x / PER_ROW, share = slot / rows_at_once, column = (threadIdx.x % PER_ROW) * 4;
    for (int r0 = static_cast<int>(blockIdx.y) * rows_at_once; r0 < tile_rows; r0 += static_cast<int>(gridDim.y) * rows_at_once) {
        const int in_tile = r0 + slot - share * rows_at_once, row = tile * ROWS + in_tile;
        const bool mine_row = in_tile < tile_rows && share < shares;
        const int n = static_cast<int>(p.G.quotient(row)), h = head * G + row - n * G;
        const int64_t place = (static_cast<int64_t>(seq) * p.N + n) * p.H + h;
        T* const out = static_cast<T*>(p.out) + place * p.D;
        if (mine_row && in_tile >= live && share == 0) {
            if (column < p.D) *reinterpret_cast<Quad*>(out + column) = Quad{};
            if (p.lse && column == 0) p.lse[place] = -kInf;
        }
        if (whole || r0 >= live) continue;
        const bool busy = mine_row && in_tile < live;
        const int shared_row = beam * static_cast<int>(p.beam_rows.d) + row;
        const int shared_item = group_items + shared_row / ROWS;
        int4 common = make_int4(0, -1, 0, 0);
        if (own.z && busy) common = p.info[shared_item];
        const int mine = own.y - own.x + 1, pieces = mine + common.y - common.x + 1;
        float top = -kInf, total = 0.0f, total_l = 0.0f;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = share; busy && i0 < pieces; i0 += AT_ONCE * shares) {
            float m[AT_ONCE], l[AT_ONCE], ll[AT_ONCE];
            f32x4 o[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int at = min(i0 + i * shares, pieces - 1);
                const bool is_own = at < mine;
                const int w = is_own ? own.x + at : common.x + at - mine, r = (is_own ? row : shared_row) % ROWS;
                const float* const part =
                    p.partial + slot_of(p, w, is_own ? own_item : shared_item, w == (is_own ? own.x : common.x)) * X::kSlot;
                m[i] = part[ROWS * DP + r];
                l[i] = part[ROWS * DP + ROWS + r];
                ll[i] = part[ROWS * DP + 2 * ROWS + r];
                o[i] = *reinterpret_cast<const f32x4*>(part + r * DP + column);
            }
            float next = top;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (m[i] != m[i]) again = 1;
                next = fmaxf(next, m[i]);
            }
            const auto weight = [&](float y) { return y == -kInf ? 0.0f : __builtin_amdgcn_exp2f((y - next) * p.scale); };
            const float by = weight(top);
            top = next;
            total *= by;
            total_l *= by;
            sum *= by;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                // a piece that saw nothing holds zeros; its total is no number where
                // all of its scores were none
                if (i0 + i * shares >= pieces || (m[i] == -kInf && l[i] == 0.0f)) continue;
                const float piece_by = m[i] == -kInf ? 1.0f : weight(m[i]);
                total = __builtin_fmaf(piece_by, l[i], total);
                total_l = __builtin_fmaf(piece_by, ll[i], total_l);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(piece_by, o[i][e], sum[e]);
            }
        }
        if (shares > 1) {
            __syncthreads();
            sums[threadIdx.x] = sum;
            tops[threadIdx.x] = top;
            totals[threadIdx.x] = total;
            totals_l[threadIdx.x] = total_l;
            __syncthreads();
            if (share == 0) {
                const int step = rows_at_once * PER_ROW;
                float next = top;
                for (int i = 1; i < shares; ++i) next = fmaxf(next, tops[threadIdx.x + i * step]);
                const auto weight = [&](float y) { return y == -kInf ? 1.0f : __builtin_amdgcn_exp2f((y - next) * p.scale); };
                const float by = weight(top);
                total *= by;
                total_l *= by;
                sum *= by;
                for (int i = 1; i < shares; ++i) {
                    const int at = threadIdx.x + i * step;
                    const float share_by = weight(tops[at]);
                    total = __builtin_fmaf(share_by, totals[at], total);
                    total_l = __builtin_fmaf(share_by, totals_l[at], total_l);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(share_by, sums[at][e], sum[e]);
                }
                top = next;
            }
        }
        if (!busy || share != 0) continue;
        const bool any = total > 0.0f || total != total;
        const float by = any ? 1.0f / total : 0.0f;
        if (column < p.D) *reinterpret_cast<Quad*>(out + column) = __builtin_convertvector(sum * by, Quad);
        if (p.lse && column == 0)
            p.lse[place] = any ? (top * p.scale + (__builtin_amdgcn_logf(total_l) - X::kLift)) * 0.693147180559945309f : -kInf;
    }
    __syncthreads();
    if (!again) return;
    for (int r0 = static_cast<int>(blockIdx.y) * rows_at_once; r0 < live; r0 += static_cast<int>(gridDim.y) * rows_at_once)
        for (int r = r0; r < min(r0 + rows_at_once, live); ++r) {
            const int row = tile * ROWS + r, n = static_cast<int>(p.G.quotient(row));
            plain_row<DTYPE>(p, seq, s, n, head, head * G + row - n * G, reinterpret_cast<float*>(sums), tops);
        }
}

template <int DTYPE, int DP, int SHAPE>
hipError_t launch_shape(const AttendParams& p, hipStream_t stream) {
    // a workgroup for each item too, where the kernel may want it
    int workgroups = p.grid;
    const int64_t tiles = static_cast<int64_t>(p.S) * p.Hkv * p.own_tiles;
    if (Dims<DTYPE, DP, SHAPE>::kRowWaves > 1 && !p.shared && tiles >= 2 * workgroups) workgroups = static_cast<int>(tiles);
    attend_kernel<DTYPE, DP, SHAPE><<<workgroups, kAttendThreads, 0, stream>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int kAtOnce = kAttendThreads / (DP / 4);
    const int rows = min(attend_rows(SHAPE), p.N * static_cast<int>(p.G.d)), items = p.S * p.Hkv * p.own_tiles;
    const dim3 grid(static_cast<unsigned>(items),
                    static_cast<unsigned>(min((rows + kAtOnce - 1) / kAtOnce, max(1, 8192 / items))));
    attend_join<DTYPE, DP, SHAPE><<<grid, kAttendThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <int DTYPE, int DP>
hipError_t launch_dim(const AttendParams& p, int shape, hipStream_t stream) {
    switch (shape) {
        case kRows16: return launch_shape<DTYPE, DP, kRows16>(p, stream);
        case kRows32: return launch_shape<DTYPE, DP, kRows32>(p, stream);
        case kRows64: return launch_shape<DTYPE, DP, kRows64>(p, stream);
        default: return launch_shape<DTYPE, DP, attend_most(DTYPE, DP)>(p, stream);
    }
}

template <int DTYPE, int DP>
AttendSizes dim_sizes(int shape) {
    const auto of = [](auto x) { return AttendSizes{decltype(x)::kResident, decltype(x)::kSlot, decltype(x)::kKeys}; };
    switch (shape) {
        case kRows16: return of(Dims<DTYPE, DP, kRows16>{});
        case kRows32: return of(Dims<DTYPE, DP, kRows32>{});
        case kRows64: return of(Dims<DTYPE, DP, kRows64>{});
        default: return of(Dims<DTYPE, DP, attend_most(DTYPE, DP)>{});
    }
}

}  // namespace attend

template <int DTYPE>
AttendSizes attend_sizes(int dim, int shape) {
    switch (dim) {
        case 64: return attend::dim_sizes<DTYPE, 64>(shape);
        case 128: return attend::dim_sizes<DTYPE, 128>(shape);
        case 192: return attend::dim_sizes<DTYPE, 192>(shape);
        default: return attend::dim_sizes<DTYPE, 256>(shape);
    }
}

template <int DTYPE>
hipError_t launch_attend(const AttendParams& p, int dim, int shape, hipStream_t stream) {
    switch (dim) {
        case 64: return attend::launch_dim<DTYPE, 64>(p, shape, stream);
        case 128: return attend::launch_dim<DTYPE, 128>(p, shape, stream);
        case 192: return attend::launch_dim<DTYPE, 192>(p, shape, stream);
        default: return attend::launch_dim<DTYPE, 256>(p, shape, stream);
    }
}

}  // namespace dbs_hip
