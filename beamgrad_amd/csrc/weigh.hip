// SPDX-License-Identifier: MIT
//
// The attention that the tokens of a paged cache get, summed over those that
// ask (include/beamgrad_state.h): what an eviction goes by.
//
// Mathematics. With the log-sums that the attention left, a weight is
// e^(scale q . k - lse) at once, without a pass for the softmax, and a key's sum needs
// no other key. The exponent is one product and sum in units of log 2, fma(q . k, scale log2 e, -lse log2 e): its
// second term is rounded by itself, so a weight is off by up to 2^-24 (|scale q . k| + |lse|) of its own beside the
// score's rounding. Q K^T is made of 16 x 16 blocks; a lane gets four rows of one key, adds
// their weights up, and a key's four lanes join at the end. Rows and their sums are in
// a fixed order.
//
// Few rows (single tokens, trees): the queries stay, in registers or LDS, and the keys pass,
// several blocks of a wavefront on their way: bound by HBM, with more rows by LDS. Many rows (the
// ends of prompts): the keys stay, in registers, and the queries pass through LDS: bound by the
// exponentials and what surrounds them. Either way the call's work lies in one line, and each workgroup
// takes an equal stretch of it, whatever the lengths (they are on the device, so the host
// cannot plan with them).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <iterator>
#include <type_traits>

#include "attend.hpp"
#include "beamgrad_state.h"
#include "engine.hpp"
#include "matrix.hpp"
#include "paged.hpp"
#include "regions.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kSequences = kThreads;  // of a launch: a thread of each workgroup reads one's length
constexpr int kNone = INT32_MIN;      // below every token
constexpr float kLog2e = 1.44269504088896341f;

// of a lambda: its captures and arrays stay in registers
#define BEAMGRAD_INLINE __attribute__((always_inline))

template <int DTYPE, int DP>
struct Dims {
    static constexpr int kSize = DTYPE == DBS_CUDA_DTYPE_F32 ? 4 : 2;
    static constexpr int kChunks = DP * kSize / 16;  // 16-byte chunks of a row
    static constexpr int kRowBytes = kChunks * 16;
    static constexpr int kSteps = kChunks / 4;  // matrix steps of a block
    // Rows of queries that lie in LDS at once, 16 KB of them. Chunk c of row r lies at
    // c ^ (r & kSwizzle): reads of one chunk of 16 rows meet different banks.
    static constexpr int kRows = kRowBytes >= 768 ? 16 : kRowBytes >= 384 ? 32 : 16384 / kRowBytes;
    static constexpr int kSwizzle = kChunks % 16 == 0 ? 15 : 7;
    static constexpr int kLoads = kRows * kChunks / kThreads;  // of a thread, for them
    // And where keys pass more of them: 64 KB, and what the bits of a tree leave room for.
    static constexpr int kMoreRows = kRowBytes <= 128 ? 384 : 65536 / kRowBytes / 32 * 32;
    // Keys that stay: blocks of 16 of a wavefront, 64 registers of a lane.
    static constexpr int kBlocks = kSteps >= 16 ? 1 : kSteps >= 6 ? 2 : kSteps >= 4 ? 4 : 8;
    static constexpr int kKeys = 16 * kBlocks;
    static constexpr int kTile = 4 * kKeys;  // of a workgroup
    // Keys that pass: blocks of a wavefront that are on their way.
    static constexpr int kAhead = kSteps >= 12 ? 1 : kSteps >= 6 ? 2 : kSteps >= 4 ? 3 : 6;
    static constexpr int kFewResident = kSteps >= 6 ? 3 : 4;  // workgroups of a CU
};
constexpr int kPass = 64;  // keys that pass a workgroup at once

// A stretch that begins within a tile, whose sums others have parts of.
struct Piece {
    int s, head, tile_key;
    int first;  // the stretch that has the tile's first rows; -1: this one does not end the tile
};

struct Weigh {
    const char* q;
    const char* k;
    int64_t qs, qn, qh, kp, kt, kh;  // strides in bytes
    int64_t ws, wh;                  // of the weights, in elements
    PageSpan span;
    const int32_t* pages;
    const int32_t* lengths;
    const int32_t* counts;
    const int32_t* parents;
    const float* lse;
    float* weights;
    // of many rows, two of each stretch: of the tile it starts in the middle of, and of the
    // one it does not finish
    Piece* pieces;   // [stretches]
    float* partial;  // [stretches][2][kTile]
    int32_t S, N, H, D, Hkv;
    Divider G;    // heads of a cache head
    float scale;  // times log2(e)
    bool even;    // the heads of a cache head divide 16, and a place's rows lie within 32 bits
};

// Which of a block's weights count: all, those of the keys up to the token that asks, or
// those that a tree's token sees.
enum { kPlain, kChain, kTree };
typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Asking {
    int length, count;
    __device__ __forceinline__ int prefix() const { return length - count; }
};

__device__ __forceinline__ Asking asking(const Weigh& p, int s) {
    const int length = p.span.length(p.lengths[s]), count = p.counts ? p.counts[s] : p.N;
    return {length, min(max(count, 0), min(p.N, length))};
}

// x, of which the compiler knows nothing: what is computed from it stays where it is
// used and takes no registers elsewhere.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Waits for loads, those to LDS too, and LDS operations.
__device__ __forceinline__ void wait_all() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t lo = uniform(static_cast<int>(x)), hi = uniform(static_cast<int>(x >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) char global_char;

// What a workgroup knows of the call's sequences, and how the line of their work lies:
// all of one cache head's after the other's, or of one sequence's heads.
struct Board {
    int64_t first[kSequences + 1];  // work ahead of each sequence
    int length[kSequences], count[kSequences];
    int64_t sum[4];
};

// Fills the board; sequence s is thread s's, work(asking) what it has. Returns all of it.
template <class Work>
__device__ __forceinline__ int64_t fill_board(const Weigh& p, Board& b, Work work) {
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    Asking a{0, 0};
    if (tid < p.S) a = asking(p, tid);
    b.length[tid] = a.length;
    b.count[tid] = a.count;
    int64_t upto = a.count > 0 ? work(a) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_up(static_cast<uint32_t>(upto), d), hi = __shfl_up(static_cast<uint32_t>(upto >> 32), d);
        if (lane >= d) upto += static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    }
    if (lane == 63) b.sum[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += b.sum[w];
    b.first[tid + 1] = upto;
    if (tid == 0) b.first[0] = 0;
    __syncthreads();
    return uniform(b.first[kSequences]);
}

// The sequence whose work place `at` of the line is.
__device__ __forceinline__ int sequence_at(const Board& b, int64_t at) {
    int s = 0;
#pragma unroll
    for (int d = kSequences / 2; d > 0; d >>= 1)
        if (b.first[s + d] <= at) s += d;
    return uniform(s);
}

// Which asking tokens each one sees, as bits; both arrays in LDS. Ends with no barrier.
__device__ __forceinline__ void see(const Weigh& p, int s, int count, int16_t* up, uint32_t* sees, int words, int from, int until) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const int32_t parent = p.parents[static_cast<int64_t>(s) * p.N + i];
        up[i] = static_cast<int16_t>(parent >= 0 && parent < i ? parent : -1);
        for (int k = 0; k < words; ++k) sees[i * words + k] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kThreads)
        for (int at = i; at >= 0; at = up[at]) {
            const int bit = at - from;
            if (at >= from && at < until) sees[i * words + bit / 32] |= 1u << (bit & 31);
        }
}

// ---------------------------------------------------------------------------
// Few rows: the keys pass
// ---------------------------------------------------------------------------

// Line: 64 keys each, of a sequence's cache heads one after the other, of the sequences.
// Each wavefront has its own 16 keys of them and several such blocks' reads on their way, so
// that nothing waits for the others. 32 single tokens over caches of 2000 to 16000, 8 heads
// of 128 in bfloat16: 124 us, 621 MB, 5.0 TB/s. Five trees of 45 tokens, 135 rows of width 72
// in float16, over 300 to 2700: 12.8 us, most of it dependent reads (lengths, pages, keys) and
// the rows' way into LDS.
// ROWS: at most. 16 are one block, and lie in registers.
template <int DTYPE, int DP, int ROWS>
__global__ __launch_bounds__(kThreads, (ROWS > Dims<DTYPE, DP>::kRows ? 2 : Dims<DTYPE, DP>::kFewResident)) void weigh_few(const Weigh p) {
    using E = Elem<DTYPE>;
    using Frag = typename E::Frag;
    using X = Dims<DTYPE, DP>;
    constexpr int STEPS = X::kSteps, AHEAD = X::kAhead, WORDS = ROWS / 32 > 0 ? ROWS / 32 : 1;
    constexpr bool ONE = ROWS == 16;
    constexpr bool kHeld = ONE && STEPS <= 8;  // the queries fit registers
    constexpr float kInf = __builtin_inff();
    __shared__ __attribute__((aligned(16))) char queries[ROWS * X::kRowBytes];
    __shared__ __attribute__((aligned(16))) float row_lse[ROWS];  // -lse * log2(e)
    __shared__ __attribute__((aligned(16))) int row_token[ROWS];  // kNone: no row, or one that gives nothing
    __shared__ uint32_t sees[ROWS * WORDS];
    __shared__ int16_t up[ROWS];
    __shared__ Board board;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), quad = lane >> 4, col = lane & 15;
    const int bytes = p.D * X::kSize, G = static_cast<int>(p.G.d);
    const int64_t total = p.Hkv * fill_board(p, board, [](const Asking& a) { return static_cast<int64_t>((a.length + kPass - 1) / kPass); });
    const int64_t each = (total + gridDim.x - 1) / gridDim.x, stop = min(total, (blockIdx.x + 1) * each);
    int64_t at = blockIdx.x * each;
    while (at < stop) {
        // the stretch's keys of one sequence and head
        const int s = sequence_at(board, uniform(at / p.Hkv));
        const Asking a{uniform(board.length[s]), uniform(board.count[s])};
        const int tiles = (a.length + kPass - 1) / kPass, prefix = a.prefix(), rows = a.count * G;
        const int64_t off = at - p.Hkv * uniform(board.first[s]);
        const int head = uniform(static_cast<int>(off / tiles)), begin = uniform(static_cast<int>(off - static_cast<int64_t>(head) * tiles));
        const int end = uniform(static_cast<int>(min(static_cast<int64_t>(tiles), begin + (stop - at))));
        at += end - begin;

        Frag keys[AHEAD][STEPS];
        float old[AHEAD];
        bool there[AHEAD];
        const int32_t* const pages = p.pages + static_cast<int64_t>(s) * p.span.P;
        float* const weights = p.weights + s * p.ws + head * p.wh;
        const auto key_of = [&](int tile) { return tile * kPass + wave * 16 + col; };
        const auto page_of = [&](int tile) {
            const int key = key_of(tile);
            return tile < end && key < a.length ? pages[p.span.page.quotient(key)] : -1;
        };
        const auto fetch = [&](int i, int tile, int page) BEAMGRAD_INLINE {
            const int key = key_of(tile);
            there[i] = p.span.is_page(page);
            const char* const from = p.k + max(page, 0) * p.kp + (key - static_cast<int>(p.span.page.quotient(key) * p.span.page.d)) * p.kt + head * p.kh + quad * 16;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                u32x4 x = {0, 0, 0, 0};
                if (there[i] && (j * 4 + quad) * 16 < bytes) x = *reinterpret_cast<const u32x4*>(from + j * 64);
                keys[i][j] = __builtin_bit_cast(Frag, x);
            }
            old[i] = there[i] && quad == 0 && key < prefix ? weights[key] : 0.0f;
        };
        int page[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) page[i] = page_of(begin + i);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            fetch(i, begin + i, page[i]);
            page[i] = page_of(begin + i + AHEAD);
        }

        __syncthreads();  // the rows before are done with
        const char* const q0 = p.q + s * p.qs + static_cast<int64_t>(head) * G * p.qh;
        for (int i = tid; i < ROWS * X::kChunks; i += kThreads) {
            const int row = i / X::kChunks, c = i - row * X::kChunks, token = static_cast<int>(p.G.quotient(row)), g = row - token * G;
            u32x4 x = {0, 0, 0, 0};
            if (row < rows && c * 16 < bytes) x = *reinterpret_cast<const u32x4*>(q0 + token * p.qn + g * p.qh + c * 16);
            *reinterpret_cast<u32x4*>(queries + row * X::kRowBytes + (c ^ (row & X::kSwizzle)) * 16) = x;
        }
        for (int row = tid; row < ROWS; row += kThreads) {
            const int token = static_cast<int>(p.G.quotient(row));
            float l = -kInf;
            if (row < rows) l = p.lse[(static_cast<int64_t>(s) * p.N + token) * p.H + head * G + (row - token * G)];
            row_lse[row] = l == -kInf ? l : -l * kLog2e;
            row_token[row] = l == -kInf ? kNone : token;
        }
        if (p.parents) see(p, s, a.count, up, sees, WORDS, 0, a.count);
        __syncthreads();

        const auto query_of = [&](int block, Frag* query) {
            const char* const row = queries + (block * 16 + col) * X::kRowBytes;
#pragma unroll
            for (int j = 0; j < STEPS; ++j)
                query[j] = *reinterpret_cast<const Frag*>(row + ((j * 4 + quad) ^ (col & X::kSwizzle)) * 16);
        };
        Frag held[STEPS];
        if (kHeld) query_of(0, held);
        const int blocks = ONE ? 1 : (rows + 15) / 16;
        const auto weigh = [&](int i, int tile) BEAMGRAD_INLINE {
            const int key = key_of(tile), asks = key - prefix;
            const bool seen = p.parents && (tile + 1) * kPass > prefix;
            float sum = 0.0f;
            for (int b = 0; b < blocks; ++b) {
                const f32x4 l = *reinterpret_cast<const f32x4*>(&row_lse[b * 16 + quad * 4]);
                const i32x4 t = *reinterpret_cast<const i32x4*>(&row_token[b * 16 + quad * 4]);
                f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (kHeld) {
#pragma unroll
                    for (int j = 0; j < STEPS; ++j) score = E::mma(held[j], keys[i][j], score);
                } else {
                    Frag query[STEPS];
                    query_of(b, query);
#pragma unroll
                    for (int j = 0; j < STEPS; ++j) score = E::mma(query[j], keys[i][j], score);
                }
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    e[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[k], p.scale, l[k]));
                    bool visible = asks <= t[k];
                    if (seen && asks >= 0 && t[k] >= 0) visible = asks < a.count && (sees[t[k] * WORDS + asks / 32] >> (asks & 31) & 1);
                    e[k] = visible ? e[k] : 0.0f;
                }
                sum += (e[0] + e[1]) + (e[2] + e[3]);
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (quad == 0 && there[i]) weights[key] = old[i] + sum;
        };
        for (int tile = begin; tile < end; tile += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (tile + i >= end) break;
                weigh(i, tile + i);
                fetch(i, tile + i + AHEAD, page[i]);
                page[i] = page_of(tile + i + 2 * AHEAD);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows: the keys stay
// ---------------------------------------------------------------------------

// Line: blocks of 16 rows, of a sequence's tiles of keys one after the other, of the
// sequences, of the cache heads. Rows of tokens ahead of a tile's first key see none of
// it, and are not in the line. 64 keys stay with a wavefront, so that a block of queries
// that is read from LDS serves 16 matrix instructions of width 128; a score costs the vector
// unit a product, an exponential and a sum. Two prompts' ends of 512 tokens over 7700 and
// 15100 of 32 heads of 128 in bfloat16: 145 us under a trace, 99 GFLOP, 680 TFLOP/s (a call, its join with it, 141 us
// repeated without a pause, 129 among calls with other inputs); with 2048
// over 16000 in eight 820; in float32 835 us, 119 TFLOP/s. The vector unit is busy for 64 % of the time and the matrix unit for
// 36 %: neither is the limit by itself, but a wavefront's products of a block and what is computed
// from them stand one after the other, and only two more wavefronts share its SIMD. With constant operands, which
// take less power, the 820 are 990. Queries read a block ahead, blocks without a loop and raised priority around
// the products changed nothing; products of 32 x 32 and a block's products among the exponentials
// of the one before were not tried.
template <int DTYPE, int DP>
__global__ __launch_bounds__(kThreads, 3) void weigh_many(const Weigh p) {
    using E = Elem<DTYPE>;
    using Frag = typename E::Frag;
    using X = Dims<DTYPE, DP>;
    constexpr int STEPS = X::kSteps, KB = X::kBlocks, ROWS = X::kRows, TILE = X::kTile, WORDS = TILE / 32;
    constexpr float kInf = __builtin_inff();
    extern __shared__ char tree[];  // with parents: [N][WORDS], which of the tile's keys a token sees, then the parents
    // two places, by name: a wait for what is read of one is not a wait for what is on its
    // way to the other
    __shared__ __attribute__((aligned(1024))) char queries0[ROWS * X::kRowBytes];
    __shared__ __attribute__((aligned(1024))) char queries1[ROWS * X::kRowBytes];
    __shared__ __attribute__((aligned(16))) float row_lse[2][ROWS];  // -lse * log2(e)
    __shared__ __attribute__((aligned(16))) int row_token[2][ROWS];  // kNone: no row, or one that gives nothing
    __shared__ int odd[2][ROWS / 16];  // a block of rows that holds such
    __shared__ Board board;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), quad = lane >> 4, col = lane & 15;
    const int bytes = p.D * X::kSize, G = static_cast<int>(p.G.d);
    if (bytes < X::kRowBytes)  // what no query fills stays zero
        for (int i = tid; i < ROWS * X::kChunks; i += kThreads) {
            reinterpret_cast<u32x4*>(queries0)[i] = u32x4{0, 0, 0, 0};
            reinterpret_cast<u32x4*>(queries1)[i] = u32x4{0, 0, 0, 0};
        }
    // of a sequence: its blocks of rows, tiles that all of them see keys of, and the blocks
    // that see none of a later tile
    const auto blocks_of = [&](const Asking& a) { return (a.count * G + 15) / 16; };
    const auto whole_of = [&](const Asking& a) {
        const int tiles = (a.length + TILE - 1) / TILE;
        return p.parents ? tiles : min(tiles, a.prefix() / TILE + 1);
    };
    const auto ahead_of = [&](const Asking& a, int tile) { return static_cast<int>((static_cast<int64_t>(tile) * TILE - a.prefix()) * G / 16); };
    const int64_t line = fill_board(p, board, [&](const Asking& a) {
        const int tiles = (a.length + TILE - 1) / TILE, blocks = blocks_of(a), whole = whole_of(a);
        int64_t n = static_cast<int64_t>(whole) * blocks;
        for (int t = whole; t < tiles; ++t) n += blocks - ahead_of(a, t);
        return n;
    });
    const int64_t total = line * p.Hkv;
    const int64_t each = (total + gridDim.x - 1) / gridDim.x;
    // neighbours in the line, which share a head's queries, on one of the card's eight parts
    const int stretch = static_cast<int>(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const int64_t stop = min(total, (stretch + 1) * each);
    int64_t at = stretch * each;
    if (tid == 0) p.pieces[stretch] = {0, 0, 0, -1};

    // the 16-byte chunks of a place's rows that the lane fetches, where p.even
    uint32_t lane_at[X::kLoads];
#pragma unroll
    for (int i = 0; i < X::kLoads; ++i) {
        const int slot = (i * 4 + wave) * 64 + lane, row = slot / X::kChunks, c = (slot - row * X::kChunks) ^ (row & X::kSwizzle);
        const int t = static_cast<int>(p.G.quotient(row)), g = row - t * G;
        lane_at[i] = static_cast<uint32_t>(t * p.qn + g * p.qh) + c * 16;
    }
    while (at < stop) {
        // blocks [begin, end) of rows against tile `tile`, which has `units` of them
        const int head = uniform(static_cast<int>(at / line));
        int64_t off = at - head * line;
        const int s = sequence_at(board, off);
        const Asking a{uniform(board.length[s]), uniform(board.count[s])};
        off = uniform(off - board.first[s]);
        const int prefix = a.prefix(), rows = a.count * G, blocks = blocks_of(a), whole = whole_of(a);
        int tile, units = blocks, begin = 0;
        if (off < static_cast<int64_t>(whole) * blocks) {
            tile = uniform(static_cast<int>(off / blocks));
            off -= static_cast<int64_t>(tile) * blocks;
        } else {
            off -= static_cast<int64_t>(whole) * blocks;
            for (tile = whole;; ++tile) {
                begin = ahead_of(a, tile);
                units = blocks - begin;
                if (off < units) break;
                off -= units;
            }
            tile = uniform(tile);
            begin = uniform(begin);
            units = uniform(units);
        }
        const int skipped = uniform(static_cast<int>(off)), taken = uniform(static_cast<int>(min(static_cast<int64_t>(units - skipped), stop - at)));
        const bool all = taken == units;
        begin += skipped;
        const int end = begin + taken, tile_key = tile * TILE, key0 = tile_key + wave * X::kKeys;
        if (skipped > 0 && tid == 0)
            p.pieces[stretch] = {s, head, tile_key, skipped + taken == units ? static_cast<int>((at - skipped) / each) : -1};
        at += taken;

        // rows from block `from` on, to a place of LDS: their queries on their way, the rest in registers
        const char* const q0 = p.q + s * p.qs + static_cast<int64_t>(head) * G * p.qh;
        float lse = -kInf;
        int token = kNone;
        const auto stage = [&](char* queries, int from) BEAMGRAD_INLINE {
            // where the rows of a token lie in one block, a lane's place in a chunk is the same in all
            const char* const rows_at = q0 + static_cast<int64_t>(from * 16 / G) * p.qn;
            if (p.even && from * 16 + ROWS <= rows && bytes == X::kRowBytes) {
#pragma unroll
                for (int i = 0; i < X::kLoads; ++i)
                    __builtin_amdgcn_global_load_lds((global_char*)(rows_at + lane_at[i]), (lds_char*)(queries + (i * 4 + wave) * 1024), 16, 0, 0);
            } else {
                const int here = opaque(lane);
#pragma unroll
                for (int i = 0; i < X::kLoads; ++i) {
                    const int slot = (i * 4 + wave) * 64 + here, row = slot / X::kChunks, c = (slot - row * X::kChunks) ^ (row & X::kSwizzle);
                    const int r = from * 16 + row, t = static_cast<int>(p.G.quotient(r)), g = r - t * G;
                    if (r < rows && c * 16 < bytes)
                        __builtin_amdgcn_global_load_lds((global_char*)(q0 + t * p.qn + g * p.qh + c * 16),
                                                         (lds_char*)(queries + (i * 4 + wave) * 1024), 16, 0, 0);
                }
            }
            lse = -kInf;
            const int r = from * 16 + tid;
            if (tid < ROWS && r < rows) {
                token = static_cast<int>(p.G.quotient(r));
                lse = p.lse[(static_cast<int64_t>(s) * p.N + token) * p.H + head * G + (r - token * G)];
            }
        };
        const auto write_rows = [&](int place) BEAMGRAD_INLINE {
            const bool none = lse == -kInf;
            const uint64_t which = __ballot(none);
            if (tid < ROWS) {
                row_lse[place][tid] = none ? lse : -lse * kLog2e;
                row_token[place][tid] = none ? kNone : token;
                if (col == 0) odd[place][tid >> 4] = (which >> lane & 0xffff) != 0;
            }
        };
        // the keys
        Frag keys[KB][STEPS];
        bool there[KB];
        {
            int page[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int key = key0 + b * 16 + col;
                page[b] = -1;
                if (key < a.length) page[b] = p.pages[static_cast<int64_t>(s) * p.span.P + p.span.page.quotient(key)];
            }
            __syncthreads();  // the tile before is done with LDS
            stage(queries0, begin);
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int key = key0 + b * 16 + col;
                there[b] = p.span.is_page(page[b]);
                const int in_page = key - static_cast<int>(p.span.page.quotient(key) * p.span.page.d);
                const char* const from = p.k + max(page[b], 0) * p.kp + in_page * p.kt + head * p.kh + quad * 16;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    u32x4 x = {0, 0, 0, 0};
                    if (there[b] && (i * 4 + quad) * 16 < bytes) x = *reinterpret_cast<const u32x4*>(from + i * 64);
                    keys[b][i] = __builtin_bit_cast(Frag, x);
                }
            }
        }
        uint32_t* const sees = reinterpret_cast<uint32_t*>(tree);
        const bool asked = tile_key + TILE > prefix;  // some of the tile's keys ask themselves
        if (p.parents && asked) see(p, s, a.count, reinterpret_cast<int16_t*>(sees + p.N * WORDS), sees, WORDS, tile_key - prefix, tile_key - prefix + TILE);
        const bool asks_itself = key0 + X::kKeys > prefix;
        float sums[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) sums[b] = 0.0f;
        write_rows(0);
        // a chunk of rows, which lies in `queries`, while the next one comes to `others`
        const auto chunk_of = [&](int chunk, auto which, const char* queries, char* others) BEAMGRAD_INLINE {
            constexpr int place = decltype(which)::value;
            wait_all();
            __syncthreads();
            const bool more = chunk + ROWS / 16 < end;
            if (more) stage(others, chunk + ROWS / 16);
            const int n = min(ROWS / 16, end - chunk);
            const auto block = [&](int b, auto mask) BEAMGRAD_INLINE {
                constexpr int MASK = decltype(mask)::value;
                Frag query[STEPS];
                const char* const row = queries + (b * 16 + col) * X::kRowBytes;
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
                    query[i] = *reinterpret_cast<const Frag*>(row + ((i * 4 + quad) ^ (col & X::kSwizzle)) * 16);
                const f32x4 l = *reinterpret_cast<const f32x4*>(&row_lse[place][b * 16 + quad * 4]);
                i32x4 t = {0, 0, 0, 0};
                if constexpr (MASK != kPlain) t = *reinterpret_cast<const i32x4*>(&row_token[place][b * 16 + quad * 4]);
                f32x4 score[KB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) score[kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) score[kb] = E::mma(query[i], keys[kb][i], score[kb]);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[kb][i], p.scale, l[i]));
                    if constexpr (MASK != kPlain) {
                        const int asks = key0 + kb * 16 + col - prefix;  // the asking token that the key is
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            bool visible = asks <= t[i];
                            if constexpr (MASK == kTree) {
                                const int bit = wave * X::kKeys + kb * 16 + col;  // the key's place in the tile
                                const uint32_t of = sees[max(t[i], 0) * WORDS + bit / 32] >> (bit & 31);
                                visible = asks < 0 ? visible : visible && (of & 1);
                            }
                            e[i] = visible ? e[i] : 0.0f;
                        }
                    }
                    sums[kb] += (e[0] + e[1]) + (e[2] + e[3]);
                }
            };
            int any = asks_itself;
#pragma unroll
            for (int b = 0; b < ROWS / 16; ++b) any |= odd[place][b];
            if (n == ROWS / 16 && !uniform(any)) {
#pragma unroll 1
                for (int b = 0; b < ROWS / 16; ++b) block(b, std::integral_constant<int, kPlain>{});
            } else {
#pragma unroll 1
                for (int b = 0; b < n; ++b) {
                    if (p.parents && asks_itself) {
                        block(b, std::integral_constant<int, kTree>{});
                        continue;
                    }
                    const int strange = uniform(odd[place][b]);
                    const int first_token = uniform(row_token[place][b * 16]), last_token = uniform(row_token[place][b * 16 + 15]);
                    if (asks_itself && !strange && last_token < key0 - prefix) continue;  // none sees any
                    if (strange || (asks_itself && first_token < key0 + X::kKeys - 1 - prefix))
                        block(b, std::integral_constant<int, kChain>{});
                    else
                        block(b, std::integral_constant<int, kPlain>{});
                }
            }
            if (more) write_rows(place ^ 1);
        };
        for (int chunk = begin; chunk < end; chunk += 2 * (ROWS / 16)) {
            chunk_of(chunk, std::integral_constant<int, 0>{}, queries0, queries1);
            if (chunk + ROWS / 16 < end) chunk_of(chunk + ROWS / 16, std::integral_constant<int, 1>{}, queries1, queries0);
        }
        // the four lanes of a key
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            sums[b] += __shfl_xor(sums[b], 16);
            sums[b] += __shfl_xor(sums[b], 32);
            if (quad != b % 4) continue;
            if (!all) {
                p.partial[(static_cast<int64_t>(stretch) * 2 + (skipped > 0 ? 0 : 1)) * TILE + wave * X::kKeys + b * 16 + col] = sums[b];
            } else if (there[b]) {
                const int key = key0 + b * 16 + col;
                float* const to = p.weights + s * p.ws + head * p.wh + key;
                *to = key < prefix ? *to + sums[b] : sums[b];
            }
        }
    }
}

// x: a stretch that ends a tile which others began: what they have of it, in order. 5 us, most
// of it a launch and three dependent reads.
__global__ __launch_bounds__(kThreads) void weigh_join(const Weigh p, const int tile) {
    const Piece piece = p.pieces[blockIdx.x];
    if (piece.first < 0) return;
    const Asking a = asking(p, piece.s);
    for (int i = threadIdx.x; i < tile; i += kThreads) {
        const int key = piece.tile_key + i;
        if (key >= a.length || !p.span.is_page(p.pages[static_cast<int64_t>(piece.s) * p.span.P + p.span.page.quotient(key)])) continue;
        float* const to = p.weights + piece.s * p.ws + piece.head * p.wh + key;
        float sum = key < a.prefix() ? *to : 0.0f;
        for (int v = piece.first; v <= static_cast<int>(blockIdx.x); ++v) sum += p.partial[(static_cast<int64_t>(v) * 2 + (v == piece.first ? 1 : 0)) * tile + i];
        *to = sum;
    }
}

// ---------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------

bool multiple16(int64_t stride, int64_t size) { return stride >= 0 && stride <= int64_t{1} << 40 && stride * size % 16 == 0; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int element_size(int data_type) { return data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2; }

bool valid_sizes(const BeamgradWeights* a) {
    if (!a || (a->data_type != DBS_CUDA_DTYPE_F32 && a->data_type != DBS_CUDA_DTYPE_F16 && a->data_type != DBS_CUDA_DTYPE_BF16)) return false;
    if (a->sequences <= 0 || a->tokens <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->page_tokens <= 0 || a->n_pages <= 0 || a->table_pages <= 0)
        return false;
    if (a->head_dim <= 0 || a->head_dim > kAttendMaxDim || a->head_dim % 8 != 0 || a->heads % a->kv_heads != 0 || a->kv_heads > 65535) return false;
    if (a->parents && a->tokens > kAttendMaxTree) return false;
    if (!std::isfinite(a->scale * kLog2e) || !(a->scale > 0.0f)) return false;
    if ((static_cast<int64_t>(a->table_pages) + 1) * a->page_tokens > INT32_MAX - 65536) return false;
    if (static_cast<double>(a->tokens) * a->heads > 1.0e9) return false;
    const int64_t places = static_cast<int64_t>(a->table_pages) * a->page_tokens;
    for (int i = 0; i < 2; ++i)
        if (a->weight_strides[i] < 0 || a->weight_strides[i] > int64_t{1} << 40) return false;
    // the places of two heads, or sequences, lie apart
    const int64_t ws = a->weight_strides[0], wh = a->weight_strides[1];
    const bool heads_inner = (a->kv_heads == 1 || wh >= places) && (a->sequences == 1 || ws >= (a->kv_heads - 1) * wh + places);
    const bool heads_outer = (a->sequences == 1 || ws >= places) && (a->kv_heads == 1 || wh >= (a->sequences - 1) * ws + places);
    if (!heads_inner && !heads_outer) return false;
    for (int i = 0; i < 3; ++i)
        if (!multiple16(a->q_strides[i], element_size(a->data_type)) || !multiple16(a->k_strides[i], element_size(a->data_type))) return false;
    return true;
}

int64_t places_of(const BeamgradWeights& a) { return static_cast<int64_t>(a.table_pages) * a.page_tokens; }
int64_t rows_of(const BeamgradWeights& a) { return static_cast<int64_t>(a.tokens) * (a.heads / a.kv_heads); }

struct Form {
    const void* kernel;
    bool many;
    int tile, resident, rounds;  // keys of a tile of many; workgroups of a CU, and how often
};
template <int DTYPE, int DP>
Form form_of_width(int64_t rows, int64_t passes) {
    using X = Dims<DTYPE, DP>;
    if (rows <= 16) return {reinterpret_cast<const void*>(weigh_few<DTYPE, DP, 16>), false, 0, X::kFewResident, 4};
    if (rows <= X::kRows) return {reinterpret_cast<const void*>(weigh_few<DTYPE, DP, X::kRows>), false, 0, X::kFewResident, 4};
    // More rows pass each key through more of LDS than keys that stay, but begin sooner and need no
    // join: so up to this many matrix instructions of a wavefront altogether, and for wide heads,
    // of whose keys few can stay, always. us, with 64 rows at most and with all of them: 135 rows
    // of width 72 in float16 over 6 x 300 to 2700 21.6, 26; 180 of 128 in bfloat16 over one of 2700
    // 15.9, 19.4, over 6 x 2700 to 8000 59.6, 55; 128 in float32 (8 steps) over 6 x 8000 108, 125.
    if (rows <= X::kMoreRows && (X::kSteps >= 8 || passes * ((rows + 15) / 16) * X::kSteps <= 1 << 17))
        return {reinterpret_cast<const void*>(weigh_few<DTYPE, DP, X::kMoreRows>), false, 0, 2, 1};
    return {reinterpret_cast<const void*>(weigh_many<DTYPE, DP>), true, X::kTile, 3, 2};
}
template <int DTYPE>
Form form_of(int dim, int64_t rows, int64_t passes) {
    switch ((dim + 63) / 64) {
        case 1: return form_of_width<DTYPE, 64>(rows, passes);
        case 2: return form_of_width<DTYPE, 128>(rows, passes);
        case 3: return form_of_width<DTYPE, 192>(rows, passes);
        default: return form_of_width<DTYPE, 256>(rows, passes);
    }
}
Form form_of(const BeamgradWeights& a) {
    const int64_t rows = rows_of(a), passes = std::min(a.sequences, kSequences) * static_cast<int64_t>(a.kv_heads) * ((places_of(a) + kPass - 1) / kPass);
    switch (a.data_type) {
        case DBS_CUDA_DTYPE_F32: return form_of<DBS_CUDA_DTYPE_F32>(a.head_dim, rows, passes);
        case DBS_CUDA_DTYPE_F16: return form_of<DBS_CUDA_DTYPE_F16>(a.head_dim, rows, passes);
        default: return form_of<DBS_CUDA_DTYPE_BF16>(a.head_dim, rows, passes);
    }
}

// The weights are written while queries, keys and log-sums are read.
bool lies_apart(const BeamgradWeights& a) {
    const int64_t size = element_size(a.data_type), *q = a.q_strides, *k = a.k_strides, *w = a.weight_strides, wide = sizeof(float);
    const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    const Region weights{at(a.weights), {a.sequences, a.kv_heads}, {w[0] * wide, w[1] * wide}, places_of(a) * wide};
    const Region read[] = {{at(a.q), {a.sequences, a.tokens}, {q[0] * size, q[1] * size}, ((a.heads - 1) * q[2] + a.head_dim) * size},
                           {at(a.k), {a.n_pages, a.page_tokens}, {k[0] * size, k[1] * size}, ((a.kv_heads - 1) * k[2] + a.head_dim) * size},
                           {at(a.lse), {1, 1}, {0, 0}, static_cast<int64_t>(a.sequences) * a.tokens * a.heads * wide}};
    return std::all_of(std::begin(read), std::end(read), [&](const Region& r) { return apart(weights, r); });
}

// Workgroups of a launch, a multiple of eight. The card holds three of many rows on a CU
// (two with a large tree's table), but of three that share a CU the oldest runs fastest:
// twice as many, in equal stretches, are done sooner (two prompts' ends of 512 tokens over
// 7700 and 15100, 32 heads of 128, bfloat16: 143 us a call, 151 with one round; more rounds
// cost more beginnings than they gain). Few rows have shorter beginnings: four rounds (32
// tokens over 2000 to 16000: 125 us, 140 with one). More rows that keys pass fill LDS of
// a CU twice, and begin longer: one round (68 rows of 128 in bfloat16 over 32 x 2700 to 8000
// 117 us, 167 with six). No more than there is work for, by the table's size.
unsigned grid_of(const BeamgradWeights& a, const Form& form, size_t lds) {
    int device = 0, cus = 0;
    if (hipGetDevice(&device) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0) {
        (void)hipGetLastError();
        cus = 256;
    }
    const int64_t most = static_cast<int64_t>(cus) * form.rounds * (lds > 14 * 1024 ? 2 : form.resident);
    const int64_t tile = form.many ? form.tile : kPass, heads = static_cast<int64_t>(std::min(a.sequences, kSequences)) * a.kv_heads;
    const double work = static_cast<double>(heads) * static_cast<double>((places_of(a) + tile - 1) / tile) * (form.many ? static_cast<double>((rows_of(a) + 15) / 16) / 3.0 : 1.0);
    return static_cast<unsigned>((std::max<int64_t>(1, static_cast<int64_t>(std::min(work, static_cast<double>(most)))) + 7) / 8 * 8);
}

size_t tree_bytes(const BeamgradWeights& a, const Form& form) {
    return a.parents && form.many ? static_cast<size_t>(a.tokens) * (form.tile / 32 * sizeof(uint32_t) + sizeof(int16_t)) : 0;
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_accumulate_weights_workspace_size(const BeamgradWeights* args) {
    if (!valid_sizes(args)) return -1;
    const Form form = form_of(*args);
    return form.many ? grid_of(*args, form, tree_bytes(*args, form)) * static_cast<int64_t>(sizeof(Piece) + 2 * form.tile * sizeof(float)) : 0;
}

DBS_CUDA_EXPORT int beamgrad_accumulate_weights(const BeamgradWeights* args, void* workspace, int64_t workspace_bytes,
                                                void* stream_ptr) {
    if (!valid_sizes(args)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const BeamgradWeights& a = *args;
    const int64_t bytes = beamgrad_accumulate_weights_workspace_size(args);
    if (!a.q || !a.k || !a.pages || !a.lengths || !a.lse || !a.weights || !aligned16(a.q) || !aligned16(a.k) || bytes < 0 ||
        (bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < bytes)) || !lies_apart(a))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Form form = form_of(a);
    const int64_t size = element_size(a.data_type);
    Weigh p{};
    p.qs = a.q_strides[0] * size, p.qn = a.q_strides[1] * size, p.qh = a.q_strides[2] * size;
    p.kp = a.k_strides[0] * size, p.kt = a.k_strides[1] * size, p.kh = a.k_strides[2] * size;
    p.k = static_cast<const char*>(a.k);
    p.ws = a.weight_strides[0], p.wh = a.weight_strides[1];
    p.span = {Divider::of(static_cast<uint32_t>(a.page_tokens)), a.n_pages, a.table_pages};
    const size_t lds = tree_bytes(a, form);
    const unsigned grid = grid_of(a, form, lds);
    p.pieces = static_cast<Piece*>(workspace);
    p.partial = reinterpret_cast<float*>(p.pieces + grid);
    p.N = a.tokens, p.H = a.heads, p.D = a.head_dim, p.Hkv = a.kv_heads;
    p.G = Divider::of(static_cast<uint32_t>(a.heads / a.kv_heads));
    p.scale = a.scale * kLog2e;
    p.even = 16 % p.G.d == 0 && p.qn <= INT32_MAX / 256 && p.qh <= INT32_MAX / 32;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = hipSuccess;
    for (int s0 = 0; s0 < a.sequences && e == hipSuccess; s0 += kSequences) {
        p.S = std::min(kSequences, a.sequences - s0);
        p.q = static_cast<const char*>(a.q) + s0 * p.qs;
        p.pages = a.pages + static_cast<int64_t>(s0) * a.table_pages;
        p.lengths = a.lengths + s0;
        p.counts = a.counts ? a.counts + s0 : nullptr;
        p.parents = a.parents ? a.parents + static_cast<int64_t>(s0) * a.tokens : nullptr;
        p.lse = a.lse + static_cast<int64_t>(s0) * a.tokens * a.heads;
        p.weights = a.weights + s0 * p.ws;
        void* arguments[] = {&p};
        e = hipLaunchKernel(form.kernel, dim3(grid), dim3(kThreads), arguments, lds, stream);
        if (e == hipSuccess && form.many) {
            weigh_join<<<grid, kThreads, 0, stream>>>(p, form.tile);
            e = hipGetLastError();
        }
    }
    return finish_call(stream, e);
}

}  // extern "C"
