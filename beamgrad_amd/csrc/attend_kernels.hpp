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
// operands' 16 bits for the matrix instruction (float32 inputs: not at all); l
// sums the unrounded values.
#pragma once

#include "attend.hpp"
#include "dbs_cuda.h"

namespace dbs_hip {
namespace attend {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) char global_char;

template <int DTYPE>
struct Elem;
template <>
struct Elem<DBS_CUDA_DTYPE_BF16> {
    using T = __bf16;
    using Frag = bf16x8;
    using Quad = bf16x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem<DBS_CUDA_DTYPE_F16> {
    using T = _Float16;
    using Frag = f16x8;
    using Quad = f16x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem<DBS_CUDA_DTYPE_F32> {
    using T = float;
    using Frag = f32x4;
    using Quad = f32x4;
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// Sizes of a kernel.
template <int DTYPE, int DP, int SHAPE>
struct Dims {
    static constexpr bool k32 = DTYPE == DBS_CUDA_DTYPE_F32;
    static constexpr int kSize = k32 ? 4 : 2;
    static constexpr int kRowBlocks = SHAPE == kRows16 ? 1 : 2;  // of 16 rows, of a wavefront
    static constexpr int kRowWaves = SHAPE == kRows128 ? 4 : SHAPE == kRows64 ? 2 : 1;
    static constexpr int kKeyWaves = 4 / kRowWaves;
    static constexpr int kRows = 16 * kRowBlocks * kRowWaves;
    static_assert(kRows == attend_rows(SHAPE));
    // Keys of a wavefront's tile: 32 fill the 16-bit matrix instruction's depth
    // for P V, 16 the float32 one's. A tile shared by four wavefronts is twice
    // as long where LDS holds two workgroups of it, for half the barriers.
    static constexpr int kKeys = SHAPE == kRows128 ? (k32 ? 32 : DP <= 128 ? 64 : 32) : (k32 ? 16 : 32);
    static constexpr int kKeyBlocks = kKeys / 16;
    static constexpr int kChunks = DP * kSize / 16;  // 16-byte chunks of a row
    static constexpr int kRowBytes = kChunks * 16;
    static constexpr int kSteps = kChunks / 4;  // matrix steps of a key block's scores
    static constexpr int kDimBlocks = DP / 16;
    static constexpr int kRegion = kKeys * kRowBytes;  // of keys or values of a wavefront's tile
    static constexpr int kLoads = kKeys * kChunks / 64 / kRowWaves;  // 16-byte loads a lane makes of a region
    // Chunk c of row r lies at c ^ (r & kSwizzle): reads of one chunk of many
    // rows meet different banks.
    static constexpr int kSwizzle = kChunks % 16 == 0 ? 15 : 7;
    static constexpr int kTile = 2 * kKeyWaves * kRegion;
    static constexpr int kAccs = kDimBlocks * kRowBlocks;
    static constexpr int kMerge = kKeyWaves > 1 ? kAccs * 4 * 64 * 16 : 0;
    static constexpr int kLds = kTile > kMerge ? kTile : kMerge;
    static constexpr int kTokens = kRows;  // of a tile of rows, at most
    static constexpr int kSlot = kRows * (DP + 2);  // floats of a partial result
    // workgroups of a CU: what its 160 KB of LDS hold, at most 4
    static constexpr int kFit = (160 * 1024) / (kLds + kTokens * (kAttendMaxTree / 8) + 2 * kAttendMaxTree + 8 * kKeyWaves * kRows);
    static constexpr int kResident = kFit >= 2 ? 2 : 1;
};

// The place of a piece's partial result. Without shared pages a workgroup
// leaves at most two: of the item it starts in the middle of, and of the item
// it does not finish. With them every piece leaves one: workgroup + item grows
// from piece to piece along the line, so no two have the same.
__device__ __forceinline__ int64_t slot_of(const AttendParams& p, int64_t workgroup, int item, bool starts) {
    return p.shared ? workgroup + item : 2 * workgroup + (starts ? 1 : 0);
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
    const int lo = __shfl(static_cast<int>(x), lane), hi = __shfl(static_cast<int>(x >> 32), lane);
    return static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) | static_cast<uint32_t>(lo));
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(x));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---------------------------------------------------------------------------
// Sequences, groups and their units
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

// Tokens that the beams of a group share, in whole pages.
__device__ __forceinline__ int shared_tokens(const AttendParams& p, int group, int& leader) {
    leader = -1;
    if (!p.shared) return 0;
    int least = INT32_MAX;
    for (int k = p.K - 1; k >= 0; --k) {
        const Sequence s = sequence(p, group * p.K + k);
        if (s.count > 0) {
            least = min(least, s.prefix());
            leader = group * p.K + k;
        }
    }
    if (leader < 0) return 0;
    const int n = min(max(p.shared[group], 0), least);
    return static_cast<int>(p.span.page.quotient(n) * p.span.page.d);
}

// The keys that row tile `tile` of a sequence has to read end here: all of
// them with a tree; in a chain, those up to its last token's.
template <int ROWS>
__device__ __forceinline__ int key_end(const AttendParams& p, const Sequence& s, int tile) {
    if (p.parents) return s.length;
    return s.prefix() + min(s.count, ((tile + 1) * ROWS - 1) / p.G + 1);
}

template <int ROWS, int KEYS>
__device__ __forceinline__ int64_t own_units(const AttendParams& p, const Sequence& s, int from) {
    const int tiles = (s.count * p.G + ROWS - 1) / ROWS;
    if (p.parents || tiles == 1) return static_cast<int64_t>(tiles) * ((s.length - from + KEYS - 1) / KEYS);
    int64_t units = 0;
    for (int t = 0; t < tiles; ++t) units += (key_end<ROWS>(p, s, t) - from + KEYS - 1) / KEYS;
    return units;
}

struct Group {
    int shared, leader;
    int64_t head_units; // of one cache head
};

template <int ROWS, int KEYS>
__device__ __forceinline__ Group group_of(const AttendParams& p, int group) {
    Group g;
    g.shared = shared_tokens(p, group, g.leader);
    g.head_units = static_cast<int64_t>(p.shared_tiles) * ((g.shared + KEYS - 1) / KEYS);
    for (int k = 0; k < p.K; ++k) {
        const Sequence s = sequence(p, group * p.K + k);
        if (s.count > 0) g.head_units += own_units<ROWS, KEYS>(p, s, g.shared);
    }
    return g;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += shfl64(x, (threadIdx.x & 63) ^ off);
    return x;
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
__global__ __launch_bounds__(kAttendThreads, (Dims<DTYPE, DP, SHAPE>::kResident)) void attend_kernel(const AttendParams p) {
    using E = Elem<DTYPE>;
    using T = typename E::T;
    using Frag = typename E::Frag;
    using Quad = typename E::Quad;
    using X = Dims<DTYPE, DP, SHAPE>;
    constexpr int RB = X::kRowBlocks, KB = X::kKeyBlocks, KEYS = X::kKeys, DB = X::kDimBlocks, ROWS = X::kRows;
    constexpr int WK = X::kKeyWaves, WR = X::kRowWaves;
    constexpr float kInf = __builtin_inff();

    __shared__ __attribute__((aligned(1024))) char lds[X::kLds];
    __shared__ float stats[2][WK][ROWS];
    __shared__ uint32_t sees[X::kTokens * (kAttendMaxTree / 32)];
    __shared__ int16_t up[kAttendMaxTree];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int quad = lane >> 4, col = lane & 15;
    const int wr = wave % WR, wk = wave / WR;

    // this workgroup's stretch of the units
    int64_t total = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64)
        total += wave_sum64(g0 + lane < p.groups ? group_of<ROWS, KEYS>(p, g0 + lane).head_units * p.Hkv : 0);
    total = uniform64(total);
    int64_t each = (total + p.grid - 1) / p.grid;
    each = (max(each, int64_t{1}) + WK - 1) / WK * WK;
    // neighbours share keys, so they lie on one XCD: workgroups go round the
    // eight of them
    const int64_t busy = (total + each - 1) / each, per_xcd = (busy + 7) / 8;
    const int64_t mine = static_cast<int64_t>(blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per_xcd || mine >= busy) return;
    int64_t at = mine * each;
    const int64_t stop = min(at + each, total);

    // the group it starts in
    int group = 0;
    int64_t base = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        const int64_t units = g0 + lane < p.groups ? group_of<ROWS, KEYS>(p, g0 + lane).head_units * p.Hkv : 0;
        int64_t upto = units;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t before = shfl64(upto, max(lane - off, 0));
            if (lane >= off) upto += before;
        }
        const uint64_t past = __ballot(base + upto > at);
        if (past) {
            const int first = __builtin_ctzll(past);
            group = g0 + first;
            base = uniform64(base + shfl64(upto - units, first));
            break;
        }
        base = uniform64(base + shfl64(upto, 63));
    }

    while (at < stop) {
        Group g = group_of<ROWS, KEYS>(p, group);
        g.head_units = uniform64(g.head_units);
        while (at - base >= g.head_units * p.Hkv) {
            base += g.head_units * p.Hkv;
            g = group_of<ROWS, KEYS>(p, ++group);
            g.head_units = uniform64(g.head_units);
        }
        // the item at `at`, and the piece of it in the stretch
        Piece w;
        int64_t start = at - base;  // first in the group, then the item's first unit
        w.head = static_cast<int>(start / g.head_units);
        int64_t off = start - w.head * g.head_units;  // within the head, then within the item
        const int head_item = group * p.items + w.head * (p.shared_tiles + p.K * p.own_tiles);
        int64_t units;
        const int shared_units = (g.shared + KEYS - 1) / KEYS;
        int from = 0, end;
        if (off < static_cast<int64_t>(p.shared_tiles) * shared_units) {
            w.shared = true;
            w.tile = static_cast<int>(off / shared_units);
            off -= static_cast<int64_t>(w.tile) * shared_units;
            units = shared_units;
            end = g.shared;
            w.seq = g.leader;
            w.own = sequence(p, w.seq);
            w.item = head_item + w.tile;
        } else {
            w.shared = false;
            off -= static_cast<int64_t>(p.shared_tiles) * shared_units;
            from = g.shared;
            int k = 0;
            for (;; ++k) {
                w.own = sequence(p, group * p.K + k);
                const int64_t u = w.own.count > 0 ? own_units<ROWS, KEYS>(p, w.own, from) : 0;
                if (off < u) break;
                off -= u;
            }
            w.seq = group * p.K + k;
            for (w.tile = 0;; ++w.tile) {
                end = key_end<ROWS>(p, w.own, w.tile);
                units = (end - from + KEYS - 1) / KEYS;
                if (off < units) break;
                off -= units;
            }
            w.item = head_item + p.shared_tiles + k * p.own_tiles + w.tile;
        }
        off = uniform64(off);
        units = uniform64(units);
        w.seq = uniform(w.seq);
        w.tile = uniform(w.tile);
        w.item = uniform(w.item);
        start = at - off;
        const int64_t until = min(start + units, stop);
        w.key0 = uniform(from + static_cast<int>(off) * KEYS);
        w.end = uniform(min(end, from + static_cast<int>(until - start) * KEYS));
        w.starts = at == start;
        w.whole = w.starts && until == start + units && !(p.shared && g.shared > 0);
        if (w.starts && threadIdx.x == 0)
            p.info[w.item] = make_int4(static_cast<int>(mine), static_cast<int>((start + units - 1) / each),
                                       g.shared > 0, 0);
        at = until;

        // ---- the piece's rows ----
        const int prefix = w.own.prefix();
        int token[RB];     // of the sequence's asking tokens
        int64_t place[RB]; // of the row in out and lse, in rows; -1: no such row
        Frag q[RB][X::kSteps];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            int r = w.tile * ROWS + (wr * RB + rb) * 16 + col;
            int seq = w.seq, count = w.own.count;
            if (w.shared) {
                const int beam = r / (p.N * p.G);
                r -= beam * p.N * p.G;
                seq = group * p.K + beam;
                count = beam < p.K ? sequence(p, seq).count : 0;
            }
            const int n = r / p.G, h = w.head * p.G + (r - n * p.G);
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
        const int first_token = w.tile * ROWS / p.G;
        if (!w.shared) masked_from = prefix + (p.parents ? 0 : first_token + 1);
        const int words = (p.N + 31) >> 5;
        if (p.parents && w.end > masked_from) {
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
        char* const k_lds = lds + wk * X::kRegion;
        char* const v_lds = lds + (WK + wk) * X::kRegion;
        const char* const k_head = static_cast<const char*>(p.k) + w.head * p.kh;
        const char* const v_head = static_cast<const char*>(p.v) + w.head * p.vh;
        const int32_t* const row_pages = p.pages + static_cast<int64_t>(w.seq) * p.span.P;
        const int chunks = p.D * X::kSize / 16;

        f32x4 o[DB][RB];
        float m[RB], l[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m[rb] = -kInf;
            l[rb] = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db][rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        const int rounds = (w.end - w.key0 + WK * KEYS - 1) / (WK * KEYS);
        for (int round = 0; round < rounds; ++round) {
            const int first = w.key0 + (round * WK + wk) * KEYS;
            if (WR == 1 && first >= w.end) break;  // no barriers below
            // the places of this tile's tokens: lane i has token first + i
            int64_t k_at = -1, v_at = -1;
            if (lane < KEYS && first + lane < w.end) {
                const uint32_t page = p.span.page.quotient(first + lane);
                const uint32_t in = first + lane - page * p.span.page.d;
                const int32_t entry = row_pages[page];
                if (p.span.is_page(entry)) {
                    k_at = entry * p.kp + in * p.kt;
                    v_at = entry * p.vp + in * p.vt;
                }
            }
            const uint64_t there = __ballot(k_at >= 0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (WR > 1) __syncthreads();
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
                for (int i = 0; i < X::kLoads; ++i) {
                    const int block = i * WR + wr;  // of 64 chunks
                    const int c = block * 64 + lane, row = c / X::kChunks, chunk = (c % X::kChunks) ^ (row & X::kSwizzle);
                    const int64_t from_row = shfl64(kv ? v_at : k_at, row);
                    char* const to = (kv ? v_lds : k_lds) + block * 1024;
                    if (from_row >= 0 && chunk < chunks)
                        __builtin_amdgcn_global_load_lds((global_char*)((kv ? v_head : k_head) + from_row + chunk * 16),
                                                         (lds_char*)to, 16, 0, 0);
                    else  // what no token fills must not be a NaN or an infinity
                        *reinterpret_cast<f32x4*>(to + lane * 16) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (WR > 1) __syncthreads();

            // scores: s[kb][rb][i] of key 16 kb + 4 quad + i and row col of block rb
            f32x4 s[KB][RB];
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
            const bool masked = there != (KEYS == 64 ? ~uint64_t{0} : (uint64_t{1} << KEYS) - 1) ||
                                first + KEYS > masked_from;
            if (masked) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = kb * 16 + quad * 4 + i;
                        const bool in = (there >> key) & 1;
                        const int drafted = first + key - prefix;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            bool seen = in;
                            if (in && first + key >= masked_from) {
                                if (p.parents)
                                    seen = token[rb] < p.N &&
                                           ((sees[(token[rb] - first_token) * words + (drafted >> 5)] >> (drafted & 31)) & 1);
                                else
                                    seen = drafted <= token[rb];
                            }
                            if (!seen) s[kb][rb][i] = -kInf;
                        }
                    }
            }
            // the maximum, raised where a tile's passes it by 2^8
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float top = s[0][rb][0];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kb][rb][i]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const bool raise = (m[rb] == -kInf && top > -kInf) || (top - m[rb]) * p.scale > 8.0f;
                if (__any(raise)) {
                    const float next = raise ? top : m[rb];
                    // nothing seen yet: the sums are zero
                    const float by = !raise ? 1.0f : m[rb] == -kInf ? 0.0f : __builtin_amdgcn_exp2f((m[rb] - next) * p.scale);
                    m[rb] = next;
                    l[rb] *= by;
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db][rb] *= by;
                }
                const float shift = m[rb] == -kInf ? 0.0f : -m[rb] * p.scale;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][rb][i], p.scale, shift));
                        s[kb][rb][i] = e;
                        l[rb] += e;
                    }
            }
            // A value that is no number or infinite, of a token that some rows
            // of the tile do not see, must not reach them as 0 * inf.
            bool careful = false;
            if (masked && first + KEYS > masked_from) {
                bool odd = false;
                for (int c = lane; c < KEYS * X::kChunks; c += 64) {
                    const Frag x = *reinterpret_cast<const Frag*>(v_lds + c * 16);
#pragma unroll
                    for (int e = 0; e < 16 / X::kSize; ++e) {
                        const float f = static_cast<float>(x[e]);
                        odd |= !(__builtin_fabsf(f) < kInf);
                    }
                }
                careful = __any(odd);
            }
            if (!careful) {
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
#pragma unroll
                    for (int pair = 0; pair < KB / 2; ++pair) {
                        Frag pr[RB];
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            const Quad lo = __builtin_convertvector(s[2 * pair][rb], Quad);
                            const Quad hi = __builtin_convertvector(s[2 * pair + 1][rb], Quad);
                            pr[rb] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                        }
                        // lane 4 j + c of a quad reads half a chunk of row j of
                        // four, and gets column `col` of the sixteen
                        const int row = pair * 32 + quad * 4 + (col >> 2), half = (col & 3) >> 1, byte = (col & 1) * 8;
#pragma unroll
                        for (int db = 0; db < DB; ++db) {
                            Frag a;
                            i16x4 part[2];
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const int r = row + 16 * t;
                                part[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) i16x4*)(v_lds + r * X::kRowBytes +
                                                                              ((db * 2 + half) ^ (r & X::kSwizzle)) * 16 + byte));
                            }
                            a = __builtin_bit_cast(Frag, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb) o[db][rb] = E::mma(a, pr[rb], o[db][rb]);
                        }
                    }
                }
            } else {
                for (int key = 0; key < KEYS; ++key) {
                    float e[RB];
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        e[rb] = 0.0f;
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (key == kb * 16 + quad * 4 + i) e[rb] = s[kb][rb][i];
                        e[rb] = __shfl(e[rb], ((key >> 2) & 3) * 16 + col);
                    }
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int byte = (db * 16 + quad * 4 + i) * X::kSize;
                            const float x = static_cast<float>(*reinterpret_cast<const T*>(
                                v_lds + key * X::kRowBytes + ((byte >> 4) ^ (key & X::kSwizzle)) * 16 + (byte & 15)));
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb)
                                if (e[rb] != 0.0f) o[db][rb][i] = __builtin_fmaf(e[rb], x, o[db][rb][i]);
                        }
                }
            }
        }

        // ---- the piece's result ----
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            l[rb] += __shfl_xor(l[rb], 16);
            l[rb] += __shfl_xor(l[rb], 32);
        }
        if constexpr (WK > 1) {
            // the wavefronts along the keys: rescaled to their common maximum
            // and summed through LDS, each wavefront a share of the sums
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                if (quad == 0) {
                    stats[0][wk][(wr * RB + rb) * 16 + col] = m[rb];
                    stats[1][wk][(wr * RB + rb) * 16 + col] = l[rb];
                }
            __syncthreads();
            f32x4* const sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int r = (wr * RB + rb) * 16 + col;
                float top = -kInf, sum = 0.0f;
#pragma unroll
                for (int i = 0; i < WK; ++i) top = fmaxf(top, stats[0][i][r]);
                const auto weight = [&](float x) { return x == -kInf ? 0.0f : __builtin_amdgcn_exp2f((x - top) * p.scale); };
#pragma unroll
                for (int i = 0; i < WK; ++i) sum = __builtin_fmaf(weight(stats[0][i][r]), stats[1][i][r], sum);
                const float by = weight(m[rb]);
#pragma unroll
                for (int db = 0; db < DB; ++db) sums[(wave * X::kAccs + db * RB + rb) * 64 + lane] = o[db][rb] * by;
                m[rb] = top;
                l[rb] = sum;
            }
            __syncthreads();
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                if (db % WK != wk) continue;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < WK; ++i) sum += sums[((i * WR + wr) * X::kAccs + db * RB + rb) * 64 + lane];
                    o[db][rb] = sum;
                }
            }
            __syncthreads();  // before the next piece's tiles
        }
        float* const part = p.partial + slot_of(p, mine, w.item, w.starts) * X::kSlot;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            if (place[rb] < 0) continue;
            const int r = (wr * RB + rb) * 16 + col;
            if (w.whole) {
                const float by = l[rb] > 0.0f || l[rb] != l[rb] ? 1.0f / l[rb] : 0.0f;
                T* const out = static_cast<T*>(p.out) + place[rb] * p.D;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (db % WK != wk) continue;
                    const int d = db * 16 + quad * 4;
                    if (d < p.D) *reinterpret_cast<Quad*>(out + d) = __builtin_convertvector(o[db][rb] * by, Quad);
                }
                if (p.lse && wk == 0 && quad == 0)
                    p.lse[place[rb]] = l[rb] > 0.0f || l[rb] != l[rb]
                                           ? (m[rb] * p.scale + __builtin_amdgcn_logf(l[rb])) * 0.693147180559945309f
                                           : -kInf;
            } else {
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    if (db % WK != wk) continue;
                    *reinterpret_cast<f32x4*>(part + r * DP + db * 16 + quad * 4) = o[db][rb];
                }
                if (wk == 0 && quad == 0) {
                    part[ROWS * DP + r] = m[rb];
                    part[ROWS * DP + ROWS + r] = l[rb];
                }
            }
        }
    }
}

// The rows' results where they are not whole: a wavefront takes a row, and
// each lane some of its columns. A row that asks nothing gets 0 and -inf.
template <int DTYPE, int DP, int SHAPE>
__global__ __launch_bounds__(kAttendThreads) void attend_join(const AttendParams p) {
    using T = typename Elem<DTYPE>::T;
    using X = Dims<DTYPE, DP, SHAPE>;
    constexpr int ROWS = X::kRows, PER = DP / 64;
    constexpr float kInf = __builtin_inff();
    const int lane = threadIdx.x & 63;
    const int64_t rows = static_cast<int64_t>(p.S) * p.N * p.H;
    const int64_t place = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (place >= rows) return;
    const int h = static_cast<int>(place % p.H);
    const int64_t sn = place / p.H;
    const int n = static_cast<int>(sn % p.N), seq = static_cast<int>(sn / p.N);
    T* const out = static_cast<T*>(p.out) + place * p.D;
    const Sequence s = sequence(p, seq);
    if (n >= s.count) {
        for (int d = lane; d < p.D; d += 64) out[d] = static_cast<T>(0.0f);
        if (p.lse && lane == 0) p.lse[place] = -kInf;
        return;
    }
    const int group = seq / p.K, beam = seq % p.K, head = h / p.G, in_head = h % p.G;
    const int head_item = group * p.items + head * (p.shared_tiles + p.K * p.own_tiles);
    const int own_row = n * p.G + in_head, shared_row = beam * p.N * p.G + own_row;
    const int own_item = head_item + p.shared_tiles + beam * p.own_tiles + own_row / ROWS;
    const int4 own = p.info[own_item];
    if (own.x == own.y && !own.z) return;

    float top = -kInf, total = 0.0f, sum[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] = 0.0f;
    const auto take = [&](const int4& info, int item, int r) {
        for (int w = info.x; w <= info.y; ++w) {
            const float* const part = p.partial + slot_of(p, w, item, w == info.x) * X::kSlot;
            const float m = part[ROWS * DP + r], l = part[ROWS * DP + ROWS + r];
            if (m == -kInf && l == 0.0f) continue;
            const float next = fmaxf(top, m);
            const float old = top == -kInf ? 0.0f : __builtin_amdgcn_exp2f((top - next) * p.scale);
            const float by = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f((m - next) * p.scale);
            top = next;
            total = total * old + l * by;
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[i] = sum[i] * old + part[r * DP + i * 64 + lane] * by;
        }
    };
    if (own.z) {
        const int item = head_item + shared_row / ROWS;
        take(p.info[item], item, shared_row % ROWS);
    }
    take(own, own_item, own_row % ROWS);
    const bool any = total > 0.0f || total != total;
    const float by = any ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (i * 64 + lane < p.D) out[i * 64 + lane] = static_cast<T>(sum[i] * by);
    if (p.lse && lane == 0)
        p.lse[place] = any ? (top * p.scale + __builtin_amdgcn_logf(total)) * 0.693147180559945309f : -kInf;
}

template <int DTYPE, int DP, int SHAPE>
hipError_t launch_shape(const AttendParams& p, hipStream_t stream) {
    attend_kernel<DTYPE, DP, SHAPE><<<p.grid, kAttendThreads, 0, stream>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t rows = static_cast<int64_t>(p.S) * p.N * p.H;
    attend_join<DTYPE, DP, SHAPE><<<static_cast<unsigned>((rows + 3) / 4), kAttendThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <int DTYPE, int DP>
hipError_t launch_dim(const AttendParams& p, int shape, hipStream_t stream) {
    switch (shape) {
        case kRows16: return launch_shape<DTYPE, DP, kRows16>(p, stream);
        case kRows32: return launch_shape<DTYPE, DP, kRows32>(p, stream);
        case kRows64: return launch_shape<DTYPE, DP, kRows64>(p, stream);
        default: return launch_shape<DTYPE, DP, kRows128>(p, stream);
    }
}

template <int DTYPE, int DP>
void dim_sizes(int shape, int& resident, int& slot) {
    switch (shape) {
        case kRows16: resident = Dims<DTYPE, DP, kRows16>::kResident, slot = Dims<DTYPE, DP, kRows16>::kSlot; break;
        case kRows32: resident = Dims<DTYPE, DP, kRows32>::kResident, slot = Dims<DTYPE, DP, kRows32>::kSlot; break;
        case kRows64: resident = Dims<DTYPE, DP, kRows64>::kResident, slot = Dims<DTYPE, DP, kRows64>::kSlot; break;
        default: resident = Dims<DTYPE, DP, kRows128>::kResident, slot = Dims<DTYPE, DP, kRows128>::kSlot; break;
    }
}

}  // namespace attend

template <int DTYPE>
void attend_sizes(int dim, int shape, int& resident, int& slot) {
    switch (dim) {
        case 64: return attend::dim_sizes<DTYPE, 64>(shape, resident, slot);
        case 128: return attend::dim_sizes<DTYPE, 128>(shape, resident, slot);
        case 192: return attend::dim_sizes<DTYPE, 192>(shape, resident, slot);
        default: return attend::dim_sizes<DTYPE, 256>(shape, resident, slot);
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
