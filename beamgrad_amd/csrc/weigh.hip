// SPDX-License-Identifier: MIT
//
// The attention that the tokens of a paged cache get, summed over those that
// ask (include/beamgrad_state.h): what an eviction goes by.
//
// Mathematics. With the log-sums that the attention left, a weight is
// e^(scale q . k - lse) at once, without a pass for the softmax, and a key's sum needs
// no other key. So keys are what stays: a wavefront holds its keys in registers as
// the second operand of Q K^T and lets all rows of queries pass; a lane gets four
// rows of one key, whose weights it adds up. The four lanes of a key join once, at the
// end. Rows and their sums are in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attend.hpp"
#include "beamgrad_state.h"
#include "engine.hpp"
#include "matrix.hpp"
#include "paged.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kSequences = kThreads;  // of a launch: a thread of each workgroup reads one's length
constexpr int kChunk = 16;            // blocks of 16 rows whose places a workgroup holds
constexpr int kMaxSplits = 32;
constexpr int kJoinThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;

template <int DTYPE, int DP>
struct Dims {
    static constexpr int kSize = DTYPE == DBS_CUDA_DTYPE_F32 ? 4 : 2;
    static constexpr int kSteps = DP * kSize / 64;  // matrix steps of a block
    // blocks of 16 keys that a wavefront holds: 64 registers of a lane
    static constexpr int kBlocks = kSteps >= 16 ? 1 : kSteps >= 8 ? 2 : kSteps >= 6 ? 2 : kSteps >= 4 ? 4 : 8;
    static constexpr int kKeys = 16 * kBlocks;  // of a wavefront
    static constexpr int kTile = 4 * kKeys;     // of a workgroup
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
    float* partial;  // [splits][S][Hkv][places], where the rows are split
    int64_t places;
    int32_t S, N, H, Hkv, D, splits;
    Divider G;
    float scale;  // times log2(e)
};

struct Asking {
    int length, count;
    __device__ __forceinline__ int prefix() const { return length - count; }
};

__device__ __forceinline__ Asking asking(const Weigh& p, int s) {
    const int length = p.span.length(p.lengths[s]), count = p.counts ? p.counts[s] : p.N;
    return {length, min(max(count, 0), min(p.N, length))};
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Item: a tile of keys of a sequence and cache head, and of its rows a split.
template <int DTYPE, int DP>
__global__ __launch_bounds__(kThreads) void weigh_kernel(const Weigh p) {
    using E = Elem<DTYPE>;
    using Frag = typename E::Frag;
    using X = Dims<DTYPE, DP>;
    constexpr int STEPS = X::kSteps, KB = X::kBlocks;
    constexpr float kInf = __builtin_inff();
    extern __shared__ char tree[];  // with parents: [N][kTile / 32] words, which keys a token sees, then the parents
    __shared__ int first[kSequences + 1], sum[4];
    __shared__ int64_t row_at[kChunk * 16];
    __shared__ __attribute__((aligned(16))) float row_lse[kChunk * 16];  // -lse * log2(e); of no row: -inf
    __shared__ int row_token[kChunk * 16];

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), quad = lane >> 4, col = lane & 15;
    // tiles of keys ahead of each sequence
    {
        int tiles = 0;
        if (tid < p.S) {
            const Asking a = asking(p, tid);
            tiles = a.count > 0 ? (a.length + X::kTile - 1) / X::kTile : 0;
        }
        int upto = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        if (lane == 63) sum[wave] = upto;
        __syncthreads();
        for (int w = 0; w < wave; ++w) upto += sum[w];
        first[tid + 1] = upto;
        if (tid == 0) first[0] = 0;
        __syncthreads();
    }
    const int64_t items = static_cast<int64_t>(uniform(first[kSequences])) * p.Hkv * p.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t of_heads = item / p.Hkv;
        const int head = static_cast<int>(item - of_heads * p.Hkv), tile = static_cast<int>(of_heads / p.splits);
        const int split = static_cast<int>(of_heads - static_cast<int64_t>(tile) * p.splits);
        int s = 0;
#pragma unroll
        for (int d = kSequences / 2; d > 0; d >>= 1)
            if (first[s + d] <= tile) s += d;
        s = uniform(s);
        const Asking a = asking(p, s);
        const int tile_key = (tile - uniform(first[s])) * X::kTile, key0 = tile_key + wave * X::kKeys, prefix = a.prefix();
        // the keys
        Frag keys[KB][STEPS];
        bool there[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int key = key0 + b * 16 + col;
            int page = -1, column = 0;
            if (key < a.length) {
                column = static_cast<int>(p.span.page.quotient(key));
                const int32_t entry = p.pages[static_cast<int64_t>(s) * p.span.P + column];
                page = p.span.is_page(entry) ? entry : -1;
            }
            there[b] = page >= 0;
            const char* const from = p.k + max(page, 0) * p.kp + (key - column * static_cast<int>(p.span.page.d)) * p.kt + head * p.kh + quad * 16;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                u32x4 x = {0, 0, 0, 0};
                if (there[b] && (i * 4 + quad) * 16 < p.D * X::kSize) x = *reinterpret_cast<const u32x4*>(from + i * 64);
                keys[b][i] = __builtin_bit_cast(Frag, x);
            }
        }
        float sums[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) sums[b] = 0.0f;

        const int G = static_cast<int>(p.G.d), rows = a.count * G, blocks = (rows + 15) / 16;
        const int each = (blocks + p.splits - 1) / p.splits, end = min(blocks, (split + 1) * each);
        int begin = split * each;
        uint32_t* const sees = reinterpret_cast<uint32_t*>(tree);
        if (p.parents) {
            int16_t* const up = reinterpret_cast<int16_t*>(sees + p.N * (X::kTile / 32));
            __syncthreads();
            if (tile_key + X::kTile > prefix) {
                for (int i = tid; i < a.count; i += kThreads) {
                    const int32_t parent = p.parents[static_cast<int64_t>(s) * p.N + i];
                    up[i] = static_cast<int16_t>(parent >= 0 && parent < i ? parent : -1);
                    for (int w = 0; w < X::kTile / 32; ++w) sees[i * (X::kTile / 32) + w] = 0;
                }
                __syncthreads();
                for (int i = tid; i < a.count; i += kThreads)
                    for (int at = i; at >= 0; at = up[at]) {
                        const int bit = prefix + at - tile_key;
                        if (bit >= 0 && bit < X::kTile) sees[i * (X::kTile / 32) + bit / 32] |= 1u << (bit & 31);
                    }
            }
        } else {
            // rows of tokens ahead of the tile's first key see none of it
            begin = max(begin, max(0, tile_key - prefix) * G / 16);
        }
        const bool masked = key0 + X::kKeys > prefix;  // some of the wavefront's keys ask themselves
        const char* const q0 = p.q + s * p.qs + static_cast<int64_t>(head) * G * p.qh + quad * 16;
        for (int chunk = begin; chunk < end; chunk += kChunk) {
            __syncthreads();
            {
                const int r = chunk * 16 + tid, token = static_cast<int>(p.G.quotient(min(r, rows - 1))), g = r - token * G;
                const bool live = r < rows;
                float l = -kInf;
                if (live) l = p.lse[(static_cast<int64_t>(s) * p.N + token) * p.H + head * G + g];
                row_lse[tid] = l == -kInf ? l : -l * kLog2e;
                row_at[tid] = live ? token * p.qn + g * p.qh : -1;
                row_token[tid] = live ? token : -1;
            }
            __syncthreads();
            const int n = min(kChunk, end - chunk);
            Frag next[STEPS];
            const auto fetch = [&](int b) {
                const int64_t at = row_at[b * 16 + col];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    u32x4 x = {0, 0, 0, 0};
                    if (at >= 0 && (i * 4 + quad) * 16 < p.D * X::kSize) x = *reinterpret_cast<const u32x4*>(q0 + at + i * 64);
                    next[i] = __builtin_bit_cast(Frag, x);
                }
            };
            fetch(0);
            for (int b = 0; b < n; ++b) {
                Frag query[STEPS];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) query[i] = next[i];
                if (b + 1 < n) fetch(b + 1);
                const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_lse[b * 16 + quad * 4]);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) score = E::mma(query[i], keys[kb][i], score);
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i], p.scale, lse[i]));
                    if (masked) {
                        const int asks = key0 + kb * 16 + col - prefix;  // the asking token that the key is
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int token = row_token[b * 16 + quad * 4 + i];
                            bool visible = asks <= token;
                            if (p.parents && asks >= 0) {
                                const int bit = asks + prefix - tile_key;
                                visible = token >= 0 && (sees[token * (X::kTile / 32) + bit / 32] >> (bit & 31) & 1);
                            }
                            w[i] = visible ? w[i] : 0.0f;
                        }
                    }
                    sums[kb] += (w[0] + w[1]) + (w[2] + w[3]);
                }
            }
        }
        // the four lanes of a key
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            sums[b] += __shfl_xor(sums[b], 16);
            sums[b] += __shfl_xor(sums[b], 32);
            const int key = key0 + b * 16 + col;
            if (quad != b % 4 || !there[b]) continue;
            if (p.splits > 1) {
                p.partial[((static_cast<int64_t>(split) * p.S + s) * p.Hkv + head) * p.places + key] = sums[b];
            } else {
                float* const to = p.weights + s * p.ws + head * p.wh + key;
                *to = key < prefix ? *to + sums[b] : sums[b];
            }
        }
    }
}

// x: places of sequence z, head y.
__global__ __launch_bounds__(kJoinThreads) void weigh_join(const Weigh p) {
    const int s = blockIdx.z, head = blockIdx.y, key = blockIdx.x * kJoinThreads + threadIdx.x;
    const Asking a = asking(p, s);
    if (a.count == 0 || key >= a.length ||
        !p.span.is_page(p.pages[static_cast<int64_t>(s) * p.span.P + p.span.page.quotient(key)]))
        return;
    float* const to = p.weights + s * p.ws + head * p.wh + key;
    float sum = key < a.prefix() ? *to : 0.0f;
    for (int i = 0; i < p.splits; ++i) sum += p.partial[((static_cast<int64_t>(i) * p.S + s) * p.Hkv + head) * p.places + key];
    *to = sum;
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

struct Form {
    int tile;
    const void* kernel;
};
template <int DTYPE>
Form form_of(int dim) {
    switch ((dim + 63) / 64) {
        case 1: return {Dims<DTYPE, 64>::kTile, reinterpret_cast<const void*>(weigh_kernel<DTYPE, 64>)};
        case 2: return {Dims<DTYPE, 128>::kTile, reinterpret_cast<const void*>(weigh_kernel<DTYPE, 128>)};
        case 3: return {Dims<DTYPE, 192>::kTile, reinterpret_cast<const void*>(weigh_kernel<DTYPE, 192>)};
        default: return {Dims<DTYPE, 256>::kTile, reinterpret_cast<const void*>(weigh_kernel<DTYPE, 256>)};
    }
}
Form form_of(const BeamgradWeights& a) {
    switch (a.data_type) {
        case DBS_CUDA_DTYPE_F32: return form_of<DBS_CUDA_DTYPE_F32>(a.head_dim);
        case DBS_CUDA_DTYPE_F16: return form_of<DBS_CUDA_DTYPE_F16>(a.head_dim);
        default: return form_of<DBS_CUDA_DTYPE_BF16>(a.head_dim);
    }
}

int64_t places_of(const BeamgradWeights& a) { return static_cast<int64_t>(a.table_pages) * a.page_tokens; }

// Many rows over few keys: the rows are split, into eight blocks of 16 at least, so
// that the card's workgroups have an item each.
int splits_of(const BeamgradWeights& a, int tile) {
    constexpr int64_t kWanted = 1024, kLeast = 8;
    const int64_t sequences = std::min<int64_t>(a.sequences, kSequences);
    const int64_t items = sequences * a.kv_heads * ((places_of(a) + tile - 1) / tile);
    const int64_t blocks = (static_cast<int64_t>(a.tokens) * (a.heads / a.kv_heads) + 15) / 16;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(kWanted + items - 1) / items, blocks / kLeast, kMaxSplits})));
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_accumulate_weights_workspace_size(const BeamgradWeights* args) {
    if (!valid_sizes(args)) return -1;
    const int splits = splits_of(*args, form_of(*args).tile);
    return splits == 1 ? 0
                       : static_cast<int64_t>(splits) * std::min(args->sequences, kSequences) * args->kv_heads * places_of(*args) *
                             static_cast<int64_t>(sizeof(float));
}

DBS_CUDA_EXPORT int beamgrad_accumulate_weights(const BeamgradWeights* args, void* workspace, int64_t workspace_bytes,
                                                void* stream_ptr) {
    if (!valid_sizes(args)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const BeamgradWeights& a = *args;
    const int64_t bytes = beamgrad_accumulate_weights_workspace_size(args);
    if (!a.q || !a.k || !a.pages || !a.lengths || !a.lse || !a.weights || !aligned16(a.q) || !aligned16(a.k) || bytes < 0 ||
        (bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < bytes)))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const Form form = form_of(a);
    const int64_t size = element_size(a.data_type);
    Weigh p{};
    p.qs = a.q_strides[0] * size, p.qn = a.q_strides[1] * size, p.qh = a.q_strides[2] * size;
    p.kp = a.k_strides[0] * size, p.kt = a.k_strides[1] * size, p.kh = a.k_strides[2] * size;
    p.k = static_cast<const char*>(a.k);
    p.ws = a.weight_strides[0], p.wh = a.weight_strides[1];
    p.span = {Divider::of(static_cast<uint32_t>(a.page_tokens)), a.n_pages, a.table_pages};
    p.partial = static_cast<float*>(workspace);
    p.places = places_of(a);
    p.N = a.tokens, p.H = a.heads, p.Hkv = a.kv_heads, p.D = a.head_dim;
    p.splits = splits_of(a, form.tile);
    p.G = Divider::of(static_cast<uint32_t>(a.heads / a.kv_heads));
    p.scale = a.scale * kLog2e;
    const size_t lds = a.parents ? static_cast<size_t>(a.tokens) * (form.tile / 32 * sizeof(uint32_t) + sizeof(int16_t)) : 0;
    // tiles of a launch in 31 bits, whatever the lengths
    const int64_t tiles = (p.places + form.tile - 1) / form.tile;
    const int batch = static_cast<int>(std::min<int64_t>(kSequences, std::max<int64_t>(1, INT32_MAX / tiles)));
    int device = 0, cus = 256, resident = 4;
    if (hipGetDevice(&device) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) (void)hipGetLastError();
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = hipSuccess;
    for (int s0 = 0; s0 < a.sequences && e == hipSuccess; s0 += batch) {
        p.S = std::min(batch, a.sequences - s0);
        p.q = static_cast<const char*>(a.q) + s0 * p.qs;
        p.pages = a.pages + static_cast<int64_t>(s0) * a.table_pages;
        p.lengths = a.lengths + s0;
        p.counts = a.counts ? a.counts + s0 : nullptr;
        p.parents = a.parents ? a.parents + static_cast<int64_t>(s0) * a.tokens : nullptr;
        p.lse = a.lse + static_cast<int64_t>(s0) * a.tokens * a.heads;
        p.weights = a.weights + s0 * p.ws;
        const double most = static_cast<double>(p.S) * p.Hkv * p.splits * static_cast<double>(tiles);
        const unsigned grid = static_cast<unsigned>(std::min<double>(most, static_cast<double>(cus) * resident));
        void* arguments[] = {&p};
        e = hipLaunchKernel(form.kernel, dim3(grid), dim3(kThreads), arguments, lds, stream);
        if (e == hipSuccess && p.splits > 1) {
            weigh_join<<<dim3(static_cast<unsigned>((p.places + kJoinThreads - 1) / kJoinThreads), static_cast<unsigned>(p.Hkv), static_cast<unsigned>(p.S)),
                         kJoinThreads, 0, stream>>>(p);
            e = hipGetLastError();
        }
    }
    return finish_call(stream, e);
}

}  // extern "C"
