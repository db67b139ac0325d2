// SPDX-License-Identifier: MIT
//
// Dense states of a search (recurrent states, caches without pages) brought
// into the order of its new beams, and the gradient of that
// (include/beamgrad_state.h). Copies: bound by HBM, so every row is written
// once and every row that a beam continues is read once (again only from L2).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "beamgrad_state.h"
#include "engine.hpp"
#include "paged.hpp"
#include "regions.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kStatesOfLaunch = 64;   // whose addresses one launch's arguments hold
constexpr int kMaxBeams = 4096;
constexpr int kTileBytes = 16 * 1024; // of LDS, for a tile of an example's rows: eight workgroups a CU
constexpr int kMostTileBytes = 64 * 1024;
constexpr int kAtOnce = 4;            // 16-byte reads of a thread in flight

// States of one row length.
struct StateSet {
    const char* from[kStatesOfLaunch];
    char* to[kStatesOfLaunch];
    int64_t row_bytes;
    int32_t n;
};

// x: 16-byte chunks of the rows of example y of state z, one after the other. A
// training step's 12 states of 8 KB rows, 8 examples of 5 beams: 5 us, latency.
__global__ __launch_bounds__(kThreads) void reorder_kernel(const StateSet set, const void* parents, const bool i64,
                                                           const int K, const Divider chunks) {
    const char* const from = set.from[blockIdx.z] + static_cast<int64_t>(blockIdx.y) * K * set.row_bytes;
    char* const to = set.to[blockIdx.z] + static_cast<int64_t>(blockIdx.y) * K * set.row_bytes;
    u32x4 x[kAtOnce];
    char* out[kAtOnce];
    int64_t left[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
        const int64_t at = (static_cast<int64_t>(blockIdx.x) * kAtOnce + i) * kThreads + threadIdx.x;
        out[i] = nullptr;
        if (at >= static_cast<int64_t>(K) * chunks.d) continue;
        const int64_t k = chunks.quotient(static_cast<uint32_t>(at));
        const int64_t byte = (at - k * chunks.d) * 16;
        const int p = parent_of(parents, i64, static_cast<int64_t>(blockIdx.y) * K + k, K);
        left[i] = set.row_bytes - byte;
        out[i] = to + k * set.row_bytes + byte;
        x[i] = p < 0 ? u32x4{0, 0, 0, 0} : load16(from + p * set.row_bytes + byte, left[i]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
        if (out[i]) store16(out[i], x[i], left[i]);
}

// In place: a workgroup takes `width` bytes of every row of example y of state
// z, reads those that move into LDS, and writes them where they go. Rows that
// stay are neither read nor written, unless another continues them too.
// With tiles of 16 KB all of a thread's reads are in flight together, and eight
// workgroups fit a CU: 16 examples of 8 beams, 24 states of 64 KB rows in 75 us,
// 4.1 TB/s (100 us with 64 KB of LDS a workgroup).
__global__ __launch_bounds__(kThreads) void reorder_inplace(const StateSet set, const void* parents, const bool i64,
                                                            const int K, const Divider chunks) {
    extern __shared__ u32x4 tile[];  // K rows of the tile, then the two arrays below
    int16_t* const parent = reinterpret_cast<int16_t*>(tile + K * chunks.d);
    uint8_t* const moves = reinterpret_cast<uint8_t*>(parent + K);  // a row that another one continues
    char* const rows = set.to[blockIdx.z] + static_cast<int64_t>(blockIdx.y) * K * set.row_bytes;
    const int64_t byte0 = static_cast<int64_t>(blockIdx.x) * chunks.d * 16;
    for (int k = threadIdx.x; k < K; k += kThreads) moves[k] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < K; k += kThreads) {
        const int p = parent_of(parents, i64, static_cast<int64_t>(blockIdx.y) * K + k, K);
        parent[k] = static_cast<int16_t>(p);
        if (p >= 0 && p != k) moves[p] = 1;
    }
    __syncthreads();
    const int items = K * static_cast<int>(chunks.d);
    for (int i0 = threadIdx.x; i0 < items; i0 += kThreads * kAtOnce) {
        u32x4 x[kAtOnce];
        bool there[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int i = i0 + j * kThreads, k = static_cast<int>(chunks.quotient(i));
            const int64_t byte = byte0 + (i - k * static_cast<int>(chunks.d)) * 16;
            there[j] = i < items && moves[k] && byte < set.row_bytes;
            if (there[j]) x[j] = load16(rows + k * set.row_bytes + byte, set.row_bytes - byte);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (there[j]) tile[i0 + j * kThreads] = x[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += kThreads) {
        const int k = static_cast<int>(chunks.quotient(i)), c = i - k * static_cast<int>(chunks.d), p = parent[k];
        const int64_t byte = byte0 + c * 16;
        if (p != k && byte < set.row_bytes)
            store16(rows + k * set.row_bytes + byte, p < 0 ? u32x4{0, 0, 0, 0} : tile[p * static_cast<int>(chunks.d) + c], set.row_bytes - byte);
    }
}

// The gradient: x covers the 16-byte chunks of the rows of example y of state
// z; a thread sums its chunk over the rows that continue its row, in 32 bits
// and in their order, so the sum does not depend on the launch.
template <class T>
__global__ __launch_bounds__(kThreads) void reorder_backward(const StateSet set, const void* parents, const bool i64,
                                                             const int K, const Divider chunks) {
    constexpr int kEach = 16 / sizeof(T);
    __shared__ int16_t parent[kMaxBeams];
    for (int k = threadIdx.x; k < K; k += kThreads)
        parent[k] = static_cast<int16_t>(parent_of(parents, i64, static_cast<int64_t>(blockIdx.y) * K + k, K));
    __syncthreads();
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (at >= static_cast<int64_t>(K) * chunks.d) return;
    const int64_t row = chunks.quotient(static_cast<uint32_t>(at));
    const int64_t byte = (at - row * chunks.d) * 16, left = set.row_bytes - byte;
    const char* const from = set.from[blockIdx.z] + static_cast<int64_t>(blockIdx.y) * K * set.row_bytes + byte;
    float sum[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum[e] = 0.0f;
    for (int k = 0; k < K; ++k) {
        if (parent[k] != row) continue;
        const u32x4 x = load16(from + k * set.row_bytes, left);
        T v[kEach];
        __builtin_memcpy(v, &x, 16);
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] += static_cast<float>(v[e]);
    }
    T v[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = static_cast<T>(sum[e]);
    u32x4 x;
    __builtin_memcpy(&x, v, 16);
    store16(set.to[blockIdx.z] + (static_cast<int64_t>(blockIdx.y) * K + row) * set.row_bytes + byte, x, left);
}

// The states in sets of one row length, as many as a launch's arguments hold.
template <class Bytes, class Each>
hipError_t over_states(const void* const* from, void* const* to, int n, Bytes bytes, Each each) {
    for (int i = 0; i < n; ++i) {
        bool seen = false;
        for (int j = 0; j < i && !seen; ++j) seen = bytes(j) == bytes(i);
        StateSet set{};
        set.row_bytes = bytes(i);
        for (int j = i; j < n && !seen; ++j) {
            if (bytes(j) == bytes(i)) {
                set.from[set.n] = static_cast<const char*>(from[j]);
                set.to[set.n] = static_cast<char*>(to[j]);
                ++set.n;
            }
            if (set.n == kStatesOfLaunch || (j + 1 == n && set.n > 0)) {
                const hipError_t e = each(set);
                if (e != hipSuccess) return e;
                set.n = 0;
            }
        }
    }
    return hipSuccess;
}

// Examples beyond the 65535 of a grid's y are refused.
bool valid_states(const void* const* from, void* const* to, const int64_t* size, int n, const void* parents, int examples,
                  int beams) {
    if (n < 0 || !parents || examples <= 0 || examples > 65535 || beams <= 0 || beams > kMaxBeams) return false;
    if (n > 0 && (!from || !to || !size)) return false;
    for (int i = 0; i < n; ++i)
        if (!from[i] || !to[i] || size[i] <= 0 || size[i] > INT32_MAX || (size[i] / 4 + 1) * beams > INT32_MAX - 65536) return false;
    return true;
}

// A state that lies where another is written would be moved twice, and in no
// order. `bytes(i)`: of a row.
template <class Bytes>
bool lie_apart(const void* const* from, void* const* to, int n, Bytes bytes, int examples, int beams, bool inplace) {
    const auto whole = [&](const void* base, int i) {
        return Region{reinterpret_cast<uintptr_t>(base), {1, 1}, {0, 0}, bytes(i) * beams * examples};
    };
    return all_apart(n, [&](int i) { return whole(to[i], i); }, inplace ? 0 : n, [&](int i) { return whole(from[i], i); });
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int beamgrad_reorder_states(const void* const* from, void* const* to, const int64_t* row_bytes, int n,
                                            const void* parents, int parents_i64, int examples, int beams,
                                            void* stream_ptr) {
    if (!valid_states(from, to, row_bytes, n, parents, examples, beams)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    bool inplace = n > 0 && from[0] == to[0];
    for (int i = 0; i < n; ++i)
        if ((from[i] == to[i]) != inplace) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!lie_apart(from, to, n, [&](int i) { return row_bytes[i]; }, examples, beams, inplace)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const hipError_t e = over_states(from, to, n, [&](int i) { return row_bytes[i]; }, [&](const StateSet& set) {
        const int64_t chunks = (set.row_bytes + 15) / 16;
        const unsigned y = static_cast<unsigned>(examples), z = static_cast<unsigned>(set.n);
        if (inplace) {
            // many beams: narrower pieces of their rows, of 256 bytes while LDS has room
            const int64_t room = std::max<int64_t>(kTileBytes / beams, std::min<int64_t>(kMostTileBytes / beams, 256)) / 16;
            const int64_t of_tile = std::max<int64_t>(1, std::min<int64_t>(chunks, room));
            const size_t lds = static_cast<size_t>(beams) * (static_cast<size_t>(of_tile) * 16 + 3);
            reorder_inplace<<<dim3(static_cast<unsigned>((chunks + of_tile - 1) / of_tile), y, z), kThreads, lds, stream>>>(
                set, parents, parents_i64 != 0, beams, Divider::of(static_cast<uint32_t>(of_tile)));
        } else {
            const int64_t each = kThreads * kAtOnce;
            reorder_kernel<<<dim3(static_cast<unsigned>((beams * chunks + each - 1) / each), y, z), kThreads, 0, stream>>>(
                set, parents, parents_i64 != 0, beams, Divider::of(static_cast<uint32_t>(chunks)));
        }
        return hipGetLastError();
    });
    return finish_call(stream, e);
}

DBS_CUDA_EXPORT int beamgrad_reorder_states_backward(const void* const* from, void* const* to, const int64_t* elements,
                                                     int n, int data_type, const void* parents, int parents_i64,
                                                     int examples, int beams, void* stream_ptr) {
    if (!valid_states(from, to, elements, n, parents, examples, beams) ||
        (data_type != DBS_CUDA_DTYPE_F32 && data_type != DBS_CUDA_DTYPE_F16 && data_type != DBS_CUDA_DTYPE_BF16))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int size = data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2;
    if (!lie_apart(from, to, n, [&](int i) { return elements[i] * size; }, examples, beams, false)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    const hipError_t e = over_states(from, to, n, [&](int i) { return elements[i] * size; }, [&](const StateSet& set) {
        const int64_t chunks = (set.row_bytes + 15) / 16;
        const dim3 grid(static_cast<unsigned>((beams * chunks + kThreads - 1) / kThreads), static_cast<unsigned>(examples),
                        static_cast<unsigned>(set.n));
        const auto launch = [&](auto* kernel) {
            kernel<<<grid, kThreads, 0, stream>>>(set, parents, parents_i64 != 0, beams, Divider::of(static_cast<uint32_t>(chunks)));
        };
        if (data_type == DBS_CUDA_DTYPE_F32)
            launch(reorder_backward<float>);
        else if (data_type == DBS_CUDA_DTYPE_F16)
            launch(reorder_backward<_Float16>);
        else
            launch(reorder_backward<__bf16>);
        return hipGetLastError();
    });
    return finish_call(stream, e);
}

}  // extern "C"
