// SPDX-License-Identifier: MIT
//
// Rotary positions of queries and keys, and their gradient, which is the same
// with the angles' signs changed (include/beamgrad_state.h).
//
// Mathematics. A token's angle position * frequency is a product of 64 bits,
// its rounding error kept, less the nearest multiple of pi / 2 (whose own
// rounding error is kept too): what is left lies within pi / 4 (1.05 at angles of 2^50, whose
// multiple is rounded itself), in 64 bits. Its sine and cosine are 32-bit Taylor sums, with what the argument
// lost in its rounding to 32 bits put back by the other one. They are computed
// once for a token and a tensor, and serve all of its heads.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <iterator>
#include <new>
#include <type_traits>

#include "beamgrad_state.h"
#include "engine.hpp"
#include "paged.hpp"
#include "regions.hpp"
#include "rows.hpp"

using namespace dbs_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;        // of a head
constexpr int64_t kMostTokens = int64_t{1} << 26;      // of a call
constexpr int64_t kTokensOfLaunch = int64_t{1} << 24;  // a launch has fewer than 2^32 threads
constexpr int64_t kMostStride = int64_t{1} << 40;
constexpr int kTensorsOfLaunch = 16;  // whose addresses one launch's arguments hold

struct Heads {
    const char* from;
    char* to;
    int64_t from_stride[3], to_stride[3];  // sequence, token, head, in bytes
    int32_t row_bytes;
    Divider units_of_head, units_of_token;
};

struct Turn {
    Heads of[kTensorsOfLaunch];
    const void* positions;
    const double* frequencies;
    const int32_t* counts;
    int64_t position_stride[2];  // in elements
    Divider tokens, pairs;       // tokens of a sequence, pairs of a head
    int64_t first, all;          // the launch's first token, and the end of its tokens
    float scale;
    bool i64, inverse, inplace;
};

// Cosine and sine of position * frequency.
__device__ __forceinline__ float2 unit_of(double position, double frequency) {
    constexpr double kTwoOverPi = 0.63661977236758134308, kHalfPi = 1.57079632679489661923, kHalfPiRest = 6.12323399573676603587e-17;
    const double a = position * frequency, rest = __builtin_fma(position, frequency, -a);
    const double k = __builtin_rint(a * kTwoOverPi);
    const double r = __builtin_fma(-k, kHalfPiRest, __builtin_fma(-k, kHalfPi, a)) + rest;
    const int quadrant = static_cast<int>(k - 4.0 * __builtin_floor(k * 0.25));
    const float x = static_cast<float>(r), low = static_cast<float>(r - static_cast<double>(x)), y = x * x;
    float s = __builtin_fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = __builtin_fmaf(y, s, 1.0f / 120.0f);
    s = __builtin_fmaf(y, s, -1.0f / 6.0f);
    s = __builtin_fmaf(x * y, s, x);
    float c = __builtin_fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = __builtin_fmaf(y, c, -1.0f / 720.0f);
    c = __builtin_fmaf(y, c, 1.0f / 24.0f);
    c = __builtin_fmaf(y, c, -0.5f);
    c = __builtin_fmaf(y, c, 1.0f);
    const float sine = __builtin_fmaf(low, c, s), cosine = __builtin_fmaf(-low, s, c);
    const float u = quadrant & 1 ? sine : cosine, v = quadrant & 1 ? cosine : sine;
    return {quadrant == 1 || quadrant == 2 ? -u : u, quadrant >= 2 ? -v : v};
}

// A value of n elements of T at any address.
template <class T, int N>
struct Run {
    T x[N];
};
template <class T, int N>
__device__ __forceinline__ Run<T, N> load_run(const char* from) {
    typedef typename std::conditional<sizeof(T) * N == 32, uint32_t __attribute__((ext_vector_type(8))),
        typename std::conditional<sizeof(T) * N == 16, u32x4, typename std::conditional<sizeof(T) * N == 8, uint64_t,
        typename std::conditional<sizeof(T) * N == 4, uint32_t, uint16_t>::type>::type>::type>::type W;
    const W w = *reinterpret_cast<const typename Unaligned<W>::type*>(from);
    Run<T, N> r;
    __builtin_memcpy(&r, &w, sizeof(w));
    return r;
}
template <class T, int N>
__device__ __forceinline__ void store_run(char* to, const Run<T, N>& r) {
    typedef typename std::conditional<sizeof(T) * N == 32, uint32_t __attribute__((ext_vector_type(8))),
        typename std::conditional<sizeof(T) * N == 16, u32x4, typename std::conditional<sizeof(T) * N == 8, uint64_t,
        typename std::conditional<sizeof(T) * N == 4, uint32_t, uint16_t>::type>::type>::type>::type W;
    W w;
    __builtin_memcpy(&w, &r, sizeof(w));
    *reinterpret_cast<typename Unaligned<W>::type*>(to) = w;
}

// x: TOKENS tokens; y: a tensor. A thread has PAIRS pairs of a head, or 16 bytes
// behind what turns. The table of a token's angles costs some 60 operations for each pair, of
// 64 bits most of them, and is made once for all heads of a tensor; beside it the
// kernel is bound by HBM: queries and keys of 16384 tokens, 40 heads of 128 in bfloat16,
// in 62 us, 5.4 TB/s. 32 tokens: 3.7 us, a launch and two dependent reads. PAIRS divides the pairs of a head,
// so an odd number of them goes pair by pair: 63 of 64 pairs turned of those queries and keys, the last two
// values copied, 201 us (in place 91); 62 of 64, two at once, 127 (61).
template <class T, int PAIRS, bool INTERLEAVED, int TOKENS>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const Turn p) {
    extern __shared__ float2 units[];  // [TOKENS][pairs]
    __shared__ bool live[TOKENS];
    const Heads& h = p.of[blockIdx.y];
    const int64_t first = p.first + static_cast<int64_t>(blockIdx.x) * TOKENS;
    const int here = static_cast<int>(min(p.all - first, static_cast<int64_t>(TOKENS))), pairs = p.pairs.d;
    const auto place = [&](int t, int64_t& s) {
        const uint32_t token = static_cast<uint32_t>(first + t), of = p.tokens.quotient(token);
        s = of;
        return static_cast<int64_t>(token - of * p.tokens.d);
    };
    for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
        const int t = p.pairs.quotient(i), f = i - t * pairs;
        int64_t s;
        const int64_t n = place(t, s);
        const bool lives = !p.counts || n < p.counts[s];
        if (f == 0) live[t] = lives;
        if (!lives) continue;
        const int64_t at = s * p.position_stride[0] + n * p.position_stride[1];
        const double position = p.i64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                      : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
        const float2 u = unit_of(position, p.frequencies[f]);
        units[i] = {u.x * p.scale, (p.inverse ? -u.y : u.y) * p.scale};
    }
    __syncthreads();
    const int items = here * static_cast<int>(h.units_of_token.d);
    const int turning = pairs / PAIRS;
    for (int i = threadIdx.x; i < items; i += kThreads) {
        const int t = h.units_of_token.quotient(i), in_token = i - t * static_cast<int>(h.units_of_token.d);
        const int head = h.units_of_head.quotient(in_token), unit = in_token - head * static_cast<int>(h.units_of_head.d);
        int64_t s;
        const int64_t n = place(t, s);
        const char* const from = h.from + s * h.from_stride[0] + n * h.from_stride[1] + head * h.from_stride[2];
        char* const to = h.to + s * h.to_stride[0] + n * h.to_stride[1] + head * h.to_stride[2];
        const bool lives = live[t];
        if (!lives && p.inplace) continue;
        if (unit >= turning) {
            const int byte = 2 * pairs * static_cast<int>(sizeof(T)) + (unit - turning) * 16, left = h.row_bytes - byte;
            store16(to + byte, lives ? load16(from + byte, left) : u32x4{0, 0, 0, 0}, left);
            continue;
        }
        const float2* const u = units + t * pairs + unit * PAIRS;
        if constexpr (INTERLEAVED) {
            const int byte = 2 * unit * PAIRS * static_cast<int>(sizeof(T));
            Run<T, 2 * PAIRS> x{};
            if (lives) x = load_run<T, 2 * PAIRS>(from + byte);
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                if (!lives) break;
                const float a = static_cast<float>(x.x[2 * j]), b = static_cast<float>(x.x[2 * j + 1]);
                x.x[2 * j] = static_cast<T>(__builtin_fmaf(a, u[j].x, -(b * u[j].y)));
                x.x[2 * j + 1] = static_cast<T>(__builtin_fmaf(a, u[j].y, b * u[j].x));
            }
            store_run<T, 2 * PAIRS>(to + byte, x);
        } else {
            const int byte = unit * PAIRS * static_cast<int>(sizeof(T)), half = pairs * static_cast<int>(sizeof(T));
            Run<T, PAIRS> x{}, y{};
            if (lives) {
                x = load_run<T, PAIRS>(from + byte);
                y = load_run<T, PAIRS>(from + half + byte);
            }
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                if (!lives) break;
                const float a = static_cast<float>(x.x[j]), b = static_cast<float>(y.x[j]);
                x.x[j] = static_cast<T>(__builtin_fmaf(a, u[j].x, -(b * u[j].y)));
                y.x[j] = static_cast<T>(__builtin_fmaf(a, u[j].y, b * u[j].x));
            }
            store_run<T, PAIRS>(to + byte, x);
            store_run<T, PAIRS>(to + half + byte, y);
        }
    }
}

// ---------------------------------------------------------------------------
// Checks and launches
// ---------------------------------------------------------------------------

int element_size(int data_type) { return data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2; }

// The heads that are written of tensor i. Sequences, tokens and heads lie in whatever order: a step that
// continues the one within it is one with it. Where all three are left, what lies between
// the rows of the innermost counts as written. False: these rows meet, or reach further than addresses do.
bool region_of(const BeamgradRotary& a, int i, Region& r) {
    struct Dim {
        int64_t n, stride;
        bool operator<(const Dim& other) const { return stride < other.stride; }
    };
    const int64_t size = element_size(a.data_type), *st = a.to_strides + 3 * i;
    Dim all[] = {{a.sequences, st[0] * size}, {a.tokens, st[1] * size}, {a.heads[i], st[2] * size}}, left[3];
    std::sort(std::begin(all), std::end(all));
    int64_t run = a.head_dim[i] * size, next = run;  // next: where what lies innermost would go on
    int levels = 0;
    for (const Dim& d : all) {
        if (d.n == 1) continue;
        if (d.stride != next) {
            left[levels++] = d;
        } else if (levels > 0) {
            left[levels - 1].n *= d.n;
        }
        if (__builtin_mul_overflow(d.n, d.stride, &next)) return false;
        if (levels == 0) run = next;
    }
    if (levels == 3) {
        if (left[0].stride < run) return false;
        run += (left[0].n - 1) * left[0].stride;
        left[0] = left[1], left[1] = left[2], levels = 2;
    }
    r = {reinterpret_cast<uintptr_t>(a.to[i]), {1, 1}, {0, 0}, run};
    for (int d = 0; d < levels; ++d) {
        r.n[1 - d] = left[d].n;
        r.stride[1 - d] = left[d].stride;
    }
    return true;
}

bool valid(const BeamgradRotary* a) {
    if (!a || a->reserved != 0 || a->sequences <= 0 || a->tokens <= 0 || a->pairs <= 0 || a->n < 0 ||
        static_cast<int64_t>(a->sequences) * a->tokens >= kMostTokens)
        return false;
    if (a->data_type != DBS_CUDA_DTYPE_F32 && a->data_type != DBS_CUDA_DTYPE_F16 && a->data_type != DBS_CUDA_DTYPE_BF16) return false;
    if (!a->positions || !a->frequencies || (a->n > 0 && (!a->from || !a->to || !a->heads || !a->head_dim || !a->from_strides || !a->to_strides)))
        return false;
    for (int i = 0; i < a->n; ++i) {
        if (!a->from[i] || !a->to[i] || a->heads[i] <= 0 || a->heads[i] > 1 << 16 || a->head_dim[i] > kMaxDim ||
            a->head_dim[i] < 2 * static_cast<int64_t>(a->pairs))
            return false;
        for (int d = 0; d < 3; ++d)
            if (a->from_strides[3 * i + d] < 0 || a->to_strides[3 * i + d] < 0 || a->from_strides[3 * i + d] > kMostStride ||
                a->to_strides[3 * i + d] > kMostStride)
                return false;
        if ((a->from[i] == a->to[i]) != (a->from[0] == a->to[0])) return false;
        if (a->from[i] == a->to[i])
            for (int d = 0; d < 3; ++d)
                if (a->from_strides[3 * i + d] != a->to_strides[3 * i + d]) return false;
    }
    return true;
}

// What is written lies apart, and in what is read only where it is the same.
bool lie_apart(const BeamgradRotary& a) {
    const bool inplace = a.from[0] == a.to[0];
    Region r;
    for (int i = 0; i < a.n; ++i)
        if (!region_of(a, i, r)) return false;
    const auto written = [&](int i) {
        Region to;
        region_of(a, i, to);
        return to;
    };
    const auto read = [&](int i) {
        const int64_t size = element_size(a.data_type), *st = a.from_strides + 3 * i;
        return Region{reinterpret_cast<uintptr_t>(a.from[i]), {a.sequences, a.tokens}, {st[0] * size, st[1] * size},
                      ((a.heads[i] - 1) * st[2] + a.head_dim[i]) * size};
    };
    return all_apart(a.n, written, inplace ? 0 : a.n, read);
}

template <class T, int PAIRS, bool INTERLEAVED>
void launch(Turn& p, int tensors, hipStream_t stream) {
    // Two tokens a workgroup give every thread work between the table and the end, one
    // gives few tokens more workgroups. 2103 tokens of 20 heads of 72, float32: 9.5 us with
    // one, 7.9 with two, 9.6 with four; 16384 of 40 heads of 128, bfloat16: 62 with two or four.
    constexpr int64_t many = 512;
    const size_t table = p.pairs.d * sizeof(float2);
    const int64_t all = p.all;
    for (p.first = 0; p.first < all; p.first += kTokensOfLaunch) {
        p.all = std::min(all, p.first + kTokensOfLaunch);
        const int64_t here = p.all - p.first;
        if (all >= many)
            rotary_kernel<T, PAIRS, INTERLEAVED, 2><<<dim3(static_cast<unsigned>((here + 1) / 2), tensors), kThreads, 2 * table, stream>>>(p);
        else
            rotary_kernel<T, PAIRS, INTERLEAVED, 1><<<dim3(static_cast<unsigned>(here), tensors), kThreads, table, stream>>>(p);
    }
    p.all = all;
}

template <class T, int PAIRS>
void launch_layout(Turn& p, bool interleaved, int tensors, hipStream_t stream) {
    if (interleaved)
        launch<T, PAIRS, true>(p, tensors, stream);
    else
        launch<T, PAIRS, false>(p, tensors, stream);
}

template <class T>
void launch_pairs(Turn& p, int each, bool interleaved, int tensors, hipStream_t stream) {
    if (each == 8) {
        if constexpr (sizeof(T) == 2) launch_layout<T, 8>(p, interleaved, tensors, stream);
    } else if (each == 4) {
        launch_layout<T, 4>(p, interleaved, tensors, stream);
    } else if (each == 2) {
        launch_layout<T, 2>(p, interleaved, tensors, stream);
    } else {
        launch_layout<T, 1>(p, interleaved, tensors, stream);
    }
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int beamgrad_rotary(const BeamgradRotary* args, void* stream_ptr) try {
    if (!valid(args) || (args->n > 0 && !lie_apart(*args))) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const BeamgradRotary& a = *args;
    const int size = element_size(a.data_type);
    Turn p{};
    p.positions = a.positions;
    p.frequencies = a.frequencies;
    p.counts = a.counts;
    p.position_stride[0] = a.position_strides[0], p.position_stride[1] = a.position_strides[1];
    p.tokens = Divider::of(static_cast<uint32_t>(a.tokens));
    p.pairs = Divider::of(static_cast<uint32_t>(a.pairs));
    p.all = static_cast<int64_t>(a.sequences) * a.tokens;
    p.scale = a.scale;
    p.i64 = a.positions_i64 != 0;
    p.inverse = a.inverse != 0;
    p.inplace = a.n > 0 && a.from[0] == a.to[0];
    // 16 bytes of each of a pair's sides, or as much as divides them
    int each = 16 / size;
    while (a.pairs % each != 0) each /= 2;
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = hipSuccess;
    for (int first = 0; first < a.n && e == hipSuccess; first += kTensorsOfLaunch) {
        const int n = std::min(kTensorsOfLaunch, a.n - first);
        for (int j = 0; j < n; ++j) {
            const int i = first + j;
            Heads& h = p.of[j];
            h.from = static_cast<const char*>(a.from[i]);
            h.to = static_cast<char*>(a.to[i]);
            for (int d = 0; d < 3; ++d) {
                h.from_stride[d] = a.from_strides[3 * i + d] * size;
                h.to_stride[d] = a.to_strides[3 * i + d] * size;
            }
            h.row_bytes = a.head_dim[i] * size;
            const int copied = p.inplace ? 0 : ((a.head_dim[i] - 2 * a.pairs) * size + 15) / 16;
            const uint32_t units = static_cast<uint32_t>(a.pairs / each + copied);
            h.units_of_head = Divider::of(units);
            h.units_of_token = Divider::of(units * static_cast<uint32_t>(a.heads[i]));
        }
        if (a.data_type == DBS_CUDA_DTYPE_F32)
            launch_pairs<float>(p, each, a.interleaved != 0, n, stream);
        else if (a.data_type == DBS_CUDA_DTYPE_F16)
            launch_pairs<_Float16>(p, each, a.interleaved != 0, n, stream);
        else
            launch_pairs<__bf16>(p, each, a.interleaved != 0, n, stream);
        e = hipGetLastError();
    }
    return finish_call(stream, e);
} catch (const std::bad_alloc&) {
    return DBS_CUDA_STATUS_OUT_OF_MEMORY;
}

}  // extern "C"
