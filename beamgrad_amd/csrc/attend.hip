// SPDX-License-Identifier: MIT
//
// The C entry of attention over a paged cache (include/beamgrad_state.h):
// checks, the choice of a kernel, its workspace.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "attend.hpp"
#include "beamgrad_state.h"
#include "engine.hpp"

using namespace dbs_hip;

namespace {

bool multiple16(int64_t stride, int64_t size) { return stride >= 0 && stride * size % 16 == 0; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Sizes, strides and what the kernels take for granted.
bool valid_sizes(const BeamgradAttention* a) {
    if (!a || a->reserved != 0) return false;
    if (a->data_type != DBS_CUDA_DTYPE_F32 && a->data_type != DBS_CUDA_DTYPE_F16 && a->data_type != DBS_CUDA_DTYPE_BF16)
        return false;
    if (a->sequences <= 0 || a->tokens <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->beams <= 0 || a->page_tokens <= 0 ||
        a->n_pages <= 0 || a->table_pages <= 0)
        return false;
    if (a->head_dim <= 0 || a->head_dim > kAttendMaxDim || a->head_dim % 8 != 0) return false;
    if (a->heads % a->kv_heads != 0 || a->sequences % a->beams != 0) return false;
    if (a->parents && a->tokens > kAttendMaxTree) return false;
    if (!std::isfinite(a->scale * 1.44269504088896341f) || !(a->scale > 0.0f)) return false;
    // places of a sequence's tokens, rows of a group and of the call in 31 bits
    if ((static_cast<int64_t>(a->table_pages) + 1) * a->page_tokens > INT32_MAX - 65536) return false;
    if (static_cast<double>(a->tokens) * a->heads * a->beams > 1.0e9) return false;
    if (static_cast<double>(a->tokens) * a->heads * a->sequences > 2.0e9) return false;
    const int64_t size = a->data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2;
    for (int i = 0; i < 3; ++i)
        // (a page's stride in 16 bytes has 32 bits)
        if (a->k_strides[i] > (int64_t{1} << 33) || a->v_strides[i] > (int64_t{1} << 33) || !multiple16(a->q_strides[i], size) || !multiple16(a->k_strides[i], size) || !multiple16(a->v_strides[i], size))
            return false;
    return true;
}

struct Plan {
    int dim, shape;
    AttendSizes sizes;
    int batch;  // sequences of a launch
    int64_t info_bytes, bytes;  // bytes < 0: more items than a launch has
};

int multiprocessors() {
    int device = 0, cus = 0;
    if (hipGetDevice(&device) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0) {
        (void)hipGetLastError();
        return 256;
    }
    return cus;
}

int64_t tiles_of(int64_t rows, int tile) { return (rows + tile - 1) / tile; }

// Items of a launch: a workgroup of 256 threads each, of which HIP takes 2^32.
constexpr int64_t kMostItems = (int64_t{1} << 24) - 1;
// Partial results of a launch whose sequences share pages, where that is more than
// one group's. 256 MB are 4000 tiles of 128 rows and 128 columns, several for each
// workgroup of the card, so that a further launch costs little beside them.
constexpr int64_t kPartialBytes = int64_t{256} << 20;

Plan plan_of(const BeamgradAttention& a, AttendParams& p) {
    Plan plan;
    plan.dim = (a.head_dim + 63) / 64 * 64;
    p.N = a.tokens;
    p.H = a.heads;
    p.Hkv = a.kv_heads;
    p.G = Divider::of(static_cast<uint32_t>(a.heads / a.kv_heads));
    p.D = a.head_dim;
    const int64_t rows = static_cast<int64_t>(p.N) * p.G.d;
    p.beam_rows = Divider::of(static_cast<uint32_t>(rows));
    // A group reads its shared pages together where its beams' own tiles would be more
    // than 8/7 of what that takes: beams that fill tiles by themselves gain nothing by
    // it, and leave a partial result for every tile. 8 beams over 16 prompts of 4000, 8 cache
    // heads of 128, bfloat16, us together and apart: 112 rows a beam (7 tiles, 8) 495, 411;
    // 256 rows 1163, 837; 132 rows (9 tiles, 16) 711, 815. At 6/5 of the tiles it is one or
    // the other (0.74 to 1.57 of the time), at 8/7 and below apart is 0.95 to 2.1 times as
    // fast. A group whose lengths one workgroup cannot hold reads them once for each beam.
    const int most = attend_rows(attend_most(a.data_type, plan.dim));
    const bool together = a.shared && a.beams > 1 && a.beams <= kAttendSequences &&
                          7 * a.beams * tiles_of(rows, most) > 8 * tiles_of(rows * a.beams, most);
    p.K = together ? a.beams : 1;
    p.shared = together ? a.shared : nullptr;
    // the smallest tile that takes the rows that read a page together: fewer
    // rows than the tile cost matrix instructions, more read the cache again
    plan.shape = kRows16;
    while (plan.shape < attend_most(a.data_type, plan.dim) && attend_rows(plan.shape) < rows * p.K) ++plan.shape;
    const int tile = attend_rows(plan.shape);
    const int64_t shared_tiles = together ? tiles_of(rows * p.K, tile) : 0, own_tiles = tiles_of(rows, tile);
    p.shared_tiles = static_cast<int>(shared_tiles);
    p.own_tiles = static_cast<int>(own_tiles);
    switch (a.data_type) {
        case DBS_CUDA_DTYPE_F32: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_F32>(plan.dim, plan.shape); break;
        case DBS_CUDA_DTYPE_F16: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_F16>(plan.dim, plan.shape); break;
        default: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_BF16>(plan.dim, plan.shape); break;
    }
    // groups of a launch
    const int64_t slot_bytes = plan.sizes.slot * static_cast<int64_t>(sizeof(float));
    const int64_t group_items = (shared_tiles + p.K * own_tiles) * p.Hkv;
    int64_t groups = std::min<int64_t>(a.sequences, kAttendSequences) / p.K;
    groups = std::min(groups, std::max<int64_t>(1, kMostItems / group_items));
    if (together) groups = std::min(groups, std::max<int64_t>(1, kPartialBytes / (group_items * slot_bytes)));
    // launches of like size
    const int64_t launches = tiles_of(a.sequences / p.K, static_cast<int>(groups));
    groups = tiles_of(a.sequences / p.K, static_cast<int>(launches));
    plan.batch = static_cast<int>(groups) * p.K;
    const int64_t items = groups * group_items;
    if (items > kMostItems) {
        plan.bytes = -1;
        return plan;
    }
    p.head_items = static_cast<int>(items / p.Hkv);
    // units in 30 bits, whatever the lengths
    const double keys = static_cast<double>(a.table_pages) * a.page_tokens;
    p.unit_shift = 0;
    while (static_cast<double>(items) * (std::ldexp(keys / plan.sizes.keys, -p.unit_shift) + 1.0) > 1.0e9) ++p.unit_shift;
    p.grid = (multiprocessors() * plan.sizes.resident + 7) / 8 * 8;
    plan.info_bytes = items * static_cast<int64_t>(sizeof(int4));
    const int64_t slots = together ? p.grid + items : 2 * static_cast<int64_t>(p.grid);
    plan.bytes = plan.info_bytes + slots * slot_bytes;
    return plan;
}

}  // namespace

extern "C" {

DBS_CUDA_EXPORT int64_t beamgrad_tree_attention_workspace_size(const BeamgradAttention* args) {
    if (!valid_sizes(args)) return -1;
    AttendParams p{};
    return plan_of(*args, p).bytes;
}

DBS_CUDA_EXPORT int beamgrad_tree_attention(const BeamgradAttention* args, void* workspace, int64_t workspace_bytes,
                                            void* stream_ptr) {
    if (!valid_sizes(args)) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const BeamgradAttention& a = *args;
    if (!a.q || !a.k || !a.v || !a.pages || !a.lengths || !a.out || !workspace) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) || !aligned16(workspace))
        return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    AttendParams p{};
    const Plan plan = plan_of(a, p);
    if (plan.bytes < 0 || workspace_bytes < plan.bytes) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
    const int64_t size = a.data_type == DBS_CUDA_DTYPE_F32 ? 4 : 2;
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.qs = a.q_strides[0] * size, p.qn = a.q_strides[1] * size, p.qh = a.q_strides[2] * size;
    p.kp = a.k_strides[0] * size, p.kt = a.k_strides[1] * size, p.kh = a.k_strides[2] * size;
    p.vp = a.v_strides[0] * size, p.vt = a.v_strides[1] * size, p.vh = a.v_strides[2] * size;
    p.kp16 = static_cast<uint32_t>(p.kp / 16), p.kt16 = static_cast<uint32_t>(p.kt / 16);
    p.vp16 = static_cast<uint32_t>(p.vp / 16), p.vt16 = static_cast<uint32_t>(p.vt / 16);
    p.span = {Divider::of(static_cast<uint32_t>(a.page_tokens)), a.n_pages, a.table_pages};
    p.pages = a.pages;
    p.lengths = a.lengths;
    p.counts = a.counts;
    p.parents = a.parents;
    p.scale = a.scale * 1.44269504088896341f;
    // finite at the smallest scales: -inf plus it has to be -inf
    p.slack = std::min((a.data_type == DBS_CUDA_DTYPE_F16 ? 7.0f : 8.0f) / p.scale, std::numeric_limits<float>::max());
    p.out = a.out;
    p.lse = a.lse;
    p.info = static_cast<int4*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.info_bytes);
    hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
    hipError_t e = hipSuccess;
    for (int s0 = 0; s0 < a.sequences && e == hipSuccess; s0 += plan.batch) {
        AttendParams b = p;
        b.S = std::min(plan.batch, a.sequences - s0);
        const int64_t rows = static_cast<int64_t>(s0) * p.N * p.H;
        b.q = static_cast<const char*>(p.q) + s0 * p.qs;
        b.pages += static_cast<int64_t>(s0) * p.span.P;
        b.lengths += s0;
        if (b.counts) b.counts += s0;
        if (b.parents) b.parents += static_cast<int64_t>(s0) * p.N;
        if (b.shared) b.shared += s0 / p.K;
        b.out = static_cast<char*>(p.out) + rows * p.D * size;
        if (b.lse) b.lse += rows;
        switch (a.data_type) {
            case DBS_CUDA_DTYPE_F32: e = launch_attend<DBS_CUDA_DTYPE_F32>(b, plan.dim, plan.shape, stream); break;
            case DBS_CUDA_DTYPE_F16: e = launch_attend<DBS_CUDA_DTYPE_F16>(b, plan.dim, plan.shape, stream); break;
            default: e = launch_attend<DBS_CUDA_DTYPE_BF16>(b, plan.dim, plan.shape, stream); break;
        }
    }
    return finish_call(stream, e);
}

}  // extern "C"
