// SPDX-License-Identifier: MIT
//
// The C entry of attention over a paged cache (include/beamgrad_state.h):
// checks, the choice of a kernel, its workspace.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

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
    int64_t info_bytes, bytes;
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

Plan plan_of(const BeamgradAttention& a, AttendParams& p) {
    Plan plan;
    plan.dim = (a.head_dim + 63) / 64 * 64;
    p.N = a.tokens;
    p.H = a.heads;
    p.Hkv = a.kv_heads;
    p.G = Divider::of(static_cast<uint32_t>(a.heads / a.kv_heads));
    p.D = a.head_dim;
    // a group whose lengths one workgroup cannot hold reads its shared pages
    // once for each beam
    p.K = a.shared && a.beams <= kAttendSequences ? a.beams : 1;
    p.shared = p.K > 1 ? a.shared : nullptr;
    plan.batch = std::min(a.sequences, kAttendSequences / p.K * p.K);
    // the smallest tile that takes the rows that read a page together: fewer
    // rows than the tile cost matrix instructions, more read the cache again
    const int64_t rows = static_cast<int64_t>(p.N) * p.G.d, together = rows * p.K;
    p.beam_rows = Divider::of(static_cast<uint32_t>(rows));
    plan.shape = kRows16;
    while (plan.shape < attend_most(a.data_type, plan.dim) && attend_rows(plan.shape) < together) ++plan.shape;
    const int tile = attend_rows(plan.shape);
    p.shared_tiles = p.shared ? static_cast<int>((together + tile - 1) / tile) : 0;
    p.own_tiles = static_cast<int>((rows + tile - 1) / tile);
    p.head_items = plan.batch / p.K * (p.shared_tiles + p.K * p.own_tiles);
    switch (a.data_type) {
        case DBS_CUDA_DTYPE_F32: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_F32>(plan.dim, plan.shape); break;
        case DBS_CUDA_DTYPE_F16: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_F16>(plan.dim, plan.shape); break;
        default: plan.sizes = attend_sizes<DBS_CUDA_DTYPE_BF16>(plan.dim, plan.shape); break;
    }
    // units in 30 bits, whatever the lengths
    const double keys = static_cast<double>(a.table_pages) * a.page_tokens;
    p.unit_shift = 0;
    while (static_cast<double>(p.head_items) * p.Hkv * (std::ldexp(keys / plan.sizes.keys, -p.unit_shift) + 1.0) > 1.0e9)
        ++p.unit_shift;
    p.grid = (multiprocessors() * plan.sizes.resident + 7) / 8 * 8;
    const int64_t items = static_cast<int64_t>(p.head_items) * p.Hkv;
    plan.info_bytes = items * static_cast<int64_t>(sizeof(int4));
    const int64_t slots = p.shared ? p.grid + items : 2 * static_cast<int64_t>(p.grid);
    plan.bytes = plan.info_bytes + slots * plan.sizes.slot * static_cast<int64_t>(sizeof(float));
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
    if (workspace_bytes < plan.bytes) return DBS_CUDA_STATUS_INVALID_ARGUMENT;
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
