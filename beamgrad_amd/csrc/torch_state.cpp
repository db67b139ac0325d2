// SPDX-License-Identifier: MIT
//
// The torch.ops.beamgrad operators of a model's state in a search: attention
// over a paged cache, its pages, reordering of dense states
// (include/beamgrad_state.h has the C entries). Part of beamgrad_amd._C_hip.
//
// Every operator checks its arguments in one function that needs no GPU. The
// CPU key runs the checks and then refuses the call, so a wrong argument has its
// message wherever the tensors are. Nothing is read back and nothing waits:
// page tables stay on the device, and the calls can be captured into a graph.
#include <torch/all.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <limits>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "beamgrad_state.h"
#include "regions.hpp"
#include "torch_engine.hpp"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using Tensors = std::vector<Tensor>;

constexpr int64_t kI32Max = std::numeric_limits<int32_t>::max();

void* current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

void check_status(int code, const char* what) {
    if (code == DBS_CUDA_STATUS_OK) return;
    TORCH_CHECK_VALUE(code != DBS_CUDA_STATUS_INVALID_ARGUMENT, "beamgrad HIP ", what, ": invalid argument");
    TORCH_CHECK(false, "beamgrad HIP ", what, " failed: ", dbs_cuda_status_string(code));
}

[[noreturn]] void refuse_cpu(const char* what, const Tensor& t) {
    TORCH_CHECK(false, "beamgrad::", what, " runs on the GPU (HIP) only, got a tensor on ", t.device());
}

// A contiguous tensor from the caching allocator, without a trip through the
// dispatcher (a call makes several, and small calls take as long as their host work).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
}

// Operators without a derivative, at the Autograd key: what a torch.func
// transform wraps is still seen here.
void refuse_derivatives(const Tensor& t, const c10::OperatorHandle& op) {
    const auto name = [&] {
        const std::string what = op.schema().name().substr(sizeof("beamgrad::") - 1);
        return what == "reorder_states_" ? "reorder_states(inplace=True)" : what;
    };
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), "beamgrad_amd.", name(),
                " has no gradient: call it under torch.no_grad() or on detached tensors");
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "beamgrad_amd.", name(),
                " has no forward-mode derivative, and would drop a tensor's tangent: call it on the tensors' primals");
}

void no_derivative(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
    for (const c10::IValue& argument : torch::jit::last(*stack, op.schema().arguments().size())) {
        if (argument.isTensor()) {
            refuse_derivatives(argument.toTensor(), op);
        } else if (argument.isTensorList()) {
            for (const auto& t : argument.toListRef()) refuse_derivatives(t.toTensor(), op);
        }
    }
    op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// Written in place: an autograd graph that saved such a tensor notices.
void written(at::TensorList tensors) {
    for (const Tensor& t : tensors)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int data_type(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32) return DBS_CUDA_DTYPE_F32;
    if (t.scalar_type() == torch::kFloat16) return DBS_CUDA_DTYPE_F16;
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kBFloat16, name, " must be float32, float16 or bfloat16, got ",
                      t.scalar_type());
    return DBS_CUDA_DTYPE_BF16;
}

bool index_type(const Tensor& t) { return t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64; }

void check_index(const Tensor& t, at::IntArrayRef shape, const Tensor& with, const char* name) {
    TORCH_CHECK_VALUE(index_type(t) && t.sizes() == shape && t.device() == with.device(), name,
                      " must be an int32 or int64 ", shape, " tensor on the same device, got ", t.scalar_type(), " ", t.sizes(),
                      " on ", t.device());
}

// An index tensor as the kernels read it; numbers past 32 bits stay out of range.
Tensor as_i32(const Tensor& t) {
    const Tensor whole = t.contiguous();
    if (whole.scalar_type() == torch::kInt32) return whole;
    Tensor out = fresh(whole.sizes(), torch::kInt32, whole);
    check_status(beamgrad_narrow_indices(whole.const_data_ptr<int64_t>(), out.data_ptr<int32_t>(), whole.numel(), current_stream()),
                 "index conversion");
    return out;
}
const int32_t* i32(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

// ---------------------------------------------------------------------------
// Page tables and pools
// ---------------------------------------------------------------------------

void check_pages(const Tensor& pages, const Tensor& lengths) {
    TORCH_CHECK_VALUE(pages.numel() <= int64_t{1} << 30, "pages is too large: more than 2**30 entries, ", pages.sizes());
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.scalar_type() == torch::kInt32 && pages.is_contiguous() &&
                          pages.numel() > 0,
                      "pages must be a contiguous int32 [S, P] tensor, got ", pages.scalar_type(), " ", pages.sizes());
    TORCH_CHECK_VALUE(lengths.scalar_type() == torch::kInt32 && lengths.dim() == 1 &&
                          lengths.size(0) == pages.size(0) && lengths.is_contiguous() && lengths.device() == pages.device(),
                      "lengths must be a contiguous int32 [S] = [", pages.size(0), "] tensor on the same device, got ",
                      lengths.scalar_type(), " ", lengths.sizes());
}

void check_table(const Tensor& pages, const Tensor& lengths, const Tensor& refs) {
    check_pages(pages, lengths);
    TORCH_CHECK_VALUE(refs.dim() == 1 && refs.scalar_type() == torch::kInt32 && refs.is_contiguous() &&
                          refs.numel() > 0 && refs.numel() <= kI32Max && refs.device() == pages.device(),
                      "refs must be a contiguous int32 [pages of the pool] tensor on the same device, got ",
                      refs.scalar_type(), " ", refs.sizes());
}

void check_span(const Tensor& pages, int64_t page_tokens) {
    TORCH_CHECK_VALUE(page_tokens > 0, "a page must hold at least one token, got ", page_tokens);
    TORCH_CHECK_VALUE((pages.size(1) + 1) <= (kI32Max - 65536) / page_tokens,
                      "a sequence's pages must hold fewer than 2**31 tokens, got ", pages.size(1), " of ", page_tokens);
}

struct Pools {
    std::vector<void*> base;
    std::vector<int64_t> row_bytes, page_stride, token_stride;
    BeamgradPools c{};

    void bind() {
        c.base = base.data();
        c.row_bytes = row_bytes.data();
        c.page_stride = page_stride.data();
        c.token_stride = token_stride.data();
        c.n = static_cast<int32_t>(base.size());
    }
};

// Whether a token's row of t (the dimensions from `from` on) is one run.
bool row_contiguous(const Tensor& t, int64_t from) {
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d >= from; --d) {
        if (t.size(d) != 1 && t.stride(d) != run) return false;
        run *= t.size(d);
    }
    return true;
}

int64_t row_elements(const Tensor& t, int64_t from) {
    int64_t n = 1;
    for (int64_t d = from; d < t.dim(); ++d) n *= t.size(d);
    return n;
}

// Whether b lies as a does: most pools of a cache do, and are checked once.
bool laid_out_alike(const Tensor& a, const Tensor& b) {
    return a.sizes() == b.sizes() && a.strides() == b.strides() && a.scalar_type() == b.scalar_type() &&
           a.device() == b.device();
}

void check_pools(const Tensors& pools, const Tensor& pages, int64_t n_pages) {
    for (size_t i = 0; i < pools.size(); ++i) {
        const Tensor& t = pools[i];
        if (i > 0 && laid_out_alike(pools[i - 1], t)) continue;
        TORCH_CHECK_VALUE(t.dim() >= 3 && t.numel() > 0, "pools[", i, "] must be a [pages, tokens of a page, ...] tensor, got ",
                          t.sizes());
        TORCH_CHECK_VALUE(t.device() == pages.device(), "pools[", i, "] is on ", t.device(), ", the page table on ",
                          pages.device());
        TORCH_CHECK_VALUE(t.size(1) == pools[0].size(1) && t.size(0) == (n_pages < 0 ? pools[0].size(0) : n_pages), "pools[", i,
                          "] must have ", n_pages < 0 ? pools[0].size(0) : n_pages, " pages of ", pools[0].size(1),
                          " tokens, got ", t.sizes());
        TORCH_CHECK_VALUE(row_contiguous(t, 2), "a token's row of pools[", i, "] must be contiguous");
        TORCH_CHECK_VALUE(t.size(0) <= kI32Max, "pools[", i, "] has too many pages");
        // a page or token that lies where another does would be written twice
        TORCH_CHECK_VALUE((t.size(1) == 1 || t.stride(1) >= row_elements(t, 2)) && (t.size(0) == 1 || t.stride(0) > 0),
                          "the pages and tokens of pools[", i, "] overlap");
    }
    if (!pools.empty()) check_span(pages, pools[0].size(1));
}

// Pools whose memory meets, or news that lie in one, which the C entries refuse:
// with the numbers of two.
dbs_hip::Region rows_of(const Tensor& t) {
    const int64_t size = static_cast<int64_t>(t.element_size());
    return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), {t.size(0), t.size(1)}, {t.stride(0) * size, t.stride(1) * size},
            row_elements(t, 2) * size};
}

void check_pools_apart(const Tensors& pools, const Tensors& news) {
    std::vector<dbs_hip::Region> written, read;
    std::vector<size_t> at;  // in news: those that are no copy
    for (const Tensor& t : pools) written.push_back(rows_of(t));
    for (size_t i = 0; i < news.size(); ++i)
        if (row_contiguous(news[i], 2)) {
            read.push_back(rows_of(news[i]));
            at.push_back(i);
        }
    const dbs_hip::Meeting m = dbs_hip::find_meeting(written, read);
    if (m.first < 0) return;
    TORCH_CHECK_VALUE(!m.reads, "news[", at[m.second], "] and pools[", m.first, "] share memory");
    TORCH_CHECK_VALUE(m.first != m.second, "the pages and tokens of pools[", m.first, "] overlap");
    TORCH_CHECK_VALUE(false, "pools[", m.first, "] and pools[", m.second, "] share memory");
}

Pools bind_pools(const Tensors& pools, int64_t n_pages, int64_t page_tokens) {
    Pools p;
    p.base.reserve(pools.size());
    p.row_bytes.reserve(pools.size());
    p.page_stride.reserve(pools.size());
    p.token_stride.reserve(pools.size());
    for (size_t i = 0; i < pools.size(); ++i) {
        const Tensor& t = pools[i];
        p.base.push_back(t.data_ptr());
        if (i > 0 && laid_out_alike(pools[i - 1], t)) {
            p.row_bytes.push_back(p.row_bytes.back());
            p.page_stride.push_back(p.page_stride.back());
            p.token_stride.push_back(p.token_stride.back());
            continue;
        }
        const int64_t size = static_cast<int64_t>(t.element_size());
        p.row_bytes.push_back(row_elements(t, 2) * size);
        p.page_stride.push_back(t.stride(0) * size);
        p.token_stride.push_back(t.stride(1) * size);
    }
    p.bind();
    p.c.n_pages = static_cast<int32_t>(n_pages);
    p.c.page_tokens = static_cast<int32_t>(page_tokens);
    return p;
}

BeamgradTable bind_table(const Tensor& pages, const Tensor& lengths, const Tensor& refs) {
    return {const_cast<int32_t*>(pages.const_data_ptr<int32_t>()), const_cast<int32_t*>(lengths.const_data_ptr<int32_t>()),
            const_cast<int32_t*>(refs.const_data_ptr<int32_t>())};
}

int narrow(int64_t n) { return static_cast<int>(n); }

using TableOut = std::tuple<Tensor, Tensor, Tensor>;

struct NewTable {
    Tensor pages, lengths, refs;
    NewTable(const Tensor& p, const Tensor& l, const Tensor& r)
        : pages(fresh(p.sizes(), torch::kInt32, p)), lengths(fresh(l.sizes(), torch::kInt32, p)), refs(fresh(r.sizes(), torch::kInt32, p)) {}
    BeamgradTable bind() const { return bind_table(pages, lengths, refs); }
    TableOut take() { return {std::move(pages), std::move(lengths), std::move(refs)}; }
};

Tensor workspace(int64_t bytes, const Tensor& like) {
    TORCH_CHECK_VALUE(bytes >= 0, "beamgrad HIP: unsupported problem size (see the limits in beamgrad_state.h)");
    return fresh({bytes > 0 ? bytes : 1}, torch::kUInt8, like);
}

// --- fork ---

void check_fork(const Tensors& pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& parents) {
    check_table(pages, lengths, refs);
    TORCH_CHECK_VALUE(!pools.empty(), "pools must hold at least one pool");
    check_pools(pools, pages, refs.numel());
    check_index(parents, {pages.size(0)}, pages, "parents");
}

TableOut fork_pages_cpu(Tensors pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& parents) {
    check_fork(pools, pages, lengths, refs, parents);
    check_pools_apart(pools, {});
    refuse_cpu("fork_pages", pages);
}

TableOut fork_pages_hip(Tensors pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& parents) {
    check_fork(pools, pages, lengths, refs, parents);
    const at::OptionalDeviceGuard guard(pages.device());
    const Tensor par = parents.contiguous();
    const Pools p = bind_pools(pools, refs.numel(), pools[0].size(1));
    NewTable to(pages, lengths, refs);
    const int64_t bytes = beamgrad_fork_pages_workspace_size(narrow(pages.size(0)));
    const Tensor ws = workspace(bytes, pages);
    const BeamgradTable from = bind_table(pages, lengths, refs), out = to.bind();
    const int status = beamgrad_fork_pages(&p.c, &from, par.const_data_ptr(), par.scalar_type() == torch::kInt64,
                                           narrow(pages.size(0)), narrow(pages.size(1)), &out, ws.data_ptr(), bytes, current_stream());
    if (status == DBS_CUDA_STATUS_INVALID_ARGUMENT) check_pools_apart(pools, {});
    check_status(status, "fork_pages");
    written(pools);
    return to.take();
}

// --- extend ---

void check_extend(const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& counts, int64_t page_tokens) {
    check_table(pages, lengths, refs);
    check_span(pages, page_tokens);
    check_index(counts, {pages.size(0)}, pages, "counts");
}

TableOut extend_pages_cpu(const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& counts, int64_t page_tokens) {
    check_extend(pages, lengths, refs, counts, page_tokens);
    refuse_cpu("extend_pages", pages);
}

TableOut extend_pages_hip(const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& counts, int64_t page_tokens) {
    check_extend(pages, lengths, refs, counts, page_tokens);
    const at::OptionalDeviceGuard guard(pages.device());
    const Tensor n = as_i32(counts);
    NewTable to(pages, lengths, refs);
    const int64_t bytes = beamgrad_extend_pages_workspace_size(narrow(refs.numel()));
    const Tensor ws = workspace(bytes, pages);
    const BeamgradTable from = bind_table(pages, lengths, refs), out = to.bind();
    check_status(beamgrad_extend_pages(&from, i32(n), narrow(pages.size(0)), narrow(pages.size(1)), narrow(refs.numel()),
                                       narrow(page_tokens), &out, ws.data_ptr(), bytes, current_stream()),
                 "extend_pages");
    return to.take();
}

// --- write ---

void check_write(const Tensors& pools, const Tensors& news, const Tensor& pages, const Tensor& lengths, const OptTensor& counts) {
    check_pages(pages, lengths);
    TORCH_CHECK_VALUE(!pools.empty() && pools.size() == news.size(), "pools and news must be as many, and at least one, got ",
                      pools.size(), " and ", news.size());
    check_pools(pools, pages, -1);
    for (size_t i = 0; i < news.size(); ++i) {
        const Tensor &n = news[i], &p = pools[i];
        if (i > 0 && laid_out_alike(news[i - 1], n) && laid_out_alike(pools[i - 1], p)) continue;
        bool same = n.dim() == p.dim() && n.dim() >= 3 && n.size(0) == pages.size(0) && n.size(1) > 0 && n.size(1) == news[0].size(1);
        for (int64_t d = 2; same && d < n.dim(); ++d) same = n.size(d) == p.size(d);
        TORCH_CHECK_VALUE(same, "news[", i, "] must be [S, N, ...] with the row of pools[", i, "], got ", n.sizes(), " for ", p.sizes());
        TORCH_CHECK_VALUE(n.scalar_type() == p.scalar_type() && n.device() == p.device(), "news[", i, "] must have the type and device of pools[",
                          i, "], got ", n.scalar_type(), " for ", p.scalar_type());
    }
    if (counts) check_index(*counts, {pages.size(0)}, pages, "counts");
}

void write_tokens_cpu(Tensors pools, Tensors news, const Tensor& pages, const Tensor& lengths, const OptTensor& counts) {
    check_write(pools, news, pages, lengths, counts);
    check_pools_apart(pools, news);
    refuse_cpu("write_tokens", pages);
}

void write_tokens_hip(Tensors pools, Tensors news, const Tensor& pages, const Tensor& lengths, const OptTensor& counts) {
    check_write(pools, news, pages, lengths, counts);
    const at::OptionalDeviceGuard guard(pages.device());
    const Tensor n = counts ? as_i32(*counts) : Tensor();
    const Pools p = bind_pools(pools, pools[0].size(0), pools[0].size(1));
    std::vector<const void*> from;
    std::vector<int64_t> strides;
    from.reserve(news.size());
    strides.reserve(2 * news.size());
    bool plain = true;
    for (size_t i = 0; i < news.size(); ++i) {
        Tensor& t = news[i];
        if (plain && i > 0 && laid_out_alike(news[i - 1], t)) {
            from.push_back(t.const_data_ptr());
            strides.push_back(strides[strides.size() - 2]);
            strides.push_back(strides[strides.size() - 2]);
            continue;
        }
        plain = row_contiguous(t, 2);
        if (!plain) t = t.contiguous();
        from.push_back(t.const_data_ptr());
        strides.push_back(t.stride(0) * static_cast<int64_t>(t.element_size()));
        strides.push_back(t.stride(1) * static_cast<int64_t>(t.element_size()));
    }
    const int status = beamgrad_write_tokens(&p.c, from.data(), strides.data(), i32(pages), i32(lengths), i32(n), narrow(pages.size(0)),
                                             narrow(pages.size(1)), narrow(news[0].size(1)), current_stream());
    if (status == DBS_CUDA_STATUS_INVALID_ARGUMENT) check_pools_apart(pools, news);
    check_status(status, "write_tokens");
    written(pools);
}

// --- keep ---

void check_keep(const Tensors& pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& drafted,
                const Tensor& keep, const Tensor& kept) {
    check_table(pages, lengths, refs);
    TORCH_CHECK_VALUE(!pools.empty(), "pools must hold at least one pool");
    check_pools(pools, pages, refs.numel());
    check_index(drafted, {pages.size(0)}, pages, "drafted");
    TORCH_CHECK_VALUE(keep.dim() == 2 && keep.size(1) > 0, "keep must be [S, A] = [", pages.size(0), ", A >= 1], got ", keep.sizes());
    check_index(keep, {pages.size(0), keep.size(1)}, pages, "keep");
    check_index(kept, {pages.size(0)}, pages, "kept");
}

TableOut keep_tokens_cpu(Tensors pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& drafted,
                         const Tensor& keep, const Tensor& kept) {
    check_keep(pools, pages, lengths, refs, drafted, keep, kept);
    check_pools_apart(pools, {});
    refuse_cpu("keep_tokens", pages);
}

TableOut keep_tokens_hip(Tensors pools, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const Tensor& drafted,
                         const Tensor& keep, const Tensor& kept) {
    check_keep(pools, pages, lengths, refs, drafted, keep, kept);
    const at::OptionalDeviceGuard guard(pages.device());
    const Tensor d = as_i32(drafted), k = as_i32(keep), n = as_i32(kept);
    const Pools p = bind_pools(pools, refs.numel(), pools[0].size(1));
    NewTable to(pages, lengths, refs);
    const BeamgradTable from = bind_table(pages, lengths, refs), out = to.bind();
    const int status = beamgrad_keep_tokens(&p.c, &from, i32(d), i32(k), i32(n), narrow(pages.size(0)), narrow(pages.size(1)),
                                            narrow(k.size(1)), &out, current_stream());
    if (status == DBS_CUDA_STATUS_INVALID_ARGUMENT) check_pools_apart(pools, {});
    check_status(status, "keep_tokens");
    written(pools);
    return to.take();
}

// ---------------------------------------------------------------------------
// Attention over a paged cache
// ---------------------------------------------------------------------------

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths,
                     const OptTensor& parents, const OptTensor& counts, int64_t beams, const OptTensor& shared, double scale) {
    TORCH_CHECK_VALUE(q.dim() == 4 && q.numel() > 0, "q must be a [S, N, H, D] tensor, got ", q.sizes());
    data_type(q, "q");
    TORCH_CHECK_VALUE(k.dim() == 4 && k.numel() > 0 && v.sizes() == k.sizes(),
                      "k and v must be [pages, tokens of a page, Hkv, D] tensors of one shape, got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                      "q, k and v must have one type, got ", q.scalar_type(), ", ", k.scalar_type(), " and ", v.scalar_type());
    TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device() && pages.device() == q.device(),
                      "q, k, v and the page table must be on one device");
    check_pages(pages, lengths);
    const int64_t S = q.size(0), N = q.size(1), H = q.size(2), D = q.size(3);
    TORCH_CHECK_VALUE(pages.size(0) == S, "q has ", S, " sequences, the page table ", pages.size(0));
    TORCH_CHECK_VALUE(D == k.size(3) && D % 8 == 0 && D <= 256, "the heads' width must be one multiple of 8 up to 256, got ", D,
                      " and ", k.size(3));
    TORCH_CHECK_VALUE(H % k.size(2) == 0, "q's ", H, " heads must be a multiple of the cache's ", k.size(2));
    check_span(pages, k.size(1));
    TORCH_CHECK_VALUE(k.size(0) <= kI32Max, "the pool has too many pages");
    if (counts) check_index(*counts, {S}, q, "counts");
    if (parents) {
        check_index(*parents, {S, N}, q, "parents");
        TORCH_CHECK_VALUE(N <= 512, "a tree holds at most 512 drafted tokens, got ", N);
    }
    TORCH_CHECK_VALUE(beams >= 1 && S % beams == 0, "beams must divide the ", S, " sequences, got ", beams);
    if (shared) check_index(*shared, {S / beams}, q, "shared");
    TORCH_CHECK_VALUE(std::isfinite(scale) && scale > 0.0 && std::isfinite(static_cast<float>(scale)) &&
                          static_cast<float>(scale) > 0.0f,
                      "scale must be positive and finite, got ", scale);
    const double rows = static_cast<double>(N) * static_cast<double>(H);
    TORCH_CHECK_VALUE(rows * static_cast<double>(S) <= 2.0e9 && rows * static_cast<double>(beams) <= 1.0e9, "q is too large");
    const auto cache = [&](const Tensor& t, const char* name) {
        const int64_t size = static_cast<int64_t>(t.element_size());
        bool fits = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
        for (int d = 0; d < 3; ++d) fits = fits && (t.size(d) == 1 || t.stride(d) * size % 16 == 0);
        TORCH_CHECK_VALUE(fits, name, "'s rows must be contiguous and begin at multiples of 16 bytes, got strides ", t.strides());
    };
    cache(k, "k");
    cache(v, "v");
}

// strides of the first three dimensions; of a dimension of one entry, 0
void strides_of(const Tensor& t, int64_t* to) {
    for (int d = 0; d < 3; ++d) to[d] = t.size(d) == 1 ? 0 : t.stride(d);
}

std::tuple<Tensor, Tensor> tree_attention_cpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths,
                                              const OptTensor& parents, const OptTensor& counts, int64_t beams, const OptTensor& shared,
                                              double scale, bool) {
    check_attention(q, k, v, pages, lengths, parents, counts, beams, shared, scale);
    refuse_cpu("tree_attention", q);
}

std::tuple<Tensor, Tensor> tree_attention_hip(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths,
                                              const OptTensor& parents, const OptTensor& counts, int64_t beams, const OptTensor& shared,
                                              double scale, bool with_lse) {
    check_attention(q, k, v, pages, lengths, parents, counts, beams, shared, scale);
    const at::OptionalDeviceGuard guard(q.device());
    Tensor query = q;
    const int64_t size = static_cast<int64_t>(q.element_size());
    bool fits = q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) fits = fits && (q.size(d) == 1 || q.stride(d) * size % 16 == 0);
    if (!fits) query = q.clone(at::MemoryFormat::Contiguous);
    Tensor par, num, sh;
    if (parents) par = as_i32(*parents);
    if (counts) num = as_i32(*counts);
    if (shared) sh = as_i32(*shared);
    Tensor out = fresh(q.sizes(), q.scalar_type(), q);
    Tensor lse = with_lse ? fresh({q.size(0), q.size(1), q.size(2)}, torch::kFloat32, q) : fresh({0}, torch::kFloat32, q);
    BeamgradAttention a{};
    a.q = query.const_data_ptr();
    a.k = k.const_data_ptr();
    a.v = v.const_data_ptr();
    a.data_type = data_type(q, "q");
    a.sequences = narrow(q.size(0));
    a.tokens = narrow(q.size(1));
    a.heads = narrow(q.size(2));
    a.kv_heads = narrow(k.size(2));
    a.head_dim = narrow(q.size(3));
    a.beams = narrow(beams);
    a.page_tokens = narrow(k.size(1));
    a.n_pages = narrow(k.size(0));
    a.table_pages = narrow(pages.size(1));
    strides_of(query, a.q_strides);
    strides_of(k, a.k_strides);
    strides_of(v, a.v_strides);
    a.pages = i32(pages);
    a.lengths = i32(lengths);
    a.counts = i32(num);
    a.parents = i32(par);
    a.shared = i32(sh);
    a.scale = static_cast<float>(scale);
    a.out = out.data_ptr();
    a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
    const int64_t bytes = beamgrad_tree_attention_workspace_size(&a);
    const Tensor ws = workspace(bytes, q);
    check_status(beamgrad_tree_attention(&a, ws.data_ptr(), bytes, current_stream()), "tree_attention");
    return {out, lse};
}

// ---------------------------------------------------------------------------
// Reordering of dense states
// ---------------------------------------------------------------------------

void check_states(const Tensors& states, const Tensor& parents, const char* name) {
    TORCH_CHECK_VALUE(parents.dim() == 2 && index_type(parents) && parents.numel() > 0,
                      "parents must be an int32 or int64 [B, K] tensor, got ", parents.scalar_type(), " ", parents.sizes());
    TORCH_CHECK_VALUE(parents.size(1) <= 4096 && parents.size(0) <= 65535, "parents must have at most 65535 examples of 4096 beams, got ",
                      parents.sizes());
    for (size_t i = 0; i < states.size(); ++i) {
        const Tensor& t = states[i];
        if (i > 0 && laid_out_alike(states[i - 1], t)) continue;
        TORCH_CHECK_VALUE(t.dim() >= 2 && t.size(0) == parents.size(0) && t.size(1) == parents.size(1), name, "[", i,
                          "] must be [B, K, ...] = [", parents.size(0), ", ", parents.size(1), ", ...], got ", t.sizes());
        TORCH_CHECK_VALUE(t.device() == parents.device(), name, "[", i, "] is on ", t.device(), ", parents on ", parents.device());
        TORCH_CHECK_VALUE(row_elements(t, 1) * static_cast<int64_t>(t.element_size()) / 4 <= kI32Max - 131072, name, "[", i,
                          "] is too large for one example: ", t.sizes());
    }
}

void check_inplace(const Tensors& states) {
    for (size_t i = 0; i < states.size(); ++i)
        TORCH_CHECK_VALUE(states[i].is_contiguous(), "states[", i, "] must be contiguous to be reordered in place");
}

// States whose memory meets, which the C entry refuses: with the numbers of two.
void check_states_apart(const Tensors& states) {
    std::vector<dbs_hip::Region> written;
    std::vector<size_t> at;  // in states: those that are not empty
    for (size_t i = 0; i < states.size(); ++i)
        if (states[i].numel() > 0) {
            written.push_back({reinterpret_cast<uintptr_t>(states[i].const_data_ptr()), {1, 1}, {0, 0},
                               states[i].numel() * static_cast<int64_t>(states[i].element_size())});
            at.push_back(i);
        }
    const dbs_hip::Meeting m = dbs_hip::find_meeting(written, {});
    TORCH_CHECK_VALUE(m.first < 0, "states[", at[m.first], "] and states[", at[m.second], "] share memory");
}

struct StateRows {
    std::vector<const void*> from;
    std::vector<void*> to;
    std::vector<int64_t> size;  // of a row
    void add(const Tensor& source, const Tensor& target, int64_t row) {
        from.push_back(source.const_data_ptr());
        to.push_back(target.data_ptr());
        size.push_back(row);
    }
};

Tensors reorder_states_cpu(Tensors states, const Tensor& parents) {
    check_states(states, parents, "states");
    refuse_cpu("reorder_states", parents);
}

int run_reorder(const StateRows& rows, const Tensor& parents) {
    const Tensor par = parents.contiguous();
    return beamgrad_reorder_states(rows.from.data(), rows.to.data(), rows.size.data(), narrow(static_cast<int64_t>(rows.from.size())),
                                   par.const_data_ptr(), par.scalar_type() == torch::kInt64, narrow(par.size(0)), narrow(par.size(1)),
                                   current_stream());
}

Tensors reorder_states_hip(Tensors states, const Tensor& parents) {
    check_states(states, parents, "states");
    const at::OptionalDeviceGuard guard(parents.device());
    Tensors out;
    StateRows rows;
    for (Tensor& t : states) {
        t = t.contiguous();
        out.push_back(fresh(t.sizes(), t.scalar_type(), t));
        if (t.numel() > 0) rows.add(t, out.back(), row_elements(t, 2) * static_cast<int64_t>(t.element_size()));
    }
    check_status(run_reorder(rows, parents), "reorder_states");
    return out;
}

void reorder_states_inplace_cpu(Tensors states, const Tensor& parents) {
    check_states(states, parents, "states");
    check_inplace(states);
    check_states_apart(states);
    refuse_cpu("reorder_states_", parents);
}

void reorder_states_inplace_hip(Tensors states, const Tensor& parents) {
    check_states(states, parents, "states");
    check_inplace(states);
    const at::OptionalDeviceGuard guard(parents.device());
    StateRows rows;
    for (const Tensor& t : states)
        if (t.numel() > 0) rows.add(t, t, row_elements(t, 2) * static_cast<int64_t>(t.element_size()));
    const int status = run_reorder(rows, parents);
    if (status == DBS_CUDA_STATUS_INVALID_ARGUMENT) check_states_apart(states);
    check_status(status, "reorder_states");
    written(states);
}

void check_grads(const Tensors& grads, const Tensor& parents) {
    check_states(grads, parents, "grads");
    for (const Tensor& t : grads) {
        data_type(t, "grads");
        TORCH_CHECK_VALUE(t.scalar_type() == grads[0].scalar_type(), "grads must have one type");
    }
}

Tensors reorder_states_backward_cpu(Tensors grads, const Tensor& parents) {
    check_grads(grads, parents);
    refuse_cpu("reorder_states_backward", parents);
}

Tensors reorder_states_backward_hip(Tensors grads, const Tensor& parents) {
    check_grads(grads, parents);
    const at::OptionalDeviceGuard guard(parents.device());
    Tensors out;
    StateRows rows;
    for (Tensor& t : grads) {
        t = t.contiguous();
        out.push_back(fresh(t.sizes(), t.scalar_type(), t));
        if (t.numel() > 0) rows.add(t, out.back(), row_elements(t, 2));
    }
    if (rows.from.empty()) return out;
    const Tensor par = parents.contiguous();
    check_status(beamgrad_reorder_states_backward(rows.from.data(), rows.to.data(), rows.size.data(),
                                                  narrow(static_cast<int64_t>(rows.from.size())), data_type(grads[0], "grads"),
                                                  par.const_data_ptr(), par.scalar_type() == torch::kInt64, narrow(par.size(0)),
                                                  narrow(par.size(1)), current_stream()),
                 "reorder_states_backward");
    return out;
}

// Whether a living graph holds the leaf's gradient accumulator with a stream
// that is not the current one.
bool leaf_of_another_stream(const Tensor& leaf) {
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!accumulator || !leaf.is_cuda()) return false;
    const auto stream = accumulator->stream();
    // by number: the two sides name the device's type differently on ROCm
    return stream && stream->id() != c10::hip::getCurrentHIPStream(leaf.device().index()).id();
}

// Whether the backward from `node` on reaches such a leaf, over whatever operators.
// During a backward, along the nodes that it runs alone: the others hand nothing over.
bool reaches_leaf_of_another_stream(const torch::autograd::Node* node) {
    const auto* const runs = torch::autograd::get_current_graph_task_exec_info();
    std::vector<const torch::autograd::Node*> open{node};
    std::unordered_set<const torch::autograd::Node*> seen{node};
    while (!open.empty()) {
        const torch::autograd::Node* const at = open.back();
        open.pop_back();
        for (const auto& edge : at->next_edges()) {
            torch::autograd::Node* const next = edge.function.get();
            if (!next || !seen.insert(next).second) continue;
            if (runs && !runs->empty()) {
                const auto info = runs->find(next);
                if (info == runs->end() || !info->second.should_execute()) continue;
            }
            const auto* const leaf = dynamic_cast<const torch::autograd::AccumulateGrad*>(next);
            if (leaf && leaf_of_another_stream(leaf->variable)) return true;
            open.push_back(next);
        }
    }
    return false;
}

bool backward_reaches_leaf_of_another_stream(const Tensor& output) {
    const auto& node = output.grad_fn();
    return node && reaches_leaf_of_another_stream(node.get());
}

// In a capture: torch hands a leaf's gradient over on the stream that the leaf's
// accumulator was made on. Where a living graph of another stream holds it, that
// stream joins the capture and the capture's end ends the process.
// Gradients without memory (meta and fake tensors) are in no capture, and may be of
// a device that is not there.
void refuse_foreign_leaves(const torch::autograd::Node* node, const Tensors& grads) {
    bool there = false;
    for (const Tensor& g : grads) there |= g.defined() && g.is_cuda() && !g.unsafeGetTensorImpl()->is_python_dispatch();
    if (!there || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    TORCH_CHECK(!reaches_leaf_of_another_stream(node),
                "beamgrad_amd.reorder_states: a captured backward reaches a leaf that a living graph of another "
                "stream uses; drop that graph (its outputs and losses) before the capture");
}

Tensors call_reorder(const Tensors& states, const Tensor& parents) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("beamgrad::reorder_states", "")
                               .typed<Tensors(Tensors, const Tensor&)>();
    return op.call(states, parents);
}
Tensors call_gather(const Tensors& grads, const Tensor& parents) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("beamgrad::reorder_states_backward", "")
                               .typed<Tensors(Tensors, const Tensor&)>();
    return op.call(grads, parents);
}

// The states in the order of the new beams (or, back, their gradients): what
// comes in for output i goes to input i, by the other of the two operators, which
// records in its turn where a graph of the backward is made.
class ReorderNode : public torch::autograd::Node {
   public:
    ReorderNode(const Tensors& inputs, const Tensor& parents, bool gathers)
        : Node(torch::autograd::collect_next_edges(inputs)), parents_(parents, false), gathers_(gathers) {}

    std::string name() const override { return gathers_ ? "ReorderStatesBackwardBackward" : "ReorderStatesBackward"; }
    void release_variables() override { parents_.reset_data(); }

   protected:
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        refuse_foreign_leaves(this, grads);
        const Tensor parents = parents_.unpack(shared_from_this());
        torch::autograd::variable_list out(grads.size());
        std::vector<bool> done(grads.size());
        for (size_t i = 0; i < grads.size(); ++i) {  // one call for each type
            if (done[i] || !grads[i].defined() || !task_should_compute_output(i)) continue;
            Tensors some;
            std::vector<size_t> at;
            for (size_t j = i; j < grads.size(); ++j) {
                if (done[j] || !grads[j].defined() || grads[j].scalar_type() != grads[i].scalar_type() ||
                    !task_should_compute_output(j))
                    continue;
                done[j] = true;
                some.push_back(grads[j]);
                at.push_back(j);
            }
            const Tensors got = gathers_ ? call_reorder(some, parents) : call_gather(some, parents);
            for (size_t j = 0; j < at.size(); ++j) out[at[j]] = got[j];
        }
        return out;
    }

   private:
    torch::autograd::SavedVariable parents_;
    bool gathers_;
};

// The operator's outputs, those of inputs that require a gradient recorded.
Tensors recorded(const Tensors& inputs, const Tensor& parents, bool gathers) {
    Tensors taking;
    for (const Tensor& t : inputs)
        if (t.requires_grad()) taking.push_back(t);
    const auto node = std::shared_ptr<ReorderNode>(new ReorderNode(taking, parents, gathers), torch::autograd::deleteNode);
    Tensors out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = gathers ? call_gather(inputs, parents) : call_reorder(inputs, parents);
    }
    for (size_t i = 0; i < inputs.size(); ++i)
        if (inputs[i].requires_grad()) torch::autograd::set_history(out[i], node);
    return out;
}

bool records(const Tensors& tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : tensors)
        if (t.requires_grad()) return true;
    return false;
}

// The map is linear: an output's tangent is the input's, moved as it is. The
// tangents go through the whole operator, which records a gradient of them too.
Tensors with_tangents(const Tensors& inputs, const Tensor& parents, bool gathers, Tensors out) {
    Tensors tangents;
    std::vector<size_t> at;
    for (size_t i = 0; i < inputs.size(); ++i) {
        if (!torch::autograd::isFwGradDefined(inputs[i])) continue;
        tangents.push_back(inputs[i]._fw_grad(/*level=*/0));
        at.push_back(i);
    }
    if (tangents.empty()) return out;
    const Tensors moved = gathers ? call_gather(tangents, parents) : call_reorder(tangents, parents);
    for (size_t j = 0; j < at.size(); ++j) out[at[j]]._set_fw_grad(moved[j], /*level=*/0, /*is_inplace_op=*/false);
    return out;
}

Tensors reorder_states_autograd(Tensors states, const Tensor& parents) {
    if (records(states)) {
        for (const Tensor& t : states)
            TORCH_CHECK_TYPE(!t.requires_grad() || t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kFloat16 ||
                                 t.scalar_type() == torch::kBFloat16,
                             "reorder_states has a gradient for float32, float16 and bfloat16 states, not ", t.scalar_type());
        return with_tangents(states, parents, false, recorded(states, parents, false));
    }
    Tensors out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = call_reorder(states, parents);
    }
    return with_tangents(states, parents, false, std::move(out));
}

Tensors reorder_states_backward_autograd(Tensors grads, const Tensor& parents) {
    if (records(grads)) return with_tangents(grads, parents, true, recorded(grads, parents, true));
    Tensors out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = call_gather(grads, parents);
    }
    return with_tangents(grads, parents, true, std::move(out));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(beamgrad, m) {
    m.def(
        "tree_attention(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor lengths, Tensor? parents, Tensor? counts, int beams, "
        "Tensor? shared, float scale, bool with_lse) -> (Tensor, Tensor)");
    m.def(
        "fork_pages(Tensor(a!)[] pools, Tensor pages, Tensor lengths, Tensor refs, Tensor parents) -> (Tensor, Tensor, Tensor)");
    m.def("extend_pages(Tensor pages, Tensor lengths, Tensor refs, Tensor counts, int page_tokens) -> (Tensor, Tensor, Tensor)");
    m.def("write_tokens(Tensor(a!)[] pools, Tensor[] news, Tensor pages, Tensor lengths, Tensor? counts) -> ()");
    m.def(
        "keep_tokens(Tensor(a!)[] pools, Tensor pages, Tensor lengths, Tensor refs, Tensor drafted, Tensor keep, Tensor kept) -> "
        "(Tensor, Tensor, Tensor)");
    m.def("reorder_states(Tensor[] states, Tensor parents) -> Tensor[]");
    m.def("reorder_states_(Tensor(a!)[] states, Tensor parents) -> ()");
    m.def("reorder_states_backward(Tensor[] grads, Tensor parents) -> Tensor[]");
    m.def("leaf_of_another_stream(Tensor leaf) -> bool", &leaf_of_another_stream);
    m.def("backward_reaches_leaf_of_another_stream(Tensor output) -> bool", &backward_reaches_leaf_of_another_stream);
}

TORCH_LIBRARY_IMPL(beamgrad, CUDA, m) {
    m.impl("tree_attention", &tree_attention_hip);
    m.impl("fork_pages", &fork_pages_hip);
    m.impl("extend_pages", &extend_pages_hip);
    m.impl("write_tokens", &write_tokens_hip);
    m.impl("keep_tokens", &keep_tokens_hip);
    m.impl("reorder_states", &reorder_states_hip);
    m.impl("reorder_states_", &reorder_states_inplace_hip);
    m.impl("reorder_states_backward", &reorder_states_backward_hip);
}

TORCH_LIBRARY_IMPL(beamgrad, Autograd, m) {
    m.impl("reorder_states", &reorder_states_autograd);
    m.impl("reorder_states_backward", &reorder_states_backward_autograd);
    for (const char* name : {"tree_attention", "fork_pages", "write_tokens", "keep_tokens", "reorder_states_"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}

// Checked, then refused.
TORCH_LIBRARY_IMPL(beamgrad, CPU, m) {
    m.impl("tree_attention", &tree_attention_cpu);
    m.impl("fork_pages", &fork_pages_cpu);
    m.impl("extend_pages", &extend_pages_cpu);
    m.impl("write_tokens", &write_tokens_cpu);
    m.impl("keep_tokens", &keep_tokens_cpu);
    m.impl("reorder_states", &reorder_states_cpu);
    m.impl("reorder_states_", &reorder_states_inplace_cpu);
    m.impl("reorder_states_backward", &reorder_states_backward_cpu);
}
