// SPDX-License-Identifier: MIT
//
// What the torch operators of a model's state and scores share: checks of page
// tables, pools and indices, tensors of the caching allocator, and the refusals of
// derivatives and captures that torch would not survive.
#pragma once

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

namespace beamgrad_torch {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using Tensors = std::vector<Tensor>;

constexpr int64_t kI32Max = std::numeric_limits<int32_t>::max();

inline void* current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

inline void check_status(int code, const char* what) {
    if (code == DBS_CUDA_STATUS_OK) return;
    TORCH_CHECK_VALUE(code != DBS_CUDA_STATUS_INVALID_ARGUMENT, "beamgrad HIP ", what, ": invalid argument");
    TORCH_CHECK(false, "beamgrad HIP ", what, " failed: ", dbs_cuda_status_string(code));
}

[[noreturn]] inline void refuse_cpu(const char* what, const Tensor& t) {
    TORCH_CHECK(false, "beamgrad::", what, " runs on the GPU (HIP) only, got a tensor on ", t.device());
}

// A contiguous tensor from the caching allocator, without a trip through the
// dispatcher (a call makes several, and small calls take as long as their host work).
inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
}

// Operators without a derivative, at the Autograd key: what a torch.func
// transform wraps is still seen here.
inline void refuse_derivatives(const Tensor& t, const c10::OperatorHandle& op) {
    const auto name = [&] {
        const std::string what = op.schema().name().substr(sizeof("beamgrad::") - 1);
        return what == "reorder_states_" ? "reorder_states(inplace=True)" : what;
    };
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), "beamgrad_amd.", name(),
                " has no gradient: call it under torch.no_grad() or on detached tensors");
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "beamgrad_amd.", name(),
                " has no forward-mode derivative, and would drop a tensor's tangent: call it on the tensors' primals");
}

inline void no_derivative(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
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
inline void written(at::TensorList tensors) {
    for (const Tensor& t : tensors)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

inline int data_type(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32) return DBS_CUDA_DTYPE_F32;
    if (t.scalar_type() == torch::kFloat16) return DBS_CUDA_DTYPE_F16;
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kBFloat16, name, " must be float32, float16 or bfloat16, got ",
                      t.scalar_type());
    return DBS_CUDA_DTYPE_BF16;
}

inline bool index_type(const Tensor& t) { return t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64; }

inline void check_index(const Tensor& t, at::IntArrayRef shape, const Tensor& with, const char* name) {
    TORCH_CHECK_VALUE(index_type(t) && t.sizes() == shape && t.device() == with.device(), name,
                      " must be an int32 or int64 ", shape, " tensor on the same device, got ", t.scalar_type(), " ", t.sizes(),
                      " on ", t.device());
}

// An index tensor as the kernels read it; numbers past 32 bits stay out of range.
inline Tensor as_i32(const Tensor& t) {
    const Tensor whole = t.contiguous();
    if (whole.scalar_type() == torch::kInt32) return whole;
    Tensor out = fresh(whole.sizes(), torch::kInt32, whole);
    check_status(beamgrad_narrow_indices(whole.const_data_ptr<int64_t>(), out.data_ptr<int32_t>(), whole.numel(), current_stream()),
                 "index conversion");
    return out;
}
inline const int32_t* i32(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

// ---------------------------------------------------------------------------
// Page tables and pools
// ---------------------------------------------------------------------------

inline void check_pages(const Tensor& pages, const Tensor& lengths) {
    TORCH_CHECK_VALUE(pages.numel() <= int64_t{1} << 30, "pages is too large: more than 2**30 entries, ", pages.sizes());
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.scalar_type() == torch::kInt32 && pages.is_contiguous() &&
                          pages.numel() > 0,
                      "pages must be a contiguous int32 [S, P] tensor, got ", pages.scalar_type(), " ", pages.sizes());
    TORCH_CHECK_VALUE(lengths.scalar_type() == torch::kInt32 && lengths.dim() == 1 &&
                          lengths.size(0) == pages.size(0) && lengths.is_contiguous() && lengths.device() == pages.device(),
                      "lengths must be a contiguous int32 [S] = [", pages.size(0), "] tensor on the same device, got ",
                      lengths.scalar_type(), " ", lengths.sizes());
}

inline void check_table(const Tensor& pages, const Tensor& lengths, const Tensor& refs) {
    check_pages(pages, lengths);
    TORCH_CHECK_VALUE(refs.dim() == 1 && refs.scalar_type() == torch::kInt32 && refs.is_contiguous() &&
                          refs.numel() > 0 && refs.numel() <= kI32Max && refs.device() == pages.device(),
                      "refs must be a contiguous int32 [pages of the pool] tensor on the same device, got ",
                      refs.scalar_type(), " ", refs.sizes());
}

inline void check_span(const Tensor& pages, int64_t page_tokens) {
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
inline bool row_contiguous(const Tensor& t, int64_t from) {
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d >= from; --d) {
        if (t.size(d) != 1 && t.stride(d) != run) return false;
        run *= t.size(d);
    }
    return true;
}

inline int64_t row_elements(const Tensor& t, int64_t from) {
    int64_t n = 1;
    for (int64_t d = from; d < t.dim(); ++d) n *= t.size(d);
    return n;
}

// Whether b lies as a does: most pools of a cache do, and are checked once.
inline bool laid_out_alike(const Tensor& a, const Tensor& b) {
    return a.sizes() == b.sizes() && a.strides() == b.strides() && a.scalar_type() == b.scalar_type() &&
           a.device() == b.device();
}

inline void check_pools(const Tensors& pools, const Tensor& pages, int64_t n_pages) {
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
inline dbs_hip::Region rows_of(const Tensor& t) {
    const int64_t size = static_cast<int64_t>(t.element_size());
    return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), {t.size(0), t.size(1)}, {t.stride(0) * size, t.stride(1) * size},
            row_elements(t, 2) * size};
}

inline void check_pools_apart(const Tensors& pools, const Tensors& news) {
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

inline Pools bind_pools(const Tensors& pools, int64_t n_pages, int64_t page_tokens) {
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

inline BeamgradTable bind_table(const Tensor& pages, const Tensor& lengths, const Tensor& refs) {
    return {const_cast<int32_t*>(pages.const_data_ptr<int32_t>()), const_cast<int32_t*>(lengths.const_data_ptr<int32_t>()),
            const_cast<int32_t*>(refs.const_data_ptr<int32_t>())};
}

inline int narrow(int64_t n) { return static_cast<int>(n); }

using TableOut = std::tuple<Tensor, Tensor, Tensor>;

struct NewTable {
    Tensor pages, lengths, refs;
    NewTable(const Tensor& p, const Tensor& l, const Tensor& r)
        : pages(fresh(p.sizes(), torch::kInt32, p)), lengths(fresh(l.sizes(), torch::kInt32, p)), refs(fresh(r.sizes(), torch::kInt32, p)) {}
    BeamgradTable bind() const { return bind_table(pages, lengths, refs); }
    TableOut take() { return {std::move(pages), std::move(lengths), std::move(refs)}; }
};

inline Tensor workspace(int64_t bytes, const Tensor& like) {
    TORCH_CHECK_VALUE(bytes >= 0, "beamgrad HIP: unsupported problem size (see the limits in beamgrad_state.h)");
    return fresh({bytes > 0 ? bytes : 1}, torch::kUInt8, like);
}

// strides of the first three dimensions; of a dimension of one entry, 0
inline void strides_of(const Tensor& t, int64_t* to) {
    for (int d = 0; d < 3; ++d) to[d] = t.size(d) == 1 ? 0 : t.stride(d);
}


// Whether a living graph holds the leaf's gradient accumulator with a stream
// that is not the current one.
inline bool leaf_of_another_stream(const Tensor& leaf) {
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!accumulator || !leaf.is_cuda()) return false;
    const auto stream = accumulator->stream();
    // by number: the two sides name the device's type differently on ROCm
    return stream && stream->id() != c10::hip::getCurrentHIPStream(leaf.device().index()).id();
}

// Whether the backward from `node` on reaches such a leaf, over whatever operators.
// During a backward, along the nodes that it runs alone: the others hand nothing over.
inline bool reaches_leaf_of_another_stream(const torch::autograd::Node* node) {
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

inline bool backward_reaches_leaf_of_another_stream(const Tensor& output) {
    const auto& node = output.grad_fn();
    return node && reaches_leaf_of_another_stream(node.get());
}

// In a capture: torch hands a leaf's gradient over on the stream that the leaf's
// accumulator was made on. Where a living graph of another stream holds it, that
// stream joins the capture and the capture's end ends the process.
// Gradients without memory (meta and fake tensors) are in no capture, and may be of
// a device that is not there.
inline void refuse_foreign_leaves(const torch::autograd::Node* node, const Tensors& grads, const char* what) {
    bool there = false;
    for (const Tensor& g : grads) there |= g.defined() && g.is_cuda() && !g.unsafeGetTensorImpl()->is_python_dispatch();
    if (!there || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    TORCH_CHECK(!reaches_leaf_of_another_stream(node),
                "beamgrad_amd.", what, ": a captured backward reaches a leaf that a living graph of another "
                "stream uses; drop that graph (its outputs and losses) before the capture");
}

}  // namespace beamgrad_torch
