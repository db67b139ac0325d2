// SPDX-License-Identifier: MIT
//
// The torch.ops.beamgrad operators of a model's state in a search: attention
// over a paged cache, its pages, eviction from it, reordering of dense states
// (include/beamgrad_state.h has the C entries). Part of beamgrad_amd._C_hip.
//
// Every operator checks its arguments in one function that needs no GPU. The
// CPU key runs the checks and then refuses the call, so a wrong argument has its
// message wherever the tensors are. Nothing is read back and nothing waits:
// page tables stay on the device, and the calls can be captured into a graph.
#include "torch_state.hpp"

namespace {

using namespace beamgrad_torch;

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

// Queries whose heads are contiguous and begin at multiples of 16 bytes: q, or a copy.
Tensor aligned_rows(const Tensor& q) {
    const int64_t size = static_cast<int64_t>(q.element_size());
    bool fits = q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) fits = fits && (q.size(d) == 1 || q.stride(d) * size % 16 == 0);
    return fits ? q : q.clone(at::MemoryFormat::Contiguous);
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
    const Tensor query = aligned_rows(q);
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
// Eviction by the attention that tokens got
// ---------------------------------------------------------------------------

void check_weights_shape(const Tensor& w, at::IntArrayRef shape, const Tensor& with, const std::string& name) {
    TORCH_CHECK_VALUE(w.scalar_type() == torch::kFloat32 && w.sizes() == shape && w.device() == with.device(), name, " must be a float32 ", shape,
                      " tensor (sequences, heads, places of a sequence's pages) on the same device, got ", w.scalar_type(), " ", w.sizes(), " on ",
                      w.device());
}

void check_accumulate(const Tensor& weights, const Tensor& q, const Tensor& k, const Tensor& lse, const Tensor& pages, const Tensor& lengths,
                      const OptTensor& parents, const OptTensor& counts, double scale) {
    check_attention(q, k, k, pages, lengths, parents, counts, 1, c10::nullopt, scale);
    check_weights_shape(weights, {q.size(0), k.size(2), pages.size(1) * k.size(1)}, q, "weights");
    TORCH_CHECK_VALUE(weights.size(2) == 1 || weights.stride(2) == 1, "weights' places must be contiguous, got strides ", weights.strides());
    const auto nested = [&](int64_t inner, int64_t outer) {  // one dimension's places lie apart, and all of them along the other
        const int64_t run = (weights.size(inner) - 1) * weights.stride(inner) + weights.size(2);
        return (weights.size(inner) == 1 || weights.stride(inner) >= weights.size(2)) && (weights.size(outer) == 1 || weights.stride(outer) >= run);
    };
    TORCH_CHECK_VALUE(nested(1, 0) || nested(0, 1), "weights' sequences and heads overlap, got strides ", weights.strides());
    TORCH_CHECK_VALUE(lse.scalar_type() == torch::kFloat32 && lse.sizes() == q.sizes().slice(0, 3) && lse.device() == q.device(),
                      "lse must be a float32 ", q.sizes().slice(0, 3), " tensor on q's device, got ", lse.scalar_type(), " ", lse.sizes(), " on ",
                      lse.device());
    TORCH_CHECK_VALUE(k.size(2) <= 65535, "a cache must have at most 65535 heads, got ", k.size(2));
}

void accumulate_weights_cpu(const Tensor& weights, const Tensor& q, const Tensor& k, const Tensor& lse, const Tensor& pages, const Tensor& lengths,
                            const OptTensor& parents, const OptTensor& counts, double scale) {
    check_accumulate(weights, q, k, lse, pages, lengths, parents, counts, scale);
    refuse_cpu("accumulate_weights", q);
}

void accumulate_weights_hip(const Tensor& weights, const Tensor& q, const Tensor& k, const Tensor& lse, const Tensor& pages, const Tensor& lengths,
                            const OptTensor& parents, const OptTensor& counts, double scale) {
    check_accumulate(weights, q, k, lse, pages, lengths, parents, counts, scale);
    const at::OptionalDeviceGuard guard(q.device());
    const Tensor query = aligned_rows(q), sums = lse.contiguous();
    Tensor par, num;
    if (parents) par = as_i32(*parents);
    if (counts) num = as_i32(*counts);
    BeamgradWeights a{};
    a.q = query.const_data_ptr();
    a.k = k.const_data_ptr();
    a.data_type = data_type(q, "q");
    a.sequences = narrow(q.size(0));
    a.tokens = narrow(q.size(1));
    a.heads = narrow(q.size(2));
    a.kv_heads = narrow(k.size(2));
    a.head_dim = narrow(q.size(3));
    a.page_tokens = narrow(k.size(1));
    a.n_pages = narrow(k.size(0));
    a.table_pages = narrow(pages.size(1));
    a.scale = static_cast<float>(scale);
    strides_of(query, a.q_strides);
    strides_of(k, a.k_strides);
    for (int d = 0; d < 2; ++d) a.weight_strides[d] = weights.size(d) == 1 ? 0 : weights.stride(d);
    a.pages = i32(pages);
    a.lengths = i32(lengths);
    a.counts = i32(num);
    a.parents = i32(par);
    a.lse = sums.const_data_ptr<float>();
    a.weights = weights.data_ptr<float>();
    const int64_t bytes = beamgrad_accumulate_weights_workspace_size(&a);
    Tensor ws;
    if (bytes != 0) ws = workspace(bytes, q);
    const int status = beamgrad_accumulate_weights(&a, bytes != 0 ? ws.data_ptr() : nullptr, bytes, current_stream());
    TORCH_CHECK_VALUE(status != DBS_CUDA_STATUS_INVALID_ARGUMENT, "weights must share no memory with q, k or lse");
    check_status(status, "accumulate_weights");
    written({weights});
}

using EvictOut = std::tuple<Tensor, Tensor, Tensor, Tensors>;

void check_evict(const Tensors& pools, const Tensors& weights, const Tensor& pages, const Tensor& lengths, const Tensor& refs,
                 const OptTensor& budgets, int64_t budget, int64_t recent, int64_t first) {
    check_table(pages, lengths, refs);
    TORCH_CHECK_VALUE(!pools.empty(), "pools must hold at least one pool");
    check_pools(pools, pages, refs.numel());
    TORCH_CHECK_VALUE(!weights.empty() && pools.size() % weights.size() == 0, "the pools must be a multiple of the weights, and those at least one, got ",
                      pools.size(), " and ", weights.size());
    TORCH_CHECK_VALUE(weights[0].dim() == 3 && weights[0].size(1) >= 1 && weights[0].size(1) <= 1024, "weights[0] must be [S, heads, places], got ",
                      weights[0].sizes());
    const int64_t S = pages.size(0), G = weights[0].size(1), places = pages.size(1) * pools[0].size(1);
    TORCH_CHECK_VALUE(S <= 65535, "a table must have at most 65535 sequences for evict_tokens, got ", S);
    for (size_t i = 0; i < weights.size(); ++i) {
        check_weights_shape(weights[i], {S, G, places}, pages, "weights[" + std::to_string(i) + "]");
    }
    for (size_t i = 0; i < pools.size(); ++i) {
        TORCH_CHECK_VALUE(G == 1 || pools[i].size(2) == G, "weights of ", G, " heads need pools [pages, tokens of a page, ", G, ", ...], got pools[", i,
                          "] ", pools[i].sizes());
        TORCH_CHECK_VALUE(row_elements(pools[i], 2) * static_cast<int64_t>(pools[i].element_size()) <= 2 << 20, "a token's row of pools[", i,
                          "] must be at most 2 MB, got ", pools[i].sizes());
    }
    if (budgets) check_index(*budgets, {S}, pages, "budget");
    TORCH_CHECK_VALUE(budgets || (budget >= 0 && budget <= kI32Max), "budget must be in [0, 2**31), got ", budget);
    TORCH_CHECK_VALUE(recent >= 0 && recent <= kI32Max, "recent must be in [0, 2**31), got ", recent);
    TORCH_CHECK_VALUE(first >= 0 && first <= kI32Max, "first must be in [0, 2**31), got ", first);
}

EvictOut evict_tokens_cpu(Tensors pools, Tensors weights, const Tensor& pages, const Tensor& lengths, const Tensor& refs,
                          const OptTensor& budgets, int64_t budget, int64_t recent, int64_t first) {
    check_evict(pools, weights, pages, lengths, refs, budgets, budget, recent, first);
    check_pools_apart(pools, {});
    refuse_cpu("evict_tokens", pages);
}

EvictOut evict_tokens_hip(Tensors pools, Tensors weights, const Tensor& pages, const Tensor& lengths, const Tensor& refs, const OptTensor& budgets,
                          int64_t budget, int64_t recent, int64_t first) {
    check_evict(pools, weights, pages, lengths, refs, budgets, budget, recent, first);
    const at::OptionalDeviceGuard guard(pages.device());
    const Tensor most = budgets ? as_i32(*budgets) : Tensor();
    const Pools p = bind_pools(pools, refs.numel(), pools[0].size(1));
    Tensors out;
    std::vector<const float*> source;
    std::vector<float*> target;
    std::vector<int64_t> strides;
    for (Tensor& w : weights) {
        if (w.size(2) != 1 && w.stride(2) != 1) w = w.contiguous();
        out.push_back(fresh(w.sizes(), torch::kFloat32, w));
        source.push_back(w.const_data_ptr<float>());
        target.push_back(out.back().data_ptr<float>());
        for (int d = 0; d < 2; ++d) strides.push_back(w.size(d) == 1 ? 0 : w.stride(d));
    }
    BeamgradEviction a{};
    a.weights = source.data();
    a.weight_strides = strides.data();
    a.to_weights = target.data();
    a.n_weights = narrow(static_cast<int64_t>(weights.size()));
    a.heads = narrow(weights[0].size(1));
    a.budgets = i32(most);
    a.budget = narrow(budget);
    a.recent = narrow(recent);
    a.first = narrow(first);
    NewTable to(pages, lengths, refs);
    const BeamgradTable from = bind_table(pages, lengths, refs), table = to.bind();
    const int64_t bytes = beamgrad_evict_tokens_workspace_size(&p.c, &a, narrow(pages.size(0)), narrow(pages.size(1)));
    const Tensor ws = workspace(bytes, pages);
    const int status = beamgrad_evict_tokens(&p.c, &a, &from, narrow(pages.size(0)), narrow(pages.size(1)), &table, ws.data_ptr(), bytes, current_stream());
    if (status == DBS_CUDA_STATUS_INVALID_ARGUMENT) check_pools_apart(pools, {});
    check_status(status, "evict_tokens");
    written(pools);
    return {std::move(to.pages), std::move(to.lengths), std::move(to.refs), std::move(out)};
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
        refuse_foreign_leaves(this, grads, "reorder_states");
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
    m.def(
        "accumulate_weights(Tensor(a!) weights, Tensor q, Tensor k, Tensor lse, Tensor pages, Tensor lengths, Tensor? parents, "
        "Tensor? counts, float scale) -> ()");
    m.def(
        "evict_tokens(Tensor(a!)[] pools, Tensor[] weights, Tensor pages, Tensor lengths, Tensor refs, Tensor? budgets, int budget, "
        "int recent, int first) -> (Tensor, Tensor, Tensor, Tensor[])");
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
    m.impl("accumulate_weights", &accumulate_weights_hip);
    m.impl("evict_tokens", &evict_tokens_hip);
    m.impl("reorder_states", &reorder_states_hip);
    m.impl("reorder_states_", &reorder_states_inplace_hip);
    m.impl("reorder_states_backward", &reorder_states_backward_hip);
}

TORCH_LIBRARY_IMPL(beamgrad, Autograd, m) {
    m.impl("reorder_states", &reorder_states_autograd);
    m.impl("reorder_states_backward", &reorder_states_backward_autograd);
    for (const char* name : {"tree_attention", "fork_pages", "write_tokens", "keep_tokens", "accumulate_weights", "evict_tokens", "reorder_states_"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}

// Checked, then refused.
TORCH_LIBRARY_IMPL(beamgrad, CPU, m) {
    m.impl("tree_attention", &tree_attention_cpu);
    m.impl("fork_pages", &fork_pages_cpu);
    m.impl("extend_pages", &extend_pages_cpu);
    m.impl("write_tokens", &write_tokens_cpu);
    m.impl("keep_tokens", &keep_tokens_cpu);
    m.impl("accumulate_weights", &accumulate_weights_cpu);
    m.impl("evict_tokens", &evict_tokens_cpu);
    m.impl("reorder_states", &reorder_states_cpu);
    m.impl("reorder_states_", &reorder_states_inplace_cpu);
    m.impl("reorder_states_backward", &reorder_states_backward_cpu);
}
