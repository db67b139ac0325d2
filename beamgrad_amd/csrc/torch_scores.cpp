// SPDX-License-Identifier: MIT
//
// The torch.ops.beamgrad operator of log-probabilities of given tokens and its
// gradient (include/beamgrad_score.h has the C entries). Part of beamgrad_amd._C_hip.
//
// As in torch_state.cpp, arguments are checked by functions that need no GPU, the
// CPU key runs the checks and refuses the call, and nothing is read back.
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "beamgrad_score.h"
#include "torch_state.hpp"

namespace {

using namespace beamgrad_torch;
using Outputs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

constexpr int64_t kMaxTop = 64;

void check_scores(const Tensor& logits, const Tensor& tokens, int64_t top) {
    data_type(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, "logits must be a [..., V] tensor, got ", logits.sizes());
    const int64_t V = logits.size(-1);
    TORCH_CHECK_VALUE(V <= int64_t{1} << 30, "logits must have at most 2**30 tokens, got ", V);
    check_index(tokens, logits.sizes().slice(0, static_cast<size_t>(logits.dim() - 1)), logits, "tokens");
    TORCH_CHECK_VALUE(tokens.numel() < int64_t{1} << 24, "logits must have fewer than 2**24 rows, got ", tokens.numel());
    TORCH_CHECK_VALUE(top >= 0 && top <= kMaxTop && top <= V, "top must be in [0, ", std::min(kMaxTop, V), "], got ", top);
}

// The rows of logits as [outer, inner, V]; a copy where their strides are others.
Tensor bind_rows(const Tensor& logits, BeamgradTokenLogprobs& a) {
    const int64_t V = logits.size(-1);
    int64_t n[2] = {1, 1}, stride[2] = {0, 0};
    int levels = 0;
    bool fits = V == 1 || logits.stride(-1) == 1;
    for (int64_t d = logits.dim() - 2; d >= 0 && fits; --d) {  // the inner ones first
        if (logits.size(d) == 1) continue;
        if (levels > 0 && logits.stride(d) == stride[levels - 1] * n[levels - 1]) {
            n[levels - 1] *= logits.size(d);
        } else if (levels == 2) {
            fits = false;
        } else {
            n[levels] = logits.size(d);
            stride[levels++] = logits.stride(d);
        }
    }
    Tensor rows = logits;
    if (!fits) {
        rows = logits.contiguous();
        n[0] = rows.numel() / V, n[1] = 1;
        stride[0] = V, stride[1] = 0;
    }
    a.logits = rows.const_data_ptr();
    a.data_type = data_type(rows, "logits");
    a.outer = narrow(n[1]);
    a.inner = narrow(n[0]);
    a.vocab = narrow(V);
    a.strides[0] = stride[1];
    a.strides[1] = stride[0];
    return rows;
}

std::vector<int64_t> with(const Tensor& tokens, int64_t last) {
    std::vector<int64_t> sizes = tokens.sizes().vec();
    sizes.push_back(last);
    return sizes;
}

Outputs token_logprobs_cpu(const Tensor& logits, const Tensor& tokens, int64_t top, bool, bool) {
    check_scores(logits, tokens, top);
    refuse_cpu("token_logprobs", logits);
}

Outputs token_logprobs_hip(const Tensor& logits, const Tensor& tokens, int64_t top, bool entropy, bool stats) {
    check_scores(logits, tokens, top);
    const at::OptionalDeviceGuard guard(logits.device());
    Tensor lp = fresh(tokens.sizes(), torch::kFloat32, logits);
    Tensor h = entropy ? fresh(tokens.sizes(), torch::kFloat32, logits) : fresh(with(tokens, 0), torch::kFloat32, logits);
    Tensor best = fresh(with(tokens, top), torch::kFloat32, logits), which = fresh(with(tokens, top), torch::kInt64, logits);
    Tensor kept = fresh(with(tokens, stats ? 4 : 0), torch::kFloat32, logits);
    if (tokens.numel() > 0) {
        BeamgradTokenLogprobs a{};
        const Tensor rows = bind_rows(logits, a), ids = tokens.contiguous();
        a.tokens = ids.const_data_ptr();
        a.tokens_i64 = ids.scalar_type() == torch::kInt64;
        a.top = narrow(top);
        a.logprobs = lp.data_ptr<float>();
        a.entropy = entropy ? h.data_ptr<float>() : nullptr;
        a.top_logprobs = top > 0 ? best.data_ptr<float>() : nullptr;
        a.top_tokens = top > 0 ? which.data_ptr<int64_t>() : nullptr;
        a.stats = stats ? kept.data_ptr<float>() : nullptr;
        const int64_t bytes = beamgrad_token_logprobs_workspace_size(&a);
        Tensor ws;
        if (bytes != 0) ws = workspace(bytes, logits);
        check_status(beamgrad_token_logprobs(&a, bytes != 0 ? ws.data_ptr() : nullptr, bytes, current_stream()), "token_logprobs");
    }
    return {std::move(lp), std::move(h), std::move(best), std::move(which), std::move(kept)};
}

void check_gradient(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& top_tokens, const OptTensor& g,
                    const OptTensor& g_entropy, const OptTensor& g_top) {
    const auto shaped = [&](const Tensor& t, const std::vector<int64_t>& sizes, at::ScalarType type, const char* name) {
        TORCH_CHECK_VALUE(t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.device() == logits.device(), name, " must be a ",
                          type, " ", at::IntArrayRef(sizes), " tensor on the logits' device, got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    };
    TORCH_CHECK_VALUE(top_tokens.dim() == tokens.dim() + 1, "top_tokens must have one dimension more than tokens");
    check_scores(logits, tokens, top_tokens.size(-1));
    shaped(top_tokens, with(tokens, top_tokens.size(-1)), torch::kInt64, "top_tokens");
    shaped(stats, with(tokens, 4), torch::kFloat32, "stats");
    if (g) shaped(*g, tokens.sizes().vec(), torch::kFloat32, "grad_logprobs");
    if (g_entropy) shaped(*g_entropy, tokens.sizes().vec(), torch::kFloat32, "grad_entropy");
    if (g_top) shaped(*g_top, with(tokens, top_tokens.size(-1)), torch::kFloat32, "grad_top");
}

Tensor token_logprobs_backward_cpu(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& top_tokens, const OptTensor& g,
                                   const OptTensor& g_entropy, const OptTensor& g_top) {
    check_gradient(logits, tokens, stats, top_tokens, g, g_entropy, g_top);
    refuse_cpu("token_logprobs_backward", logits);
}

Tensor token_logprobs_backward_hip(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& top_tokens, const OptTensor& g,
                                   const OptTensor& g_entropy, const OptTensor& g_top) {
    check_gradient(logits, tokens, stats, top_tokens, g, g_entropy, g_top);
    const at::OptionalDeviceGuard guard(logits.device());
    Tensor out = fresh(logits.sizes(), logits.scalar_type(), logits);
    if (tokens.numel() == 0) return out;
    BeamgradTokenLogprobs a{};
    const Tensor rows = bind_rows(logits, a), ids = tokens.contiguous(), kept = stats.contiguous(), which = top_tokens.contiguous();
    const auto whole = [](const OptTensor& t) { return t ? t->contiguous() : Tensor(); };
    const Tensor g0 = whole(g), g1 = whole(g_entropy), g2 = whole(g_top);
    const auto at = [](const Tensor& t) { return t.defined() && t.numel() > 0 ? t.const_data_ptr<float>() : nullptr; };
    a.tokens = ids.const_data_ptr();
    a.tokens_i64 = ids.scalar_type() == torch::kInt64;
    a.top = narrow(top_tokens.size(-1));
    a.top_tokens = a.top > 0 ? const_cast<int64_t*>(which.const_data_ptr<int64_t>()) : nullptr;
    a.stats = const_cast<float*>(kept.const_data_ptr<float>());
    check_status(beamgrad_token_logprobs_backward(&a, at(g0), at(g1), at(g2), out.data_ptr(), current_stream()), "token_logprobs_backward");
    return out;
}

Outputs call_forward(const Tensor& logits, const Tensor& tokens, int64_t top, bool entropy, bool stats) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("beamgrad::token_logprobs", "")
                               .typed<Outputs(const Tensor&, const Tensor&, int64_t, bool, bool)>();
    return op.call(logits, tokens, top, entropy, stats);
}
Tensor call_backward(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& top_tokens, const OptTensor& g,
                     const OptTensor& g_entropy, const OptTensor& g_top) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("beamgrad::token_logprobs_backward", "")
                               .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                             const OptTensor&)>();
    return op.call(logits, tokens, stats, top_tokens, g, g_entropy, g_top);
}

// The outputs that carry a gradient are the log-probabilities, the entropy (where it
// was asked for) and the alternatives' log-probabilities.
class ScoresNode : public torch::autograd::Node {
   public:
    ScoresNode(const Tensor& logits, const Tensor& tokens, bool entropy)
        : Node(torch::autograd::collect_next_edges(logits)), logits_(logits, false), tokens_(tokens, false), entropy_(entropy) {}
    void keep(const Tensor& stats, const Tensor& top_tokens) {
        stats_ = torch::autograd::SavedVariable(stats, false);
        top_tokens_ = torch::autograd::SavedVariable(top_tokens, false);
    }

    std::string name() const override { return "TokenLogprobsBackward"; }
    void release_variables() override {
        logits_.reset_data();
        tokens_.reset_data();
        stats_.reset_data();
        top_tokens_.reset_data();
    }

   protected:
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        refuse_foreign_leaves(this, grads, "token_logprobs");
        const auto given = [&](size_t i) { return i < grads.size() && grads[i].defined() ? OptTensor(grads[i]) : OptTensor(); };
        const OptTensor g = given(0), g_entropy = entropy_ ? given(1) : OptTensor(), g_top = given(entropy_ ? 2 : 1);
        if (!g && !g_entropy && !g_top) return {Tensor()};
        const Tensor logits = logits_.unpack(), tokens = tokens_.unpack(), stats = stats_.unpack(), top_tokens = top_tokens_.unpack();
        Tensor out;
        {
            const at::NoGradGuard none;
            out = call_backward(logits, tokens, stats, top_tokens, g, g_entropy, g_top);
        }
        if (!at::GradMode::is_enabled()) return {out};
        // a graph of the backward is recorded: one that would be differentiated raises then
        const auto no_second = std::shared_ptr<torch::autograd::DelayedError>(
            new torch::autograd::DelayedError("beamgrad_amd.token_logprobs has no second derivative", 1), torch::autograd::deleteNode);
        return (*no_second)({out.detach().requires_grad_(true)});
    }

   private:
    torch::autograd::SavedVariable logits_, tokens_, stats_, top_tokens_;
    bool entropy_;
};

Outputs token_logprobs_autograd(const Tensor& logits, const Tensor& tokens, int64_t top, bool entropy, bool stats) {
    TORCH_CHECK(!torch::autograd::isFwGradDefined(logits), "beamgrad_amd.token_logprobs has no forward-mode derivative, and would drop "
                "a tensor's tangent: call it on the tensors' primals");
    const bool records = at::GradMode::is_enabled() && logits.requires_grad();
    std::shared_ptr<ScoresNode> node;
    if (records) node = std::shared_ptr<ScoresNode>(new ScoresNode(logits, tokens, entropy), torch::autograd::deleteNode);
    Outputs out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = call_forward(logits, tokens, top, entropy, stats || records);
    }
    if (!records) return out;
    torch::autograd::set_history(std::get<0>(out), node);
    if (entropy) torch::autograd::set_history(std::get<1>(out), node);
    if (top > 0) torch::autograd::set_history(std::get<2>(out), node);
    node->keep(std::get<4>(out), std::get<3>(out));
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(beamgrad, m) {
    m.def("token_logprobs(Tensor logits, Tensor tokens, int top, bool entropy, bool stats) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def(
        "token_logprobs_backward(Tensor logits, Tensor tokens, Tensor stats, Tensor top_tokens, Tensor? grad_logprobs, "
        "Tensor? grad_entropy, Tensor? grad_top) -> Tensor");
}

TORCH_LIBRARY_IMPL(beamgrad, CUDA, m) {
    m.impl("token_logprobs", &token_logprobs_hip);
    m.impl("token_logprobs_backward", &token_logprobs_backward_hip);
}

TORCH_LIBRARY_IMPL(beamgrad, Autograd, m) {
    m.impl("token_logprobs", &token_logprobs_autograd);
    m.impl("token_logprobs_backward", torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}

// Checked, then refused.
TORCH_LIBRARY_IMPL(beamgrad, CPU, m) {
    m.impl("token_logprobs", &token_logprobs_cpu);
    m.impl("token_logprobs_backward", &token_logprobs_backward_cpu);
}
