// SPDX-License-Identifier: MIT
//
// The torch.ops.beamgrad operators of rotary positions (include/beamgrad_state.h
// has the C entry). Part of beamgrad_amd._C_hip; checks as in torch_state.cpp.
#include "torch_state.hpp"

namespace {

using namespace beamgrad_torch;

constexpr int64_t kMaxDim = 1024, kMaxHeads = 65536;

struct Form {
    bool interleaved;
    double scale;
    bool inverse;
};

void check_rotary(const Tensors& heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, double scale) {
    TORCH_CHECK_VALUE(positions.dim() == 2 && index_type(positions),
                      "positions must be an int32 or int64 [S, N] tensor, got ", positions.scalar_type(), " ", positions.sizes());
    const int64_t S = positions.size(0), N = positions.size(1);
    TORCH_CHECK_VALUE(positions.numel() < int64_t{1} << 26, "positions must have fewer than 2**26 tokens, got ", positions.sizes());
    TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.numel() > 0 && frequencies.device() == positions.device() &&
                          (frequencies.scalar_type() == torch::kFloat64 || frequencies.scalar_type() == torch::kFloat32),
                      "frequencies must be a float64 or float32 [pairs] tensor on the positions' device, got ", frequencies.scalar_type(), " ",
                      frequencies.sizes(), " on ", frequencies.device());
    for (size_t i = 0; i < heads.size(); ++i) {
        const Tensor& t = heads[i];
        TORCH_CHECK_VALUE(t.dim() == 4 && t.size(0) == S && t.size(1) == N && t.size(2) > 0 && t.size(3) > 0, "tensors[", i, "] must be [S, N, H, D] = [", S, ", ", N,
                          ", H, D], got ", t.sizes());
        data_type(t, "tensors");
        TORCH_CHECK_VALUE(t.scalar_type() == heads[0].scalar_type(), "tensors must have one type, got ", heads[0].scalar_type(), " and ",
                          t.scalar_type());
        TORCH_CHECK_VALUE(t.device() == positions.device(), "tensors[", i, "] is on ", t.device(), ", positions on ", positions.device());
        TORCH_CHECK_VALUE(2 * frequencies.numel() <= t.size(3) && t.size(3) <= kMaxDim, "the heads of tensors[", i, "] must be from ",
                          2 * frequencies.numel(), " (two for each frequency) to ", kMaxDim, " wide, got ", t.size(3));
        TORCH_CHECK_VALUE(t.size(2) <= kMaxHeads, "tensors[", i, "] must have at most ", kMaxHeads, " heads, got ", t.size(2));
        for (int64_t d = 0; d < 3; ++d)
            TORCH_CHECK_VALUE(t.size(d) == 1 || t.stride(d) <= int64_t{1} << 40, "tensors[", i, "]'s strides are too large: ", t.strides());
    }
    if (counts) check_index(*counts, {S}, positions, "counts");
    TORCH_CHECK_VALUE(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), "scale must be finite, got ", scale);
}

void check_inplace(const Tensors& heads) {
    for (size_t i = 0; i < heads.size(); ++i)
        TORCH_CHECK_VALUE(heads[i].size(3) == 1 || heads[i].stride(3) == 1, "the heads of tensors[", i, "] must be contiguous to be turned in place");
}

int run_rotary(const Tensors& from, const Tensors& to, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, const Form& form) {
    constexpr unsigned kUsual = 4;  // tensors without memory of their own (small calls take as long as their host work)
    const size_t count = from.size();
    c10::SmallVector<const void*, kUsual> source(count);
    c10::SmallVector<void*, kUsual> target(count);
    c10::SmallVector<int32_t, kUsual> heads(count), dims(count);
    c10::SmallVector<int64_t, 3 * kUsual> source_strides(3 * count), target_strides(3 * count);
    for (size_t i = 0; i < count; ++i) {
        source[i] = from[i].const_data_ptr();
        target[i] = to[i].data_ptr();
        heads[i] = narrow(from[i].size(2));
        dims[i] = narrow(from[i].size(3));
        strides_of(from[i], &source_strides[3 * i]);
        strides_of(to[i], &target_strides[3 * i]);
    }
    const bool ready = frequencies.scalar_type() == torch::kFloat64 && frequencies.is_contiguous();
    const Tensor f = ready ? frequencies : frequencies.to(torch::kFloat64).contiguous(), n = counts ? as_i32(*counts) : Tensor();
    BeamgradRotary a{};
    a.from = source.data();
    a.to = target.data();
    a.heads = heads.data();
    a.head_dim = dims.data();
    a.from_strides = source_strides.data();
    a.to_strides = target_strides.data();
    a.n = narrow(static_cast<int64_t>(count));
    a.data_type = data_type(from[0], "tensors");
    a.sequences = narrow(positions.size(0));
    a.tokens = narrow(positions.size(1));
    a.pairs = narrow(f.numel());
    a.interleaved = form.interleaved;
    a.inverse = form.inverse;
    a.scale = static_cast<float>(form.scale);
    a.positions = positions.const_data_ptr();
    a.position_strides[0] = positions.size(0) == 1 ? 0 : positions.stride(0);
    a.position_strides[1] = positions.size(1) == 1 ? 0 : positions.stride(1);
    a.positions_i64 = positions.scalar_type() == torch::kInt64;
    a.frequencies = f.const_data_ptr<double>();
    a.counts = i32(n);
    return beamgrad_rotary(&a, current_stream());
}

Tensors rotary_cpu(Tensors heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, bool, double scale, bool) {
    check_rotary(heads, positions, frequencies, counts, scale);
    refuse_cpu("rotary", positions);
}

Tensors rotary_hip(Tensors heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, bool interleaved, double scale,
                   bool inverse) {
    check_rotary(heads, positions, frequencies, counts, scale);
    if (heads.empty()) return {};
    const at::OptionalDeviceGuard guard(positions.device());
    Tensors out;
    for (Tensor& t : heads) {
        if (t.size(3) != 1 && t.stride(3) != 1) t = t.contiguous();
        out.push_back(fresh(t.sizes(), t.scalar_type(), t));
    }
    if (positions.numel() == 0) return out;
    check_status(run_rotary(heads, out, positions, frequencies, counts, {interleaved, scale, inverse}), "rotary");
    return out;
}

void rotary_inplace_cpu(Tensors heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, bool, double scale, bool) {
    check_rotary(heads, positions, frequencies, counts, scale);
    check_inplace(heads);
    refuse_cpu("rotary_", positions);
}

void rotary_inplace_hip(Tensors heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, bool interleaved, double scale,
                        bool inverse) {
    check_rotary(heads, positions, frequencies, counts, scale);
    check_inplace(heads);
    if (heads.empty() || positions.numel() == 0) return;
    const at::OptionalDeviceGuard guard(positions.device());
    const int status = run_rotary(heads, heads, positions, frequencies, counts, {interleaved, scale, inverse});
    TORCH_CHECK_VALUE(status != DBS_CUDA_STATUS_INVALID_ARGUMENT,
                      "tensors that are turned in place must share no memory (of one whose sequences, tokens and heads lie in three unrelated steps, "
                      "what lies between the rows of the smallest step counts as its own)");
    check_status(status, "rotary");
    written(heads);
}

Tensors call_rotary(const Tensors& heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, const Form& form) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("beamgrad::rotary", "")
                               .typed<Tensors(Tensors, const Tensor&, const Tensor&, const OptTensor&, bool, double, bool)>();
    return op.call(heads, positions, frequencies, counts, form.interleaved, form.scale, form.inverse);
}

// The gradient is the operator itself by the angles' negatives; it records in its
// turn where a graph of the backward is made.
class RotaryNode : public torch::autograd::Node {
   public:
    RotaryNode(const Tensors& inputs, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, const Form& form)
        : Node(torch::autograd::collect_next_edges(inputs)), positions_(positions, false), frequencies_(frequencies, false),
          counts_(counts, false), form_(form) {}

    std::string name() const override { return "RotaryBackward"; }
    void release_variables() override {
        positions_.reset_data();
        frequencies_.reset_data();
        counts_.reset_data();
    }

   protected:
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        refuse_foreign_leaves(this, grads, "rotary");
        const Tensor positions = positions_.unpack(), frequencies = frequencies_.unpack(), counts = counts_.unpack();
        Tensors some;
        std::vector<size_t> at;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined() && task_should_compute_output(i)) {
                some.push_back(grads[i]);
                at.push_back(i);
            }
        torch::autograd::variable_list out(grads.size());
        if (some.empty()) return out;
        Form form = form_;
        form.inverse = !form.inverse;
        const Tensors got = call_rotary(some, positions, frequencies, counts.defined() ? OptTensor(counts) : OptTensor(), form);
        for (size_t i = 0; i < at.size(); ++i) out[at[i]] = got[i];
        return out;
    }

   private:
    torch::autograd::SavedVariable positions_, frequencies_, counts_;
    Form form_;
};

Tensors rotary_autograd(Tensors heads, const Tensor& positions, const Tensor& frequencies, const OptTensor& counts, bool interleaved, double scale,
                        bool inverse) {
    const Form form{interleaved, scale, inverse};
    TORCH_CHECK(!(at::GradMode::is_enabled() && frequencies.requires_grad()), "beamgrad_amd.rotary has no gradient of its frequencies");
    TORCH_CHECK(!torch::autograd::isFwGradDefined(frequencies), "beamgrad_amd.rotary has no derivative of its frequencies");
    Tensors taking, tangents;
    std::vector<size_t> moving;
    for (size_t i = 0; i < heads.size(); ++i) {
        if (at::GradMode::is_enabled() && heads[i].requires_grad()) taking.push_back(heads[i]);
        if (torch::autograd::isFwGradDefined(heads[i])) {
            tangents.push_back(heads[i]._fw_grad(/*level=*/0));
            moving.push_back(i);
        }
    }
    std::shared_ptr<RotaryNode> node;
    if (!taking.empty())
        node = std::shared_ptr<RotaryNode>(new RotaryNode(taking, positions, frequencies, counts, form), torch::autograd::deleteNode);
    Tensors out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = call_rotary(heads, positions, frequencies, counts, form);
    }
    if (node)
        for (size_t i = 0; i < heads.size(); ++i)
            if (heads[i].requires_grad()) torch::autograd::set_history(out[i], node);
    if (!tangents.empty()) {
        // the map is linear: a tangent turns as its primal does
        const Tensors turned = call_rotary(tangents, positions, frequencies, counts, form);
        for (size_t i = 0; i < moving.size(); ++i) out[moving[i]]._set_fw_grad(turned[i], /*level=*/0, /*is_inplace_op=*/false);
    }
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(beamgrad, m) {
    m.def(
        "rotary(Tensor[] tensors, Tensor positions, Tensor frequencies, Tensor? counts, bool interleaved, float scale, bool inverse) -> Tensor[]");
    m.def(
        "rotary_(Tensor(a!)[] tensors, Tensor positions, Tensor frequencies, Tensor? counts, bool interleaved, float scale, bool inverse) -> ()");
}

TORCH_LIBRARY_IMPL(beamgrad, CUDA, m) {
    m.impl("rotary", &rotary_hip);
    m.impl("rotary_", &rotary_inplace_hip);
}

TORCH_LIBRARY_IMPL(beamgrad, Autograd, m) {
    m.impl("rotary", &rotary_autograd);
    m.impl("rotary_", torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}

// Checked, then refused.
TORCH_LIBRARY_IMPL(beamgrad, CPU, m) {
    m.impl("rotary", &rotary_cpu);
    m.impl("rotary_", &rotary_inplace_cpu);
}
