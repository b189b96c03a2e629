// torch operators of the block: torch.ops.mops.embedding_lookup, grouped_matrix_product and gated_residual_norm, with
// their gradients (first derivatives; second ones are refused). CUDA tensors of float32, float64, float16 or bfloat16. Rows may lie apart
// (any strides but that of the last dimension); anything else is made contiguous. Kernels run on torch's current stream of the tensors'
// device without synchronising it, so an index out of range is not reported: its row is zero, and it gives no gradient.
#include "torch_common.hpp"

namespace {

using namespace mops_torch;

void block_types(const tensor_list& tensors) {
    const auto type = tensors[0].scalar_type();
    if (type != torch::kF64 && type != torch::kF32 && type != torch::kF16 && type != torch::kBFloat16) {
        C10_THROW_ERROR(TypeError, "Found dtype " + std::string(tensors[0].dtype().name()) +
                                       ", only float32, float64, float16 and bfloat16 are supported");
    }
    for (const auto& t : tensors) {
        if (t.scalar_type() != type) {
            C10_THROW_ERROR(TypeError, "All floating point tensors must be of the same dtype, found " +
                                           std::string(t.dtype().name()) + " and " +
                                           std::string(tensors[0].dtype().name()));
        }
    }
}

// A tensor as an array of the C ABI; no data for one that is not defined.
mops_b200_array_t array(const Tensor& t) {
    mops_b200_array_t a{};
    if (!t.defined()) return a;
    a.data = t.data_ptr();
    switch (t.scalar_type()) {
    case torch::kF64: a.type = MOPS_B200_F64; break;
    case torch::kF16: a.type = MOPS_B200_F16; break;
    case torch::kBFloat16: a.type = MOPS_B200_BF16; break;
    case torch::kI32: a.type = MOPS_B200_I32; break;
    default: a.type = MOPS_B200_F32;
    }
    a.dimensions = static_cast<int32_t>(t.dim());
    for (int64_t d = 0; d < t.dim(); d++) {
        a.shape[d] = t.size(d);
        a.stride[d] = t.stride(d);
    }
    return a;
}

// The tensor itself where the values of a row are neighbours, else a contiguous copy.
Tensor rows_of(const Tensor& t) {
    const int64_t last = t.dim() - 1;
    if (t.is_neg() || t.is_conj()) return t.resolve_neg().resolve_conj().contiguous();
    return t.stride(last) == 1 || t.size(last) <= 1 ? t : t.contiguous();
}

void checked(int status) {
    if (status != 0) throw std::runtime_error(mops_get_last_error_message());
}

Tensor empty_if(bool wanted, at::IntArrayRef sizes, const Tensor& like) {
    return wanted ? torch::empty(sizes, like.options()) : Tensor();
}

// Gradients that were not asked for are placeholders on their way out of a Function (its callers ask which they wanted).
tensor_list all_defined(tensor_list gradients, const Tensor& like) {
    for (auto& g : gradients) g = defined(g, like);
    return gradients;
}
Tensor if_needed(const Tensor& t, bool needed) { return needed ? t : Tensor(); }

// The gradients `run(args...)`; where this backward pass is itself recorded, or an argument has a forward-mode tangent, through a Function, which
// refuses to be differentiated.
template <typename Backward, typename... Args>
tensor_list first_derivative(const tensor_list& differentiable, const Args&... args) {
    bool tangent = false;
    for (const auto& t : differentiable) tangent |= t.defined() && t._fw_grad(/*level=*/0).defined();
    return at::GradMode::is_enabled() || tangent ? Backward::apply(args...) : Backward::run(args...);
}

// Whether a call leaves something to differentiate (or to refuse to). What does not, goes without a Function, whose node and saved variables take
// the host as long as the rest of a call.
bool differentiated(std::initializer_list<const Tensor*> arguments) {
    const bool recorded = at::GradMode::is_enabled();
    for (const Tensor* t : arguments)
        if (t->defined() && ((recorded && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
    return false;
}

// ====================================================================== embedding_lookup
// Arguments are replaced by what the kernels take.
Tensor run_embedding_lookup(Tensor& W, Tensor& indices, double scale, int64_t padding_index) {
    static constexpr const char* op = "embedding_lookup";
    same_device({W, indices});
    block_types({W});
    int32_indices({indices});
    ndim(W, 2, "W", op);
    ndim(indices, 1, "indices", op);
    cuda_only(W, op);
    if (padding_index < -1 || padding_index >= W.size(0))
        C10_THROW_ERROR(ValueError, "padding_index " + std::to_string(padding_index) + " is not a row of W in " + op);
    W = rows_of(W);
    indices = indices.contiguous();
    Tensor output = torch::empty({indices.size(0), W.size(1)}, W.options());
    on_stream_of(W, [&] { checked(mops_b200_cuda_embedding_lookup(array(output), array(W), array(indices), scale)); });
    return output;
}

struct EmbeddingLookupBackward : torch::autograd::Function<EmbeddingLookupBackward> {
    static tensor_list run(const Tensor& grad_output, const Tensor& indices, int64_t rows, double scale, int64_t padding_index) {
        Tensor grad_W = torch::empty({rows, grad_output.size(1)}, grad_output.options());
        on_stream_of(grad_output, [&] {
            checked(mops_b200_cuda_embedding_lookup_vjp(array(grad_W), array(grad_output), array(indices), scale,
                                                        padding_index));
        });
        return {grad_W};
    }
    static tensor_list forward(AutogradContext*, Tensor grad_output, Tensor indices, int64_t rows, double scale,
                               int64_t padding_index) {
        return run(grad_output, indices, rows, scale, padding_index);
    }
    static tensor_list backward(AutogradContext*, tensor_list) { no_second_derivative("embedding_lookup"); }
};

struct EmbeddingLookup : torch::autograd::Function<EmbeddingLookup> {
    static Tensor forward(AutogradContext* ctx, Tensor W, Tensor indices, double scale, int64_t padding_index) {
        Tensor output = run_embedding_lookup(W, indices, scale, padding_index);
        ctx->save_for_backward({indices});
        ctx->saved_data["rows"] = W.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding_index"] = padding_index;
        return output;
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        if (!ctx->needs_input_grad(0)) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const Tensor grad_output = rows_of(grads[0]);
        auto r = first_derivative<EmbeddingLookupBackward>(
            {grad_output}, grad_output, ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
            ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding_index"].toInt());
        return {r[0], Tensor(), Tensor(), Tensor()};
    }
};

// ================================================================ grouped_matrix_product
// The matrices as they are where one of their dimensions lies value by value in memory, else a contiguous copy.
Tensor matrices_of(const Tensor& W) {
    if (W.is_neg() || W.is_conj()) return W.resolve_neg().resolve_conj().contiguous();
    return W.stride(2) == 1 || W.stride(1) == 1 ? W : W.contiguous();
}

Tensor run_grouped_matrix_product(Tensor& A, Tensor& W, Tensor& offsets) {
    static constexpr const char* op = "grouped_matrix_product";
    same_device({A, W, offsets});
    block_types({A, W});
    int32_indices({offsets});
    ndim(A, 2, "A", op);
    ndim(W, 3, "W", op);
    ndim(offsets, 1, "offsets", op);
    cuda_only(A, op);
    A = rows_of(A);
    W = matrices_of(W);
    offsets = offsets.contiguous();
    Tensor output = torch::empty({A.size(0), W.size(2)}, A.options());
    on_stream_of(A, [&] { checked(mops_b200_cuda_grouped_matrix_product(array(output), array(A), array(W), array(offsets))); });
    return output;
}

struct GroupedMatrixProductBackward : torch::autograd::Function<GroupedMatrixProductBackward> {
    static tensor_list run(const Tensor& grad_output, const Tensor& A, const Tensor& W, const Tensor& offsets, bool need_A,
                           bool need_W) {
        Tensor grad_A = empty_if(need_A, A.sizes(), A), grad_W;
        if (need_W) // stored the way round that W is
            grad_W = W.stride(2) == 1 ? torch::empty(W.sizes(), W.options())
                                      : torch::empty({W.size(0), W.size(2), W.size(1)}, W.options()).transpose(1, 2);
        on_stream_of(A, [&] {
            checked(mops_b200_cuda_grouped_matrix_product_vjp(array(grad_A), array(grad_W), array(grad_output), array(A),
                                                              array(W), array(offsets)));
        });
        return {grad_A, grad_W};
    }
    static tensor_list forward(AutogradContext*, Tensor grad_output, Tensor A, Tensor W, Tensor offsets, bool need_A,
                               bool need_W) {
        return all_defined(run(grad_output, A, W, offsets, need_A, need_W), A);
    }
    static tensor_list backward(AutogradContext*, tensor_list) { no_second_derivative("grouped_matrix_product"); }
};

struct GroupedMatrixProduct : torch::autograd::Function<GroupedMatrixProduct> {
    static Tensor forward(AutogradContext* ctx, Tensor A, Tensor W, Tensor offsets) {
        Tensor output = run_grouped_matrix_product(A, W, offsets);
        ctx->save_for_backward({A, W, offsets});
        return output;
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        auto s = ctx->get_saved_variables();
        const Tensor grad_output = rows_of(grads[0]);
        auto r = first_derivative<GroupedMatrixProductBackward>({grad_output, s[0], s[1]}, grad_output, s[0], s[1], s[2],
                                                                ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        return {if_needed(r[0], ctx->needs_input_grad(0)), if_needed(r[1], ctx->needs_input_grad(1)), Tensor()};
    }
};

// =================================================================== gated_residual_norm
// (gate: none if it is not defined)
tensor_list run_gated_residual_norm(Tensor& residual, Tensor& branch, Tensor& gate, Tensor& scale, Tensor& weight_branch, Tensor& weight_output,
                                    double epsilon) {
    static constexpr const char* op = "gated_residual_norm";
    tensor_list all = {residual, branch, scale, weight_branch, weight_output};
    if (gate.defined()) all.push_back(gate);
    same_device(all);
    block_types(all);
    ndim(residual, 2, "residual", op);
    ndim(branch, 2, "branch", op);
    if (gate.defined()) ndim(gate, 2, "gate", op);
    ndim(scale, 1, "scale", op);
    ndim(weight_branch, 1, "weight_branch", op);
    ndim(weight_output, 1, "weight_output", op);
    cuda_only(residual, op);
    for (Tensor* t : {&residual, &branch, &scale, &weight_branch, &weight_output}) *t = rows_of(*t);
    if (gate.defined()) gate = rows_of(gate);
    Tensor stream = torch::empty(residual.sizes(), residual.options()), normed = torch::empty(residual.sizes(), residual.options());
    on_stream_of(residual, [&] {
        checked(mops_b200_cuda_gated_residual_norm(array(stream), array(normed), array(residual), array(branch), array(gate), array(scale),
                                                   array(weight_branch), array(weight_output), epsilon));
    });
    return {stream, normed};
}

struct GatedResidualNormBackward : torch::autograd::Function<GatedResidualNormBackward> {
    // need: one bit for each input, in order
    static tensor_list run(const Tensor& grad_stream, const Tensor& grad_normed, const Tensor& residual, const Tensor& branch,
                           const std::optional<Tensor>& optional_gate, const Tensor& scale, const Tensor& weight_branch,
                           const Tensor& weight_output, double epsilon, int64_t need) {
        const Tensor gate = optional_gate.value_or(Tensor());
        const Tensor* inputs[] = {&residual, &branch, &gate, &scale, &weight_branch, &weight_output};
        tensor_list r;
        for (int i = 0; i < 6; i++) r.push_back(need >> i & 1 ? torch::empty(inputs[i]->sizes(), residual.options()) : Tensor());
        on_stream_of(residual, [&] {
            checked(mops_b200_cuda_gated_residual_norm_vjp(
                array(r[0]), array(r[1]), array(r[2]), array(r[3]), array(r[4]), array(r[5]), array(grad_stream),
                array(grad_normed), array(residual), array(branch), array(gate), array(scale), array(weight_branch),
                array(weight_output), epsilon));
        });
        return r;
    }
    static tensor_list forward(AutogradContext*, Tensor grad_stream, Tensor grad_normed, Tensor residual, Tensor branch,
                               std::optional<Tensor> gate, Tensor scale, Tensor weight_branch, Tensor weight_output,
                               double epsilon, int64_t need) {
        return all_defined(run(grad_stream, grad_normed, residual, branch, gate, scale, weight_branch, weight_output, epsilon,
                               need),
                           residual);
    }
    static tensor_list backward(AutogradContext*, tensor_list) { no_second_derivative("gated_residual_norm"); }
};

struct GatedResidualNorm : torch::autograd::Function<GatedResidualNorm> {
    static tensor_list forward(AutogradContext* ctx, Tensor residual, Tensor branch, std::optional<Tensor> optional_gate,
                               Tensor scale, Tensor weight_branch, Tensor weight_output, double epsilon) {
        Tensor gate = optional_gate.value_or(Tensor());
        tensor_list r = run_gated_residual_norm(residual, branch, gate, scale, weight_branch, weight_output, epsilon);
        ctx->save_for_backward({residual, branch, gate, scale, weight_branch, weight_output});
        ctx->saved_data["epsilon"] = epsilon;
        return r;
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        auto s = ctx->get_saved_variables();
        const Tensor grad_stream = rows_of(grads[0]), grad_normed = rows_of(grads[1]);
        int64_t need = 0;
        size_t at = 0; // (a gate that was not given is not counted)
        for (int i = 0; i < 6; i++)
            if (s[i].defined() && ctx->needs_input_grad(at++)) need |= int64_t(1) << i;
        const std::optional<Tensor> gate = s[2].defined() ? std::optional<Tensor>(s[2]) : std::nullopt;
        auto r = first_derivative<GatedResidualNormBackward>(
            {grad_stream, grad_normed, s[0], s[1], s[2], s[3], s[4], s[5]}, grad_stream, grad_normed, s[0], s[1], gate, s[3],
            s[4], s[5], ctx->saved_data["epsilon"].toDouble(), need);
        tensor_list all;
        for (int i = 0; i < 6; i++) all.push_back(if_needed(r[i], need >> i & 1));
        all.push_back(Tensor());
        return all;
    }
};

// ------------------------------------------------------------------ registered entry points
Tensor embedding_lookup(Tensor W, Tensor indices, double scale, int64_t padding_index) {
    return differentiated({&W}) ? EmbeddingLookup::apply(W, indices, scale, padding_index)
                                : run_embedding_lookup(W, indices, scale, padding_index);
}

Tensor grouped_matrix_product(Tensor A, Tensor W, Tensor offsets) {
    return differentiated({&A, &W}) ? GroupedMatrixProduct::apply(A, W, offsets) : run_grouped_matrix_product(A, W, offsets);
}

std::tuple<Tensor, Tensor> gated_residual_norm(Tensor residual, Tensor branch, std::optional<Tensor> gate, Tensor scale,
                                               Tensor weight_branch, Tensor weight_output, double epsilon) {
    Tensor given = gate.value_or(Tensor());
    auto r = differentiated({&residual, &branch, &given, &scale, &weight_branch, &weight_output})
                 ? GatedResidualNorm::apply(residual, branch, gate, scale, weight_branch, weight_output, epsilon)
                 : run_gated_residual_norm(residual, branch, given, scale, weight_branch, weight_output, epsilon);
    return {r[0], r[1]};
}

} // namespace

TORCH_LIBRARY_FRAGMENT(mops, m) {
    m.def("embedding_lookup(Tensor W, Tensor indices, float scale=1.0, int padding_index=-1) -> Tensor", embedding_lookup);
    m.def("grouped_matrix_product(Tensor A, Tensor W, Tensor offsets) -> Tensor", grouped_matrix_product);
    m.def("gated_residual_norm(Tensor residual, Tensor branch, Tensor? gate, Tensor scale, Tensor weight_branch, "
          "Tensor weight_output, float epsilon=1e-6) -> (Tensor, Tensor)",
          gated_residual_norm);
}
