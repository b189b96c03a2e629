// grouped_gated_product on tensor cores: f16 and bf16 (gated_mma.cu), f32 (gated_split.cu).
#ifndef MOPS_B200_GATED_MMA_HPP
#define MOPS_B200_GATED_MMA_HPP

#include "grouped_mma.hpp"

namespace mops_b200 {

// A (rows x depth) is boxable, so are both halves of W (groups x depth x 2 columns, the last two either way round), each of `columns` columns.
struct GatedProblem {
    Array A, W;
    const int32_t* offsets;
    int64_t groups, rows, depth, columns;
    int32_t activation;
    bool by_columns() const { return W.stride[2] == 1; }
    // The half's first value.
    void* half(int i) const { return static_cast<unsigned char*>(W.data) + i * columns * W.stride[2] * type_bytes(W.type); }
};

// output: rows x columns, or fewer. As vjp: `to` (rows x 2 columns, 16 bits, contiguous, columns a multiple of 8) becomes dU and dV side by side; grad has real_columns
// <= columns of them.
void gated_rows_mma(const Call& call, const GatedProblem& p, const Array& output, const std::string& op);
void gated_rows_vjp_mma(const Call& call, const GatedProblem& p, void* to, const Array& grad, const std::string& op);
// The same of f32; `to` is rows x 2 columns, boxable or not.
void gated_rows_split(const Call& call, const GatedProblem& p, const Array& output, const std::string& op);
void gated_rows_vjp_split(const Call& call, const GatedProblem& p, const Array& to, const Array& grad, const std::string& op);
// grad_A = duv W^T, where that is worth cutting the depth for (few tiles of a long depth); else false.
bool multiply_rows_sliced(const Call& call, const RowsProblem& p, int64_t least, const std::string& op);

} // namespace mops_b200

#endif
