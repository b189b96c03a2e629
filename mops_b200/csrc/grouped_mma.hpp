// grouped_matrix_product on tensor cores (grouped_mma.cu): the problems, and launches that say whether they took one on.
#ifndef MOPS_B200_GROUPED_MMA_HPP
#define MOPS_B200_GROUPED_MMA_HPP

#include "arrays.hpp"

namespace mops_b200 {

// out = X (rows x depth) times, for each group, M (value (d, j) at d * depth_stride + j * column_stride, one of them 1).
struct RowsProblem {
    Array out, X, M;
    int64_t depth_stride, column_stride;
    const int32_t* offsets;
    int64_t groups, rows, depth, columns;
};

// out[g] = X[rows of g]^T Y[rows of g]; out is contiguous. factor, if any: in device memory, for 16-bit results.
struct OuterProblem {
    Array out, X, Y;
    const int32_t* offsets;
    int64_t groups;
    const float* factor = nullptr;
};

// By whichever kernels fit (grouped.cu). Arrays of 16 and 32 bits are such that the copy engine can fetch them (pack.hpp), unless straight_rows() or
// straight_outer() say that this does not matter.
void multiply_rows(const Call& call, const RowsProblem& p, const std::string& op);
void multiply_outer(const Call& call, const OuterProblem& p, const std::string& op);
// One of the last two dimensions of W lies value by value in memory.
void check_matrices(Array& W, const char* name, const std::string& op);

// A few rows in all, as single tokens are (grouped_few.cu): false if there are too many.
bool multiply_rows_few(const Call& call, const RowsProblem& p, const std::string& op);
bool multiply_outer_few(const Call& call, const OuterProblem& p, const std::string& op);
// Whether they take the arrays as they are, wherever rows begin: products of `rows` rows with the matrices M (by_columns: whose columns, not
// whose depth, are neighbours in memory), and outer products of height x columns.
bool straight_rows(const Array& M, int64_t rows, bool by_columns);
bool straight_outer(int64_t rows, int64_t groups, int64_t height, int64_t columns, int32_t type);

// On arrays that the copy engine can fetch (pack.hpp); f16 and bf16 in grouped_mma.cu, f32 in grouped_split.cu. false: not taken on
// (another type, or nothing to multiply).
bool multiply_rows_mma(const Call& call, const RowsProblem& p, const std::string& op);
bool multiply_outer_mma(const Call& call, const OuterProblem& p, const std::string& op);
bool multiply_rows_split(const Call& call, const RowsProblem& p, const std::string& op);
bool multiply_outer_split(const Call& call, const OuterProblem& p, const std::string& op);

} // namespace mops_b200

#endif
