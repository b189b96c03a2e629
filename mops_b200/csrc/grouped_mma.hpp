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

// out[g] = X[rows of g]^T Y[rows of g]; out is contiguous.
struct OuterProblem {
    Array out, X, Y;
    const int32_t* offsets;
    int64_t groups;
};

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
