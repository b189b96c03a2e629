// The stable device sort of an index (sort.cu), for operators that sort as part of a call.
#ifndef MOPS_B200_SORT_HPP
#define MOPS_B200_SORT_HPP

#include "runtime.hpp"

namespace mops_b200 {

// sorted[i] = key of indices[permutation[i]], ascending, equal keys in input order (n > 0). The key of an index is the
// index itself; that of one outside of [0, n_rows) (reported as index array 0) and that of
// `dropped` is `replacement`, which is at most n_rows.
void sort_keys(const Call& call, int32_t* sorted, int32_t* permutation, const int32_t* indices, int64_t n,
               int64_t n_rows, int32_t replacement, int32_t dropped);

} // namespace mops_b200

#endif
