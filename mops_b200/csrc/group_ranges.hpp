// Ranges of rows between the offsets of groups, kept inside of [0, rows) and in order whatever the offsets say: they are in device memory, and
// nobody has looked at them before the kernels do.
#ifndef MOPS_B200_GROUP_RANGES_HPP
#define MOPS_B200_GROUP_RANGES_HPP

#include <cstdint>

#ifdef __CUDACC__
#define MOPS_B200_BOTH_SIDES __host__ __device__ __forceinline__
#else
#define MOPS_B200_BOTH_SIDES inline
#endif

namespace mops_b200 {

struct RowRange {
    int64_t lo, hi; // lo <= hi
};

// The rows from `begin` to `end`, two offsets.
MOPS_B200_BOTH_SIDES RowRange rows_between(int64_t begin, int64_t end, int64_t rows) {
    RowRange r;
    r.lo = begin < 0 ? 0 : begin < rows ? begin : rows;
    r.hi = end < 0 ? 0 : end < rows ? end : rows;
    if (r.hi < r.lo) r.hi = r.lo;
    return r;
}

// Calls f(row) for the rows of no group: those in front of the first offset and those behind the last one, each once.
template <typename F> MOPS_B200_BOTH_SIDES void for_rows_of_no_group(int64_t first_offset, int64_t last_offset, int64_t rows, F&& f) {
    const RowRange grouped = rows_between(first_offset, last_offset, rows);
    for (int64_t r = 0; r < grouped.lo; r++) f(r);
    for (int64_t r = grouped.hi; r < rows; r++) f(r);
}

} // namespace mops_b200

#endif
