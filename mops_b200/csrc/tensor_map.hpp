// Descriptions of arrays in global memory for the copy engine's tiled copies (TMA).
#ifndef MOPS_B200_TENSOR_MAP_HPP
#define MOPS_B200_TENSOR_MAP_HPP

#include <cuda.h>

#include "arrays.hpp"

namespace mops_b200 {

// An array of f32, f16 or bf16 values (inner x outer x slices, strides in values) that is copied in boxes of 128 bytes of inner values (one
// row of shared memory, swizzled) by `box` outer ones. What lies outside of the array is read as zero and not written. boxable() says whether
// an array can be copied so.
CUtensorMap tensor_map(int32_t type, const void* data, int64_t inner, int64_t outer, int64_t slices, int64_t outer_stride,
                       int64_t slice_stride, int box);

inline bool boxable(int32_t type, const void* data, int64_t inner, int64_t outer, int64_t slices, int64_t outer_stride,
                    int64_t slice_stride) {
    const int64_t values = 16 / type_bytes(type);
    return reinterpret_cast<uintptr_t>(data) % 16 == 0 && (outer <= 1 || (outer_stride % values == 0 && outer_stride >= inner)) &&
           (slices <= 1 || (slice_stride % values == 0 && slice_stride > 0));
}

} // namespace mops_b200

#endif
