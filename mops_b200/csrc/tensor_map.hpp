// Descriptions of arrays in global memory for the copy engine's tiled copies (TMA).
#ifndef MOPS_B200_TENSOR_MAP_HPP
#define MOPS_B200_TENSOR_MAP_HPP

#include <cuda.h>

#include "arrays.hpp"

namespace mops_b200 {

// An array of 16-bit values (inner x outer x slices, strides in values) that is copied in boxes of 64 inner values (128
// bytes, one row of shared memory, swizzled) by `box` outer ones. What lies outside of the array is read as zero and not written.
// The base and the strides are multiples of 16 bytes (aligned16).
CUtensorMap tensor_map_64(int32_t type, const void* data, int64_t inner, int64_t outer, int64_t slices,
                          int64_t outer_stride, int64_t slice_stride, int box);

} // namespace mops_b200

#endif
