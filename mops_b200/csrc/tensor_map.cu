#include "tensor_map.hpp"

namespace mops_b200 {

namespace {
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        MOPS_CUDA_OK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &found));
        if (entry == nullptr) throw std::runtime_error("the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeTiled>(entry);
    }();
    return f;
}
} // namespace

CUtensorMap tensor_map(int32_t type, const void* data, int64_t inner, int64_t outer, int64_t slices,
                          int64_t outer_stride, int64_t slice_stride, int box) {
    CUtensorMap map;
    const int64_t size = type_bytes(type);
    // strides of dimensions of size 1 mean nothing, but have to look well
    if (outer == 1) outer_stride = ceil_div(inner, 16 / size) * (16 / size);
    if (slices == 1) slice_stride = outer * outer_stride;
    const cuuint64_t sizes[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(slices)};
    const cuuint64_t stride[2] = {static_cast<cuuint64_t>(outer_stride * size), static_cast<cuuint64_t>(slice_stride * size)};
    const cuuint32_t boxes[3] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(box), 1}, steps[3] = {1, 1, 1};
    const CUresult r = encode_tiled()(&map, type == MOPS_B200_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                            : type == MOPS_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                      3, const_cast<void*>(data), sizes, stride, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        throw std::runtime_error("CUDA error: cuTensorMapEncodeTiled returned " + std::to_string(static_cast<int>(r)));
    return map;
}

} // namespace mops_b200
