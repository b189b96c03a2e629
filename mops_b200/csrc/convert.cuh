// Copies of arrays in another type, row by row: operands of 16 bits widened for kernels of 32, and results rounded back.
#ifndef MOPS_B200_CONVERT_CUH
#define MOPS_B200_CONVERT_CUH

#include "arrays.hpp"

namespace mops_b200 {

constexpr int kRowThreads = 64, kRowsAtATime = 4; // of a block that goes over rows

// Launches a kernel whose blocks take kRowsAtATime rows at a time, one for each threadIdx.y.
inline dim3 row_blocks(const Call& call, int64_t rows) {
    return dim3(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(rows, kRowsAtATime), 1), int64_t(sm_count(call.device)) * 32)));
}
inline dim3 row_threads() { return dim3(kRowThreads, kRowsAtATime); }
__device__ __forceinline__ int64_t first_row() { return static_cast<int64_t>(blockIdx.x) * kRowsAtATime + threadIdx.y; }
__device__ __forceinline__ int64_t row_step() { return static_cast<int64_t>(gridDim.x) * kRowsAtATime; }

template <typename To, typename From> __device__ __forceinline__ To convert(From v) {
    if constexpr (std::is_same<To, From>::value) return v;
    else return narrow<To>(static_cast<Sum<To>>(widen(v)));
}

// to[slice][row][i] = from[slice][row][i], `slices` x `outer` rows of `inner` values.
template <typename To, typename From>
static __global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
convert_rows(To* __restrict__ to, int64_t to_slice_stride, int64_t to_stride, const From* __restrict__ from, int64_t slices, int64_t outer, int64_t inner, int64_t slice_stride,
             int64_t outer_stride) {
    for (int64_t row = first_row(); row < slices * outer; row += row_step()) {
        const int64_t slice = row / outer;
        const From* p = from + slice * slice_stride + (row - slice * outer) * outer_stride;
        To* q = to + slice * to_slice_stride + (row - slice * outer) * to_stride;
        for (int64_t i = threadIdx.x; i < inner; i += kRowThreads) q[i] = convert<To>(p[i]);
    }
}

// A contiguous copy of `a` in type To at `to`, as an array. Of 3 dimensions the last two keep the way round that they are stored.
template <typename To> Array converted(const Call& call, const Array& a, To* to, int32_t type) {
    Array r = a;
    r.data = to, r.type = type;
    const int last = a.dimensions - 1;
    const int inner = a.dimensions == 3 && a.stride[last] != 1 ? last - 1 : last, outer = a.dimensions == 3 && inner == last - 1 ? last : last - 1;
    const int64_t slices = a.dimensions == 3 ? a.shape[0] : 1;
    r.stride[inner] = 1, r.stride[outer] = a.shape[inner];
    if (a.dimensions == 3) r.stride[0] = a.shape[inner] * a.shape[outer];
    if (inner != last && a.shape[inner] == 1) r.stride[inner] = a.shape[outer]; // (columns of one value are rows of the copy: one stride of 1 alone says which way round it is)
    if (slices * a.shape[outer] * a.shape[inner] > 0)
        for_type(a.type, [&](auto zero) {
            using From = decltype(zero);
            convert_rows<To, From><<<row_blocks(call, slices * a.shape[outer]), row_threads(), 0, call.stream>>>(
                to, a.shape[inner] * a.shape[outer], a.shape[inner], static_cast<const From*>(a.data), slices, a.shape[outer], a.shape[inner], a.dimensions == 3 ? a.stride[0] : 0, a.stride[outer]);
        });
    MOPS_CUDA_OK(cudaGetLastError());
    return r;
}

// Launches a kernel that begins with after_others(), where it waits for what is in front of it on the stream: its blocks are in place when that is done.
template <typename... P, typename... A> void launch_early(const Call& call, void (*kernel)(P...), dim3 grid, dim3 block, const A&... arguments) {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    config.gridDim = grid;
    config.blockDim = block;
    config.stream = call.stream;
    MOPS_CUDA_OK(cudaLaunchKernelEx(&config, kernel, P(arguments)...));
}
__device__ __forceinline__ void after_others() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

inline int64_t values_of(const Array& a) {
    int64_t n = 1;
    for (int d = 0; d < a.dimensions; d++) n *= a.shape[d];
    return n;
}

// A contiguous array of two dimensions, or three.
inline Array contiguous(void* data, int32_t type, int64_t rows, int64_t columns) {
    Array a{};
    a.data = data, a.type = type, a.dimensions = 2;
    a.shape[0] = rows, a.shape[1] = columns, a.stride[0] = columns, a.stride[1] = 1;
    return a;
}
inline Array contiguous(void* data, int32_t type, int64_t slices, int64_t rows, int64_t columns) {
    Array a{};
    a.data = data, a.type = type, a.dimensions = 3;
    a.shape[0] = slices, a.shape[1] = rows, a.shape[2] = columns;
    a.stride[0] = rows * columns, a.stride[1] = columns, a.stride[2] = 1;
    return a;
}

} // namespace mops_b200

#endif
