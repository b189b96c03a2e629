// grouped_matrix_product: rows sorted by group, each group with a matrix of its own.
//
//   output[r,:] = A[r,:] W[g,:,:]          for offsets[g] <= r < offsets[g+1]
//   grad_A[r,:] = grad_output[r,:] W[g,:,:]^T
//   grad_W[g]   = A[rows of g]^T grad_output[rows of g]
//
// The products of 16 and 32 bits run on the tensor cores (grouped_mma.cu, grouped_split.cu). Those of f64 are computed here, by the ordinary
// arithmetic units, which are as fast as the tensor cores for f64: a block computes a tile of 64 x 64 values, 4 x 4 of them per
// thread in registers, from slices of 16 that both operands leave in shared memory. So are the zeros of empty sums. 20 000 rows of 8 groups, 256 x 256: 276 us (9.5
// TFLOP/s), gradients 296 and 406; the slices are loaded and multiplied in turn, and the gradient of W has 128 tiles for 148 SMs.
#include "arrays.hpp"
#include "block_ops.hpp"
#include "group_tiles.cuh"
#include "grouped_mma.hpp"
#include "pack.hpp"

namespace mops_b200 {
namespace {

constexpr int kTile = 64;
constexpr int kSlice = 16;
constexpr int kThreads = 256;
constexpr int kPad = 4;

// c += the product of slices a[depth][row] and b[depth][column].
template <typename S>
__device__ __forceinline__ void multiply_slices(S (&c)[4][4], const S (&a)[kSlice][kTile + kPad],
                                                const S (&b)[kSlice][kTile + kPad]) {
    const int i0 = threadIdx.x / 16 * 4, j0 = threadIdx.x % 16 * 4;
#pragma unroll
    for (int d = 0; d < kSlice; d++) {
        S x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a[d][i0 + i], y[i] = b[d][j0 + i];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) c[i][j] += x[i] * y[j];
    }
}

// A slice of a matrix whose value (d, i) is at p[d * depth_stride + i * row_stride], widened; zeros outside of [0, depth) x [0, rows).
template <typename T>
__device__ __forceinline__ void load_slice(Sum<T> (&s)[kSlice][kTile + kPad], const T* __restrict__ p, int64_t depth_stride,
                                           int64_t row_stride, int64_t depth, int64_t rows) {
    // neighbouring threads along the dimension whose values are neighbours
    const bool along_depth = depth_stride == 1;
#pragma unroll
    for (int k = 0; k < kSlice * kTile / kThreads; k++) {
        const int at = k * kThreads + threadIdx.x;
        const int d = along_depth ? at % kSlice : at / kTile, i = along_depth ? at / kSlice : at % kTile;
        s[d][i] = d < depth && i < rows ? widen(p[d * depth_stride + i * row_stride]) : Sum<T>(0);
    }
}

// out[r,:] = X[r,:] M[group of r] (depth x columns each, value (d, j) at d * depth_stride + j * column_stride).
template <typename T>
__global__ void __launch_bounds__(kThreads)
grouped_rows_plain(T* __restrict__ out, const T* __restrict__ X, int64_t stride, const T* __restrict__ M, int64_t group_stride,
             int64_t depth_stride, int64_t column_stride, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
             int64_t depth, int64_t columns, Status st) {
    __shared__ Sum<T> a[kSlice][kTile + kPad], b[kSlice][kTile + kPad];
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(offsets, groups, rows, st);
    GroupWalk<RowTiles> walk(offsets, groups, rows, -1, groups, RowTiles{kTile, 1});
    const GroupPiece piece = walk.find(blockIdx.x, threadIdx.x & 31);
    if (!piece.found) return;
    const bool in_group = piece.group >= 0 && piece.group < groups;
    const int64_t row0 = piece.lo + piece.within * kTile;
    const int64_t here = min(piece.hi - row0, int64_t(kTile));
    for (int64_t j0 = static_cast<int64_t>(blockIdx.y) * kTile; j0 < columns; j0 += static_cast<int64_t>(gridDim.y) * kTile) {
        Sum<T> c[4][4] = {};
        if (in_group) {
            const T* x = X + row0 * stride;
            const T* m = M + piece.group * group_stride + j0 * column_stride;
            for (int64_t d0 = 0; d0 < depth; d0 += kSlice) {
                load_slice<T>(a, x + d0, 1, stride, depth - d0, here);
                load_slice<T>(b, m + d0 * depth_stride, depth_stride, column_stride, depth - d0, columns - j0);
                __syncthreads();
                multiply_slices(c, a, b);
                __syncthreads();
            }
        }
        const int i0 = threadIdx.x / 16 * 4, jt = threadIdx.x % 16 * 4;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + i < here && j0 + jt + j < columns)
                    out[(row0 + i0 + i) * columns + j0 + jt + j] = narrow<T>(c[i][j]);
    }
}

// out[g] = X[rows of g]^T Y[rows of g], values (i, j) at i * columns + j.
template <typename T>
__global__ void __launch_bounds__(kThreads)
grouped_outer_plain(T* __restrict__ out, const T* __restrict__ X, int64_t x_stride, const T* __restrict__ Y, int64_t y_stride,
              const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int64_t height, int64_t columns, Status st) {
    __shared__ Sum<T> a[kSlice][kTile + kPad], b[kSlice][kTile + kPad];
    const int64_t g = blockIdx.x;
    if (g == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_offsets(offsets, groups, rows, st);
    int64_t lo, hi;
    group_bounds(offsets, groups, rows, g, lo, hi);
    for (int64_t i0 = static_cast<int64_t>(blockIdx.y) * kTile; i0 < height; i0 += static_cast<int64_t>(gridDim.y) * kTile)
        for (int64_t j0 = static_cast<int64_t>(blockIdx.z) * kTile; j0 < columns; j0 += static_cast<int64_t>(gridDim.z) * kTile) {
            Sum<T> c[4][4] = {};
            for (int64_t d0 = lo; d0 < hi; d0 += kSlice) {
                load_slice<T>(a, X + d0 * x_stride + i0, x_stride, 1, hi - d0, height - i0);
                load_slice<T>(b, Y + d0 * y_stride + j0, y_stride, 1, hi - d0, columns - j0);
                __syncthreads();
                multiply_slices(c, a, b);
                __syncthreads();
            }
            const int it = threadIdx.x / 16 * 4, jt = threadIdx.x % 16 * 4;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i0 + it + i < height && j0 + jt + j < columns)
                        out[(g * height + i0 + it + i) * columns + j0 + jt + j] = narrow<T>(c[i][j]);
        }
}

const char* const kIndexNames[] = {"offsets"};

} // namespace

void multiply_rows(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.rows == 0 || p.columns == 0 || multiply_rows_few(call, p, op) || multiply_rows_mma(call, p, op) ||
        multiply_rows_split(call, p, op))
        return;
    for_type(p.X.type, [&](auto zero) {
        using T = decltype(zero);
        const int64_t tiles = most_row_tiles(p.rows, p.groups, kTile);
        fits_int32(static_cast<size_t>(tiles), "the number of tiles", op);
        const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(std::min<int64_t>(ceil_div(p.columns, kTile), 65535)));
        grouped_rows_plain<T><<<grid, kThreads, 0, call.stream>>>(
            static_cast<T*>(p.out.data), static_cast<const T*>(p.X.data), p.X.stride[0], static_cast<const T*>(p.M.data),
            p.M.stride[0], p.depth_stride, p.column_stride, p.offsets, p.groups, p.rows, p.depth, p.columns, call.status);
        note_kernel_f("grouped_rows_plain<%s>", array_type_name<T>());
    });
    MOPS_CUDA_OK(cudaGetLastError());
}

void multiply_outer(const Call& call, const OuterProblem& p, const std::string& op) {
    const Array &out = p.out, &X = p.X, &Y = p.Y;
    const int32_t* offsets = p.offsets;
    const int64_t groups = p.groups, rows = X.shape[0], height = X.shape[1], columns = Y.shape[1];
    if (groups == 0 || height == 0 || columns == 0 || (p.factor == nullptr && multiply_outer_few(call, p, op)) || multiply_outer_mma(call, p, op) ||
        multiply_outer_split(call, p, op))
        return;
    fits_int32(static_cast<size_t>(groups), "the number of groups", op);
    for_type(X.type, [&](auto zero) {
        using T = decltype(zero);
        const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(std::min<int64_t>(ceil_div(height, kTile), 65535)),
                        static_cast<unsigned>(std::min<int64_t>(ceil_div(columns, kTile), 65535)));
        grouped_outer_plain<T><<<grid, kThreads, 0, call.stream>>>(
            static_cast<T*>(out.data), static_cast<const T*>(X.data), X.stride[0], static_cast<const T*>(Y.data), Y.stride[0],
            offsets, groups, rows, height, columns, call.status);
        note_kernel_f("grouped_outer_plain<%s>", array_type_name<T>());
    });
    MOPS_CUDA_OK(cudaGetLastError());
}

namespace {

// Sizes and types of rows (R x K), matrices (G x K x N) and offsets (G + 1).
void check_common(Array& A, Array& W, const char* w_name, Array& offsets, Array& rows, const char* rows_name,
                  const std::string& op) {
    check_floating(A.type, "A", op);
    check_array(A, "A", 2, A.type, op);
    check_array(W, w_name, 3, A.type, op);
    check_array(rows, rows_name, 2, A.type, op);
    check_array(offsets, "offsets", 1, MOPS_B200_I32, op);
    check_size(A.shape[1], "A", 1, W.shape[1], w_name, 1, op);
    check_size(rows.shape[0], rows_name, 0, A.shape[0], "A", 0, op);
    check_size(rows.shape[1], rows_name, 1, W.shape[2], w_name, 2, op);
    check_size(offsets.shape[0], "offsets", 0, W.shape[0] + 1, "the groups of W (and one)", 0, op);
    check_rows(A, "A", op);
    if (offsets.stride[0] != 1) throw std::runtime_error("offsets must be contiguous in " + op);
    for (int64_t n : {A.shape[0], A.shape[1], W.shape[0], W.shape[2]}) fits_int32(static_cast<size_t>(n), "a size", op);
}

} // namespace

// (So does one of size 1, whatever its stride; matrices of one row whose columns lie apart are columns of one value each.)
void check_matrices(Array& W, const char* name, const std::string& op) {
    if (W.shape[1] == 1 && W.stride[2] != 1) W.stride[1] = 1;
    if (W.stride[2] != 1 && W.stride[1] != 1)
        throw std::runtime_error(std::string(name) + " must have a stride of 1 in one of its last two dimensions in " + op);
}

namespace {

// Whether there are products to compute that the tensor cores take on (the other problems go to the kernels of this file).
bool on_tensor_cores(const Array& A, const Array& W) {
    return A.type != MOPS_B200_F64 && A.shape[0] > 0 && A.shape[1] > 0 && W.shape[0] > 0 && W.shape[2] > 0;
}

} // namespace

void grouped_matrix_product(Array output, Array A, Array W, Array offsets) {
    const std::string op = "cuda_grouped_matrix_product";
    check_common(A, W, "W", offsets, output, "output", op);
    check_matrices(W, "W", op);
    check_output(output, "output", op);
    if (output.shape[0] == 0 || output.shape[1] == 0) return;
    Call call = begin_call();
    Packing packing(call);
    if (on_tensor_cores(A, W) && !straight_rows(W, A.shape[0], W.stride[2] == 1)) {
        packing.add(A);
        packing.add(W);
        packing.run();
    }
    multiply_rows(call,
                  {output, A, W, W.stride[1], W.stride[2], static_cast<const int32_t*>(offsets.data), W.shape[0], A.shape[0],
                   A.shape[1], W.shape[2]},
                  op);
    packing.release();
    end_call(call, op.c_str(), kIndexNames, 1);
}

void grouped_matrix_product_vjp(Array grad_A, Array grad_W, Array grad_output, Array A, Array W, Array offsets) {
    const std::string op = "cuda_grouped_matrix_product_vjp";
    check_common(A, W, "W", offsets, grad_output, "grad_output", op);
    check_rows(grad_output, "grad_output", op);
    check_matrices(W, "W", op);
    const bool need_A = grad_A.data != nullptr, need_W = grad_W.data != nullptr;
    if (need_A) {
        check_array(grad_A, "grad_A", 2, A.type, op);
        for (int d = 0; d < 2; d++) check_size(grad_A.shape[d], "grad_A", d, A.shape[d], "A", d, op);
        check_output(grad_A, "grad_A", op);
    }
    bool turned = false; // grad_W[g] is stored column by column
    if (need_W) {
        check_array(grad_W, "grad_W", 3, A.type, op);
        for (int d = 0; d < 3; d++) check_size(grad_W.shape[d], "grad_W", d, W.shape[d], "W", d, op);
        turned = grad_W.stride[2] != 1;
        if (turned) std::swap(grad_W.shape[1], grad_W.shape[2]), std::swap(grad_W.stride[1], grad_W.stride[2]);
        check_output(grad_W, "grad_W", op);
    }
    if (!need_A && !need_W) return;
    Call call = begin_call();
    Packing packing(call);
    if (on_tensor_cores(A, W)) {
        const bool rows_packed = need_A && !straight_rows(W, A.shape[0], W.stride[1] == 1);
        const bool outer_packed = need_W && !straight_outer(A.shape[0], W.shape[0], W.shape[1], W.shape[2], A.type);
        if (rows_packed || outer_packed) packing.add(grad_output);
        if (rows_packed) packing.add(W);
        if (outer_packed) packing.add(A);
        packing.run();
    }
    const int32_t* starts = static_cast<const int32_t*>(offsets.data);
    if (need_A)
        multiply_rows(call,
                      {grad_A, grad_output, W, W.stride[2], W.stride[1], starts, W.shape[0], A.shape[0], W.shape[2], A.shape[1]},
                      op);
    if (need_W) {
        if (turned) multiply_outer(call, {grad_W, grad_output, A, starts, W.shape[0]}, op);
        else multiply_outer(call, {grad_W, A, grad_output, starts, W.shape[0]}, op);
    }
    packing.release();
    end_call(call, op.c_str(), kIndexNames, 1);
}

} // namespace mops_b200
