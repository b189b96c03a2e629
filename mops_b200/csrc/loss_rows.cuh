// linear_cross_entropy: the rows that count, and sums over parts of the vocabulary that are joined.
//
// Rows without a target take no part: those that have one are numbered in order, 0 <= i < kept, and gathered, so that neither work nor what stands in the others
// gets into the products. How many they are is known on the device only; it goes as the offsets of a single group, {0, kept}.
#ifndef MOPS_B200_LOSS_ROWS_CUH
#define MOPS_B200_LOSS_ROWS_CUH

#include "arrays.hpp"
#include "convert.cuh"

namespace mops_b200 {

struct LossRows {
    int32_t* offsets; // 0, kept
    int32_t* order;   // of the i-th kept row: its number
    int32_t* place;   // of a row: i, or -1
};

// Sums over a part of a row: the largest x and the sum of exp(x - largest).
template <typename S> struct alignas(2 * sizeof(S)) PartSum {
    S top, sum;
    __device__ __forceinline__ static PartSum none() { return {-S(INFINITY), S(0)}; }
    // What exponents are taken from: infinite sums stay infinite (not NaN) when it is 0.
    __device__ __forceinline__ static S from(S top) { return isinf(top) ? S(0) : top; }
    __device__ __forceinline__ void join(const PartSum& o) {
        const S both = fmax(top, o.top), base = from(both);
        sum = sum * exp(from(top) - base) + o.sum * exp(from(o.top) - base);
        top = both;
    }
};

// The i-th row's loss and log_sum from the sums of its parts, in their order, and x at the target. A block to a row.
template <typename S>
static __global__ void __launch_bounds__(128)
loss_join(S* __restrict__ loss, S* __restrict__ log_sum, const PartSum<S>* __restrict__ parts, int64_t n, const S* __restrict__ at_target,
          const LossRows rows) {
    __shared__ PartSum<S> of_warp[4];
    const int64_t i = blockIdx.x;
    if (i >= rows.offsets[1]) return;
    PartSum<S> all = PartSum<S>::none();
    for (int64_t p = threadIdx.x; p < n; p += 128) all.join(parts[i * n + p]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        PartSum<S> other;
        other.top = __shfl_down_sync(kFullMask, all.top, d);
        other.sum = __shfl_down_sync(kFullMask, all.sum, d);
        all.join(other);
    }
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = all;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 4; w++) all.join(of_warp[w]);
    const int64_t r = rows.order[i];
    const S value = PartSum<S>::from(all.top) + log(all.sum);
    log_sum[r] = value;
    loss[r] = value - at_target[i];
}

} // namespace mops_b200

#endif
