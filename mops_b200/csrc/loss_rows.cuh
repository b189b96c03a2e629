// linear_cross_entropy: the rows that count, and sums over parts of the vocabulary that are joined.
//
// Rows without a target take no part: those that have one are numbered in order, 0 <= i < kept, and gathered, so that neither work nor what stands in the others
// gets into the products. How many they are is known on the device only; it goes as the offsets of a single group, {0, kept}.
#ifndef MOPS_B200_LOSS_ROWS_CUH
#define MOPS_B200_LOSS_ROWS_CUH

#include "convert.cuh"

namespace mops_b200 {

struct LossRows {
    int32_t* offsets; // 0, kept
    int32_t* order;   // of the i-th kept row: its number
    int32_t* place;   // of a row: i, or -1
    int32_t* target;  // of the i-th kept row
    float* unit;      // of their gradients: the largest |grad_loss|, or |grad_loss| + |grad_log_sum| where those of sums are the larger ones
};

// Sums over a part of a row: the largest x and the sum of exp(x - largest).
template <typename S> struct alignas(2 * sizeof(S)) PartSum {
    S top, sum;
    __device__ __forceinline__ static PartSum none() { return {-S(INFINITY), S(0)}; }
    // What exponents are taken from: infinite sums stay infinite (not NaN) when it is 0.
    __device__ __forceinline__ static S from(S top) { return isinf(top) ? S(0) : top; }
    // (a sum of nothing but exp(-infinity) is 0, or NaN, whatever it is taken from)
    __device__ __forceinline__ S weight(S base) const { return top == -S(INFINITY) ? S(1) : exp(from(top) - base); }
    __device__ __forceinline__ void join(const PartSum& o) {
        const S both = fmax(top, o.top), base = from(both);
        sum = sum * weight(base) + o.sum * o.weight(base);
        top = both;
    }
};

// The i-th row's loss and log_sum from the sums of its parts, in their order, and x at the target. A block to a row. Where rows have not been numbered (no order) they
// are all there, and those without a target get their zeros here.
template <typename S>
static __global__ void __launch_bounds__(128)
loss_join(S* __restrict__ loss, S* __restrict__ log_sum, const PartSum<S>* __restrict__ parts, int64_t n, const S* __restrict__ at_target,
          const LossRows rows, const int32_t* __restrict__ targets, int64_t vocabulary, int64_t ignored, Status st) {
    __shared__ PartSum<S> of_warp[4];
    const int64_t i = blockIdx.x;
    int64_t r = i;
    if (rows.order != nullptr) {
        if (i >= rows.offsets[1]) return;
        r = rows.order[i];
    } else {
        const int64_t t = targets[i];
        if (t < 0 || t >= vocabulary || t == ignored) {
            if (threadIdx.x == 0) {
                loss[i] = log_sum[i] = S(0);
                if (t != ignored) report_bad_index(st, 0);
            }
            return;
        }
    }
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
    const S value = PartSum<S>::from(all.top) + log(all.sum);
    log_sum[r] = value;
    loss[r] = value - at_target[i];
}

inline LossRows take_rows(Scratch& room, int64_t rows) {
    room.take(static_cast<size_t>(3 * rows + 4) * sizeof(int32_t));
    int32_t* p = room.as<int32_t>();
    return {p, p + 4, p + 4 + rows, p + 4 + 2 * rows, reinterpret_cast<float*>(p + 2)};
}

// Numbers the rows that have a target (cross_entropy.cu). The others get zeros in loss and log_sum, if these are given; of gradients, if they are, the unit is found.
template <typename S>
void prepare_rows(const Call& call, const LossRows& to, S* loss, S* log_sum, const Array& targets, int64_t vocabulary, int64_t ignored, const S* grad_loss,
                  const S* grad_log_sum);

// The vocabulary's loss on tensor cores, f16 and bf16 (cross_entropy_mma.cu).
struct LossProblem {
    Array A, W, targets;
    double scale;
    int64_t ignored;
};
void loss_forward_mma(const Call& call, const LossProblem& p, const Array& loss, const Array& log_sum, const std::string& op);
void loss_backward_mma(const Call& call, const LossProblem& p, const Array& grad_A, const Array& grad_W, const Array& grad_loss, const Array& grad_log_sum, const Array& loss,
                       const Array& log_sum, const std::string& op);

} // namespace mops_b200

#endif
