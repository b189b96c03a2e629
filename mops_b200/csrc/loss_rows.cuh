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
    int32_t* doubled; // 0, 2 kept
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

// The i-th row's loss and log_sum from the sums of its parts, and x at the target. kLanes to a row (a warp, or 4 where its parts are few: 53 996 rows of one 4.5 us for 18.6, 62 070 of five 5.3 for 16.9): they find the largest first, and take one exponential for each part. Where rows have not
// been numbered (no order) they are all there, and those without a target get their zeros here.
constexpr int kJoinThreads = 128, kInFlight = 8; // parts that a lane has under way
template <typename S, int kLanes>
static __global__ void __launch_bounds__(kJoinThreads)
loss_join(S* __restrict__ loss, S* __restrict__ log_sum, const PartSum<S>* __restrict__ parts, int64_t n, int64_t all_rows, const S* __restrict__ at_target,
          const LossRows rows, const int32_t* __restrict__ targets, int64_t vocabulary, int64_t ignored, Status st) {
    after_others();
    const int lane = threadIdx.x % kLanes;
    const unsigned group = kLanes == 32 ? kFullMask : ((1u << kLanes) - 1) << (threadIdx.x & 31) / kLanes * kLanes;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
    if (i >= all_rows) return;
    int64_t r = i;
    if (rows.order != nullptr) {
        if (i >= rows.offsets[1]) return;
        r = rows.order[i];
    } else {
        const int64_t t = targets[i];
        if (t < 0 || t >= vocabulary || t == ignored) {
            if (lane == 0) {
                loss[i] = log_sum[i] = S(0);
                if (t != ignored) report_bad_index(st, 0);
            }
            return;
        }
    }
    const PartSum<S>* of_row = parts + i * n;
    S top = -S(INFINITY);
    for (int64_t p0 = lane; p0 < n; p0 += kLanes * kInFlight) {
        S v[kInFlight];
#pragma unroll
        for (int k = 0; k < kInFlight; k++) v[k] = p0 + kLanes * k < n ? of_row[p0 + kLanes * k].top : -S(INFINITY);
#pragma unroll
        for (int k = 0; k < kInFlight; k++) top = fmax(top, v[k]);
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(group, top, d));
    const S base = PartSum<S>::from(top);
    S sum = 0;
    for (int64_t p0 = lane; p0 < n; p0 += kLanes * kInFlight) { // (from the L1, or near it)
        PartSum<S> v[kInFlight];
#pragma unroll
        for (int k = 0; k < kInFlight; k++) v[k] = p0 + kLanes * k < n ? of_row[p0 + kLanes * k] : PartSum<S>::none();
#pragma unroll
        for (int k = 0; k < kInFlight; k++) sum += v[k].sum * v[k].weight(base);
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(group, sum, d);
    if (lane != 0) return;
    const S value = base + log(sum);
    log_sum[r] = value;
    loss[r] = value - at_target[i];
}
template <typename S>
void join_rows(const Call& call, const Array& loss, const Array& log_sum, const PartSum<S>* parts, int64_t n, const S* at_target, const LossRows& rows, const Array& targets,
               int64_t vocabulary, int64_t ignored) {
    const int64_t all = targets.shape[0];
    auto launch = [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value;
        launch_early(call, loss_join<S, kLanes>, static_cast<unsigned>(ceil_div(all, kJoinThreads / kLanes)), kJoinThreads, static_cast<S*>(loss.data),
                     static_cast<S*>(log_sum.data), parts, n, all, at_target, rows, static_cast<const int32_t*>(targets.data), vocabulary, ignored, call.status);
    };
    if (n <= 4 * kInFlight) launch(std::integral_constant<int, 4>());
    else launch(std::integral_constant<int, 32>());
}

inline LossRows take_rows(Scratch& room, int64_t rows) {
    room.take(static_cast<size_t>(3 * rows + 8) * sizeof(int32_t));
    int32_t* p = room.as<int32_t>();
    return {p, p + 2, p + 8, p + 8 + rows, p + 8 + 2 * rows, reinterpret_cast<float*>(p + 4)};
}

// Numbers the rows that have a target (cross_entropy.cu). The others get zeros in loss and log_sum, if these are given; of gradients, if they are, the unit is found.
template <typename S>
void prepare_rows(const Call& call, const LossRows& to, S* loss, S* log_sum, const Array& targets, int64_t vocabulary, int64_t ignored, const S* grad_loss,
                  const S* grad_log_sum);

// grad_A[r,:] = *factor (if it is given) times the sums of row place[r] (of both its rows, if `twice`), zeros for rows that have no place. Four columns to a thread; the sums have room up to a multiple of 4.
constexpr int kScatterThreads = 256;
template <typename T>
static __global__ void __launch_bounds__(kScatterThreads)
scatter_rows(T* __restrict__ to, const float* __restrict__ sums, int slices, int64_t stride, const LossRows rows, int64_t n, int columns, bool by_four,
             bool twice, const float* __restrict__ factor) {
    after_others();
    const float f = factor != nullptr ? *factor : 1.f;
    const int quads = static_cast<int>(stride / 4);
    const int64_t copies = twice ? 2 : 1, slice = copies * n * stride;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; r < n; r += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const int64_t i = rows.place[r];
#pragma unroll 2
        for (int q = threadIdx.x; q < quads; q += blockDim.x) {
            Pack<T, 4> out;
            if (i >= 0) {
                const float* from = sums + copies * i * stride + 4 * q;
                float4 v = make_float4(0, 0, 0, 0);
                for (int s = 0; s < slices; s++) {
                    float4 w = *reinterpret_cast<const float4*>(from + s * slice);
                    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                    if (twice) {
                        w = *reinterpret_cast<const float4*>(from + s * slice + stride);
                        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                    }
                }
                out.v[0] = narrow<T>(v.x * f), out.v[1] = narrow<T>(v.y * f), out.v[2] = narrow<T>(v.z * f), out.v[3] = narrow<T>(v.w * f);
            } else {
                out.v[0] = out.v[1] = out.v[2] = out.v[3] = T(0.f);
            }
            T* p = to + r * columns + 4 * q;
            if (by_four) {
                *reinterpret_cast<Pack<T, 4>*>(p) = out;
            } else { // (a column to a thread: 48 357 rows of 469 59 us for 44)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (4 * q + k < columns) p[k] = out.v[k];
            }
        }
    }
}
template <typename T>
void scatter_sums(const Call& call, T* grad_A, const float* sums, int64_t slices, int64_t stride, const LossRows& rows, int64_t n, int64_t columns, bool twice,
                  const float* factor) {
    const bool by_four = columns % 4 == 0 && reinterpret_cast<uintptr_t>(grad_A) % (4 * sizeof(T)) == 0;
    unsigned across = 32;
    while (across < kScatterThreads && across * 4 < columns) across *= 2;
    const dim3 block(across, kScatterThreads / across);
    const unsigned down = static_cast<unsigned>(std::min<int64_t>(ceil_div(n, block.y), int64_t(sm_count(call.device)) * 32));
    launch_early(call, scatter_rows<T>, down, block, grad_A, sums, static_cast<int>(slices), stride, rows, n, static_cast<int>(columns), by_four, twice, factor);
}

// Whether rows are numbered and gathered in front of a forward pass, which takes some 10 us: where all of them take 50 us or more (f32 takes eight times as long as 16 bits).
inline bool worth_gathering(int32_t type, int64_t rows, int64_t vocabulary, int64_t columns) {
    return rows >= 512 && 2.0 * rows * vocabulary * columns >= (type == MOPS_B200_F32 ? 6e9 : 5e10);
}

// The vocabulary's loss on tensor cores, f16 and bf16 (cross_entropy_mma.cu).
struct LossProblem {
    Array A, W, targets;
    double scale;
    int64_t ignored;
};
// A few rows (cross_entropy_few.cu; not f64).
bool few_loss_rows(const LossProblem& p);
void loss_forward_few(const Call& call, const LossProblem& p, const Array& loss, const Array& log_sum);
void loss_forward_mma(const Call& call, const LossProblem& p, const Array& loss, const Array& log_sum, const std::string& op);
void loss_backward_mma(const Call& call, const LossProblem& p, const Array& grad_A, const Array& grad_W, const Array& grad_loss, const Array& grad_log_sum, const Array& loss,
                       const Array& log_sum, const std::string& op);

} // namespace mops_b200

#endif
