// linear_cross_entropy: the cross entropy of a softmax over the rows of a table, without the logits.
//
//   x[r,v] = scale A[r,:] . W[v,:]
//   log_sum[r] = log sum_v exp(x[r,v]), loss[r] = log_sum[r] - x[r,t_r]
//   dx[r,v] = (grad_loss[r] + grad_log_sum[r]) exp(x[r,v] - log_sum[r]) - grad_loss[r] [v = t_r]
//   grad_A = scale dx W, grad_W = scale dx^T A
//
// A piece of the vocabulary at a time: its logits are a product into scratch memory, of which sums are taken, or which become dx where they stand and are multiplied by the
// piece's rows of W and, the other way, by A. The gradients compute the logits again. In f32 the logits are worked on where they are summed (LossStore32, GradientStore32) and
// never stored, but for few tiles of much depth. Here: f32 and f64 (and f16 and bf16 without columns); f16 and bf16 are in cross_entropy_mma.cu, a few rows in cross_entropy_few.cu.
#include "block_ops.hpp"
#include "convert.cuh"
#include "few_rows.cuh"
#include "gated_mma.hpp"
#include "grouped_mma.hpp"
#include "loss_rows.cuh"
#include "pack.hpp"
#include "parts_rows.cuh"

namespace mops_b200 {
namespace {

constexpr int kPrepareThreads = 1024, kPrepareRows = 8;
constexpr int64_t kPartColumns = 4096;             // of a part of a row's sums, at most
constexpr int64_t kMostLogits = int64_t(64) << 20; // of a piece
constexpr int64_t kLeastSteps = 4;                 // stages of depth of a slice of f32 products

// Numbers the rows that have a target, by a block, or a cluster of blocks with a part of the rows each, which count theirs first; the others get zeros, if loss is given. (16 384 rows: one block 13.8 us,
// 9 by eight; 48 285: 31 and 9.)
template <typename S>
__global__ void __launch_bounds__(kPrepareThreads)
loss_prepare(const LossRows to, S* __restrict__ loss, S* __restrict__ log_sum, const int32_t* __restrict__ targets, int64_t rows, int64_t vocabulary,
             int64_t ignored, const S* __restrict__ grad_loss, const S* __restrict__ grad_log_sum, Status st) {
    constexpr int kRuns = kPrepareRows * kPrepareThreads / 32; // of 32 rows each
    __shared__ int in_run[kRuns], in_front[kRuns + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool gradients = grad_loss != nullptr || grad_log_sum != nullptr;
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int64_t part = (rows + blocks - 1) / blocks, begin = min(rank * part, rows), end = min(begin + part, rows);
    int before = 0, all = 0;
    __shared__ int own_count;
    if (blocks > 1) {
        if (threadIdx.x == 0) own_count = 0;
        __syncthreads();
        int own = 0;
        for (int64_t r = begin + threadIdx.x; r < end; r += kPrepareThreads) {
            const int64_t t = targets[r];
            own += t >= 0 && t < vocabulary && t != ignored;
        }
        own = __reduce_add_sync(kFullMask, own);
        if (lane == 0) atomicAdd(&own_count, own);
        cluster.sync();
        for (int b = 0; b < blocks; b++) {
            const int n = *cluster.map_shared_rank(&own_count, b);
            before += b < rank ? n : 0, all += n;
        }
    }
    float largest[3] = {}; // of the gradients of losses, of sums, of both together
    bool bad = false;
    for (int64_t r0 = begin; r0 < end; r0 += kPrepareThreads * kPrepareRows) {
        int32_t target[kPrepareRows];
        unsigned kept[kPrepareRows];
#pragma unroll
        for (int k = 0; k < kPrepareRows; k++) {
            const int64_t r = r0 + k * kPrepareThreads + threadIdx.x;
            target[k] = r < end ? targets[r] : 0;
        }
#pragma unroll
        for (int k = 0; k < kPrepareRows; k++) {
            const int64_t r = r0 + k * kPrepareThreads + threadIdx.x, t = target[k];
            const bool in = r < end && t >= 0 && t < vocabulary && t != ignored;
            bad |= r < end && !in && t != ignored;
            kept[k] = __ballot_sync(kFullMask, in);
            if (lane == 0) in_run[k * (kPrepareThreads / 32) + warp] = __popc(kept[k]);
        }
        __syncthreads();
        if (warp == 0) { // the runs in front of each
            constexpr int kEach = kRuns / 32;
            int sum = 0, own[kEach];
#pragma unroll
            for (int i = 0; i < kEach; i++) own[i] = in_run[lane * kEach + i], sum += own[i];
            int up_to = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(kFullMask, up_to, d);
                if (lane >= d) up_to += v;
            }
            int at = up_to - sum;
#pragma unroll
            for (int i = 0; i < kEach; i++) in_front[lane * kEach + i] = at, at += own[i];
            if (lane == 31) in_front[kRuns] = at;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPrepareRows; k++) {
            const int64_t r = r0 + k * kPrepareThreads + threadIdx.x;
            if (r >= end) continue;
            const bool in = kept[k] >> lane & 1;
            const int i = before + in_front[k * (kPrepareThreads / 32) + warp] + __popc(kept[k] & ((1u << lane) - 1));
            to.place[r] = in ? i : -1;
            if (in) {
                to.order[i] = static_cast<int32_t>(r);
                to.target[i] = target[k];
                if (gradients) {
                    const float l = grad_loss != nullptr ? static_cast<float>(fabs(grad_loss[r])) : 0.f;
                    const float m = grad_log_sum != nullptr ? static_cast<float>(fabs(grad_log_sum[r])) : 0.f;
                    const float all[3] = {l, m, l + m};
#pragma unroll
                    for (int q = 0; q < 3; q++)
                        if (all[q] <= 3e38f) largest[q] = fmaxf(largest[q], all[q]); // (infinities keep to their rows)
                }
            } else if (loss != nullptr) {
                loss[r] = log_sum[r] = S(0);
            }
        }
        before += in_front[kRuns];
        __syncthreads();
    }
    __shared__ float most[3][kPrepareThreads / 32];
    if (gradients) {
#pragma unroll
        for (int q = 0; q < 3; q++) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) largest[q] = fmaxf(largest[q], __shfl_xor_sync(kFullMask, largest[q], d));
            if (lane == 0) most[q][warp] = largest[q];
        }
        __syncthreads();
        if (threadIdx.x < 3) {
            float m = 0;
            for (int w = 0; w < kPrepareThreads / 32; w++) m = fmaxf(m, most[threadIdx.x][w]);
            most[threadIdx.x][0] = m;
        }
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    if (threadIdx.x == 0 && rank == 0) {
        const int kept = blocks > 1 ? all : before;
        to.offsets[0] = 0, to.offsets[1] = kept, to.doubled[0] = 0, to.doubled[1] = 2 * kept;
        if (gradients) {
            for (int q = 0; q < 3; q++) {
                largest[q] = 0;
                for (int b = 0; b < blocks; b++) largest[q] = fmaxf(largest[q], *cluster.map_shared_rank(&most[q][0], b));
            }
            // (small gradients of sums are left out: 16-bit units are those of the losses', so that -1 stays -1)
            *to.unit = largest[1] <= 2 * largest[0] ? largest[0] : largest[2];
        }
    }
    if (blocks > 1) cluster.sync(); // (nobody leaves while others read what it found)
    if (bad) report_bad_index(st, 0);
}

// to[i,:] = from[order[i],:]
template <typename S>
__global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
loss_gather(S* __restrict__ to, int64_t to_stride, const S* __restrict__ from, int64_t stride, const LossRows rows, int64_t columns) {
    const int64_t kept = rows.offsets[1];
    for (int64_t i = first_row(); i < kept; i += row_step()) {
        const int64_t r = rows.order[i];
        for (int64_t c = threadIdx.x; c < columns; c += kRowThreads) to[i * to_stride + c] = from[r * stride + c];
    }
}

// to[r,:] = from[place[r],:], zeros for rows that have no place
template <typename S>
__global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
loss_scatter(S* __restrict__ to, const S* __restrict__ from, const LossRows rows, int64_t n, int64_t columns) {
    for (int64_t r = first_row(); r < n; r += row_step()) {
        const int64_t i = rows.place[r];
        for (int64_t c = threadIdx.x; c < columns; c += kRowThreads) to[r * columns + c] = i >= 0 ? from[i * columns + c] : S(0);
    }
}

template <typename S>
__global__ void __launch_bounds__(256)
add_values(S* __restrict__ to, const S* __restrict__ from, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) to[i] += from[i];
}

// The sums of parts of `part` columns of a piece's logits. A block to a part.
template <typename S>
__global__ void __launch_bounds__(256)
loss_sums(PartSum<S>* __restrict__ parts, int64_t n, int64_t first_part, S* __restrict__ at_target, const S* __restrict__ logits, int64_t columns, S scale,
          const int32_t* __restrict__ targets, int64_t first_column, int64_t part, const LossRows rows) {
    __shared__ PartSum<S> of_warp[8];
    const int64_t i = blockIdx.x, c0 = static_cast<int64_t>(blockIdx.y) * part;
    if (i >= rows.offsets[1]) return;
    const S* x = logits + i * columns;
    const int64_t end = min(c0 + part, columns);
    S top = -S(INFINITY);
    for (int64_t c = c0 + threadIdx.x; c < end; c += 256) top = fmax(top, scale * x[c]);
    const S base = PartSum<S>::from(top);
    S sum = 0;
    for (int64_t c = c0 + threadIdx.x; c < end; c += 256) sum += exp(scale * x[c] - base);
    PartSum<S> all{top, sum};
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
    for (int w = 1; w < 8; w++) all.join(of_warp[w]);
    parts[i * n + first_part + blockIdx.y] = all;
    const int64_t t = targets[rows.order[i]] - first_column;
    if (t >= c0 && t < end) at_target[i] = scale * x[t];
}

// The logits of a piece become scale dx.
template <typename S>
__global__ void __launch_bounds__(256)
loss_gradient(S* __restrict__ logits, int64_t columns, S scale, const S* __restrict__ grad_loss, const S* __restrict__ grad_log_sum,
              const S* __restrict__ log_sum, const int32_t* __restrict__ targets, int64_t first_column, int64_t part, const LossRows rows) {
    const int64_t i = blockIdx.x, c0 = static_cast<int64_t>(blockIdx.y) * part;
    if (i >= rows.offsets[1]) return;
    const int64_t r = rows.order[i], t = targets[r] - first_column;
    const S of_loss = grad_loss != nullptr ? grad_loss[r] : S(0), of_sum = grad_log_sum != nullptr ? grad_log_sum[r] : S(0);
    const S both = (of_loss + of_sum) * scale, base = log_sum[r];
    S* x = logits + i * columns;
    for (int64_t c = c0 + threadIdx.x; c < min(c0 + part, columns); c += 256) {
        S d = both * exp(scale * x[c] - base);
        if (c == t) d -= of_loss * scale;
        x[c] = d;
    }
}

// ---- f32, where the logits are summed: a lane has 64 of its row
template <int kOwn_> struct LossStoreOf {
    static constexpr bool kHalves = false, kMend = true, kAllRows = false;
    static constexpr int kOwn = kOwn_;
    struct Args {
        PartSum<float>* parts;
        int64_t n;
        float* at_target;
        const int32_t* target;
        int columns;
        float scale;
    };
    const Args& a;
    int lane;
    int64_t row = 0;
    int here = 0, first = 0, target = -1;
    __device__ LossStoreOf(const Args& a, uint32_t, int lane) : a(a), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) {
        row = r + lane, here = h, first = piece.column + half * kOwn;
        target = lane < here && piece.group >= 0 ? a.target[row] : -1;
    }
    __device__ __forceinline__ void store(float (&sum)[kOwn]) const {
        const int wide = min(a.columns - first, kOwn);
        if (wide <= 0) return;
        const int at = target - first;
        if (__any_sync(kFullMask, at >= 0 && at < wide)) {
            float x = 0;
#pragma unroll
            for (int j = 0; j < kOwn; j++)
                if (j == at) x = sum[j];
            if (at >= 0 && at < wide) a.at_target[row] = x * a.scale;
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < kOwn; j++) {
            if (wide < kOwn && j >= wide) sum[j] = -INFINITY;
            most[j % 4] = fmaxf(most[j % 4], sum[j]);
        }
        PartSum<float> part{fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * a.scale, 0.f};
        const float base = PartSum<float>::from(part.top);
        float all[4] = {};
#pragma unroll
        for (int j = 0; j < kOwn; j++) all[j % 4] += expf(fmaf(sum[j], a.scale, -base));
        part.sum = (all[0] + all[1]) + (all[2] + all[3]);
        if (lane < here) a.parts[row * a.n + first / kOwn] = part;
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {}
};

using LossStore32 = LossStoreOf<kSplitColumns / 2>;

// What dx takes of a lane's row.
struct RowGradient {
    int target = -1; // in the piece
    float base = 0, both = 0, of_loss = 0; // with the scale of the gradients
    template <typename Args> __device__ __forceinline__ void load(const Args& a, int64_t i) {
        const int64_t of = a.rows.order[i];
        target = a.rows.target[i] - a.first_column;
        const float l = a.grad_loss != nullptr ? a.grad_loss[of] : 0.f, m = a.grad_log_sum != nullptr ? a.grad_log_sum[of] : 0.f;
        base = a.log_sum[of], both = (l + m) * a.scale, of_loss = l * a.scale;
    }
};

struct GradientStore32 {
    static constexpr bool kHalves = false;
    static constexpr int kOwn = kSplitColumns / 2;
    struct Args {
        CUtensorMap map;
        float* out;
        int64_t stride;
        int columns, first_column; // of the piece
        float scale;
        const float *grad_loss, *grad_log_sum, *log_sum;
        LossRows rows;
    };
    const Args& a;
    BoxOut32 out;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, first = 0;
    RowGradient g;
    __device__ GradientStore32(const Args& a, uint32_t staging, int lane) : a(a), out{a.map, a.out, a.stride, a.columns, false}, staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) {
        row = r, here = h, first = piece.column + half * kOwn;
        if (lane < here && piece.group >= 0) g.load(a, row + lane); // (behind the last numbered row there are no numbers)
    }
    __device__ __forceinline__ void store(const float (&sum)[kOwn]) const {
#pragma unroll
        for (int c = 0; c < kOwn; c += 32) {
            if (first + c >= a.columns) return;
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = g.both * expf(fmaf(sum[c + j], a.scale, -g.base));
            const int at = g.target - first - c;
            if (__any_sync(kFullMask, at >= 0 && at < 32)) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j == at) v[j] -= g.of_loss;
            }
            out.put(v, staging, row, here, first + c, lane);
        }
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

// dx in three parts, with zeros in the rows behind the last one up to the end of the tile: products over the rows take whole stages of 64.
struct GradientParts {
    static constexpr bool kHalves = false, kMend = true, kAllRows = true;
    static constexpr int kOwn = kPartsOwn;
    struct Args {
        CUtensorMap map;
        int columns, first_column; // of the piece
        float scale;
        const float *grad_loss, *grad_log_sum, *log_sum;
        LossRows rows;
    };
    const Args& a;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, first = 0;
    RowGradient g;
    __device__ GradientParts(const Args& a, uint32_t staging, int lane) : a(a), staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) {
        row = r, here = h, first = piece.column + half * kOwn;
        if (lane < here && piece.group >= 0) g.load(a, row + lane);
    }
    __device__ __forceinline__ void store(float (&sum)[kOwn]) const {
#pragma unroll
        for (int c = 0; c < kOwn; c += 64) {
            if (first + c >= a.columns) return;
            const int at = g.target - first - c;
            const bool any = __any_sync(kFullMask, at >= 0 && at < 64);
#pragma unroll
            for (int j = 0; j < 64; j++) {
                float v = g.both * expf(fmaf(sum[c + j], a.scale, -g.base));
                if (any && j == at) v -= g.of_loss;
                sum[c + j] = lane < here ? v : 0.f;
            }
#pragma unroll
            for (int p = 0; p < kThreeParts; p++) {
                if (lane == 0) boxes_left<0>();
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t x = __float_as_uint(sum[c + 8 * k + 2 * q]), y = __float_as_uint(sum[c + 8 * k + 2 * q + 1]);
                        w[q] = split::cut_part(x, y);
                        sum[c + 8 * k + 2 * q] = __uint_as_float(x), sum[c + 8 * k + 2 * q + 1] = __uint_as_float(y);
                    }
                    smem_store16(staging + lane * kBoxRow + ((k ^ (lane & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
                }
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) box_out(a.map, first + c, static_cast<int>(row), p, staging);
            }
        }
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

const char* const kIndexNames[] = {"targets"};

} // namespace

template <typename S>
void prepare_rows(const Call& call, const LossRows& to, S* loss, S* log_sum, const Array& targets, int64_t vocabulary, int64_t ignored, const S* grad_loss,
                  const S* grad_log_sum) {
    const int64_t rows = targets.shape[0];
    Clusters clusters(call, "linear_cross_entropy", 1, rows > kPrepareThreads * kPrepareRows / 2 ? 8 : 1, 1, kPrepareThreads, 0);
    MOPS_CUDA_OK(cudaLaunchKernelEx(&clusters.config, loss_prepare<S>, to, loss, log_sum, static_cast<const int32_t*>(targets.data), rows, vocabulary, ignored, grad_loss,
                                    grad_log_sum, call.status));
    MOPS_CUDA_OK(cudaGetLastError());
}
template void prepare_rows(const Call&, const LossRows&, float*, float*, const Array&, int64_t, int64_t, const float*, const float*);

namespace {

// Sizes and types; the results have the type of sums.
void check_loss(Array& A, Array& W, Array& targets, Array& loss, Array& log_sum, double scale, const std::string& op) {
    check_floating(A.type, "A", op);
    check_array(A, "A", 2, A.type, op);
    check_array(W, "W", 2, A.type, op);
    check_array(targets, "targets", 1, MOPS_B200_I32, op);
    const int32_t sums = A.type == MOPS_B200_F64 ? MOPS_B200_F64 : MOPS_B200_F32;
    check_array(loss, "loss", 1, sums, op);
    check_array(log_sum, "log_sum", 1, sums, op);
    check_size(A.shape[1], "A", 1, W.shape[1], "W", 1, op);
    check_size(targets.shape[0], "targets", 0, A.shape[0], "A", 0, op);
    check_size(loss.shape[0], "loss", 0, A.shape[0], "A", 0, op);
    check_size(log_sum.shape[0], "log_sum", 0, A.shape[0], "A", 0, op);
    check_rows(A, "A", op);
    check_rows(W, "W", op);
    check_rows(targets, "targets", op);
    check_output(loss, "loss", op);
    check_output(log_sum, "log_sum", op);
    if (W.shape[0] == 0) throw std::runtime_error("W must have a row in " + op);
    if (!(scale > 0) || std::isinf(scale)) throw std::runtime_error("scale must be positive and finite in " + op);
    for (int64_t n : {A.shape[0], A.shape[1], W.shape[0]}) fits_int32(static_cast<size_t>(n), "a size", op);
}

unsigned blocks_for(const Call& call, int64_t n) {
    return static_cast<unsigned>(std::min<int64_t>(ceil_div(n, 256), int64_t(sm_count(call.device)) * 16));
}

// Whether operands are cut into parts beforehand, which takes a pass over them and tiles of 256 x 256: 4000 rows of 8000 x 512 169 us for 230 without, with gradients 629 for 952; 1500 of 1000 x 2048 (6 GFLOP) 102
// and 306 for 80 and 302; 4000 of 8000 x 48 74 and 323 for 57 and 294; 300 of 8000 x 512 53 and 163 for 40 and 154.
bool worth_cutting(int64_t rows, int64_t vocabulary, int64_t columns) { return rows >= 512 && columns >= 128 && 2.0 * rows * vocabulary * columns >= 8e9; }

// What forward and backward share: the rows that count, gathered and as the products want them, W likewise, and the logits of a piece.
template <typename S> struct Pieces {
    const Call& call;
    const std::string& op;
    Scratch room_rows, room_A, room_logits;
    Packing packing;
    LossRows rows;
    Array A, W, logits;
    int64_t width, part; // columns of a piece, and of a part of it
    bool fused;          // worked on where they are summed
    bool numbered;       // rows without a target have been left out
    bool in_parts;       // operands are cut beforehand
    bool sliced;         // or in slices of the depth, where tiles would leave SMs without work, to be worked on where they are stored
    PartsArray parts_A{}, parts_W{};
    Scratch room_parts_A, room_parts_W;
    static constexpr int32_t kType = sizeof(S) == 8 ? MOPS_B200_F64 : MOPS_B200_F32;

    Pieces(const Call& call, const std::string& op, const Array& a, const Array& w, bool forward)
        : call(call), op(op), room_rows(call), room_A(call), room_logits(call), packing(call), W(w), room_parts_A(call), room_parts_W(call) {
        const int64_t n = a.shape[0], columns = a.shape[1];
        W.type = kType; // (of another type there are no values)
        width = std::max<int64_t>(kMostLogits / n, 256);
        width = width >= kPartColumns ? width / kPartColumns * kPartColumns : width / 256 * 256;
        part = std::min(width, kPartColumns);
        width = std::min(width, W.shape[0]);
        fused = kType == MOPS_B200_F32 && columns > 0;
        in_parts = fused && worth_cutting(n, W.shape[0], columns);
        // (674 rows of 60 x 3040, 6 tiles: 31 us for 86, with gradients 97 for 219; 200 of 1000 x 4096, 16 tiles, 53 and 159 for 115 and 290. But 60 of 4000 x 2048, 32 tiles, 76 and 197 for 63 and 179, and
        // with less depth the host's part of three more launches is longer: 674 of 60 x 1024 43 for 37)
        const int64_t tiles = ceil_div(n, kTileRows) * ceil_div(W.shape[0], kSplitColumns), sms = sm_count(call.device);
        sliced = fused && !in_parts && columns >= 2048 && (8 * tiles <= sms || (4 * tiles <= sms && W.shape[0] <= kSplitColumns));
        numbered = !forward || !fused || in_parts || sliced || worth_gathering(kType, n, W.shape[0], columns);
        if (numbered) {
            rows = take_rows(room_rows, n);
            const int64_t stride = fused ? (columns + 3) / 4 * 4 : columns; // (as the copy engine can fetch them)
            room_A.take(static_cast<size_t>(n * stride) * sizeof(S) + 16);
            A = contiguous(room_A.as<void>(), kType, n, columns);
            A.stride[0] = stride;
        } else {
            rows = LossRows{};
            A = a;
        }
    }
    void take_logits() { room_logits.take(static_cast<size_t>(A.shape[0] * (width + 3)) * sizeof(S) + 16); }
    TileProblem problem(int64_t columns) const { return {A, rows.offsets, 1, A.shape[0], A.shape[1], columns}; }
    void gather(const Array& a) {
        if (a.shape[1] == 0) return;
        if (numbered)
            loss_gather<S><<<row_blocks(call, a.shape[0]), row_threads(), 0, call.stream>>>(static_cast<S*>(A.data), A.stride[0], static_cast<const S*>(a.data), a.stride[0], rows,
                                                                                             a.shape[1]);
        MOPS_CUDA_OK(cudaGetLastError());
        if (in_parts) {
            if constexpr (sizeof(S) == 4) {
                const int64_t outer = padded_rows(), wide = (W.shape[1] + 7) / 8 * 8;
                room_parts_A.take(static_cast<size_t>(outer * wide) * 2 * kThreeParts);
                room_parts_W.take(static_cast<size_t>(W.shape[0] * wide) * 2 * kThreeParts);
                parts_A = cut(call, room_parts_A.as<void>(), static_cast<const float*>(A.data), A.stride[0], A.shape[0], outer, A.shape[1], rows.offsets + 1);
                parts_W = cut(call, room_parts_W.as<void>(), static_cast<const float*>(W.data), W.stride[0], W.shape[0], W.shape[0], W.shape[1], nullptr);
            }
        } else if (fused) {
            packing.add(A);
            packing.add(W);
            packing.run();
        }
    }
    int64_t padded_rows() const { return ceil_div(A.shape[0], kPartsTile) * kPartsTile; }
    SplitOperands operands(int64_t v0) const { // in f32
        return {static_cast<const float*>(A.data), {static_cast<const float*>(W.data) + v0 * W.stride[0], nullptr}, A.stride[0], 0, 1, W.stride[0]};
    }
    PartsArray parts_of(int64_t v0, int64_t v1) const { // rows v0 .. v1 of W
        PartsArray p = parts_W;
        p.data = static_cast<uint16_t*>(p.data) + v0 * p.stride, p.outer = v1 - v0;
        return p;
    }
    // The rows v0 .. v1 of W as the single group's matrix, C x (v1 - v0).
    Array matrices(int64_t v0, int64_t v1) const {
        Array m = contiguous(static_cast<S*>(W.data) + v0 * W.stride[0], kType, 1, W.shape[1], v1 - v0);
        m.stride[1] = 1, m.stride[2] = W.stride[0];
        return m;
    }
    template <typename F> void for_each(F&& f) {
        take_logits();
        for (int64_t v0 = 0; v0 < W.shape[0]; v0 += width) {
            const int64_t v1 = std::min(v0 + width, W.shape[0]);
            const Array m = matrices(v0, v1);
            logits = contiguous(room_logits.as<void>(), kType, A.shape[0], v1 - v0);
            const RowsProblem problem{logits, A, m, m.stride[1], m.stride[2], rows.offsets, 1, A.shape[0], A.shape[1], v1 - v0};
            if (!sliced || !multiply_rows_sliced(call, problem, kLeastSteps, op)) multiply_rows(call, problem, op);
            const dim3 grid(static_cast<unsigned>(A.shape[0]), static_cast<unsigned>(ceil_div(v1 - v0, part)));
            f(v0, v1, grid, static_cast<S*>(logits.data));
            MOPS_CUDA_OK(cudaGetLastError());
        }
    }
};

template <typename S>
void loss_forward(const Call& call, const Array& loss, const Array& log_sum, const Array& A, const Array& W, const Array& targets, double scale,
                  int64_t ignored, const std::string& op) {
    if constexpr (sizeof(S) == 4) {
        if (A.type == MOPS_B200_F32 && few_loss_rows({A, W, targets, scale, ignored})) {
            loss_forward_few(call, {A, W, targets, scale, ignored}, loss, log_sum);
            return;
        }
    }
    Pieces<S> pieces(call, op, A, W, true);
    const int64_t n = A.shape[0], parts = ceil_div(W.shape[0], pieces.in_parts ? kPartsOwn : pieces.fused && !pieces.sliced ? LossStore32::kOwn : pieces.part);
    const int32_t* t = static_cast<const int32_t*>(targets.data);
    if (pieces.numbered) prepare_rows<S>(call, pieces.rows, static_cast<S*>(loss.data), static_cast<S*>(log_sum.data), targets, W.shape[0], ignored, nullptr, nullptr);
    pieces.gather(A);
    Scratch room(call, static_cast<size_t>(n * parts) * sizeof(PartSum<S>) + static_cast<size_t>(n) * sizeof(S));
    PartSum<S>* sums = room.as<PartSum<S>>();
    S* at_target = reinterpret_cast<S*>(sums + n * parts);
    if constexpr (sizeof(S) == 4) {
        if (pieces.in_parts) {
            using E = LossStoreOf<kPartsOwn>;
            const E::Args args{sums, parts, at_target, pieces.rows.target, static_cast<int>(W.shape[0]), static_cast<float>(scale)};
            launch_parts<false, false, E, DecodeRows>(call, op, pieces.parts_A, pieces.parts_W, pieces.rows.offsets, n, W.shape[1], W.shape[0], 1, pieces.operands(0), args);
            note_kernel("loss_rows_parts");
        } else if (pieces.fused && !pieces.sliced) {
            const LossStore32::Args args{sums, parts, at_target, pieces.numbered ? pieces.rows.target : t, static_cast<int>(W.shape[0]), static_cast<float>(scale)};
            const TileOperand w{pieces.W.data, 1, pieces.W.stride[0], 0}, operands[2] = {w, w};
            if (pieces.numbered) launch_split<false, LossStore32, DecodeRows>(call, op, pieces.problem(W.shape[0]), operands, args);
            else launch_split<false, LossStore32, DecodeTable>(call, op, pieces.problem(W.shape[0]), operands, args);
            note_kernel("loss_rows_split");
        }
    }
    if (!pieces.fused || pieces.sliced) pieces.for_each([&](int64_t v0, int64_t v1, dim3 grid, S* logits) {
        loss_sums<S><<<grid, 256, 0, call.stream>>>(sums, parts, v0 / pieces.part, at_target, logits, v1 - v0, static_cast<S>(scale), t, v0, pieces.part,
                                                     pieces.rows);
    });
    join_rows<S>(call, loss, log_sum, sums, parts, at_target, pieces.rows, targets, W.shape[0], ignored);
    note_kernel_f("loss_sums<%s>", scalar_name<S>());
}

template <typename S>
void loss_backward(const Call& call, const Array& grad_A, const Array& grad_W, const Array& grad_loss, const Array& grad_log_sum, const Array& log_sum,
                   const Array& A, const Array& W, const Array& targets, double scale, int64_t ignored, const std::string& op) {
    Pieces<S> pieces(call, op, A, W, false);
    const int64_t n = A.shape[0], columns = A.shape[1];
    const int32_t* t = static_cast<const int32_t*>(targets.data);
    prepare_rows<S>(call, pieces.rows, nullptr, nullptr, targets, W.shape[0], ignored, nullptr, nullptr);
    if (columns == 0) return;
    pieces.gather(A);
    const bool need_A = grad_A.data != nullptr, need_W = grad_W.data != nullptr;
    Scratch room_A(call), room_more(call);
    const int64_t stride_A = pieces.fused ? (columns + 3) / 4 * 4 : columns; // of the sums for grad_A
    int64_t slices = 1;
    if (pieces.in_parts && need_A) {
        slices = best_slices(ceil_div(n, kPartsTile) * ceil_div(columns, kPartsTile), sm_count(call.device) / 2, ceil_div(pieces.width, kBoxDepth), 2.5, 8,
                             static_cast<double>(n) * columns * 8);
    } else if (pieces.fused && need_A) {
        const int64_t deep = ceil_div(pieces.width, split::kDepth), tiles = ceil_div(n, kTileRows) * ceil_div(columns, kSplitColumns);
        slices = best_slices(tiles, sm_count(call.device), deep, 0.7, 16, static_cast<double>(n) * columns * 8);
    }
    const size_t bytes = static_cast<size_t>(slices * n * stride_A) * sizeof(S);
    if (need_A) room_A.take(bytes);
    if (need_A && !pieces.fused && pieces.width < W.shape[0]) room_more.take(bytes);
    auto multiply = [&](int64_t v0, int64_t v1, Array dx) {
        Array m = pieces.matrices(v0, v1), a = pieces.A;
        m.shape[1] = v1 - v0, m.shape[2] = columns; // (v1 - v0) x C
        std::swap(m.stride[1], m.stride[2]);
        Packing packing(call);
        if (pieces.fused) {
            const bool outer_packed = need_W && !straight_outer(n, 1, v1 - v0, columns, pieces.kType);
            if (need_A || outer_packed) packing.add(dx);
            if (need_A) packing.add(m);
            if (outer_packed) packing.add(a);
            packing.run();
        }
        if (need_A && pieces.fused) {
            if constexpr (sizeof(S) == 4) {
                TileProblem problem{dx, pieces.rows.offsets, 1, n, v1 - v0, columns, slices};
                const TileOperand w{m.data, m.stride[1], 1, 0}, operands[2] = {w, w};
                launch_split<true, SumStore32, DecodeRowSlices>(call, op, problem, operands, sum_args(room_A.template as<float>(), slices, n, stride_A, columns, v0 > 0));
            }
        } else if (need_A) {
            S* to = v0 == 0 ? room_A.as<S>() : room_more.as<S>();
            multiply_rows(call, {contiguous(to, pieces.kType, n, columns), dx, m, m.stride[1], 1, pieces.rows.offsets, 1, n, v1 - v0, columns}, op);
            if (v0 > 0) add_values<S><<<blocks_for(call, n * columns), 256, 0, call.stream>>>(room_A.as<S>(), to, n * columns);
        }
        if (need_W) multiply_outer(call, {contiguous(static_cast<S*>(grad_W.data) + v0 * columns, pieces.kType, 1, v1 - v0, columns), dx, a, pieces.rows.offsets, 1}, op);
        packing.release();
    };
    if (pieces.in_parts) {
        if constexpr (sizeof(S) == 4) {
            const int64_t stride = (pieces.width + 7) / 8 * 8, outer = pieces.padded_rows();
            Scratch room_dx(call, static_cast<size_t>(outer * stride) * 2 * kThreeParts), room_sums(call);
            // the products with A: straight to where they belong, if that can be, and their depth need not be cut
            const int64_t deep = ceil_div(n, kBoxDepth), tiles = ceil_div(pieces.width, kPartsTile) * ceil_div(columns, kPartsTile);
            const int64_t cuts = best_slices(tiles, sm_count(call.device) / 2, deep, 2.5, 8, static_cast<double>(pieces.width) * columns * 8);
            const bool straight = cuts == 1 && columns % 4 == 0 && reinterpret_cast<uintptr_t>(grad_W.data) % 16 == 0;
            if (need_W && !straight) room_sums.take(static_cast<size_t>(cuts * pieces.width * stride_A) * sizeof(float));
            using Sums = SumStoreOf<kPartsOwn>;
            for (int64_t v0 = 0; v0 < W.shape[0]; v0 += pieces.width) {
                const int64_t v1 = std::min(v0 + pieces.width, W.shape[0]), here = v1 - v0;
                const PartsArray dx{room_dx.as<void>(), here, outer, stride, outer * stride}, w = pieces.parts_of(v0, v1);
                const GradientParts::Args args{dx.map(32), static_cast<int>(here), static_cast<int>(v0), static_cast<float>(scale), static_cast<const float*>(grad_loss.data),
                                               static_cast<const float*>(grad_log_sum.data), static_cast<const float*>(log_sum.data), pieces.rows};
                launch_parts<false, false, GradientParts, DecodeRows>(call, op, pieces.parts_A, w, pieces.rows.offsets, n, columns, here, 1, pieces.operands(v0), args);
                if (need_A)
                    launch_parts<false, true, Sums, DecodeRowSlices>(call, op, dx, w, pieces.rows.offsets, n, here, columns, slices, {},
                                                                     sum_args<Sums>(room_A.template as<float>(), slices, n, stride_A, columns, v0 > 0));
                if (need_W) {
                    float* to = static_cast<float*>(grad_W.data) + v0 * columns;
                    launch_parts<true, true, Sums, DecodeDepth>(call, op, dx, pieces.parts_A, pieces.rows.offsets, here, n, columns, cuts, {},
                                                                sum_args<Sums>(straight ? to : room_sums.as<float>(), cuts, here, stride_A, columns, false));
                    if (!straight) add_slices<<<blocks_for(call, here * stride_A / 4), 256, 0, call.stream>>>(to, room_sums.as<float>(), static_cast<int>(cuts), here, stride_A,
                                                                                                         static_cast<int>(columns));
                }
                MOPS_CUDA_OK(cudaGetLastError());
            }
        }
    } else if (pieces.fused && !pieces.sliced) {
        if constexpr (sizeof(S) == 4) {
            pieces.take_logits();
            const int64_t stride = (pieces.width + 3) / 4 * 4;
            for (int64_t v0 = 0; v0 < W.shape[0]; v0 += pieces.width) {
                const int64_t v1 = std::min(v0 + pieces.width, W.shape[0]);
                Array dx = contiguous(pieces.room_logits.template as<void>(), pieces.kType, n, v1 - v0);
                dx.stride[0] = stride;
                const GradientStore32::Args args{tensor_map(pieces.kType, dx.data, v1 - v0, n, 1, stride, 0, 32), static_cast<float*>(dx.data), stride,
                                                 static_cast<int>(v1 - v0), static_cast<int>(v0), static_cast<float>(scale), static_cast<const float*>(grad_loss.data),
                                                 static_cast<const float*>(grad_log_sum.data), static_cast<const float*>(log_sum.data), pieces.rows};
                const TileOperand w{static_cast<float*>(pieces.W.data) + v0 * pieces.W.stride[0], 1, pieces.W.stride[0], 0}, operands[2] = {w, w};
                launch_split<false, GradientStore32, DecodeRows>(call, op, pieces.problem(v1 - v0), operands, args);
                multiply(v0, v1, dx);
                MOPS_CUDA_OK(cudaGetLastError());
            }
        }
    } else {
        pieces.for_each([&](int64_t v0, int64_t v1, dim3 grid, S* logits) {
            loss_gradient<S><<<grid, 256, 0, call.stream>>>(logits, v1 - v0, static_cast<S>(scale), static_cast<const S*>(grad_loss.data),
                                                            static_cast<const S*>(grad_log_sum.data), static_cast<const S*>(log_sum.data), t, v0, pieces.part, pieces.rows);
            multiply(v0, v1, pieces.logits);
        });
    }
    if (need_A) {
        if constexpr (sizeof(S) == 4) {
            if (pieces.fused) scatter_sums(call, static_cast<float*>(grad_A.data), room_A.template as<float>(), slices, stride_A, pieces.rows, n, columns, false, nullptr);
        }
        if (!pieces.fused) loss_scatter<S><<<row_blocks(call, n), row_threads(), 0, call.stream>>>(static_cast<S*>(grad_A.data), room_A.as<S>(), pieces.rows, n, columns);
    }
    MOPS_CUDA_OK(cudaGetLastError());
    note_kernel_f("loss_gradient<%s>", scalar_name<S>());
}

bool sixteen_bits(const Array& A) { return (A.type == MOPS_B200_F16 || A.type == MOPS_B200_BF16) && A.shape[1] > 0; }

} // namespace

void linear_cross_entropy(Array loss, Array log_sum, Array A, Array W, Array targets, double scale, int64_t ignore_index) {
    const std::string op = "cuda_linear_cross_entropy";
    check_loss(A, W, targets, loss, log_sum, scale, op);
    if (A.shape[0] == 0) return;
    Call call = begin_call();
    // Rows some at a time: the sums of their parts, one for each 64 columns at the most, shall not take more than 2 GB.
    const int64_t most = std::max<int64_t>((int64_t(1) << 31) / (ceil_div(W.shape[0], 64) * 16), 1024), n = A.shape[0];
    for (int64_t r = 0; r < n; r += most) {
        auto rows = [&](const Array& a) {
            Array part = a;
            part.data = static_cast<unsigned char*>(a.data) + r * a.stride[0] * type_bytes(a.type);
            part.shape[0] = std::min(most, n - r);
            return part;
        };
        if (sixteen_bits(A)) loss_forward_mma(call, {rows(A), W, rows(targets), scale, ignore_index}, rows(loss), rows(log_sum), op);
        else if (A.type == MOPS_B200_F64) loss_forward<double>(call, rows(loss), rows(log_sum), rows(A), W, rows(targets), scale, ignore_index, op);
        else loss_forward<float>(call, rows(loss), rows(log_sum), rows(A), W, rows(targets), scale, ignore_index, op);
    }
    end_call(call, op.c_str(), kIndexNames, 1);
}

void linear_cross_entropy_vjp(Array grad_A, Array grad_W, Array grad_loss, Array grad_log_sum, Array loss, Array log_sum, Array A, Array W,
                              Array targets, double scale, int64_t ignore_index) {
    const std::string op = "cuda_linear_cross_entropy_vjp";
    check_loss(A, W, targets, loss, log_sum, scale, op);
    auto given = [&](Array& g, const char* name) {
        if (g.data == nullptr && g.dimensions == 0) return;
        check_array(g, name, 1, loss.type, op);
        check_size(g.shape[0], name, 0, A.shape[0], "A", 0, op);
        check_output(g, name, op);
    };
    given(grad_loss, "grad_loss");
    given(grad_log_sum, "grad_log_sum");
    auto wanted = [&](Array& g, const char* name, const Array& of, const char* of_name) {
        if (g.data == nullptr) return;
        check_array(g, name, 2, A.type, op);
        for (int d = 0; d < 2; d++) check_size(g.shape[d], name, d, of.shape[d], of_name, d, op);
        check_output(g, name, op);
    };
    wanted(grad_A, "grad_A", A, "A");
    wanted(grad_W, "grad_W", W, "W");
    if (grad_A.data == nullptr && grad_W.data == nullptr) return;
    Call call = begin_call();
    if (A.shape[0] == 0) {
        if (grad_W.data != nullptr)
            MOPS_CUDA_OK(cudaMemsetAsync(grad_W.data, 0, static_cast<size_t>(values_of(grad_W) * type_bytes(grad_W.type)), call.stream));
    } else if (sixteen_bits(A)) {
        loss_backward_mma(call, {A, W, targets, scale, ignore_index}, grad_A, grad_W, grad_loss, grad_log_sum, loss, log_sum, op);
    } else if (A.type == MOPS_B200_F64) {
        loss_backward<double>(call, grad_A, grad_W, grad_loss, grad_log_sum, log_sum, A, W, targets, scale, ignore_index, op);
    } else {
        loss_backward<float>(call, grad_A, grad_W, grad_loss, grad_log_sum, log_sum, A, W, targets, scale, ignore_index, op);
    }
    end_call(call, op.c_str(), kIndexNames, 1);
}

} // namespace mops_b200
