// grouped_matrix_product for a few rows in all: single tokens, each with a matrix of its own.
//
// Nothing but the matrices counts: each of their values is read once and multiplied by the values of one or a few rows. What matters is that enough of
// them is under way on all SMs, from the first microsecond on. So a block has one tile of the output, as many blocks as fit are on an SM, and where there are too few tiles
// the depth is cut: the blocks of a cluster, each with a part of it, add up their sums through each other's shared memory.
//
// 16 bits: the tensor cores with the operands the other way round. The matrix gives the 128 rows of the accumulator, the rows of X its 16 or 64 columns, so that
// little is fetched besides the matrix. In bf16, 16 rows of 32 groups, 2048 x 1536 (12 of them used, 75 MB): 16.3 us, 4.6 TB/s, which is bounded by how fast the copies of a block
// that has just begun get under way; tiles of 128 rows, whose blocks fetch as much of X as of the matrices, 23.0 us. Two rows of 16 groups, 4096 x 1024: 8.4 and 25.7 us.
// f32, f64 and matrices whose rows begin anywhere: the ordinary units, straight from the loads. In f32 the first of them takes 43 us (3.5 TB/s; tiles of 128 rows 61), eight rows of 8 groups, 128 x 128, 4.6 (9.0); bounded
// by the loads that a block's registers can hold.
#include "few_rows.cuh"
#include "grouped_mma.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {
namespace {

// The tile's 128 columns are rows (lanes) of the accumulator, the rows of X its columns.
template <typename T, bool M_MN, int kRows>
__global__ void __launch_bounds__(kTileThreads)
few_rows_mma(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m, T* __restrict__ out,
             const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int depth, int columns, Status st) {
    extern __shared__ unsigned char raw[];
    using L = FewLayout<kRows>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int column = static_cast<int>(blockIdx.x) / parts * kTileRows;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(offsets, groups, rows, st);
    if (blockIdx.y == 0 && rank == 0) clear_others<T, kTileRows, kTileThreads>(out, offsets, groups, rows, column, columns);
    GroupWalk<FewRows> walk(offsets, groups, rows, 0, groups - 1, FewRows{kRows});
    const GroupPiece piece = walk.find(blockIdx.y, lane);
    if (!piece.found) return; // (all blocks of the cluster)
    const int64_t row = piece.lo + piece.within * kRows;
    const int here = static_cast<int>(min(piece.hi - row, int64_t(kRows)));
    const int all_steps = (depth + kBoxDepth - 1) / kBoxDepth, per = (all_steps + parts - 1) / parts;
    const int from = min(rank * per, all_steps), to = min(from + per, all_steps);
    Block<L> block(raw, st);
    block.begin(warp);
    Turn<L::kStages> stage;
    bool ok = true;
    if (threadIdx.x == 0) {
        for (int s = from; s < to; s++) {
            ok = block.wait_empty(block.rings->stages, stage);
            if (!ok) break;
            uint64_t* full = &block.rings->stages.full[stage.at];
            const uint32_t m = block.base + static_cast<uint32_t>(stage.at) * L::kStage;
            mbarrier_arrive_expect(full, L::kStage);
            if constexpr (M_MN) {
#pragma unroll
                for (int j = 0; j < kTileRows / 64; j++)
                    box_in(m + j * kBoxBytes, map_m, column + j * 64, s * kBoxDepth, static_cast<int>(piece.group), full);
            } else {
                box_in(m, map_m, s * kBoxDepth, column, static_cast<int>(piece.group), full);
            }
            box_in(m + L::kM, map_x, s * kBoxDepth, static_cast<int>(row), 0, full);
            stage.next();
        }
        block.drain(block.rings->stages, stage, to - from);
    } else if (threadIdx.x == 32) {
        constexpr uint32_t instruction = instruction_descriptor(std::is_same<T, __nv_bfloat16>::value, M_MN, false, kRows);
        for (int s = from; s < to; s++) {
            ok = block.wait_full(block.rings->stages, stage);
            if (!ok) break;
            tmem_fence_after_sync();
            const uint32_t at = block.base + static_cast<uint32_t>(stage.at) * L::kStage;
            const uint64_t m = operand_descriptor(at, kBoxBytes), x = operand_descriptor(at + L::kM, kBoxBytes);
#pragma unroll
            for (int k = 0; k < kBoxDepth / 16; k++)
                umma(block.rings->tmem, m + k * kDepthStep<M_MN>, x + k * kDepthStep<false>, instruction, s > from || k > 0);
            umma_arrive(&block.rings->stages.empty[stage.at]);
            stage.next();
        }
        if (ok) umma_arrive(&block.rings->done);
    }
    __syncwarp();
    if (lane == 0) ok = block.wait(&block.rings->done, 0);
    __syncwarp();
    tmem_fence_after_sync();
    // A column to a thread. The sums of the parts go through shared memory, where the stages were; each block of a cluster joins every parts-th row. (Written
    // into the shared memory of the one that joins them, instead of read from that of the others: 17.9 us for 12.5, 128 rows, 4096 x 1024.)
    const uint32_t accumulator = tmem_quadrant(block.rings->tmem, warp);
    float* part = reinterpret_cast<float*>(block.smem) + threadIdx.x;
    T* to_column = out + row * columns + column + threadIdx.x;
    const bool mine = column + static_cast<int>(threadIdx.x) < columns;
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 8) {
        if (r0 >= here) break;
        uint32_t v[8];
        tmem_load(accumulator + r0, v);
        tmem_wait_load();
        tmem_pin(v);
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const float sum = from < to ? __uint_as_float(v[r]) : 0.f; // (a part of no steps has left nothing in its accumulator)
            if (parts > 1) part[(r0 + r) * kTileRows] = sum;
            else if (r0 + r < here && mine) to_column[static_cast<int64_t>(r0 + r) * columns] = narrow<T>(sum);
        }
    }
    if (parts > 1) {
        cluster.sync();
        const float* parts_of[kMostParts];
#pragma unroll
        for (int b = 0; b < kMostParts; b++) parts_of[b] = cluster.map_shared_rank(part, b < parts ? b : rank);
#pragma unroll 2
        for (int r = rank; r < here; r += parts) {
            float v[kMostParts], sum = 0; // (side by side: the way to another SM and back takes its time)
#pragma unroll
            for (int b = 0; b < kMostParts; b++) v[b] = b < parts ? parts_of[b][r * kTileRows] : 0.f;
#pragma unroll
            for (int b = 0; b < kMostParts; b++) sum += v[b];
            if (mine) to_column[static_cast<int64_t>(r) * columns] = narrow<T>(sum);
        }
        cluster.sync(); // (nobody leaves while others read its sums)
    }
    block.end(warp);
}

// ---------------------------------------------------------------------------------- f32 and f64
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 4;         // of a block
constexpr int kMostRows = 64;    // of a call
constexpr int kChunk = 1024;     // values of depth of the rows that are in shared memory at a time
// (loads of a thread under way: 128 bytes where they are whole packs)
template <typename T, int N> constexpr int kInFlight = N > 1 ? 8 : 16;

template <typename T> struct Few {
    T* out;
    const T *x, *m;
    int64_t x_stride, group_stride, stride; // stride: of m, between its rows of neighbouring values
    const int32_t* offsets;
    int64_t groups, rows;
    int depth, columns;
};

// Adds up the sums of a cluster's blocks (part: kRows x kColumns in each one's shared memory) and writes them.
template <typename T, int kColumns>
__device__ __forceinline__ void join_parts(Sum<T>* part, const Few<T>& p, int64_t row, int here, int column) {
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks(), rank = cluster.block_rank();
    if (parts > 1) cluster.sync();
    else __syncthreads();
    for (int i = rank * kThreads + threadIdx.x; i < kRows * kColumns; i += parts * kThreads) {
        const int r = i / kColumns, c = i % kColumns;
        Sum<T> sum = 0;
        if (parts > 1)
            for (int b = 0; b < parts; b++) sum += cluster.map_shared_rank(part, b)[i];
        else
            sum = part[i];
        if (r < here && column + c < p.columns) p.out[(row + r) * p.columns + column + c] = narrow<T>(sum);
    }
    if (parts > 1) cluster.sync(); // (nobody leaves while others read its sums)
}

// Columns that are neighbours in memory (depth x columns). kAcross threads side by side take a pack of N columns each, the rows of such threads every kDown-th value of depth.
template <int N> constexpr int kAcross = N > 1 ? 16 : 64;
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
few_rows_columns(const __grid_constant__ Few<T> p, Status st) {
    using S = Sum<T>;
    constexpr int kAcross = mops_b200::kAcross<N>, kInFlight = mops_b200::kInFlight<T, N>, kDown = kThreads / kAcross, kColumns = kAcross * N;
    __shared__ S x[kRows][kChunk];
    __shared__ S sums[kDown][kRows * kColumns / 4]; // a quarter of the columns at a time
    __shared__ S part[kRows * kColumns];
    const int lane = threadIdx.x & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks(), rank = cluster.block_rank();
    const int column = static_cast<int>(blockIdx.x / parts) * kColumns;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(p.offsets, p.groups, p.rows, st);
    if (blockIdx.y == 0 && rank == 0) clear_others<T, kColumns, kThreads>(p.out, p.offsets, p.groups, p.rows, column, p.columns);
    GroupWalk<FewRows> walk(p.offsets, p.groups, p.rows, 0, p.groups - 1, FewRows{kRows});
    const GroupPiece piece = walk.find(blockIdx.y, lane);
    if (!piece.found) return; // (all blocks of the cluster)
    const int64_t row = piece.lo + piece.within * kRows;
    const int here = static_cast<int>(min(piece.hi - row, int64_t(kRows)));
    const int per = (p.depth + parts * kDown - 1) / (parts * kDown) * kDown;
    const int from = min(rank * per, p.depth), to = min(from + per, p.depth);
    const int across = threadIdx.x % kAcross, down = threadIdx.x / kAcross;
    const bool mine = column + across * N < p.columns;
    const T* m = p.m + piece.group * p.group_stride + column + across * N;
    S sum[kRows][N];
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int i = 0; i < N; i++) sum[r][i] = 0;
    for (int k0 = from; k0 < to; k0 += kChunk) {
        const int n = min(to - k0, kChunk);
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * n; i += kThreads) {
            const int r = i / n, k = i - r * n;
            x[r][k] = r < here ? widen(p.x[(row + r) * p.x_stride + k0 + k]) : S(0);
        }
        __syncthreads();
        if (!mine) continue;
        for (int k = down; k < n; k += kDown * kInFlight) {
            Pack<T, N> w[kInFlight];
#pragma unroll
            for (int u = 0; u < kInFlight; u++)
                if (k + u * kDown < n) w[u] = *reinterpret_cast<const Pack<T, N>*>(m + (k0 + k + u * kDown) * p.stride);
#pragma unroll
            for (int u = 0; u < kInFlight; u++) {
                if (k + u * kDown >= n) break;
#pragma unroll
                for (int r = 0; r < kRows; r++) {
                    if (r >= here) break;
                    const S v = x[r][k + u * kDown];
#pragma unroll
                    for (int i = 0; i < N; i++) sum[r][i] += v * widen(w[u].v[i]);
                }
            }
        }
    }
    // the rows of threads, then the blocks of the cluster
#pragma unroll
    for (int q = 0; q < 4; q++) {
        __syncthreads();
        if (across / (kAcross / 4) == q) {
#pragma unroll
            for (int r = 0; r < kRows; r++)
#pragma unroll
                for (int i = 0; i < N; i++) sums[down][r * (kColumns / 4) + across % (kAcross / 4) * N + i] = sum[r][i];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * kColumns / 4; i += kThreads) {
            S all = 0;
#pragma unroll
            for (int d = 0; d < kDown; d++) all += sums[d][i];
            part[i / (kColumns / 4) * kColumns + q * (kColumns / 4) + i % (kColumns / 4)] = all;
        }
    }
    join_parts<T, kColumns>(part, p, row, here, column);
}

// Depth that is neighbours in memory (columns x depth). A warp takes four columns, its lanes packs of N values of the depth.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
few_rows_depth(const __grid_constant__ Few<T> p, Status st) {
    using S = Sum<T>;
    constexpr int kOwn = 4, kColumns = kWarps * kOwn, kInFlight = 4 * mops_b200::kInFlight<T, N> / (N > 1 ? 4 : 2);
    __shared__ alignas(16) T x[kRows][kChunk];
    __shared__ S part[kRows * kColumns];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks(), rank = cluster.block_rank();
    const int column = static_cast<int>(blockIdx.x / parts) * kColumns;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(p.offsets, p.groups, p.rows, st);
    if (blockIdx.y == 0 && rank == 0) clear_others<T, kColumns, kThreads>(p.out, p.offsets, p.groups, p.rows, column, p.columns);
    GroupWalk<FewRows> walk(p.offsets, p.groups, p.rows, 0, p.groups - 1, FewRows{kRows});
    const GroupPiece piece = walk.find(blockIdx.y, lane);
    if (!piece.found) return; // (all blocks of the cluster)
    const int64_t row = piece.lo + piece.within * kRows;
    const int here = static_cast<int>(min(piece.hi - row, int64_t(kRows)));
    const int per = (p.depth + parts * N - 1) / (parts * N) * N;
    const int from = min(rank * per, p.depth), to = min(from + per, p.depth); // (whole packs: the depth is a multiple of N)
    const T* m = p.m + piece.group * p.group_stride + (column + warp * kOwn) * p.stride;
    S sum[kRows][kOwn];
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int c = 0; c < kOwn; c++) sum[r][c] = 0;
    for (int k0 = from; k0 < to; k0 += kChunk) {
        const int n = min(to - k0, kChunk);
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * n; i += kThreads) {
            const int r = i / n, k = i - r * n;
            x[r][k] = r < here ? p.x[(row + r) * p.x_stride + k0 + k] : narrow<T>(0);
        }
        __syncthreads();
        for (int k = lane * N; k < n; k += 32 * N * (kInFlight / kOwn)) {
            Pack<T, N> w[kInFlight / kOwn][kOwn];
#pragma unroll
            for (int u = 0; u < kInFlight / kOwn; u++)
#pragma unroll
                for (int c = 0; c < kOwn; c++)
                    if (k + u * 32 * N < n && column + warp * kOwn + c < p.columns)
                        w[u][c] = *reinterpret_cast<const Pack<T, N>*>(m + c * p.stride + k0 + k + u * 32 * N);
                    else
#pragma unroll
                        for (int i = 0; i < N; i++) w[u][c].v[i] = narrow<T>(0);
#pragma unroll
            for (int u = 0; u < kInFlight / kOwn; u++) {
                if (k + u * 32 * N >= n) break;
#pragma unroll
                for (int r = 0; r < kRows; r++) {
                    if (r >= here) break;
                    const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(&x[r][k + u * 32 * N]);
#pragma unroll
                    for (int c = 0; c < kOwn; c++)
#pragma unroll
                        for (int i = 0; i < N; i++) sum[r][c] += widen(v.v[i]) * widen(w[u][c].v[i]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int c = 0; c < kOwn; c++) {
            const S all = warp_sum(sum[r][c]);
            if (lane == 0) part[r * kColumns + warp * kOwn + c] = all;
        }
    join_parts<T, kColumns>(part, p, row, here, column);
}

// ------------------------------------------------------------------- outer products of few rows
// out[g] = X[rows of g]^T Y[rows of g], of which most are zero or the product of one or two rows: what counts is to write them. A thread has 16 bytes of the output at a time,
// wherever matrices and their rows begin, and adds up the products of its group's rows in f32 (f64), read through the L1, value by value, which bounds it. 16 rows of 56 groups,
// 1195 x 33 in bf16 (4.4 MB): 7 us, tiles on the tensor cores 25 and a copy of the operands. Large matrices are better off there (18 rows of 13 groups, 1754 x 2693, 123 MB: 71 us, here 89).
constexpr int kOuterTurns = 2;
template <typename T>
__global__ void __launch_bounds__(kThreads)
few_outer(T* __restrict__ out, const T* __restrict__ X, int64_t x_stride, const T* __restrict__ Y, int64_t y_stride, const int32_t* __restrict__ offsets,
          int64_t groups, int64_t rows, uint32_t columns, Divider by_columns, uint32_t values, Status st) {
    using S = Sum<T>;
    constexpr int N = kPack<T>;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(offsets, groups, rows, st);
    int64_t lo, hi;
    group_bounds(offsets, groups, rows, blockIdx.y, lo, hi);
    out += static_cast<int64_t>(blockIdx.y) * values; // the group's matrix
    // how far it begins behind a multiple of 16 bytes
    const uint32_t head = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T));
    uint32_t at = (blockIdx.x * (kThreads * kOuterTurns) + threadIdx.x) * N; // counted from there
    for (int turn = 0; turn < kOuterTurns; turn++, at += kThreads * N) {
        if (at >= values + head) break;
        if (at >= head && at + N <= values + head) {
            const uint32_t v = at - head;
            uint32_t j;
            S sum[N];
#pragma unroll
            for (int u = 0; u < N; u++) sum[u] = 0;
            if (lo < hi) {
                const uint32_t i = by_columns.divide(v);
                j = v - i * columns;
                for (int64_t r = lo; r < hi; r++) {
                    const T *x = X + r * x_stride + i, *y = Y + r * y_stride;
                    S factor = widen(*x);
                    uint32_t c = j;
#pragma unroll
                    for (int u = 0; u < N; u++) {
                        sum[u] += factor * widen(y[c]);
                        if (++c == columns) {
                            c = 0;
                            if (u + 1 < N) factor = widen(*++x);
                        }
                    }
                }
            }
            Pack<T, N> result;
#pragma unroll
            for (int u = 0; u < N; u++) result.v[u] = narrow<T>(sum[u]);
            store_through(out + v, result);
        } else { // the matrix begins or ends in here
            for (uint32_t a = max(at, head); a < min(at + N, values + head); a++) {
                const uint32_t i = by_columns.divide(a - head), j = a - head - i * columns;
                S sum = 0;
                for (int64_t r = lo; r < hi; r++) sum += widen(X[r * x_stride + i]) * widen(Y[r * y_stride + j]);
                out[a - head] = narrow<T>(sum);
            }
        }
    }
}

} // namespace

bool straight_rows(const Array& M, int64_t rows, bool by_columns) {
    const int64_t groups = M.shape[0], bytes = type_bytes(M.type);
    if (rows > kMostRows / (bytes == 2 ? 2 : 1)) return false;
    // Where many rows share matrices the tiles of 128 rows read them once for all; those of f32 take long for few rows, and the next four find the matrix in L2 (32 rows of a
    // group, 1024 x 1024: 22 us so, 30 in tiles; 4096 x 4096: 147 and 113, 8 rows 45 and 113).
    if (rows > kRows * groups && !(bytes == 4 && (rows <= 16 || (rows <= 32 && M.shape[1] * M.shape[2] <= 1 << 23)))) return false;
    if (bytes != 2) return true;
    // 16 bits: only what the copy engine cannot fetch.
    const int inner = M.stride[2] == 1 ? 2 : 1, outer = 3 - inner;
    if (boxable(M.type, M.data, M.shape[inner], M.shape[outer], groups, M.stride[outer], M.stride[0])) return false;
    // Columns one by one come at 1.3 TB/s, and copies, of all matrices, with the tensor cores behind them, at 1.5 (13 matrices of 1754 x 2693, all used: 120 and 84 us); with the depth along
    // rows it is 2 TB/s. So copies it is for large matrices by columns of which most are used.
    return !by_columns || std::min(rows, groups) * 3 <= groups * 2 || groups * M.shape[1] * M.shape[2] * bytes <= 16 << 20;
}

bool straight_outer(int64_t rows, int64_t groups, int64_t height, int64_t columns, int32_t type) {
    return rows <= 64 && rows <= 2 * groups && groups <= 65535 && groups * height * columns * type_bytes(type) <= 16 << 20;
}

bool multiply_rows_few(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.depth == 0 || p.groups == 0) return false;
    const bool mn = p.column_stride == 1;
    const int64_t stride = mn ? p.depth_stride : p.column_stride;
    const int64_t inner = mn ? p.columns : p.depth, outer = mn ? p.depth : p.columns;
    const int64_t sms = sm_count(call.device);
    if (straight_rows(p.M, p.rows, mn)) {
        for_type(p.X.type, [&](auto zero) {
            using T = decltype(zero);
            auto launch = [&](auto width) {
                constexpr int N = decltype(width)::value;
                const int64_t across = ceil_div(p.columns, mn ? kAcross<N> * N : kWarps * 4), pieces = std::min<int64_t>(p.rows, p.groups + p.rows / kRows);
                const int parts = parts_of_depth(across * pieces, sms * 4, p.depth, 128);
                const Few<T> few{static_cast<T*>(p.out.data), static_cast<const T*>(p.X.data), static_cast<const T*>(p.M.data), p.X.stride[0], p.M.stride[0],
                                 stride, p.offsets, p.groups, p.rows, static_cast<int>(p.depth), static_cast<int>(p.columns)};
                Clusters clusters(call, op, across, parts, pieces, kThreads, 0);
                MOPS_CUDA_OK(cudaLaunchKernelEx(&clusters.config, mn ? few_rows_columns<T, N> : few_rows_depth<T, N>, few, call.status));
                note_kernel_f("few_rows_%s<%s,%d>, %d parts", mn ? "columns" : "depth", array_type_name<T>(), N, parts);
            };
            if constexpr (sizeof(T) > 2)
                if (inner % kPack<T> == 0 && boxable(p.X.type, p.M.data, inner, outer, p.groups, stride, p.M.stride[0])) {
                    launch(std::integral_constant<int, kPack<T>>());
                    return;
                }
            launch(std::integral_constant<int, 1>());
        });
        return true;
    }
    if (p.X.type == MOPS_B200_F16 || p.X.type == MOPS_B200_BF16) {
        // Up to 32 rows the accumulators have 16 columns, up to 128 of deep matrices 64 (64 rows of 32 groups, 2048 x 1536: 29.5 us, with 16 columns 36.8). More rows, and
        // shallow matrices, are left to the tiles of 128 rows (200 rows of 8 groups, 2048 x 1536: 18.5 us here, 17.1 there; 48 of 2, 1024 x 1024: 11.7 and 9.8).
        if (p.rows > 32 && (p.rows > 128 || p.depth < 2048)) return false;
        auto launch = [&](auto zero, auto major, auto high) {
            using T = decltype(zero);
            constexpr bool M_MN = decltype(major)::value;
            constexpr int kRowsOf = decltype(high)::value;
            using L = FewLayout<kRowsOf>;
            const int64_t across = ceil_div(p.columns, kTileRows), pieces = std::min<int64_t>(p.rows, p.groups + p.rows / kRowsOf);
            // as many blocks as SMs (four times as many, of 16 rows of 32 groups, 2048 x 1536: 24.8 us for 16.3); to join 64 rows takes what 500 values of depth take
            const int parts = parts_of_depth(across * pieces, sms, p.depth, kRowsOf == 16 ? 128 : 512);
            const CUtensorMap x = tensor_map(p.X.type, p.X.data, p.depth, p.rows, 1, p.X.stride[0], 0, kRowsOf);
            const CUtensorMap m = tensor_map(p.X.type, p.M.data, inner, outer, p.groups, stride, p.M.stride[0], M_MN ? 64 : kTileRows);
            auto kernel = few_rows_mma<T, M_MN, kRowsOf>;
            allow_dynamic_smem(kernel, call.device, L::kBytes);
            Clusters clusters(call, op, across, parts, pieces, kTileThreads, L::kBytes);
            MOPS_CUDA_OK(cudaLaunchKernelEx(&clusters.config, kernel, x, m, static_cast<T*>(p.out.data), p.offsets, p.groups, p.rows,
                                            static_cast<int>(p.depth), static_cast<int>(p.columns), call.status));
            note_kernel_f("few_rows_mma<%s,%s,%d>, %d parts", array_type_name<T>(), M_MN ? "columns" : "depth", kRowsOf, parts);
        };
        auto by_rows = [&](auto zero, auto major) {
            if (p.rows > 32) launch(zero, major, std::integral_constant<int, 64>());
            else launch(zero, major, std::integral_constant<int, 16>());
        };
        auto by_major = [&](auto zero) {
            if (mn) by_rows(zero, std::true_type());
            else by_rows(zero, std::false_type());
        };
        if (p.X.type == MOPS_B200_BF16) by_major(__nv_bfloat16());
        else by_major(__half());
        return true;
    }
    return false;
}

bool multiply_outer_few(const Call& call, const OuterProblem& p, const std::string& op) {
    const int64_t rows = p.X.shape[0], height = p.X.shape[1], columns = p.Y.shape[1];
    if (!straight_outer(rows, p.groups, height, columns, p.X.type)) return false;
    for_type(p.X.type, [&](auto zero) {
        using T = decltype(zero);
        const int64_t values = height * columns;
        few_outer<T><<<dim3(static_cast<unsigned>(ceil_div(values + kPack<T>, int64_t(kThreads) * kOuterTurns * kPack<T>)), static_cast<unsigned>(p.groups)), kThreads, 0,
                       call.stream>>>(static_cast<T*>(p.out.data), static_cast<const T*>(p.X.data), p.X.stride[0], static_cast<const T*>(p.Y.data), p.Y.stride[0],
                                      p.offsets, p.groups, rows, static_cast<uint32_t>(columns), Divider(static_cast<uint32_t>(columns)),
                                      static_cast<uint32_t>(values), call.status);
        note_kernel_f("few_outer<%s>", array_type_name<T>());
    });
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
