// grouped_matrix_product on tensor cores, for f32.
//
// A value is split into three bf16 parts of eight bits each, by cutting bits off, so that the parts add up to the value: x = x0 + x1 +
// x2 (of values below some 2^-110 the bits under 2^-133, the smallest bf16, are lost). Of the nine products of parts the six of up to 2^-16 of the largest are computed, the small ones first; the three left out are about
// 2^-24 of the result, as a rounding to f32 is. The tensor cores add to their f32 accumulators by cutting off what does not fit, an error of one sign that
// grows with the number of additions; so an accumulator takes kRun stages (64 values of depth) and is then added, rounded, to sums in
// registers. That is the choice here: f32 results whose error is about twice that of f32 products and sums rounded one by one (K = 128, normal values: 4.0e-7 and 2.0e-7 of the norm), at two to
// three times the rate that the ordinary units could reach (74 TFLOP/s). Calls of few rows (grouped_few.cu) go to those. Sums that come out as NaN, as they do wherever an operand is infinite, are computed again by the ordinary units (repair()), so
// infinities come out as f32 arithmetic has them.
//
// The copy engine fetches boxes of f32 into one ring of stages; eight warps split them, the parts of the rows' operand go to tensor memory and those of the other to
// a second ring; one thread issues the products; eight warps add up what the accumulators hold and store the tiles. Bounded by shared memory: of a stage of 64 values of
// depth, 128 x 128, it moves 64 KB in, 64 KB out, 48 KB of parts in and 96 KB of them to the tensor cores. (With the parts of both operands in shared memory
// it was 416 KB, and 2.0 us for such a stage.) 16 384 rows of 8 groups, 1024 x 1024: 209 us (164 TFLOP/s, 0.99 P of bf16), gradients 204 and 269. Shallow products are bounded by memory and by the
// number of tiles: 100 003 rows of 20 groups, 128 x 128: 34 us, of which a tile on every SM takes 4.1 (4.5 TB/s) and beginning and end 6.5.
#include "split_block.cuh"

namespace mops_b200 {
namespace {

using namespace split;

// ---------------------------------------------------------------------------------- rows
// out[r,:] = X[r,:] M[group of r]. M_MN: the columns of M are neighbours in memory, else its depth is.
struct RowOperands {
    const float *x, *m;
    int64_t x_stride, group_stride, depth_stride, column_stride; // of m the last three
};
template <bool M_MN, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_split(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_out,
                   float* __restrict__ out, const __grid_constant__ RowOperands from, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int depth,
                   int columns, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using W = Work<false, M_MN, kColumns>;
    using L = typename W::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    W work{block};
    Supply<L> supply{block};
    Piece piece;
    if (warp < kSplitWarps) {
        fewer_registers<kSplitRegisters>();
        work.split(warp, lane);
    } else if (warp < kMultiplyWarp) {
        more_registers<kStoreRegisters>();
        const int quadrant = warp & 3, half = (warp - kSplitWarps) / 4;
        while (supply.next(piece, lane)) {
            float sum[W::kOwn];
            if (!work.collect(sum, piece.steps, quadrant, half, lane)) break;
            const int64_t row = piece.lo + quadrant * 32, column = piece.column + half * W::kOwn;
            if (work.store(sum, warp - kSplitWarps, map_out, column, static_cast<int>(row), 0, out + row * columns + column, columns, piece.hi - row,
                           columns - column, loose, lane))
                work.repair(sum, warp - kSplitWarps, lane, out + row * columns + column, columns, [&] {
                    return Terms{from.x + row * from.x_stride, from.m + piece.group * from.group_stride + column * from.column_stride, from.x_stride, 1, from.column_stride,
                                 from.depth_stride, depth, static_cast<int>(min(piece.hi - row, int64_t(32))), static_cast<int>(columns - column)};
                });
        }
    } else {
        fewer_registers<kMultiplyRegisters>();
        bool ok = true;
        if (warp == kMultiplyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0) ok = work.multiply(piece.steps);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
        } else if (warp == kPieceWarp) {
            hand_out(block, 0, lane, DecodeRows<kTileRows, kColumns>(offsets, groups, rows, columns, (depth + kDepth - 1) / kDepth, lane));
        } else if (warp == kCopyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0)
                    for (int s = 0; s < piece.steps && ok; s++)
                        ok = work.fetch(map_x, map_m, s * kDepth, static_cast<int>(piece.lo), M_MN ? piece.column : s * kDepth,
                                        M_MN ? s * kDepth : piece.column, piece.group, kDepth);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
            if (lane == 0) {
                if (ok) (void)work.fetch(map_x, map_m, 0, 0, 0, 0, 0, -1);
                block.drain(block.rings->raws, work.raw, work.fetched);
            }
        }
    }
    if (lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

// ------------------------------------------------------------------------- outer products
// out[g] = X[rows of g]^T Y[rows of g].
struct OuterOperands {
    const float *x, *y;
    int64_t x_stride, y_stride;
};
template <int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_outer_split(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                    const __grid_constant__ CUtensorMap map_out, float* __restrict__ out, float* __restrict__ parts, int64_t most_parts, const __grid_constant__ OuterOperands from,
                    const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using W = Work<true, true, kColumns>;
    using L = typename W::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    W work{block};
    Supply<L> supply{block};
    Piece piece;
    if (warp < kSplitWarps) {
        fewer_registers<kSplitRegisters>();
        work.split(warp, lane);
    } else if (warp < kMultiplyWarp) {
        more_registers<kStoreRegisters>();
        const int quadrant = warp & 3, half = (warp - kSplitWarps) / 4;
        while (supply.next(piece, lane)) {
            float sum[W::kOwn];
            if (!work.collect(sum, piece.steps, quadrant, half, lane)) break;
            const int64_t row = piece.row + quadrant * 32, column = piece.column + half * W::kOwn;
            float* to = out + (static_cast<int64_t>(piece.group) * height + row) * columns + column;
            int64_t stride = columns;
            bool odd;
            if (piece.slot >= 0) {
                // (there are more parts than there is room for only where offsets descend, which is reported)
                if (piece.slot >= most_parts) continue;
                to = parts + (piece.slot * kTileRows + quadrant * 32) * kColumns + half * W::kOwn;
                stride = kColumns;
#pragma unroll
                for (int i = 0; i < W::kOwn; i += 4)
                    *reinterpret_cast<float4*>(to + lane * kColumns + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
                odd = W::any_nan(sum);
            } else {
                // (the copy engine leaves out what lies behind the output's last row)
                odd = work.store(sum, warp - kSplitWarps, map_out, column, static_cast<int>(row), piece.group, to, columns,
                                 loose || row >= height ? height - row : 32, columns - column, loose, lane);
            }
            if (odd)
                work.repair(sum, warp - kSplitWarps, lane, to, stride, [&] {
                    return Terms{from.x + piece.lo * from.x_stride + row, from.y + piece.lo * from.y_stride + column, 1, from.x_stride, 1, from.y_stride,
                                 static_cast<int>(piece.hi - piece.lo), static_cast<int>(height - row), static_cast<int>(columns - column)};
                });
        }
    } else {
        fewer_registers<kMultiplyRegisters>();
        bool ok = true;
        if (warp == kMultiplyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0) ok = work.multiply(piece.steps);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
        } else if (warp == kPieceWarp) {
            hand_out(block, 0, lane, DecodeOuter<kTileRows, kColumns, kDepth>(offsets, groups, rows, height, columns, segment, lane));
        } else if (warp == kCopyWarp) {
            while (ok && supply.next(piece, lane)) {
                const int lo = static_cast<int>(piece.lo), hi = static_cast<int>(piece.hi);
                if (lane == 0)
                    for (int s = 0; s < piece.steps && ok; s++)
                        ok = work.fetch(map_x, map_y, piece.row, lo + s * kDepth, piece.column, lo + s * kDepth, 0, min(hi - lo - s * kDepth, kDepth));
                ok = __shfl_sync(kFullMask, ok, 0);
            }
            if (lane == 0) {
                if (ok) (void)work.fetch(map_x, map_y, 0, 0, 0, 0, 0, -1);
                block.drain(block.rings->raws, work.raw, work.fetched);
            }
        }
    }
    if (lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

} // namespace

bool multiply_rows_split(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.X.type != MOPS_B200_F32 || p.depth == 0 || p.groups == 0) return false;
    const bool mn = p.column_stride == 1;
    const int64_t stride = mn ? p.depth_stride : p.column_stride; // of M
    const int sms = sm_count(call.device);
    auto launch = [&](auto major, auto width) {
        constexpr bool M_MN = decltype(major)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, p.depth, p.rows, 1, p.X.stride[0], 0, kTileRows);
        const CUtensorMap m = M_MN ? tensor_map(p.X.type, p.M.data, p.columns, p.depth, p.groups, stride, p.M.stride[0], kDepth)
                                   : tensor_map(p.X.type, p.M.data, p.depth, p.columns, p.groups, stride, p.M.stride[0], kColumns);
        const bool loose = p.columns % 4 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, p.columns, p.rows, 1, p.columns, 0, 32);
        const int64_t tiles = most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, kColumns);
        auto kernel = grouped_rows_split<M_MN, kColumns>;
        check_registers(reinterpret_cast<const void*>(kernel), op);
        const RowOperands from{static_cast<const float*>(p.X.data), static_cast<const float*>(p.M.data), p.X.stride[0], p.M.stride[0], p.depth_stride, p.column_stride};
        launch_blocks<L>(call, op, kernel, tiles, x, m, out, static_cast<float*>(p.out.data), from, p.offsets, p.groups, p.rows,
                         static_cast<int>(p.depth), static_cast<int>(p.columns), loose, call.status);
        note_kernel_f("grouped_rows_split<%s,%d>", M_MN ? "columns" : "depth", kColumns);
    };
    auto by_width = [&](auto major) {
        if (p.columns > 64 && most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, 128) >= sms / 2)
            launch(major, std::integral_constant<int, 128>());
        else launch(major, std::integral_constant<int, 64>());
    };
    if (mn) by_width(std::true_type());
    else by_width(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

bool multiply_outer_split(const Call& call, const OuterProblem& p, const std::string& op) {
    const int64_t rows = p.X.shape[0], height = p.X.shape[1], columns = p.Y.shape[1];
    if (p.X.type != MOPS_B200_F32 || rows == 0) return false;
    const int sms = sm_count(call.device);
    auto launch = [&](auto width) {
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, height, rows, 1, p.X.stride[0], 0, kDepth);
        const CUtensorMap y = tensor_map(p.X.type, p.Y.data, columns, rows, 1, p.Y.stride[0], 0, kDepth);
        const int64_t tiles = ceil_div(height, kTileRows) * ceil_div(columns, kColumns);
        const int64_t segment = outer_segment(rows, p.groups, tiles, sms), most_parts = most_outer_parts(rows, tiles, segment);
        Scratch room(call);
        if (rows > segment) room.take(static_cast<size_t>(most_parts) * kTileRows * kColumns * sizeof(float));
        float* parts = room.as<float>();
        auto kernel = grouped_outer_split<kColumns>;
        check_registers(reinterpret_cast<const void*>(kernel), op);
        const bool loose = columns % 4 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, columns, height, p.groups, columns, height * columns, 32);
        const OuterOperands from{static_cast<const float*>(p.X.data), static_cast<const float*>(p.Y.data), p.X.stride[0], p.Y.stride[0]};
        launch_blocks<L>(call, op, kernel, tiles * (rows / segment + p.groups), x, y, out, static_cast<float*>(p.out.data), parts, most_parts, from, p.offsets,
                         p.groups, rows, static_cast<int>(height), static_cast<int>(columns), segment, loose, call.status);
        if (rows > segment) {
            join_outer<float, kTileRows, kColumns>(call, p, parts, most_parts, tiles, segment, op);
            room.free();
        }
        note_kernel_f("grouped_outer_split<%d>", kColumns);
    };
    if (columns > 64) launch(std::integral_constant<int, 128>());
    else launch(std::integral_constant<int, 64>());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
