// Products of rows of f32 on tensor cores whose sums are worked on before anything is stored: the gated layer, the loss over a table. As tile_rows.cuh for 16 bits: a storing
// warp has the sums of 32 rows, a row to a lane, of 64 columns of the tile, or (E::kHalves) of the same 32 columns of either half of the second operand.
//
// E has: kHalves, Args, and
//   E(args, staging, lane)             staging: 4 KB of shared memory of the warp's own
//   begin(piece, row, here, half)      before the sums are there. The warp's first row, how many rows it has, which half of the tile's columns
//   store(sum)
//   clear()                            rows of no group
//   end()
#ifndef MOPS_B200_SPLIT_ROWS_CUH
#define MOPS_B200_SPLIT_ROWS_CUH

#include "split_block.cuh"
#include "tile_rows.cuh"

namespace mops_b200 {

constexpr int kSplitColumns = 128; // of a tile's sums

// The operands in global memory, for sums that are computed again.
struct SplitOperands {
    const float *x, *m[2];
    int64_t x_stride, group_stride, depth_stride, column_stride; // of m the last three
};

template <bool M_MN, typename E, template <int, int> class Decode>
__global__ void __launch_bounds__(split::kThreads, 1)
split_rows(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m0, const __grid_constant__ CUtensorMap map_m1,
           const __grid_constant__ typename E::Args args, const __grid_constant__ SplitOperands from, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
           int depth, int columns, int slices, Status st) {
    extern __shared__ unsigned char raw[];
    using namespace split;
    constexpr bool kSliced = kRowSlices<Decode>;
    using W = Work<false, M_MN, kSplitColumns>;
    using L = typename W::L;
    constexpr int kTile = E::kHalves ? kSplitColumns / 2 : kSplitColumns; // columns of the result
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if constexpr (!kOneGroup<Decode>)
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
        E result(args, smem_address(block.smem + L::kStagingAt + (warp - kSplitWarps) * L::kStaging), lane);
        while (supply.next(piece, lane)) {
            const int64_t row = piece.lo + quadrant * 32;
            const int here = static_cast<int>(min(max(piece.hi - row, int64_t(0)), int64_t(32)));
            result.begin(piece, row, here, half);
            if (piece.group < 0) {
                if (half == 0) result.clear();
                continue;
            }
            float sum[W::kOwn];
            if (!work.template collect<E::kHalves>(sum, piece.steps, quadrant, half, lane)) break;
            if (here <= 0) continue;
            if (W::any_nan(sum, lane < here)) {
                RowsIn::wait();
                const int first = kSliced ? static_cast<int>(piece.slot) * kDepth : 0, deep = kSliced ? min(depth - first, piece.steps * kDepth) : depth;
                work.mend(sum, warp - kSplitWarps, lane, [&](int c) {
                    const int column = piece.column + (E::kHalves ? half * 32 : half * W::kOwn + c);
                    return Terms{from.x + row * from.x_stride + first,
                                 from.m[E::kHalves && c > 0 ? 1 : 0] + piece.group * from.group_stride + column * from.column_stride + first * from.depth_stride,
                                 from.x_stride, 1, from.column_stride, from.depth_stride, deep, here, columns - column};
                });
                result.begin(piece, row, here, half); // (what it had in the staging memory has been written over)
            }
            result.store(sum);
        }
        result.end();
    } else {
        fewer_registers<kMultiplyRegisters>();
        bool ok = true;
        if (warp == kMultiplyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0) ok = work.multiply(piece.steps);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
        } else if (warp == kPieceWarp) {
            const int steps = (depth + kDepth - 1) / kDepth;
            if constexpr (kRowSlices<Decode>) hand_out(block, 0, lane, Decode<kTileRows, kTile>(offsets, groups, rows, columns, steps, slices, lane));
            else hand_out(block, 0, lane, Decode<kTileRows, kTile>(offsets, groups, rows, columns, steps, lane));
        } else if (warp == kCopyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0)
                    for (int s = 0; s < piece.steps && ok; s++) {
                        const int deep = (kSliced ? static_cast<int>(piece.slot) + s : s) * kDepth;
                        const int inner = M_MN ? piece.column : deep, outer = M_MN ? deep : piece.column;
                        if constexpr (E::kHalves)
                            ok = work.fetch_halves(map_x, map_m0, map_m1, deep, static_cast<int>(piece.lo), inner, outer, piece.group);
                        else
                            ok = work.fetch(map_x, map_m0, deep, static_cast<int>(piece.lo), inner, outer, piece.group, kDepth);
                    }
                ok = __shfl_sync(kFullMask, ok, 0);
            }
            if (lane == 0) {
                if (ok) (void)work.fetch(map_x, map_m0, 0, 0, 0, 0, 0, -1);
                block.drain(block.rings->raws, work.raw, work.fetched);
            }
        }
    }
    __syncwarp();
    block.end(warp);
}

// 32 columns of f32 of a warp's 32 rows, as BoxOut of 64 columns of 16 bits.
struct BoxOut32 {
    const CUtensorMap& map;
    float* out;
    int64_t stride;
    int columns;
    bool loose;
    __device__ __forceinline__ void put(const float (&v)[32], uint32_t staging, int64_t row, int here, int column, int lane) const {
        if (lane == 0) boxes_left<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; j++)
            smem_store16(staging + lane * kBoxRow + ((j ^ (lane & 7)) << 4),
                         make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])));
        if (!loose && here == 32) {
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) box_out(map, column, static_cast<int>(row), 0, staging);
        } else {
            __syncwarp();
            if (column + lane < columns)
                for (int i = 0; i < here; i++)
                    out[(row + i) * stride + column + lane] = __uint_as_float(smem_load4(staging + i * kBoxRow + ((lane / 4 ^ (i & 7)) << 4) + lane % 4 * 4));
            __syncwarp();
        }
    }
    __device__ __forceinline__ void clear(int64_t row, int here, int column, int wide, int lane) const {
        for (int i = 0; i < here; i++)
            for (int c = lane; c < wide && column + c < columns; c += 32) out[(row + i) * stride + column + c] = 0.f;
    }
};

// Sums as they are, each slice of the depth in an array of its own; `add`: to what is there. Zeros for rows of no group.
template <int kOwn_> struct SumStoreOf {
    static constexpr bool kHalves = false, kMend = false, kAllRows = false;
    static constexpr int kOwn = kOwn_;
    struct Args {
        CUtensorMap map;
        float* out;
        int64_t rows, stride; // of a slice; stride: a multiple of 4
        int columns;
        bool add;
    };
    const Args& a;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0, slice = 0;
    __device__ SumStoreOf(const Args& a, uint32_t staging, int lane) : a(a), staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) { row = r, here = h, column = piece.column + half * kOwn, slice = piece.row; }
    __device__ __forceinline__ void store(const float (&sum)[kOwn]) const {
#pragma unroll
        for (int c = 0; c < kOwn; c += 32) {
            if (column + c >= a.columns) return;
            if (here == 32) {
                if (lane == 0) boxes_left<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++)
                    smem_store16(staging + lane * kBoxRow + ((j ^ (lane & 7)) << 4),
                                 make_uint4(__float_as_uint(sum[c + 4 * j]), __float_as_uint(sum[c + 4 * j + 1]), __float_as_uint(sum[c + 4 * j + 2]),
                                            __float_as_uint(sum[c + 4 * j + 3])));
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    if (a.add) box_add(a.map, column + c, static_cast<int>(row), slice, staging);
                    else box_out(a.map, column + c, static_cast<int>(row), slice, staging);
                }
            } else if (lane < here) {
                float* to = a.out + (slice * a.rows + row + lane) * a.stride + column + c;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (column + c + 4 * j < a.columns) { // (there is room up to a multiple of 4)
                        float4 v = make_float4(sum[c + 4 * j], sum[c + 4 * j + 1], sum[c + 4 * j + 2], sum[c + 4 * j + 3]);
                        if (a.add) {
                            const float4 w = *reinterpret_cast<const float4*>(to + 4 * j);
                            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                        }
                        *reinterpret_cast<float4*>(to + 4 * j) = v;
                    }
            }
        }
    }
    __device__ __forceinline__ void clear() const {
        for (int i = 0; i < here; i++)
            for (int c = lane; c < 2 * kOwn && column + c < a.columns; c += 32) a.out[(slice * a.rows + row + i) * a.stride + column + c] = 0.f;
    }
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};
using SumStore32 = SumStoreOf<kSplitColumns / 2>;
template <typename E = SumStore32> typename E::Args sum_args(float* out, int64_t slices, int64_t rows, int64_t stride, int64_t columns, bool add) {
    return {tensor_map(MOPS_B200_F32, out, columns, rows, slices, stride, rows * stride, 32), out, rows, stride, static_cast<int>(columns), add};
}

// to[r,:] = the sums of all slices (stride: a multiple of 4)
static __global__ void __launch_bounds__(256)
add_slices(float* __restrict__ to, const float* __restrict__ sums, int slices, int64_t rows, int64_t stride, int columns) {
    const int64_t quads = stride / 4, slice = rows * stride;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < rows * quads; at += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = at / quads;
        const int c = static_cast<int>(at - r * quads) * 4;
        float4 v = make_float4(0, 0, 0, 0);
        for (int s = 0; s < slices; s++) {
            const float4 w = *reinterpret_cast<const float4*>(sums + s * slice + at * 4);
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        float* p = to + r * columns + c;
        const float all[4] = {v.x, v.y, v.z, v.w};
        if (columns % 4 == 0 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
            *reinterpret_cast<float4*>(p) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (c + k < columns) p[k] = all[k];
        }
    }
}

template <bool M_MN, typename E, template <int, int> class Decode>
void launch_split(const Call& call, const std::string& op, const TileProblem& p, const TileOperand (&b)[2], const typename E::Args& args) {
    using namespace split;
    using L = Layout<kSplitColumns>;
    constexpr int kTile = E::kHalves ? kSplitColumns / 2 : kSplitColumns;
    const CUtensorMap x = tensor_map(MOPS_B200_F32, p.A.data, p.depth, p.rows, 1, p.A.stride[0], 0, kTileRows);
    auto map_of = [&](const TileOperand& o) {
        return M_MN ? tensor_map(MOPS_B200_F32, o.data, p.columns, p.depth, p.groups, o.depth_stride, o.group_stride, kDepth)
                    : tensor_map(MOPS_B200_F32, o.data, p.depth, p.columns, p.groups, o.column_stride, o.group_stride, kTile);
    };
    const CUtensorMap m0 = map_of(b[0]), m1 = E::kHalves ? map_of(b[1]) : m0;
    const SplitOperands from{static_cast<const float*>(p.A.data), {static_cast<const float*>(b[0].data), static_cast<const float*>(b[1].data)}, p.A.stride[0],
                             b[0].group_stride, b[0].depth_stride, b[0].column_stride};
    const int64_t tiles = (kOneGroup<Decode> ? ceil_div(p.rows, kTileRows) : most_row_tiles(p.rows, p.groups, kTileRows)) * ceil_div(p.columns, kTile) *
                          p.slices;
    auto kernel = split_rows<M_MN, E, Decode>;
    check_registers(reinterpret_cast<const void*>(kernel), op);
    launch_blocks<L>(call, op, kernel, tiles, x, m0, m1, args, from, p.offsets, p.groups, p.rows, static_cast<int>(p.depth), static_cast<int>(p.columns),
                     static_cast<int>(p.slices), call.status);
}

} // namespace mops_b200

#endif
