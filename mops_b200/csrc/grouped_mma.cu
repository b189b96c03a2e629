// grouped_matrix_product on tensor cores, for f16 and bf16.
//
// One block per SM works off tiles of 128 rows by kColumns columns. One warp has the copy engine fetch boxes of both operands into a ring
// of stages of 64 values of depth, one thread of another issues the products (tcgen05.mma, accumulators in tensor
// memory), and four warps move finished accumulators through shared memory to the output while the next tile is under way in
// the other half of tensor memory.
//
// Rows: a tile begins where its group's rows do, wherever that is; of a tile that reaches past the end of its group the rows
// behind it are computed and not stored. Outer products: the depth is the group's rows, and of the last stage of a
// group the rows behind its end are cleared in shared memory before they are multiplied.
#include "grouped_block.cuh"
#include "grouped_mma.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {

namespace {

constexpr int kThreads = 192;   // the copying warp, the multiplying warp, four that store
constexpr int kStoreWarps = 4;
constexpr int kStaging = 32 * kBoxRow; // bytes: 32 rows of 64 values, of one warp

// What a block keeps in shared memory.
template <int kColumns> struct Layout {
    static constexpr int kStages = kColumns == 256 ? 4 : kColumns == 128 ? 6 : 8;
    static constexpr int kA = kTileRows * kBoxRow, kB = kColumns * kBoxRow; // bytes of a stage
    static constexpr int kStage = kA + kB;
    static constexpr int kStagingAt = kStages * kStage;
    static constexpr int kRingsAt = kStagingAt + kStoreWarps * 2 * kStaging;
    static constexpr int kBytes = kRingsAt + 256 + 1024; // (boxes begin on multiples of 1024 bytes)
    static constexpr unsigned kTmem = 2 * kColumns;      // columns of tensor memory: two accumulators
    struct Rings {
        Ring<kStages> stages;
        Ring<2> accumulators;
        uint32_t tmem;
        int gave_up;
        __device__ void begin() {
            stages.begin(1, 1);
            accumulators.begin(1, kStoreWarps);
        }
    };
    static_assert(sizeof(Rings) <= 256, "room for the rings");
};

template <bool BF16> __device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Writes the 64 columns that follow `column` of a warp's 32 rows of an accumulator, `here` of which are the group's: all of them by the copy engine,
// fewer each lane its row. Where rows of the output begin anywhere (loose), a row after the other, value by value. out: the first row of the band.
template <bool BF16>
__device__ __forceinline__ void store_columns(uint32_t accumulator, uint32_t staging, int64_t& sent, const CUtensorMap& map,
                                              uint16_t* __restrict__ out, int row, int slice, int column, int columns, int here, bool loose,
                                              int lane) {
    uint32_t r[2][32];
    tmem_load(accumulator, r[0]);
    tmem_load(accumulator + 32, r[1]);
    tmem_wait_load();
    tmem_pin(r[0]);
    tmem_pin(r[1]);
    uint4 v[8];
#pragma unroll
    for (int c = 0; c < 8; c++) {
        const uint32_t* w = &r[c / 4][c % 4 * 8];
        v[c] = make_uint4(pack2<BF16>(w[0], w[1]), pack2<BF16>(w[2], w[3]), pack2<BF16>(w[4], w[5]), pack2<BF16>(w[6], w[7]));
    }
    if (loose || here == 32) {
        const uint32_t to = staging + static_cast<uint32_t>(sent & 1) * kStaging;
        if (!loose && lane == 0) boxes_left<1>();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; c++) smem_store16(to + lane * kBoxRow + ((c ^ (lane & 7)) << 4), v[c]);
        if (loose) {
            __syncwarp();
            const int wide = columns - column;
            for (int i = 0; i < here; i++) {
                uint16_t* p = out + static_cast<int64_t>(i) * columns + column;
#pragma unroll
                for (int h = 0; h < 64; h += 32) {
                    const int c = h + lane;
                    if (c < wide) p[c] = smem_load2(to + i * kBoxRow + ((c / 8 ^ (i & 7)) << 4) + c % 8 * 2);
                }
            }
        } else {
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) box_out(map, column, row, slice, to);
        }
        sent++;
    } else if (lane < here) {
        uint4* to = reinterpret_cast<uint4*>(out + static_cast<int64_t>(lane) * columns + column);
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (column + c * 8 < columns) to[c] = v[c]; // (columns are a multiple of 8 here)
    }
}

// ---------------------------------------------------------------------------------- rows
// out[r,:] = X[r,:] M[group of r]. M_MN: the columns of M are neighbours in memory, else its depth is.
template <bool BF16, bool M_MN, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_mma(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m,
                 const __grid_constant__ CUtensorMap map_out, uint16_t* __restrict__ out, const int32_t* __restrict__ offsets,
                 int64_t groups, int64_t rows, int depth, int columns, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using L = Layout<kColumns>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    const int64_t column_tiles = (columns + kColumns - 1) / kColumns;
    const int steps = (depth + kBoxDepth - 1) / kBoxDepth;
    GroupWalk<RowTiles> walk(offsets, groups, rows, -1, groups, RowTiles{kTileRows, column_tiles});
    Turn<L::kStages> stage;
    Turn<2> tile;     // accumulator
    int64_t sent = 0; // boxes that this warp has fetched or stored
    auto stage_at = [&] { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    for (int64_t want = blockIdx.x;; want += gridDim.x) {
        const GroupPiece piece = walk.find(want, lane);
        if (!piece.found) break;
        int64_t tile_row, tile_column;
        banded(piece.within, (piece.hi - piece.lo + kTileRows - 1) / kTileRows, column_tiles, tile_row, tile_column);
        const int64_t row = piece.lo + tile_row * kTileRows;
        const int column = static_cast<int>(tile_column) * kColumns;
        const bool in_group = piece.group >= 0 && piece.group < groups;
        bool ok = true;
        if (warp == 0) {
            if (lane == 0 && in_group) {
                for (int s = 0; s < steps && ok; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(), b = a + L::kA;
                    mbarrier_arrive_expect(full, L::kStage);
                    box_in(a, map_x, s * kBoxDepth, static_cast<int>(row), 0, full);
                    if constexpr (M_MN) {
#pragma unroll
                        for (int j = 0; j < kColumns / 64; j++)
                            box_in(b + j * kBoxBytes, map_m, column + j * 64, s * kBoxDepth, static_cast<int>(piece.group), full);
                    } else {
                        box_in(b, map_m, s * kBoxDepth, column, static_cast<int>(piece.group), full);
                    }
                    stage.next();
                    sent++;
                }
            }
        } else if (warp == 1) {
            if (lane == 0 && in_group) {
                constexpr uint32_t instruction = instruction_descriptor(BF16, false, M_MN, kColumns);
                ok = block.wait_empty(block.rings->accumulators, tile);
                tmem_fence_after_sync();
                for (int s = 0; s < steps && ok; s++) {
                    ok = block.wait_full(block.rings->stages, stage);
                    if (!ok) break;
                    tmem_fence_after_sync();
                    const uint64_t a = operand_descriptor(stage_at(), kBoxBytes);
                    const uint64_t b = operand_descriptor(stage_at() + L::kA, kBoxBytes);
#pragma unroll
                    for (int k = 0; k < kBoxDepth / 16; k++)
                        umma(block.accumulator(tile), a + k * kDepthStep<false>, b + k * kDepthStep<M_MN>, instruction, s + k > 0);
                    umma_arrive(&block.rings->stages.empty[stage.at]);
                    stage.next();
                }
                if (ok) umma_arrive(&block.rings->accumulators.full[tile.at]);
                tile.next();
            }
        } else {
            const int quadrant = warp & 3;
            const int64_t band = row + quadrant * 32;
            const int here = static_cast<int>(min(max(piece.hi - band, int64_t(0)), int64_t(32)));
            const int wide = min(columns - column, kColumns);
            if (in_group) {
                ok = block.wait_full(block.rings->accumulators, tile);
                if (ok) {
                    tmem_fence_after_sync();
                    const uint32_t from = tmem_quadrant(block.accumulator(tile), quadrant);
                    const uint32_t staging = block.base + L::kStagingAt + quadrant * 2 * kStaging;
                    if (here > 0)
                        for (int c = 0; c < wide; c += 64)
                            store_columns<BF16>(from + c, staging, sent, map_out, out + band * columns, static_cast<int>(band), 0, column + c,
                                                        columns, here, loose, lane);
                    tmem_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(&block.rings->accumulators.empty[tile.at]);
                }
                tile.next();
            } else { // rows of no group
                for (int i = 0; i < here; i++)
                    for (int c = lane; c < wide; c += 32) out[(band + i) * columns + column + c] = 0;
            }
        }
        if (!__shfl_sync(kFullMask, ok, 0)) break;
    }
    if (warp == 0 && lane == 0) block.drain(block.rings->stages, stage, sent);
    if (warp >= 2 && lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

// ------------------------------------------------------------------------- outer products
// out[g] = X[rows of g]^T Y[rows of g].
template <bool BF16, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_outer_mma(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                  const __grid_constant__ CUtensorMap map_out, uint16_t* __restrict__ out, float* __restrict__ parts, int64_t most_parts,
                  const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment,
                  bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using L = Layout<kColumns>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    const int64_t row_tiles = (height + kTileRows - 1) / kTileRows, column_tiles = (columns + kColumns - 1) / kColumns;
    const int64_t tiles = row_tiles * column_tiles;
    GroupWalk<OuterPieces> walk(offsets, groups, rows, 0, groups - 1, OuterPieces{segment, tiles});
    Turn<L::kStages> stage;
    Turn<2> tile;
    int64_t sent = 0;
    auto stage_at = [&] { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    for (int64_t want = blockIdx.x;; want += gridDim.x) {
        const GroupPiece piece = walk.find(want, lane);
        if (!piece.found) break;
        const int64_t part = piece.within / tiles;
        int64_t tile_row, tile_column;
        banded(piece.within - part * tiles, row_tiles, column_tiles, tile_row, tile_column);
        const int row = static_cast<int>(tile_row) * kTileRows, column = static_cast<int>(tile_column) * kColumns;
        const int64_t lo = piece.lo + part * segment, hi = min(lo + segment, piece.hi);
        const int steps = static_cast<int>((hi - lo + kBoxDepth - 1) / kBoxDepth);
        bool ok = true;
        if (warp == 0) {
            if (lane == 0) {
                for (int s = 0; s < steps && ok; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(), b = a + L::kA;
                    const int at = static_cast<int>(lo) + s * kBoxDepth;
                    mbarrier_arrive_expect(full, L::kStage);
#pragma unroll
                    for (int i = 0; i < kTileRows / 64; i++) box_in(a + i * kBoxBytes, map_x, row + i * 64, at, 0, full);
#pragma unroll
                    for (int j = 0; j < kColumns / 64; j++) box_in(b + j * kBoxBytes, map_y, column + j * 64, at, 0, full);
                    stage.next();
                    sent++;
                }
            }
        } else if (warp == 1) {
            if (steps > 0) {
                constexpr uint32_t instruction = instruction_descriptor(BF16, true, true, kColumns);
                if (lane == 0) ok = block.wait_empty(block.rings->accumulators, tile);
                ok = __shfl_sync(kFullMask, ok, 0);
                tmem_fence_after_sync();
                for (int s = 0; s < steps && ok; s++) {
                    const int64_t left = hi - lo - int64_t(s) * kBoxDepth;
                    if (lane == 0 || left < kBoxDepth) ok = block.wait_full(block.rings->stages, stage);
                    ok = __all_sync(kFullMask, ok);
                    if (!ok) break;
                    if (left < kBoxDepth) { // the rows behind are of another group
                        const uint32_t from = static_cast<uint32_t>(left) * kBoxRow;
                        for (uint32_t box = 0; box < L::kStage; box += kBoxBytes)
                            for (uint32_t at = from + lane * 16; at < kBoxBytes; at += 32 * 16)
                                smem_store16(stage_at() + box + at, make_uint4(0, 0, 0, 0));
                        async_proxy_fence();
                        __syncwarp();
                    }
                    if (lane == 0) {
                        tmem_fence_after_sync();
                        const uint64_t a = operand_descriptor(stage_at(), kBoxBytes);
                        const uint64_t b = operand_descriptor(stage_at() + L::kA, kBoxBytes);
#pragma unroll
                        for (int k = 0; k < kBoxDepth / 16; k++)
                            umma(block.accumulator(tile), a + k * kDepthStep<true>, b + k * kDepthStep<true>, instruction, s + k > 0);
                        umma_arrive(&block.rings->stages.empty[stage.at]);
                    }
                    stage.next();
                    __syncwarp();
                }
                if (lane == 0 && ok) umma_arrive(&block.rings->accumulators.full[tile.at]);
                tile.next();
            }
        } else {
            const int quadrant = warp & 3;
            const int band = row + quadrant * 32, wide = min(columns - column, kColumns);
            if (steps > 0) ok = block.wait_full(block.rings->accumulators, tile);
            if (ok) {
                const uint32_t from = tmem_quadrant(block.accumulator(tile), quadrant);
                const uint32_t staging = block.base + L::kStagingAt + quadrant * 2 * kStaging;
                tmem_fence_after_sync();
                if (piece.hi - piece.lo > segment) {
                    const int64_t slot = parts_before(offsets, groups, rows, piece.group, OuterParts{segment, tiles}, lane) + piece.within;
                    float* to = parts + (slot * kTileRows + quadrant * 32 + lane) * kColumns;
                    // (there are more parts than there is room for only where offsets descend, which is reported)
                    for (int c = 0; c < wide && slot < most_parts; c += 32) {
                        uint32_t r[32];
                        tmem_load(from + c, r);
                        tmem_wait_load();
                        tmem_pin(r);
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            *reinterpret_cast<uint4*>(to + c + 4 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    }
                } else {
                    const int here = min(height - band, 32);
                    uint16_t* to = out + (piece.group * height + band) * static_cast<int64_t>(columns);
                    if (here > 0 && steps > 0) {
                        // (the copy engine leaves out what lies behind the output's last row)
                        for (int c = 0; c < wide; c += 64)
                            store_columns<BF16>(from + c, staging, sent, map_out, to, band, static_cast<int>(piece.group),
                                                        column + c, columns, loose ? here : 32, loose, lane);
                    } else { // a group without rows
                        for (int i = 0; i < here; i++)
                            for (int c = lane; c < wide; c += 32) to[static_cast<int64_t>(i) * columns + column + c] = 0;
                    }
                }
                if (steps > 0) {
                    tmem_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbarrier_arrive(&block.rings->accumulators.empty[tile.at]);
                    tile.next();
                }
            }
        }
        if (!__shfl_sync(kFullMask, ok, 0)) break;
    }
    if (warp == 0 && lane == 0) block.drain(block.rings->stages, stage, sent);
    if (warp >= 2 && lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

} // namespace

bool multiply_rows_mma(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.X.type != MOPS_B200_F16 && p.X.type != MOPS_B200_BF16) return false;
    const bool mn = p.column_stride == 1;
    const int64_t stride = mn ? p.depth_stride : p.column_stride; // of M
    if (p.depth == 0 || p.groups == 0) return false;
    const bool loose = p.columns % 8 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
    const int sms = sm_count(call.device);
    auto launch = [&](auto type, auto major, auto width) {
        constexpr bool BF16 = decltype(type)::value, M_MN = decltype(major)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, p.depth, p.rows, 1, p.X.stride[0], 0, kTileRows);
        const CUtensorMap m = M_MN ? tensor_map(p.X.type, p.M.data, p.columns, p.depth, p.groups, stride, p.M.stride[0], 64)
                                   : tensor_map(p.X.type, p.M.data, p.depth, p.columns, p.groups, stride, p.M.stride[0], kColumns);
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, p.columns, p.rows, 1, p.columns, 0, 32);
        const int64_t tiles = most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, kColumns);
        auto kernel = grouped_rows_mma<BF16, M_MN, kColumns>;
        allow_dynamic_smem(kernel, call.device, L::kBytes);
        kernel<<<static_cast<unsigned>(std::min<int64_t>(tiles, sms)), kThreads, L::kBytes, call.stream>>>(
            x, m, out, static_cast<uint16_t*>(p.out.data), p.offsets, p.groups, p.rows, static_cast<int>(p.depth),
            static_cast<int>(p.columns), loose, call.status);
        note_kernel_f("grouped_rows_mma<%s,%s,%d>", BF16 ? "bf16" : "f16", M_MN ? "columns" : "depth", kColumns);
    };
    auto by_width = [&](auto type, auto major) {
        // The wider the tile, the fewer times X is fetched; the narrower, the more blocks share the work.
        const int64_t row_tiles = most_row_tiles(p.rows, p.groups, kTileRows);
        if (p.columns > 128 && row_tiles * ceil_div(p.columns, 256) >= sms) launch(type, major, std::integral_constant<int, 256>());
        else if (p.columns > 64 && row_tiles * ceil_div(p.columns, 128) >= sms / 2) launch(type, major, std::integral_constant<int, 128>());
        else launch(type, major, std::integral_constant<int, 64>());
    };
    auto by_major = [&](auto type) {
        if (mn) by_width(type, std::true_type());
        else by_width(type, std::false_type());
    };
    if (p.X.type == MOPS_B200_BF16) by_major(std::true_type());
    else by_major(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

bool multiply_outer_mma(const Call& call, const OuterProblem& p, const std::string& op) {
    if (p.X.type != MOPS_B200_F16 && p.X.type != MOPS_B200_BF16) return false;
    const int64_t rows = p.X.shape[0], height = p.X.shape[1], columns = p.Y.shape[1];
    if (rows == 0) return false;
    const bool loose = columns % 8 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
    const int sms = sm_count(call.device);
    auto launch = [&](auto type, auto width) {
        constexpr bool BF16 = decltype(type)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, height, rows, 1, p.X.stride[0], 0, 64);
        const CUtensorMap y = tensor_map(p.X.type, p.Y.data, columns, rows, 1, p.Y.stride[0], 0, 64);
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, columns, height, p.groups, columns, height * columns, 32);
        const int64_t tiles = ceil_div(height, kTileRows) * ceil_div(columns, kColumns);
        const int64_t segment = outer_segment(rows, tiles, sms), most_parts = most_outer_parts(rows, tiles, segment);
        float* parts = rows > segment ? static_cast<float*>(scratch_alloc(call, static_cast<size_t>(most_parts) * kTileRows * kColumns * sizeof(float)))
                                      : nullptr;
        auto kernel = grouped_outer_mma<BF16, kColumns>;
        allow_dynamic_smem(kernel, call.device, L::kBytes);
        const int64_t pieces = tiles * (rows / segment + p.groups);
        kernel<<<static_cast<unsigned>(std::min<int64_t>(pieces, sms)), kThreads, L::kBytes, call.stream>>>(
            x, y, out, static_cast<uint16_t*>(p.out.data), parts, most_parts, p.offsets, p.groups, rows, static_cast<int>(height),
            static_cast<int>(columns), segment, loose, call.status);
        if (rows > segment) {
            join_outer<T, kColumns>(call, p, parts, most_parts, tiles, segment, op);
            scratch_free(call, parts);
        }
        note_kernel_f("grouped_outer_mma<%s,%d>", BF16 ? "bf16" : "f16", kColumns);
    };
    auto by_width = [&](auto type) {
        if (columns > 128) launch(type, std::integral_constant<int, 256>());
        else if (columns > 64) launch(type, std::integral_constant<int, 128>());
        else launch(type, std::integral_constant<int, 64>());
    };
    if (p.X.type == MOPS_B200_BF16) by_width(std::true_type());
    else by_width(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
