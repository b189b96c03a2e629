// Products of rows on tensor cores (f16, bf16) whose accumulators are worked on before anything is stored: the gated layer, the loss over a table.
//
// A block has an SM to itself, or two multiply as a pair, and works off tiles of kRows rows by kColumns columns of accumulators, as in grouped_mma.cu: a warp has the copy engine
// fetch boxes of both operands into a ring of stages, one thread issues the products, a warp works out pieces of work ahead of the others. What becomes of a finished accumulator is up to E,
// by warps of which two (or one) take the 32 rows of a quadrant, while the next tile is under way in the other half of tensor memory. The second operand may come in two halves (E::kHalves), each with
// a map of its own: kColumns / 2 columns of either stand in an accumulator, so that a lane finds both of its values in its own row. Of a pair the first block fetches one and the second the other.
//
// E has: kHalves, kAllRows (whether it stores also where the warp has no rows), kStoreWarps (4 or 8), kStaging (bytes of shared memory of each of them), Args (among the kernel's arguments), and
//   E(args, staging, lane)                            what a storing warp keeps
//   begin(piece, row, here, part)                     before the accumulator is there: what can be loaded (of rows of no group nothing: piece.group < 0). The warp's first row, how many it
//                                                     has, and its part of the columns
//   store(accumulator, part)                          the warp's part of the columns (0 of 1, or of 2). A slice of the depth may have no stages (piece.steps == 0): then nothing has been summed, and the
//                                                     accumulator has what stood there before
//   clear()                                           rows of no group
//   end()                                             before the block leaves
#ifndef MOPS_B200_TILE_ROWS_CUH
#define MOPS_B200_TILE_ROWS_CUH

#include "grouped_block.cuh"
#include "tensor_map.hpp"

namespace mops_b200 {

constexpr int kFirstStoreWarp = 4;
constexpr int kTilePieceWarp = 2;

template <int kColumns, bool kPaired, typename E> struct TileLayout {
    static constexpr bool kPair = kPaired, kRepairs = false;
    static constexpr int kOwnColumns = kPair ? kColumns / 2 : kColumns; // that a block fetches
    static constexpr int kRows = kPair ? 2 * kTileRows : kTileRows;     // of a tile
    static constexpr int kTileColumns = E::kHalves ? kColumns / 2 : kColumns; // of the result
    static constexpr int kA = kTileRows * kBoxRow, kB = kOwnColumns * kBoxRow, kStage = kA + kB; // bytes of a stage
    static constexpr int kStagingAll = E::kStoreWarps * E::kStaging;
    static constexpr int kMostStages = (226 * 1024 - 2048 - kStagingAll) / kStage, kStages = kMostStages < 8 ? kMostStages : 8;
    static constexpr int kStagingAt = kStages * kStage;
    static constexpr int kRingsAt = kStagingAt + kStagingAll;
    static constexpr int kPieces = 3; // known ahead
    static constexpr int kThreads = (kFirstStoreWarp + E::kStoreWarps) * 32;
    static constexpr int kBytes = kRingsAt + 512 + 1024; // (boxes begin on multiples of 1024 bytes)
    static constexpr unsigned kTmem = 2 * kColumns;      // columns of tensor memory: two accumulators
    struct Rings {
        Ring<kStages> stages;
        Ring<2> accumulators;
        Pieces<kPieces> pieces;
        uint32_t tmem;
        int gave_up;
        __device__ void begin() {
            stages.begin(kPair ? 2 : 1, 1);
            accumulators.begin(1, (kPair ? 2 : 1) * E::kStoreWarps);
            pieces.begin(2 + E::kStoreWarps, kPair);
        }
    };
    static_assert(sizeof(Rings) <= 512, "room for the rings");
};

// What a pair and a block by itself do differently.
template <typename L> struct Hands {
    // A stage's barrier, on which both blocks of a pair count, is that of the first; so are those that say that accumulators are free.
    __device__ static __forceinline__ void expect(uint64_t* full, uint32_t bytes) {
        if constexpr (L::kPair) pair_arrive_expect(first_of_pair(full), bytes);
        else mbarrier_arrive_expect(full, bytes);
    }
    __device__ static __forceinline__ void fetch(uint32_t to, const CUtensorMap& map, int inner, int outer, int slice, uint64_t* full) {
        if constexpr (L::kPair) pair_box_in(to, map, inner, outer, slice, first_of_pair(full));
        else box_in(to, map, inner, outer, slice, full);
    }
    __device__ static __forceinline__ void arrive(uint64_t* bar) {
        if constexpr (L::kPair) pair_arrive(first_of_pair(bar));
        else mbarrier_arrive(bar);
    }
    __device__ static __forceinline__ void multiply(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
        if constexpr (L::kPair) pair_umma(accumulator, a, b, instruction, add);
        else umma(accumulator, a, b, instruction, add);
    }
    __device__ static __forceinline__ void multiplied(uint64_t* bar) { // to be told to both
        if constexpr (L::kPair) pair_umma_arrive(bar);
        else umma_arrive(bar);
    }
};

template <bool BF16> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Where 64 columns of 16 bits of a warp's 32 rows go: by the copy engine where there are all 32 rows, else each lane its row; where rows of the
// output begin anywhere (loose), a row after the other, value by value. The warp has kBytes of shared memory for them.
struct BoxOut {
    static constexpr int kBytes = 32 * kBoxRow;
    const CUtensorMap& map;
    uint16_t* out; // the array's first value
    int64_t stride;
    int columns;   // of the array
    bool loose;
    __device__ __forceinline__ void put(const uint4 (&v)[8], uint32_t staging, int64_t row, int here, int column, int lane) const {
        if (loose || here == 32) {
            if (!loose && lane == 0) boxes_left<0>();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; c++) smem_store16(staging + lane * kBoxRow + ((c ^ (lane & 7)) << 4), v[c]);
            if (loose) {
                __syncwarp();
                const int wide = columns - column;
                for (int i = 0; i < here; i++) {
                    uint16_t* p = out + (row + i) * stride + column;
#pragma unroll
                    for (int h = 0; h < 64; h += 32) {
                        const int c = h + lane;
                        if (c < wide) p[c] = smem_load2(staging + i * kBoxRow + ((c / 8 ^ (i & 7)) << 4) + c % 8 * 2);
                    }
                }
                __syncwarp();
            } else {
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) box_out(map, column, static_cast<int>(row), 0, staging);
            }
        } else if (lane < here) {
            uint4* to = reinterpret_cast<uint4*>(out + (row + lane) * stride + column);
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (column + c * 8 < columns) to[c] = v[c]; // (columns are a multiple of 8 here, or there is room up to one)
        }
    }
    // zeros
    __device__ __forceinline__ void clear(int64_t row, int here, int column, int wide, int lane) const {
        for (int i = 0; i < here; i++)
            for (int c = lane; c < wide && column + c < columns; c += 32) out[(row + i) * stride + column + c] = 0;
    }
};

// As box_out, but added (f32) to what is there.
__device__ __forceinline__ void box_add(const CUtensorMap& map, int inner, int outer, int slice, uint32_t smem) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(&map), "r"(inner), "r"(outer),
                 "r"(slice), "r"(smem)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}

// Rows of 128 bytes that a warp has in its staging memory before its accumulator is there: a row for each lane, laid out as a box is.
struct RowsIn {
    // from: the first row's first byte, all on multiples of 16 bytes. `here` rows; the others are left as they are.
    __device__ static __forceinline__ void fetch(uint32_t staging, const void* from, int64_t stride, int here, int lane) {
        if (lane == 0) boxes_left<0>();
        __syncwarp();
        const int c = lane % 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = i * 4 + lane / 8;
            if (r < here)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(staging + r * kBoxRow + ((c ^ (r & 7)) << 4)),
                             "l"(static_cast<const unsigned char*>(from) + r * stride + c * 16)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
    __device__ static __forceinline__ void wait() {
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        __syncwarp();
    }
    __device__ static __forceinline__ uint4 chunk(uint32_t staging, int c, int lane) { return smem_load16(staging + lane * kBoxRow + ((c ^ (lane & 7)) << 4)); }
};

// All rows, as a single group without offsets. (Where there are offsets they are walked for a single group, too: for reasons that have not been found the same kernels take 12 to 15 % longer with this in the
// place of the walk; 16 384 rows of 50 021 x 1024: 1260 for 1110 us.)
template <int kRows, int kColumns> struct DecodeTable {
    int64_t row_tiles, column_tiles, kept;
    int steps;
    __device__ DecodeTable(const int32_t*, int64_t, int64_t rows, int64_t columns, int steps, int)
        : column_tiles((columns + kColumns - 1) / kColumns), steps(steps) {
        kept = rows;
        row_tiles = (kept + kRows - 1) / kRows;
    }
    __device__ bool operator()(int64_t want, Piece& p) const {
        if (want >= row_tiles * column_tiles) return false;
        int64_t tile_row, tile_column;
        banded(want, row_tiles, column_tiles, tile_row, tile_column);
        p.lo = tile_row * kRows, p.hi = kept, p.slot = -1;
        p.group = 0, p.row = 0, p.column = static_cast<int>(tile_column) * kColumns;
        p.steps = steps;
        return true;
    }
};

// Tiles of groups' rows, each with the depth cut into slices of `slice_steps` stages (the last ones may have fewer, or none): a piece's first stage is in p.slot, its slice in p.row.
template <int kRows, int kColumns> struct DecodeRowSlices {
    DecodeRows<kRows, kColumns> rows;
    int slices, slice_steps, all_steps;
    __device__ DecodeRowSlices(const int32_t* offsets, int64_t groups, int64_t rows, int64_t columns, int steps, int slices, int lane)
        : rows(offsets, groups, rows, columns, steps, lane), slices(slices), slice_steps((steps + slices - 1) / slices), all_steps(steps) {}
    __device__ bool operator()(int64_t want, Piece& p) {
        const int64_t tile = want / slices;
        const int slice = static_cast<int>(want - tile * slices);
        if (!rows(tile, p)) return false;
        p.slot = min(slice * slice_steps, all_steps), p.row = slice;
        if (p.group >= 0) p.steps = min(slice_steps, all_steps - static_cast<int>(p.slot));
        return true;
    }
};
template <template <int, int> class Decode> constexpr bool kRowSlices = std::is_same<Decode<1, 1>, DecodeRowSlices<1, 1>>::value;
template <template <int, int> class Decode> constexpr bool kOneGroup = std::is_same<Decode<1, 1>, DecodeTable<1, 1>>::value;

// Tiles of height x columns whose depth is the rows that offsets[1] says, cut into slices: an outer product over the rows of a single group.
template <int kRows, int kColumns> struct DecodeDepth {
    int64_t row_tiles, column_tiles;
    int slices, slice_steps, all_steps;
    __device__ DecodeDepth(const int32_t* offsets, int64_t most_rows, int64_t height, int64_t columns, int, int slices, int)
        : row_tiles((height + kRows - 1) / kRows), column_tiles((columns + kColumns - 1) / kColumns), slices(slices) {
        all_steps = static_cast<int>((rows_between(0, __ldg(offsets + 1), most_rows).hi + kBoxDepth - 1) / kBoxDepth);
        slice_steps = (all_steps + slices - 1) / slices;
    }
    __device__ bool operator()(int64_t want, Piece& p) const {
        const int64_t tile = want / slices;
        const int slice = static_cast<int>(want - tile * slices);
        if (tile >= row_tiles * column_tiles) return false;
        int64_t tile_row, tile_column;
        banded(tile, row_tiles, column_tiles, tile_row, tile_column);
        p.lo = tile_row * kRows, p.hi = INT32_MAX, p.group = 0;
        p.slot = min(slice * slice_steps, all_steps), p.row = slice, p.column = static_cast<int>(tile_column) * kColumns;
        p.steps = min(slice_steps, all_steps - static_cast<int>(p.slot));
        return true;
    }
};
template <template <int, int> class Decode> constexpr bool kOfDepth = std::is_same<Decode<1, 1>, DecodeDepth<1, 1>>::value;

// a_bytes: of a box of the first operand, which may have fewer than 128 rows where there are no more (what stands in the others does not matter). B_MN: the columns of the second operand are
// neighbours in memory, else its depth is. map_b1: its second half. rows, depth: of an outer product (DecodeDepth) the height, and the most rows there may be; the rows of both operands are the depth then,
// and those behind the last one, up to a whole stage, are zeros.
template <bool BF16, bool B_MN, int kColumns, bool kPair, typename E, template <int, int> class Decode>
__global__ void __launch_bounds__(TileLayout<kColumns, kPair, E>::kThreads, 1)
tile_rows(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b0, const __grid_constant__ CUtensorMap map_b1, int a_bytes,
          const __grid_constant__ typename E::Args args, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int depth, int columns, int slices, Status st) {
    extern __shared__ unsigned char raw[];
    using L = TileLayout<kColumns, kPair, E>;
    using H = Hands<L>;
    constexpr bool A_MN = kOfDepth<Decode>, kSliced = kRowSlices<Decode> || kOfDepth<Decode>;
    const int rank = kPair ? static_cast<int>(pair_rank()) : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if constexpr (!kOneGroup<Decode> && !kOfDepth<Decode>)
        if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);
    auto stage_at = [&](const Turn<L::kStages>& stage) { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    if (warp == kTilePieceWarp) {
        const int steps = (depth + kBoxDepth - 1) / kBoxDepth;
        if constexpr (kOfDepth<Decode>) hand_out(block, rank, lane, Decode<L::kRows, L::kTileColumns>(offsets, depth, rows, columns, steps, slices, lane));
        else if constexpr (kSliced) hand_out(block, rank, lane, Decode<L::kRows, L::kTileColumns>(offsets, groups, rows, columns, steps, slices, lane));
        else hand_out(block, rank, lane, Decode<L::kRows, L::kTileColumns>(offsets, groups, rows, columns, steps, lane));
    } else if (warp == 0) {
        Supply<L> supply{block};
        Turn<L::kStages> stage;
        int64_t sent = 0;
        for (Piece piece; supply.next(piece, lane);) {
            bool ok = true;
            if (lane == 0 && piece.group >= 0) {
                const int row = static_cast<int>(min(piece.lo + rank * kTileRows, rows));
                for (int s = 0; s < piece.steps; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(stage), b = a + L::kA;
                    const int deep = (kSliced ? static_cast<int>(piece.slot) + s : s) * kBoxDepth;
                    H::expect(full, static_cast<uint32_t>(a_bytes) + L::kB);
                    if constexpr (A_MN) {
                        const int first = static_cast<int>(piece.lo) + rank * kTileRows; // (a multiple of 64 whatever the number of rows is)
                        H::fetch(a, map_a, first, deep, 0, full);
                        H::fetch(a + kBoxBytes, map_a, first + 64, deep, 0, full);
                    } else {
                        H::fetch(a, map_a, deep, row, 0, full);
                    }
                    if constexpr (!E::kHalves) {
                        const int column = piece.column + rank * L::kOwnColumns;
                        if constexpr (B_MN) {
#pragma unroll
                            for (int j = 0; j < L::kOwnColumns / 64; j++) H::fetch(b + j * kBoxBytes, map_b0, column + j * 64, deep, piece.group, full);
                        } else {
                            H::fetch(b, map_b0, deep, column, piece.group, full);
                        }
                    } else if constexpr (kPair) {
                        const CUtensorMap& map = rank == 0 ? map_b0 : map_b1;
                        if constexpr (B_MN) {
#pragma unroll
                            for (int j = 0; j < L::kOwnColumns / 64; j++) H::fetch(b + j * kBoxBytes, map, piece.column + j * 64, deep, piece.group, full);
                        } else {
                            H::fetch(b, map, deep, piece.column, piece.group, full);
                        }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const CUtensorMap& map = half == 0 ? map_b0 : map_b1;
                            const uint32_t to = b + half * (L::kB / 2);
                            if constexpr (B_MN) {
#pragma unroll
                                for (int j = 0; j < kColumns / 128; j++) H::fetch(to + j * kBoxBytes, map, piece.column + j * 64, deep, piece.group, full);
                            } else {
                                H::fetch(to, map, deep, piece.column, piece.group, full);
                            }
                        }
                    }
                    stage.next();
                    sent++;
                }
            }
            if (!__shfl_sync(kFullMask, ok, 0)) break;
        }
        if (lane == 0) block.drain(block.rings->stages, stage, sent);
    } else if (warp == 1) {
        Supply<L> supply{block};
        Turn<L::kStages> stage;
        Turn<2> tile;
        for (Piece piece; supply.next(piece, lane);) {
            bool ok = true;
            if (lane == 0 && piece.group >= 0 && rank == 0) {
                constexpr uint32_t instruction = instruction_descriptor(BF16, A_MN, B_MN, kColumns, L::kRows);
                ok = block.wait_empty(block.rings->accumulators, tile);
                tmem_fence_after_sync();
                for (int s = 0; s < piece.steps && ok; s++) {
                    ok = block.wait_full(block.rings->stages, stage);
                    if (!ok) break;
                    tmem_fence_after_sync();
                    const uint64_t a = operand_descriptor(stage_at(stage), kBoxBytes), b = operand_descriptor(stage_at(stage) + L::kA, kBoxBytes);
#pragma unroll
                    for (int k = 0; k < kBoxDepth / 16; k++)
                        H::multiply(block.accumulator(tile), a + k * kDepthStep<A_MN>, b + k * kDepthStep<B_MN>, instruction, s + k > 0);
                    H::multiplied(&block.rings->stages.empty[stage.at]);
                    stage.next();
                }
                if (ok) H::multiplied(&block.rings->accumulators.full[tile.at]);
                tile.next();
            }
            if (!__shfl_sync(kFullMask, ok, 0)) break;
        }
    } else if (warp >= kFirstStoreWarp) {
        const int quadrant = warp & 3, part = (warp - kFirstStoreWarp) / 4;
        Supply<L> supply{block};
        Turn<2> tile;
        E work(args, block.base + L::kStagingAt + (warp - kFirstStoreWarp) * E::kStaging, lane);
        for (Piece piece; supply.next(piece, lane);) {
            const int64_t row = piece.lo + rank * kTileRows + quadrant * 32;
            const int here = static_cast<int>(min(max(min(piece.hi, kOfDepth<Decode> ? rows : piece.hi) - row, int64_t(0)), int64_t(32)));
            work.begin(piece, row, here, part);
            if (piece.group < 0) {
                if (part == 0) work.clear();
                continue;
            }
            if (!__all_sync(kFullMask, block.wait_full(block.rings->accumulators, tile))) break;
            tmem_fence_after_sync();
            if (here > 0 || E::kAllRows) work.store(tmem_quadrant(block.accumulator(tile), quadrant), part);
            tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) H::arrive(&block.rings->accumulators.empty[tile.at]);
            tile.next();
        }
        work.end();
    }
    __syncwarp();
    block.end(warp);
}

// How many slices the depth of a product (of `steps` stages, microseconds each; slices of `least` stages at least) is cut into, each with sums of its own: so many that the last round of `workers` is nearly
// full, for what the sums (bytes, written and read again) take at some 4 TB/s.
inline int64_t best_slices(int64_t tiles, int64_t workers, int64_t steps, double microseconds, int64_t least, double bytes) {
    int64_t best = 1;
    double shortest = 1e30;
    for (int64_t s = 1; s <= 64 && (s == 1 || steps / s >= least); s++) {
        const int64_t per = ceil_div(steps, s);
        const double time = static_cast<double>(ceil_div(tiles * ceil_div(steps, per), workers)) * (per * microseconds + 1.0) + s * bytes / 4e6;
        if (time < shortest) shortest = time, best = s;
    }
    return ceil_div(steps, ceil_div(steps, best)); // (none without steps, of so many; where a product of fewer is cut into as many slices, the last ones may have none)
}

// What a launch takes from its problem; `columns`: of the result.
struct TileProblem {
    Array A;            // rows x depth, boxable
    const int32_t* offsets;
    int64_t groups, rows, depth, columns;
    int64_t slices = 1; // of the depth (DecodeRowSlices)
};

// The second operand, or a half of it: value (d, j) of group g at g * group_stride + d * depth_stride + j * column_stride, boxable.
struct TileOperand {
    const void* data;
    int64_t depth_stride, column_stride, group_stride;
    bool by_columns() const { return column_stride == 1; }
};

template <bool BF16, bool B_MN, int kColumns, bool kPair, typename E, template <int, int> class Decode>
void launch_tiles(const Call& call, const std::string& op, const TileProblem& p, const TileOperand (&b)[2], const typename E::Args& args) {
    using L = TileLayout<kColumns, kPair, E>;
    constexpr int32_t type = BF16 ? MOPS_B200_BF16 : MOPS_B200_F16;
    int box = kTileRows;
    if (!kPair && !kOfDepth<Decode>)
        while (box > 16 && p.rows <= box / 2) box /= 2;
    constexpr bool kDeep = kOfDepth<Decode>;
    const CUtensorMap a = kDeep ? tensor_map(type, p.A.data, p.rows, p.depth, 1, p.A.stride[0], 0, 64) : tensor_map(type, p.A.data, p.depth, p.rows, 1, p.A.stride[0], 0, box);
    auto map_of = [&](const TileOperand& o) {
        return B_MN ? tensor_map(type, o.data, p.columns, p.depth, p.groups, o.depth_stride, o.group_stride, 64)
                    : tensor_map(type, o.data, p.depth, p.columns, p.groups, o.column_stride, o.group_stride, E::kHalves ? kColumns / 2 : L::kOwnColumns);
    };
    const CUtensorMap b0 = map_of(b[0]), b1 = E::kHalves ? map_of(b[1]) : b0;
    const int64_t tiles = (kOneGroup<Decode> || kDeep ? ceil_div(p.rows, L::kRows) : most_row_tiles(p.rows, p.groups, L::kRows)) * ceil_div(p.columns, L::kTileColumns) * p.slices;
    launch_blocks<L>(call, op, tile_rows<BF16, B_MN, kColumns, kPair, E, Decode>, tiles, a, b0, b1, box * kBoxRow, args, p.offsets, p.groups, p.rows,
                     static_cast<int>(p.depth), static_cast<int>(p.columns), static_cast<int>(p.slices), call.status);
}

} // namespace mops_b200

#endif
