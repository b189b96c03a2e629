// grouped_matrix_product on tensor cores, for f16 and bf16.
//
// A block has an SM to itself and works off tiles of 128 rows by kColumns columns. One warp has the copy engine fetch boxes of both operands into a ring
// of stages of 64 values of depth, one thread of another issues the products (tcgen05.mma, accumulators in tensor
// memory), and four warps move finished accumulators through shared memory to the output while the next tile is under way in
// the other half of tensor memory.
//
// Pairs: shared memory bounds such a block: of a stage of 128 x 256 it takes 48 KB in and gives 48 KB to the tensor cores in 512 clocks,
// 192 bytes a clock, and it moves some 140. Two blocks that multiply together (cta_group::2), 256 rows by 256 columns, take half of the columns' operand
// each: 128 bytes a clock. Where there are enough rows to a group, pairs do the work.
//
// 16 384 rows of 8 groups, 2048 x 4096 in bf16 (275 GFLOP): 200 us, gradients 199 (A) and 229 us (W), 1.38 and 1.20 PFLOP/s; bounded by the tensor cores at the clock that the
// power limit leaves, the last of them also by the copies of two operands whose depth does not lie along rows. 8192 rows of 16 groups, 2048 x 1536: 52 us for some 430 tiles, three rounds of 148, of which
// shared memory by the figures above explains 34.
//
// Sums are the tensor cores' own, in f32, to the end of the depth: they cut off what does not fit where f32 would round. Of results in bf16 some 0.2 % are the neighbour of the value nearest to the exact one; the
// largest error is that of sums that are rounded.
//
// Rows: a tile begins where its group's rows do, wherever that is; of a tile that reaches past the end of its group the rows
// behind it are computed and not stored. Outer products: the depth is the group's rows; of those that do not fill a stage the ones behind the group's
// end are cleared in shared memory, by a warp that does nothing else, before they are multiplied.
#include "grouped_block.cuh"
#include "grouped_mma.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {

namespace {

constexpr int kThreads = 256;   // the copying warp, the multiplying warp, four that store, the one that clears, the one that gets pieces
constexpr int kClearWarp = 6, kPieceWarp = 7;
constexpr int kStoreWarps = 4;
constexpr int kStaging = 32 * kBoxRow; // bytes: 32 rows of 64 values, of one warp

// What a block keeps in shared memory.
template <int kColumns, bool kPaired> struct Layout {
    static constexpr bool kPair = kPaired, kRepairs = false;
    static constexpr int kOwnColumns = kPair ? kColumns / 2 : kColumns; // that a block fetches
    static constexpr int kRows = kPair ? 2 * kTileRows : kTileRows;     // of a tile
    static constexpr int kStages = kOwnColumns == 256 ? 4 : kOwnColumns == 128 ? 6 : 8;
    static constexpr int kA = kTileRows * kBoxRow, kB = kOwnColumns * kBoxRow; // bytes of a stage
    static constexpr int kStage = kA + kB;
    static constexpr int kStagingAt = kStages * kStage;
    static constexpr int kRingsAt = kStagingAt + kStoreWarps * 2 * kStaging;
    static constexpr int kPieces = 3;                    // known ahead
    static constexpr int kThreads = mops_b200::kThreads;
    static constexpr int kBytes = kRingsAt + 512 + 1024; // (boxes begin on multiples of 1024 bytes)
    static constexpr unsigned kTmem = 2 * kColumns;      // columns of tensor memory: two accumulators
    struct Rings {
        Ring<kStages> stages;
        Ring<2> accumulators;
        uint64_t to_clear[kStages]; // the copies of stages that are cleared in part before they count as full
        Pieces<kPieces> pieces;
        uint32_t tmem;
        int gave_up;
        __device__ void begin() {
            stages.begin(kPair ? 2 : 1, 1);
            accumulators.begin(1, kPair ? 2 * kStoreWarps : kStoreWarps);
            pieces.begin(kPieceWarp, kPair);
            for (int i = 0; i < kStages; i++) mbarrier_init(&to_clear[i], 1);
        }
    };
    static_assert(sizeof(Rings) <= 512, "room for the rings");
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
// fewer each lane its row. Where rows of the output begin anywhere (loose), a row after the other, value by value. out: the first row of the band. kScaled: times `factor`.
template <bool BF16, bool kScaled = false>
__device__ __forceinline__ void store_columns(uint32_t accumulator, uint32_t staging, int64_t& sent, const CUtensorMap& map,
                                              uint16_t* __restrict__ out, int row, int slice, int column, int columns, int here, bool loose,
                                              int lane, float factor = 1.f) {
    uint32_t r[2][32];
    tmem_load(accumulator, r[0]);
    tmem_load(accumulator + 32, r[1]);
    tmem_wait_load();
    tmem_pin(r[0]);
    tmem_pin(r[1]);
    if constexpr (kScaled) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 32; j++) r[h][j] = __float_as_uint(__uint_as_float(r[h][j]) * factor);
    }
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

// What a pair and a block by itself do differently.
template <typename L> struct Hand {
    // A stage's barrier, on which both blocks of a pair count, is that of the first; so are those that say that accumulators are free.
    __device__ static __forceinline__ void expect(uint64_t* full) {
        if constexpr (L::kPair) pair_arrive_expect(first_of_pair(full), L::kStage);
        else mbarrier_arrive_expect(full, L::kStage);
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

// ---------------------------------------------------------------------------------- rows
// out[r,:] = X[r,:] M[group of r]. M_MN: the columns of M are neighbours in memory, else its depth is.
template <bool BF16, bool M_MN, int kColumns, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_mma(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m,
                 const __grid_constant__ CUtensorMap map_out, uint16_t* __restrict__ out, const int32_t* __restrict__ offsets,
                 int64_t groups, int64_t rows, int depth, int columns, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using L = Layout<kColumns, kPair>;
    using H = Hand<L>;
    const int rank = kPair ? static_cast<int>(pair_rank()) : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    if (warp == kPieceWarp)
        hand_out(block, rank, lane, DecodeRows<L::kRows, kColumns>(offsets, groups, rows, columns, (depth + kBoxDepth - 1) / kBoxDepth, lane));
    Supply<L> supply{block};
    Turn<L::kStages> stage;
    Turn<2> tile;     // accumulator
    int64_t sent = 0; // boxes that this warp has fetched or stored
    auto stage_at = [&] { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    for (Piece piece; warp < kPieceWarp && supply.next(piece, lane);) {
        const int64_t row = piece.lo + rank * kTileRows; // of this block's half
        const int column = piece.column, steps = piece.steps;
        const bool in_group = piece.group >= 0;
        bool ok = true;
        if (warp == 0) {
            if (lane == 0 && in_group) {
                for (int s = 0; s < steps && ok; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(), b = a + L::kA;
                    const int own_column = column + rank * L::kOwnColumns;
                    H::expect(full);
                    H::fetch(a, map_x, s * kBoxDepth, static_cast<int>(min(row, rows)), 0, full);
                    if constexpr (M_MN) {
#pragma unroll
                        for (int j = 0; j < L::kOwnColumns / 64; j++)
                            H::fetch(b + j * kBoxBytes, map_m, own_column + j * 64, s * kBoxDepth, piece.group, full);
                    } else {
                        H::fetch(b, map_m, s * kBoxDepth, own_column, piece.group, full);
                    }
                    stage.next();
                    sent++;
                }
            }
        } else if (warp == 1) {
            if (lane == 0 && in_group && rank == 0) {
                constexpr uint32_t instruction = instruction_descriptor(BF16, false, M_MN, kColumns, L::kRows);
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
                        H::multiply(block.accumulator(tile), a + k * kDepthStep<false>, b + k * kDepthStep<M_MN>, instruction, s + k > 0);
                    H::multiplied(&block.rings->stages.empty[stage.at]);
                    stage.next();
                }
                if (ok) H::multiplied(&block.rings->accumulators.full[tile.at]);
                tile.next();
            }
        } else if (warp < kClearWarp) {
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
                    if (lane == 0) H::arrive(&block.rings->accumulators.empty[tile.at]);
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
    if (warp >= 2 && warp < kClearWarp && lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

// ------------------------------------------------------------------------- outer products
// out[g] = X[rows of g]^T Y[rows of g], kScaled: times *factor.
template <bool BF16, int kColumns, bool kPair, bool kScaled>
__global__ void __launch_bounds__(kThreads, 1)
grouped_outer_mma(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                  const __grid_constant__ CUtensorMap map_out, uint16_t* __restrict__ out, float* __restrict__ parts, int64_t most_parts,
                  const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment,
                  bool loose, const float* __restrict__ factor, Status st) {
    extern __shared__ unsigned char raw[];
    using L = Layout<kColumns, kPair>;
    using H = Hand<L>;
    const int rank = kPair ? static_cast<int>(pair_rank()) : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);
    const float scaled = kScaled ? __ldg(factor) : 1.f;

    if (warp == kPieceWarp)
        hand_out(block, rank, lane, DecodeOuter<L::kRows, kColumns, kBoxDepth>(offsets, groups, rows, height, columns, segment, lane));
    Supply<L> supply{block};
    Turn<L::kStages> stage;
    Turn<2> tile;
    int64_t sent = 0;
    unsigned cleared = 0; // a bit for each place of the ring: the round of its to_clear
    auto stage_at = [&] { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    for (Piece piece; warp < kPieceWarp && supply.next(piece, lane);) {
        const int row = piece.row + rank * kTileRows, column = piece.column, steps = piece.steps;
        const int64_t lo = piece.lo, hi = piece.hi;
        // the rows that do not fill a stage come first: they are cleared while the tile before is multiplied
        const int left = static_cast<int>((hi - lo) % kBoxDepth);
        bool ok = true;
        if (warp == 0) {
            if (lane == 0) {
                for (int s = 0; s < steps && ok; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(), b = a + L::kA;
                    const int at = static_cast<int>(left == 0 ? lo + int64_t(s) * kBoxDepth : s == 0 ? hi - left : lo + int64_t(s - 1) * kBoxDepth);
                    const int own_column = column + rank * L::kOwnColumns;
                    if (s > 0 || left == 0) {
                        H::expect(full);
#pragma unroll
                        for (int i = 0; i < kTileRows / 64; i++) H::fetch(a + i * kBoxBytes, map_x, row + i * 64, at, 0, full);
#pragma unroll
                        for (int j = 0; j < L::kOwnColumns / 64; j++) H::fetch(b + j * kBoxBytes, map_y, own_column + j * 64, at, 0, full);
                    } else { // to the clearing warp first
                        uint64_t* copied = &block.rings->to_clear[stage.at];
                        mbarrier_arrive_expect(copied, L::kStage);
#pragma unroll
                        for (int i = 0; i < kTileRows / 64; i++) box_in(a + i * kBoxBytes, map_x, row + i * 64, at, 0, copied);
#pragma unroll
                        for (int j = 0; j < L::kOwnColumns / 64; j++) box_in(b + j * kBoxBytes, map_y, own_column + j * 64, at, 0, copied);
                    }
                    stage.next();
                    sent++;
                }
            }
        } else if (warp == 1) {
            if (lane == 0 && rank == 0 && steps > 0) {
                constexpr uint32_t instruction = instruction_descriptor(BF16, true, true, kColumns, L::kRows);
                ok = block.wait_empty(block.rings->accumulators, tile);
                tmem_fence_after_sync();
                for (int s = 0; s < steps && ok; s++) {
                    const bool cut = s == 0 && left > 0;
                    if (kPair && cut) ok = block.template wait<true>(&block.rings->stages.full[stage.at], stage.round); // cleared by both
                    else ok = block.wait_full(block.rings->stages, stage);
                    if (!ok) break;
                    tmem_fence_after_sync();
                    const uint64_t a = operand_descriptor(stage_at(), kBoxBytes);
                    const uint64_t b = operand_descriptor(stage_at() + L::kA, kBoxBytes);
#pragma unroll
                    for (int k = 0; k < kBoxDepth / 16; k++)
                        if (!cut || k * 16 < left)
                            H::multiply(block.accumulator(tile), a + k * kDepthStep<true>, b + k * kDepthStep<true>, instruction, s + k > 0);
                    H::multiplied(&block.rings->stages.empty[stage.at]);
                    stage.next();
                }
                if (ok) H::multiplied(&block.rings->accumulators.full[tile.at]);
                tile.next();
            }
        } else if (warp == kClearWarp) {
            if (left > 0) {
                if (lane == 0) ok = block.wait(&block.rings->to_clear[stage.at], cleared >> stage.at & 1);
                ok = __shfl_sync(kFullMask, ok, 0);
                if (ok) ok = block.wait(&block.rings->to_clear[stage.at], cleared >> stage.at & 1); // (so that every lane has seen it)
                ok = __all_sync(kFullMask, ok);
                cleared ^= 1u << stage.at;
                if (ok) { // the rows behind are of another group; 16 of them are multiplied at a time
                    const uint32_t from = static_cast<uint32_t>(left) * kBoxRow, to = static_cast<uint32_t>(left + 15) / 16 * 16 * kBoxRow;
                    for (uint32_t box = 0; box < L::kStage; box += kBoxBytes)
                        for (uint32_t at = from + lane * 16; at < to; at += 32 * 16)
                            smem_store16(stage_at() + box + at, make_uint4(0, 0, 0, 0));
                    async_proxy_fence();
                    __syncwarp();
                    if (lane == 0) H::arrive(&block.rings->stages.full[stage.at]);
                }
            }
            stage.skip(steps);
        } else {
            const int quadrant = warp & 3;
            const int band = row + quadrant * 32, wide = min(columns - column, kColumns);
            if (steps > 0) ok = block.wait_full(block.rings->accumulators, tile);
            if (ok) {
                const uint32_t from = tmem_quadrant(block.accumulator(tile), quadrant);
                const uint32_t staging = block.base + L::kStagingAt + quadrant * 2 * kStaging;
                tmem_fence_after_sync();
                if (piece.slot >= 0) {
                    float* to = parts + (piece.slot * L::kRows + rank * kTileRows + quadrant * 32 + lane) * kColumns;
                    // (there are more parts than there is room for only where offsets descend, which is reported)
                    for (int c = 0; c < wide && piece.slot < most_parts; c += 32) {
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
                    uint16_t* to = out + (static_cast<int64_t>(piece.group) * height + band) * columns;
                    if (here > 0 && steps > 0) {
                        // (the copy engine leaves out what lies behind the output's last row)
                        for (int c = 0; c < wide; c += 64)
                            store_columns<BF16, kScaled>(from + c, staging, sent, map_out, to, band, piece.group,
                                                         column + c, columns, loose ? here : 32, loose, lane, scaled);
                    } else if (!loose) { // a group without rows
                        for (int i = 0; i < here; i++)
                            for (int c = lane * 8; c < wide; c += 32 * 8) *reinterpret_cast<uint4*>(to + static_cast<int64_t>(i) * columns + column + c) = make_uint4(0, 0, 0, 0);
                    } else {
                        for (int i = 0; i < here; i++)
                            for (int c = lane; c < wide; c += 32) to[static_cast<int64_t>(i) * columns + column + c] = 0;
                    }
                }
                if (steps > 0) {
                    tmem_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) H::arrive(&block.rings->accumulators.empty[tile.at]);
                    tile.next();
                }
            }
        }
        if (!__shfl_sync(kFullMask, ok, 0)) break;
    }
    if (warp == 0 && lane == 0) block.drain(block.rings->stages, stage, sent);
    if (warp >= 2 && warp < kClearWarp && lane == 0) boxes_left<0>();
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
    auto launch = [&](auto type, auto major, auto width, auto paired) {
        constexpr bool BF16 = decltype(type)::value, M_MN = decltype(major)::value, kPair = decltype(paired)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns, kPair>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, p.depth, p.rows, 1, p.X.stride[0], 0, kTileRows);
        const CUtensorMap m = M_MN ? tensor_map(p.X.type, p.M.data, p.columns, p.depth, p.groups, stride, p.M.stride[0], 64)
                                   : tensor_map(p.X.type, p.M.data, p.depth, p.columns, p.groups, stride, p.M.stride[0], L::kOwnColumns);
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, p.columns, p.rows, 1, p.columns, 0, 32);
        const int64_t tiles = most_row_tiles(p.rows, p.groups, L::kRows) * ceil_div(p.columns, kColumns);
        launch_blocks<L>(call, op, grouped_rows_mma<BF16, M_MN, kColumns, kPair>, tiles, x, m, out, static_cast<uint16_t*>(p.out.data), p.offsets,
                         p.groups, p.rows, static_cast<int>(p.depth), static_cast<int>(p.columns), loose, call.status);
        note_kernel_f("grouped_rows_mma<%s,%s,%d,%s>", BF16 ? "bf16" : "f16", M_MN ? "columns" : "depth", kColumns, kPair ? "pair" : "block");
    };
    auto by_width = [&](auto type, auto major) {
        using std::integral_constant;
        // The wider the tile, the fewer times X is fetched; the narrower, the more blocks share the work.
        const int64_t row_tiles = most_row_tiles(p.rows, p.groups, kTileRows);
        // Half of a tile for each group is rows that are not there, on average; a pair computes its tiles in some 0.8 of the time
        // that two blocks take for theirs.
        const int64_t of_blocks = ceil_div((2 * p.rows / kTileRows + p.groups) * ceil_div(p.columns, 256), 2 * sms);
        const int64_t of_pairs = ceil_div((p.rows / kTileRows + p.groups) * ceil_div(p.columns, 256), sms);
        if (p.columns > 128 && row_tiles * ceil_div(p.columns, 256) >= sms) {
            if (4 * of_pairs <= 5 * of_blocks - 1) launch(type, major, integral_constant<int, 256>(), std::true_type());
            else launch(type, major, integral_constant<int, 256>(), std::false_type());
        } else if (p.columns > 64 && row_tiles * ceil_div(p.columns, 128) >= sms / 2) {
            launch(type, major, integral_constant<int, 128>(), std::false_type());
        } else {
            launch(type, major, integral_constant<int, 64>(), std::false_type());
        }
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
    auto launch_as = [&](auto type, auto width, auto paired, auto with_factor) {
        constexpr bool BF16 = decltype(type)::value, kPair = decltype(paired)::value, kScaled = decltype(with_factor)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns, kPair>;
        using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, height, rows, 1, p.X.stride[0], 0, 64);
        const CUtensorMap y = tensor_map(p.X.type, p.Y.data, columns, rows, 1, p.Y.stride[0], 0, 64);
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, columns, height, p.groups, columns, height * columns, 32);
        const int64_t tiles = ceil_div(height, L::kRows) * ceil_div(columns, kColumns);
        const int64_t segment = outer_segment(rows, p.groups, tiles, kPair ? sms / 2 : sms), most_parts = most_outer_parts(rows, tiles, segment);
        Scratch room(call);
        if (rows > segment) room.take(static_cast<size_t>(most_parts) * L::kRows * kColumns * sizeof(float));
        float* parts = room.as<float>();
        launch_blocks<L>(call, op, grouped_outer_mma<BF16, kColumns, kPair, kScaled>, tiles * (rows / segment + p.groups), x, y, out,
                         static_cast<uint16_t*>(p.out.data), parts, most_parts, p.offsets, p.groups, rows, static_cast<int>(height),
                         static_cast<int>(columns), segment, loose, p.factor, call.status);
        if (rows > segment) {
            join_outer<T, L::kRows, kColumns>(call, p, parts, most_parts, tiles, segment, op);
            room.free();
        }
        note_kernel_f("grouped_outer_mma<%s,%d,%s>", BF16 ? "bf16" : "f16", kColumns, kPair ? "pair" : "block");
    };
    auto launch = [&](auto type, auto width, auto paired) {
        if (p.factor != nullptr) launch_as(type, width, paired, std::true_type());
        else launch_as(type, width, paired, std::false_type());
    };
    auto by_width = [&](auto type) {
        using std::integral_constant;
        if (columns > 128 && height > kTileRows) launch(type, integral_constant<int, 256>(), std::true_type());
        else if (columns > 128) launch(type, integral_constant<int, 256>(), std::false_type());
        else if (columns > 64) launch(type, integral_constant<int, 128>(), std::false_type());
        else launch(type, integral_constant<int, 64>(), std::false_type());
    };
    if (p.X.type == MOPS_B200_BF16) by_width(std::true_type());
    else by_width(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
