// Products of f32 on tensor cores whose operands have been cut into three bf16 parts beforehand (x = x0 + x1 + x2, by cutting bits off; grouped_split.cu says why six products of them and in what
// order), as arrays of three slices. Cutting takes a pass over the operands, 10 bytes a value; in return nothing stands between the copies and the products, so that pairs of blocks can multiply: tiles of 256 x 256, of
// whose stages of 64 values of depth each block takes 96 KB in and gives the tensor cores 192 KB for six products. As there, an accumulator takes a stage and is then added, rounded, to sums in
// registers. For a single group of rows, or the columns of outer products.
// 3689 rows of 8009 x 512 (182 GFLOP in six products): the loss 146 us (1.24 PFLOP/s), dx 177 (181 MB of parts are written), grad_A 143, grad_W 130, at up to 1965 MHz; gradients in steps without a pause, at
// some 1650 MHz, 5 to 15 % more.
//
// E as in split_rows.cuh, with sums of 128 columns, of the tile's first half or its second. E::kAllRows: it stores also where the warp has no rows; E::kMend: sums that are NaN are computed again.
#ifndef MOPS_B200_PARTS_ROWS_CUH
#define MOPS_B200_PARTS_ROWS_CUH

#include "split_rows.cuh"

namespace mops_b200 {

constexpr int kThreeParts = 3;
constexpr int kPartsOwn = 128; // columns of a storing warp
constexpr int kPartsTile = 256;

struct PartsLayout {
    static constexpr bool kPair = true, kRepairs = false;
    static constexpr int kOperand = kTileRows * kBoxRow; // bytes of a part of a stage, of either operand
    static constexpr int kStage = 2 * kThreeParts * kOperand, kStages = 2;
    static constexpr int kStoreWarps = 8, kStaging = BoxOut::kBytes;
    static constexpr int kStagingAt = kStages * kStage;
    static constexpr int kRingsAt = kStagingAt + kStoreWarps * kStaging;
    static constexpr int kPieces = 3;
    static constexpr int kThreads = (kFirstStoreWarp + kStoreWarps) * 32;
    static constexpr int kBytes = kRingsAt + 512 + 1024;
    static constexpr unsigned kTmem = 2 * kPartsTile;
    struct Rings {
        Ring<kStages> stages;
        Ring<2> accumulators;
        Pieces<kPieces> pieces;
        uint32_t tmem;
        int gave_up;
        __device__ void begin() {
            stages.begin(2, 1);
            accumulators.begin(1, 2 * kStoreWarps);
            pieces.begin(2 + kStoreWarps, true);
        }
    };
    static_assert(sizeof(Rings) <= 512, "room for the rings");
};

// As Work::mend (split_block.cuh): sums that are NaN are replaced by what the ordinary units make of the f32 operands. terms: of the warp's first row and column.
template <int kOwn> __device__ __noinline__ void mend_parts(float* sum, const split::Terms& all, int lane) {
#pragma unroll 1
    for (int c = 0; c < kOwn; c += 32) {
        split::Terms terms = all;
        terms.b += c * terms.b_column;
        terms.columns -= c;
#pragma unroll 1
        for (int j = 0; j < 32 && j < terms.columns; j++) {
            const float value = sum[c + j];
            unsigned bad = __ballot_sync(kFullMask, lane < terms.rows && value != value && !terms.nan_at_once(lane, j));
            for (; bad != 0; bad &= bad - 1) {
                const int i = __ffs(bad) - 1;
                const float again = terms.product(i, j, lane);
                if (lane == i) sum[c + j] = again;
            }
        }
    }
}

// rows, depth: of a product of rows; of an outer product (DecodeDepth) the height, and the most rows there may be.
template <bool A_MN, bool B_MN, typename E, template <int, int> class Decode>
__global__ void __launch_bounds__(PartsLayout::kThreads, 1)
parts_rows(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ typename E::Args args,
           const __grid_constant__ SplitOperands from, const int32_t* __restrict__ offsets, int64_t rows, int depth, int columns, int slices, Status st) {
    extern __shared__ unsigned char raw[];
    using L = PartsLayout;
    using H = Hands<L>;
    constexpr bool kSliced = kRowSlices<Decode> || kOfDepth<Decode>;
    constexpr int part_a[6] = {0, 2, 1, 0, 1, 0}, part_b[6] = {2, 0, 1, 1, 0, 0}; // small products first
    const int rank = static_cast<int>(pair_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    auto stage_at = [&](const Turn<L::kStages>& stage) { return block.base + static_cast<uint32_t>(stage.at) * L::kStage; };
    if (warp == kTilePieceWarp) {
        const int steps = (depth + kBoxDepth - 1) / kBoxDepth;
        if constexpr (kOfDepth<Decode>) hand_out(block, rank, lane, Decode<kPartsTile, kPartsTile>(offsets, depth, rows, columns, steps, slices, lane));
        else if constexpr (kSliced) hand_out(block, rank, lane, Decode<kPartsTile, kPartsTile>(offsets, 1, rows, columns, steps, slices, lane));
        else hand_out(block, rank, lane, Decode<kPartsTile, kPartsTile>(offsets, 1, rows, columns, steps, lane));
    } else if (warp == 0) {
        Supply<L> supply{block};
        Turn<L::kStages> stage;
        int64_t sent = 0;
        for (Piece piece; supply.next(piece, lane);) {
            bool ok = true;
            if (lane == 0 && piece.group >= 0) {
                const int row = static_cast<int>(min(piece.lo + rank * kTileRows, rows)), column = piece.column + rank * kTileRows;
                for (int s = 0; s < piece.steps; s++) {
                    ok = block.wait_empty(block.rings->stages, stage);
                    if (!ok) break;
                    uint64_t* full = &block.rings->stages.full[stage.at];
                    const uint32_t a = stage_at(stage), b = a + kThreeParts * L::kOperand;
                    const int deep = (kSliced ? static_cast<int>(piece.slot) + s : s) * kBoxDepth;
                    H::expect(full, L::kStage);
#pragma unroll
                    for (int p = kThreeParts - 1; p >= 0; p--) {
                        if constexpr (A_MN) {
                            // (a box begins on a multiple of 64 whatever the number of rows is)
                            const int first = static_cast<int>(piece.lo) + rank * kTileRows;
                            H::fetch(a + p * L::kOperand, map_a, first, deep, p, full);
                            H::fetch(a + p * L::kOperand + kBoxBytes, map_a, first + 64, deep, p, full);
                        } else {
                            H::fetch(a + p * L::kOperand, map_a, deep, row, p, full);
                        }
                        if constexpr (B_MN) {
                            H::fetch(b + p * L::kOperand, map_b, column, deep, p, full);
                            H::fetch(b + p * L::kOperand + kBoxBytes, map_b, column + 64, deep, p, full);
                        } else {
                            H::fetch(b + p * L::kOperand, map_b, deep, column, p, full);
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
        Turn<2> run;
        for (Piece piece; supply.next(piece, lane);) {
            bool ok = true;
            if (lane == 0 && piece.group >= 0 && rank == 0) {
                constexpr uint32_t instruction = instruction_descriptor(true, A_MN, B_MN, kPartsTile, 2 * kTileRows);
                for (int s = 0; s < piece.steps && ok; s++) {
                    ok = block.wait_empty(block.rings->accumulators, run) && block.wait_full(block.rings->stages, stage);
                    if (!ok) break;
                    tmem_fence_after_sync();
                    const uint64_t a = operand_descriptor(stage_at(stage), kBoxBytes), b = operand_descriptor(stage_at(stage) + kThreeParts * L::kOperand, kBoxBytes);
#pragma unroll
                    for (int i = 0; i < 6; i++)
#pragma unroll
                        for (int k = 0; k < kBoxDepth / 16; k++)
                            H::multiply(block.accumulator(run), a + (part_a[i] * (L::kOperand >> 4) + k * kDepthStep<A_MN>),
                                        b + (part_b[i] * (L::kOperand >> 4) + k * kDepthStep<B_MN>), instruction, i + k > 0);
                    H::multiplied(&block.rings->stages.empty[stage.at]);
                    H::multiplied(&block.rings->accumulators.full[run.at]);
                    stage.next();
                    run.next();
                }
            }
            if (!__shfl_sync(kFullMask, ok, 0)) break;
        }
    } else if (warp >= kFirstStoreWarp) {
        const int quadrant = warp & 3, half = (warp - kFirstStoreWarp) / 4;
        Supply<L> supply{block};
        Turn<2> run;
        E work(args, block.base + L::kStagingAt + (warp - kFirstStoreWarp) * L::kStaging, lane);
        for (Piece piece; supply.next(piece, lane);) {
            const int64_t row = piece.lo + rank * kTileRows + quadrant * 32;
            const int here = static_cast<int>(min(max(min(piece.hi, kOfDepth<Decode> ? rows : piece.hi) - row, int64_t(0)), int64_t(32)));
            work.begin(piece, row, here, half);
            if (piece.group < 0) {
                if (half == 0) work.clear();
                continue;
            }
            float sum[kPartsOwn];
#pragma unroll
            for (int i = 0; i < kPartsOwn; i++) sum[i] = 0;
            bool ok = true;
            for (int s = 0; s < piece.steps; s++) {
                ok = __all_sync(kFullMask, block.wait_full(block.rings->accumulators, run));
                if (!ok) break;
                tmem_fence_after_sync();
                const uint32_t at = tmem_quadrant(block.accumulator(run), quadrant) + half * kPartsOwn;
#pragma unroll
                for (int c = 0; c < kPartsOwn; c += 16) {
                    uint32_t r[2][8];
                    tmem_load(at + c, r[0]);
                    tmem_load(at + c + 8, r[1]);
                    tmem_wait_load();
                    tmem_pin(r[0]);
                    tmem_pin(r[1]);
#pragma unroll
                    for (int j = 0; j < 16; j++) sum[c + j] += __uint_as_float(r[j / 8][j % 8]);
                }
                tmem_fence_before_sync();
                __syncwarp();
                if (lane == 0) H::arrive(&block.rings->accumulators.empty[run.at]);
                run.next();
            }
            if (!ok) break;
            if (here <= 0 && !E::kAllRows) continue;
            if constexpr (E::kMend) {
                float check[4] = {};
#pragma unroll
                for (int i = 0; i < kPartsOwn; i++) check[i % 4] = fmaf(sum[i], 0.f, check[i % 4]);
                if (__any_sync(kFullMask, lane < here && isnan((check[0] + check[1]) + (check[2] + check[3])))) {
                    const int column = piece.column + half * kPartsOwn;
                    const split::Terms terms{from.x + row * from.x_stride, from.m[0] + column * from.column_stride, from.x_stride, 1, from.column_stride, from.depth_stride,
                                             depth, here, columns - column};
                    float copy[kPartsOwn]; // (in local memory: this is for sums that are infinite or NaN)
#pragma unroll
                    for (int i = 0; i < kPartsOwn; i++) copy[i] = sum[i];
                    mend_parts<kPartsOwn>(copy, terms, lane);
#pragma unroll
                    for (int i = 0; i < kPartsOwn; i++) sum[i] = copy[i];
                }
            }
            work.store(sum);
        }
        work.end();
    }
    __syncwarp();
    block.end(warp);
}

// An operand in parts: three slices, `stride` values between rows of `inner` neighbouring ones, `outer` rows.
struct PartsArray {
    void* data;
    int64_t inner, outer, stride, slice;
    CUtensorMap map(int box) const { return tensor_map(MOPS_B200_BF16, data, inner, outer, kThreeParts, stride, slice, box); }
};

template <bool A_MN, bool B_MN, typename E, template <int, int> class Decode>
void launch_parts(const Call& call, const std::string& op, const PartsArray& a, const PartsArray& b, const int32_t* offsets, int64_t rows, int64_t depth, int64_t columns,
                  int64_t slices, const SplitOperands& from, const typename E::Args& args) {
    const int64_t tiles = (ceil_div(rows, kPartsTile) + (kOfDepth<Decode> ? 0 : 2)) * ceil_div(columns, kPartsTile) * slices;
    launch_blocks<PartsLayout>(call, op, parts_rows<A_MN, B_MN, E, Decode>, tiles, a.map(A_MN ? 64 : kTileRows), b.map(B_MN ? 64 : kTileRows), args, from, offsets, rows,
                               static_cast<int>(depth), static_cast<int>(columns), static_cast<int>(slices), call.status);
}

// Cuts two values' top eight bits off each, three times: the parts of both side by side.
__device__ __forceinline__ void cut_three(float x, float y, uint32_t (&w)[kThreeParts]) {
    uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
#pragma unroll
    for (int p = 0; p < kThreeParts; p++) w[p] = split::cut_part(u, v);
}

// Rows of f32 in parts, 8 columns (a pack of each part) to a thread: all of them, or *kept and 64 of zeros behind them.
static __global__ void __launch_bounds__(256)
cut_rows(uint4* __restrict__ to, int64_t slice_packs, int64_t packs, const float* __restrict__ from, int64_t stride, int64_t rows, int columns,
         const int32_t* __restrict__ kept, bool aligned) {
    const int64_t n = kept != nullptr ? min(int64_t(*kept) + 64, rows) : rows, real = kept != nullptr ? *kept : rows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; i < n; i += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const float* p = from + i * stride;
        for (int64_t c = threadIdx.x; c < packs; c += blockDim.x) {
            alignas(16) float x[8];
            const int here = i < real ? columns - static_cast<int>(c) * 8 : 0;
            if (aligned && here >= 8) {
                *reinterpret_cast<float4*>(x) = __ldg(reinterpret_cast<const float4*>(p) + 2 * c);
                *reinterpret_cast<float4*>(x + 4) = __ldg(reinterpret_cast<const float4*>(p) + 2 * c + 1);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = k < here ? p[c * 8 + k] : 0.f;
            }
            uint32_t w[4][kThreeParts];
#pragma unroll
            for (int k = 0; k < 4; k++) cut_three(x[2 * k], x[2 * k + 1], w[k]);
#pragma unroll
            for (int q = 0; q < kThreeParts; q++) to[q * slice_packs + i * packs + c] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
        }
    }
}
// room: 6 bytes for each of `outer` x whole packs
inline PartsArray cut(const Call& call, void* room, const float* from, int64_t stride, int64_t rows, int64_t outer, int64_t columns, const int32_t* kept) {
    const int64_t packs = (columns + 7) / 8;
    unsigned across = 4;
    while (across < 32 && across < packs) across *= 2;
    const dim3 block(across, 256 / across);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(outer, block.y), int64_t(sm_count(call.device)) * 16));
    cut_rows<<<grid, block, 0, call.stream>>>(static_cast<uint4*>(room), outer * packs, packs, from, stride, kept != nullptr ? outer : rows, static_cast<int>(columns), kept,
                                              stride % 4 == 0 && reinterpret_cast<uintptr_t>(from) % 16 == 0);
    MOPS_CUDA_OK(cudaGetLastError());
    return {room, columns, outer, packs * 8, outer * packs * 8};
}

} // namespace mops_b200

#endif
