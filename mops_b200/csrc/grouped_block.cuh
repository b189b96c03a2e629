// The frame of the tensor-core kernels of grouped_matrix_product: a ring of stages in shared memory between the threads that fill them
// and the one that multiplies, two accumulators in tensor memory between that one and the warps that store, and the pieces of work
// of outer products over a group's rows.
#ifndef MOPS_B200_GROUPED_BLOCK_CUH
#define MOPS_B200_GROUPED_BLOCK_CUH

#include "arrays.hpp"
#include "group_tiles.cuh"
#include "grouped_mma.hpp"
#include "umma.cuh"

namespace mops_b200 {

constexpr int kTileRows = 128;
constexpr int kBand = 16; // tiles of rows that are taken in turn for a tile of columns, so that both stay in L2

struct Barriers {
    uint64_t full[8], empty[8], done[2], free[2];
    uint32_t tmem;
    int gave_up;
};

// Output tiles of a block of `rows` x `columns` tiles, kBand tiles of rows at a time.
__device__ __forceinline__ void banded(int64_t at, int64_t rows, int64_t columns, int64_t& row, int64_t& column) {
    const int64_t band = at / (kBand * columns);
    const int64_t high = min(int64_t(kBand), rows - band * kBand);
    const int64_t r = at - band * kBand * columns;
    column = r / high;
    row = band * kBand + (r - column * high);
}

// What the kernels share: setting up and leaving, and the turn that each side takes at the ring of stages and at the two accumulators. A
// wait that runs out is reported, and everybody leaves. L says how shared and tensor memory are laid out, how many arrivals fill
// a stage and how many free an accumulator.
template <typename L> struct Block {
    unsigned char* smem;
    Barriers* b;
    uint32_t base; // shared-memory address of the stages
    Status st;

    __device__ Block(unsigned char* raw, const Status& st) : st(st) {
        smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
        b = reinterpret_cast<Barriers*>(smem + L::kBarriersAt);
        base = smem_address(smem);
    }
    __device__ void begin(int warp) {
        if (warp == 1) tmem_alloc(&b->tmem, L::kTmem);
        if (threadIdx.x == 0) {
            for (int s = 0; s < L::kStages; s++) mbarrier_init(&b->full[s], L::kFillers), mbarrier_init(&b->empty[s], 1);
            for (int a = 0; a < 2; a++) mbarrier_init(&b->done[a], 1), mbarrier_init(&b->free[a], L::kStorers);
            b->gave_up = 0;
            mbarrier_init_fence();
        }
        tmem_fence_before_sync();
        __syncthreads();
        tmem_fence_after_sync();
    }
    __device__ void end(int warp) {
        tmem_fence_before_sync();
        __syncthreads();
        tmem_fence_after_sync();
        if (warp == 1) tmem_free(b->tmem, L::kTmem);
    }
    __device__ bool wait(uint64_t* bar, unsigned parity) {
        if (*static_cast<volatile int*>(&b->gave_up) == 0 && mbarrier_wait(bar, parity)) return true;
        if (atomicExch(&b->gave_up, 1) == 0) report_stalled(st);
        return false;
    }
    __device__ uint32_t stage(int64_t i) const { return base + static_cast<uint32_t>(i % L::kStages) * L::kStage; }
    // The copying thread, before it fills stage i; before it leaves, for the copies that nobody waited for.
    __device__ bool wait_empty(int64_t i) {
        return i < L::kStages || wait(&b->empty[i % L::kStages], static_cast<unsigned>(i / L::kStages - 1) & 1);
    }
    __device__ void drain(int64_t issued) {
        if (*static_cast<volatile int*>(&b->gave_up) == 0) return;
        for (int64_t i = issued > L::kStages ? issued - L::kStages : 0; i < issued; i++)
            (void)mbarrier_wait(&b->full[i % L::kStages], static_cast<unsigned>(i / L::kStages) & 1);
    }
    __device__ bool wait_full(int64_t i) { return wait(&b->full[i % L::kStages], static_cast<unsigned>(i / L::kStages) & 1); }
    __device__ bool wait_free(int64_t tile) { return tile < 2 || wait(&b->free[tile & 1], static_cast<unsigned>(tile / 2 - 1) & 1); }
    __device__ bool wait_done(int64_t tile) { return wait(&b->done[tile & 1], static_cast<unsigned>(tile / 2) & 1); }
    __device__ uint32_t accumulator(int64_t tile) const { return b->tmem + static_cast<uint32_t>(tile & 1) * (L::kTmem / 2); }
};

// A group's rows are cut into segments of `segment` rows; the pieces of work are (segment, tile of the output). A group of more than one segment
// leaves its tiles in `parts`, in f32, one after the other, and grouped_outer_join adds them up.
struct OuterPieces {
    int64_t segment, tiles;
    __device__ int64_t operator()(int64_t rows) const { return max((rows + segment - 1) / segment, int64_t(1)) * tiles; }
};
struct OuterParts { // of those, the ones that are left in parts
    int64_t segment, tiles;
    __device__ int64_t operator()(int64_t rows) const { return rows > segment ? (rows + segment - 1) / segment * tiles : 0; }
};
struct OuterJoins {
    int64_t segment, tiles;
    __device__ int64_t operator()(int64_t rows) const { return rows > segment ? tiles : 0; }
};

// How many parts the groups in front of `group` leave (a warp together).
__device__ __forceinline__ int64_t parts_before(const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int64_t group,
                                                OuterParts parts, int lane) {
    int64_t n = 0;
    for (int64_t g = lane; g < group; g += 32) {
        int64_t lo, hi;
        group_bounds(offsets, groups, rows, g, lo, hi);
        n += parts(hi - lo);
    }
    return warp_sum(n);
}

// Adds up the parts of a tile, in the order of the rows.
template <typename T, int kColumns>
static __global__ void __launch_bounds__(256)
grouped_outer_join(T* __restrict__ out, const float* __restrict__ parts, int64_t most_parts,
                   const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment) {
    const int lane = threadIdx.x & 31;
    const int64_t row_tiles = (height + kTileRows - 1) / kTileRows, column_tiles = (columns + kColumns - 1) / kColumns;
    const int64_t tiles = row_tiles * column_tiles;
    GroupWalk<OuterJoins> walk(offsets, groups, rows, 0, groups - 1, OuterJoins{segment, tiles});
    const GroupPiece piece = walk.find(blockIdx.x, lane);
    if (!piece.found) return;
    int64_t tile_row, tile_column;
    banded(piece.within, row_tiles, column_tiles, tile_row, tile_column);
    const int row = static_cast<int>(tile_row) * kTileRows, column = static_cast<int>(tile_column) * kColumns;
    const int64_t n = (piece.hi - piece.lo + segment - 1) / segment;
    const int64_t first = parts_before(offsets, groups, rows, piece.group, OuterParts{segment, tiles}, lane) + piece.within;
    if (first + (n - 1) * tiles >= most_parts) return;
    constexpr int kSplit = 8; // blocks to a tile
    constexpr int kValues = kTileRows * kColumns / kSplit;
    for (int at = blockIdx.y * kValues + threadIdx.x * 4; at < (blockIdx.y + 1) * kValues; at += 256 * 4) {
        const int i = at / kColumns, j = at % kColumns;
        if (row + i >= height || column + j >= columns) continue;
        float4 sum = make_float4(0, 0, 0, 0);
        const float* from = parts + (first * kTileRows + i) * kColumns + j;
        for (int64_t s = 0; s < n; s++) {
            const float4 v = *reinterpret_cast<const float4*>(from + s * tiles * kTileRows * kColumns);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        T* to = out + (piece.group * height + row + i) * columns + column + j;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (column + j + k < columns) to[k] = narrow<T>(v[k]);
    }
}

// Segments such that, were all rows in one group, there would be some four pieces of work for each SM; so no block has much more than its share,
// and few tiles are left in parts where there are many groups.
inline int64_t outer_segment(int64_t rows, int64_t tiles, int sms) {
    return std::max<int64_t>(ceil_div(rows * tiles, int64_t(sms) * 4 * kBoxDepth) * kBoxDepth, 256);
}
// Room for the parts: a group of r > segment rows leaves at most 2 r / segment of each tile.
inline int64_t most_outer_parts(int64_t rows, int64_t tiles, int64_t segment) { return tiles * (rows / segment * 2); }

template <typename T, int kColumns>
void join_outer(const Call& call, const OuterProblem& p, const float* parts, int64_t most_parts, int64_t tiles, int64_t segment,
                const std::string& op) {
    const int64_t rows = p.X.shape[0], joins = tiles * std::min<int64_t>(p.groups, rows / segment);
    fits_int32(static_cast<size_t>(joins), "the number of tiles", op);
    grouped_outer_join<T, kColumns><<<dim3(static_cast<unsigned>(joins), 8), 256, 0, call.stream>>>(
        static_cast<T*>(p.out.data), parts, most_parts, p.offsets, p.groups, rows, static_cast<int>(p.X.shape[1]),
        static_cast<int>(p.Y.shape[1]), segment);
    MOPS_CUDA_OK(cudaGetLastError());
}

} // namespace mops_b200

#endif
