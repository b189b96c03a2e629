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

// Whose turn it is in a ring of N places: a place and the parity of the round.
template <int N> struct Turn {
    int at = 0;
    unsigned round = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, round ^= 1;
    }
    __device__ __forceinline__ void skip(int n) {
        at += n;
        round ^= static_cast<unsigned>(at / N) & 1;
        at %= N;
    }
};

// Between those who fill the places of a ring and those who empty them.
template <int N> struct Ring {
    uint64_t full[N], empty[N];
    __device__ void begin(unsigned fillers, unsigned emptiers) {
        for (int i = 0; i < N; i++) mbarrier_init(&full[i], fillers), mbarrier_init(&empty[i], emptiers);
    }
};

// Output tiles of a block of `rows` x `columns` tiles, kBand tiles of rows at a time.
__device__ __forceinline__ void banded(int64_t at, int64_t rows, int64_t columns, int64_t& row, int64_t& column) {
    const int64_t band = at / (kBand * columns);
    const int64_t high = min(int64_t(kBand), rows - band * kBand);
    const int64_t r = at - band * kBand * columns;
    column = r / high;
    row = band * kBand + (r - column * high);
}

// What the kernels share: setting up, waiting and leaving. A wait that runs out is reported, and everybody leaves. L says how shared memory is
// laid out, how many columns of tensor memory there are, what the rings are (L::Rings, with begin(), `tmem` and `gave_up`), and whether two blocks
// work as a pair (L::kPair), and whether warps compute sums again (L::kRepairs): how long others wait for them, `patience`, then grows by the time that takes.
constexpr long long kPatience = 2000000000; // clocks
template <typename L> struct Block {
    unsigned char* smem;
    typename L::Rings* rings;
    uint32_t base; // shared-memory address of the stages
    Status st;

    __device__ Block(unsigned char* raw, const Status& st) : st(st) {
        smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
        rings = reinterpret_cast<typename L::Rings*>(smem + L::kRingsAt);
        base = smem_address(smem);
    }
    __device__ void begin(int warp) {
        if (warp == 1) {
            if constexpr (L::kPair) pair_tmem_alloc(&rings->tmem, L::kTmem);
            else tmem_alloc(&rings->tmem, L::kTmem);
        }
        if (threadIdx.x == 0) {
            rings->begin();
            rings->gave_up = 0;
            mbarrier_init_fence();
        }
        sync();
    }
    __device__ void sync() {
        tmem_fence_before_sync();
        __syncthreads();
        if constexpr (L::kPair) pair_sync(); // (neither block leaves while the other may reach into its memory)
        tmem_fence_after_sync();
    }
    __device__ void end(int warp) {
        sync();
        if (warp == 1) {
            if constexpr (L::kPair) pair_tmem_free(rings->tmem, L::kTmem);
            else tmem_free(rings->tmem, L::kTmem);
        }
    }
    template <bool kOfPair> __device__ __forceinline__ static bool passed(uint64_t* bar, unsigned parity) {
        if constexpr (kOfPair) return mbarrier_try_wait_pair(bar, parity);
        else return mbarrier_try_wait(bar, parity);
    }
    // For about a second, as mbarrier_wait. kOfPair: for what threads of the other block have written, too.
    template <bool kOfPair = false> __device__ __forceinline__ bool wait(uint64_t* bar, unsigned parity) {
        if (passed<kOfPair>(bar, parity)) return true;
        const long long start = clock64();
        if constexpr (L::kRepairs) {
            while (clock64() - start < *static_cast<volatile long long*>(&rings->patience))
                if (passed<kOfPair>(bar, parity)) return true;
            *static_cast<volatile long long*>(&rings->patience) = 0; // (of everybody)
        } else {
            while (*static_cast<volatile int*>(&rings->gave_up) == 0 && clock64() - start < kPatience)
                if (passed<kOfPair>(bar, parity)) return true;
        }
        if (atomicExch(&rings->gave_up, 1) == 0) report_stalled(st);
        return false;
    }
    template <int N> __device__ __forceinline__ bool wait_full(Ring<N>& ring, const Turn<N>& turn) {
        return wait(&ring.full[turn.at], turn.round);
    }
    template <int N> __device__ __forceinline__ bool wait_empty(Ring<N>& ring, const Turn<N>& turn) { // (a fresh one is empty)
        return wait(&ring.empty[turn.at], turn.round ^ 1);
    }
    // The copying thread, before it leaves when somebody gave up: the copies that may be under way, at most one for each place. A place
    // that has none is full or waits in vain.
    template <int N> __device__ void drain(Ring<N>& ring, Turn<N> turn, int64_t issued) {
        if (*static_cast<volatile int*>(&rings->gave_up) == 0) return;
        for (int i = 0; i < N && i < issued; i++) {
            // the place before this turn, filled in its round
            turn.at = turn.at == 0 ? N - 1 : turn.at - 1;
            if (turn.at == N - 1) turn.round ^= 1;
            (void)mbarrier_wait(&ring.full[turn.at], turn.round);
        }
    }
    __device__ uint32_t accumulator(const Turn<2>& turn) const { return rings->tmem + static_cast<uint32_t>(turn.at) * (L::kTmem / 2); }
};

// ------------------------------------------------------------------ pieces of work
// A piece of work, as everybody in a block needs it.
struct alignas(16) Piece {
    int64_t lo, hi;  // rows of the tile's group from its first row on (of the first block, in a pair); outer products: the rows of its segment
    int64_t slot;    // outer products: where its part goes, -1 if it is the whole
    int group;       // -1: rows of no group
    int row, column; // outer products: the tile's first row and column
    int steps;       // stages
};

// A warp of each block gets pieces and works out what they are, while the others are at the ones before: to find a piece among groups takes a microsecond or two
// of divisions and sums over lanes, which, done by the warps that copy, multiply and store, left the tensor cores idle between tiles. The first
// piece is the one that the block (or pair) was launched for, then come those of blocks that have not begun; so all SMs are done at about the same
// time, whatever their pieces take. L::kPieces pieces are known ahead; L::kReaders warps read them.
template <int kPieces> struct Pieces {
    Ring<kPieces> ring;
    Piece piece[kPieces];
    Ring<1> answers;
    uint4 answer; // whose work was taken over
    __device__ void begin(unsigned readers, bool pair) {
        ring.begin(1, readers);
        answers.begin(1, pair ? 2 : 1);
    }
};

// The warp that gets them. decode(index, piece) says whether there is such a piece, and which (all lanes).
template <typename L, typename Decode> __device__ __forceinline__ void hand_out(Block<L>& block, int rank, int lane, Decode decode) {
    auto& pieces = block.rings->pieces;
    Turn<1> asked;
    Turn<L::kPieces> turn;
    int64_t want = blockIdx.x / (L::kPair ? 2 : 1);
    auto publish = [&](const Piece& p) {
        bool ok = true;
        if (lane == 0) {
            ok = block.wait_empty(pieces.ring, turn);
            if (ok) {
                pieces.piece[turn.at] = p;
                mbarrier_arrive(&pieces.ring.full[turn.at]);
            }
        }
        turn.next();
        return __shfl_sync(kFullMask, ok, 0) != 0;
    };
    for (;;) {
        // the next one is on its way while this one is worked out; of a pair the first block asks, and both are told
        bool ok = true;
        if (lane == 0) {
            if (rank == 0) ok = block.wait_empty(pieces.answers, asked);
            if (ok) mbarrier_arrive_expect(&pieces.answers.full[0], 16);
            if (ok && rank == 0) take_over<L::kPair>(&pieces.answer, &pieces.answers.full[0]);
        }
        if (!__shfl_sync(kFullMask, ok, 0)) return;
        Piece p;
        if (decode(want, p) && !publish(p)) {
            if (lane == 0) (void)mbarrier_wait(&pieces.answers.full[0], asked.round); // (the answer that is on its way into shared memory)
            return;
        }
        int taken = -1;
        if (lane == 0) {
            ok = block.wait_full(pieces.answers, asked);
            if (ok) {
                taken = taken_over(&pieces.answer);
                async_proxy_fence();
                if constexpr (L::kPair) pair_arrive(first_of_pair(&pieces.answers.empty[0]));
                else mbarrier_arrive(&pieces.answers.empty[0]);
            }
        }
        asked.next();
        taken = __shfl_sync(kFullMask, taken, 0);
        if (taken < 0) break;
        want = taken / (L::kPair ? 2 : 1);
    }
    Piece end{};
    end.steps = -1;
    (void)publish(end);
}

// The other warps: the next piece, if there is one.
template <typename L> struct Supply {
    Block<L>& block;
    Turn<L::kPieces> turn;
    __device__ __forceinline__ bool next(Piece& p, int lane) {
        auto& pieces = block.rings->pieces;
        const bool ok = block.wait_full(pieces.ring, turn);
        if (ok) p = pieces.piece[turn.at];
        else p.steps = -1;
        // (the vote waits for the loads: an arrival would overtake them)
        const bool all = __all_sync(kFullMask, ok && p.lo >= 0 && p.slot >= -1 && p.steps >= -1);
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&pieces.ring.empty[turn.at]);
        turn.next();
        return all && p.steps >= 0;
    }
};

// The pieces of products of rows: tiles of kRows rows by kColumns columns.
template <int kRows, int kColumns> struct DecodeRows {
    GroupWalk<RowTiles> walk;
    int64_t column_tiles;
    int steps, lane;
    __device__ DecodeRows(const int32_t* offsets, int64_t groups, int64_t rows, int64_t columns, int steps, int lane)
        : walk(offsets, groups, rows, -1, groups, RowTiles{kRows, (columns + kColumns - 1) / kColumns}),
          column_tiles((columns + kColumns - 1) / kColumns), steps(steps), lane(lane) {}
    __device__ bool operator()(int64_t want, Piece& p) {
        const GroupPiece piece = walk.find(want, lane);
        if (!piece.found) return false;
        int64_t tile_row, tile_column;
        banded(piece.within, (piece.hi - piece.lo + kRows - 1) / kRows, column_tiles, tile_row, tile_column);
        const bool in_group = piece.group >= 0 && piece.group < walk.groups;
        p.lo = piece.lo + tile_row * kRows, p.hi = piece.hi, p.slot = -1;
        p.group = in_group ? static_cast<int>(piece.group) : -1;
        p.row = 0, p.column = static_cast<int>(tile_column) * kColumns;
        p.steps = in_group ? steps : 0;
        return true;
    }
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

// The pieces of outer products: (segment, tile), kDepth rows to a stage.
template <int kRows, int kColumns, int kDepth> struct DecodeOuter {
    int64_t row_tiles, column_tiles, tiles, segment;
    GroupWalk<OuterPieces> walk;
    int lane;
    __device__ DecodeOuter(const int32_t* offsets, int64_t groups, int64_t rows, int64_t height, int64_t columns, int64_t segment, int lane)
        : row_tiles((height + kRows - 1) / kRows), column_tiles((columns + kColumns - 1) / kColumns), tiles(row_tiles * column_tiles),
          segment(segment), walk(offsets, groups, rows, 0, groups - 1, OuterPieces{segment, tiles}), lane(lane) {}
    __device__ bool operator()(int64_t want, Piece& p) {
        const GroupPiece piece = walk.find(want, lane);
        if (!piece.found) return false;
        const int64_t part = piece.within / tiles;
        int64_t tile_row, tile_column;
        banded(piece.within - part * tiles, row_tiles, column_tiles, tile_row, tile_column);
        p.lo = piece.lo + part * segment, p.hi = min(p.lo + segment, piece.hi);
        p.slot = piece.hi - piece.lo > segment
                     ? parts_before(walk.offsets, walk.groups, walk.rows, piece.group, OuterParts{segment, tiles}, lane) + piece.within
                     : -1;
        p.group = static_cast<int>(piece.group);
        p.row = static_cast<int>(tile_row) * kRows, p.column = static_cast<int>(tile_column) * kColumns;
        p.steps = static_cast<int>((p.hi - p.lo + kDepth - 1) / kDepth);
        return true;
    }
};

// Adds up the parts of a tile, in the order of the rows.
template <typename T, int kRows, int kColumns>
static __global__ void __launch_bounds__(256)
grouped_outer_join(T* __restrict__ out, const float* __restrict__ parts, int64_t most_parts,
                   const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment,
                   const float* __restrict__ factor) {
    const int lane = threadIdx.x & 31;
    const int64_t row_tiles = (height + kRows - 1) / kRows, column_tiles = (columns + kColumns - 1) / kColumns;
    const int64_t tiles = row_tiles * column_tiles;
    GroupWalk<OuterJoins> walk(offsets, groups, rows, 0, groups - 1, OuterJoins{segment, tiles});
    const GroupPiece piece = walk.find(blockIdx.x, lane);
    if (!piece.found) return;
    int64_t tile_row, tile_column;
    banded(piece.within, row_tiles, column_tiles, tile_row, tile_column);
    const int row = static_cast<int>(tile_row) * kRows, column = static_cast<int>(tile_column) * kColumns;
    const int64_t n = (piece.hi - piece.lo + segment - 1) / segment;
    const int64_t first = parts_before(offsets, groups, rows, piece.group, OuterParts{segment, tiles}, lane) + piece.within;
    if (first + (n - 1) * tiles >= most_parts) return;
    for (int at = (blockIdx.y * 256 + threadIdx.x) * 4; at < kRows * kColumns; at += gridDim.y * 1024) { // four values at a time
        const int i = at / kColumns, j = at % kColumns;
        if (row + i >= height || column + j >= columns) continue;
        const float* from = parts + (first * kRows + i) * kColumns + j;
        float4 sum = make_float4(0, 0, 0, 0);
        int64_t s = 0;
        constexpr int kInFlight = 8;
        for (; s + kInFlight <= n; s += kInFlight) {
            float4 v[kInFlight];
#pragma unroll
            for (int k = 0; k < kInFlight; k++) v[k] = *reinterpret_cast<const float4*>(from + (s + k) * tiles * kRows * kColumns);
#pragma unroll
            for (int k = 0; k < kInFlight; k++) sum.x += v[k].x, sum.y += v[k].y, sum.z += v[k].z, sum.w += v[k].w;
        }
        for (; s < n; s++) {
            const float4 v = *reinterpret_cast<const float4*>(from + s * tiles * kRows * kColumns);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        T* to = out + (piece.group * height + row + i) * columns + column + j;
        if (factor != nullptr) sum.x *= *factor, sum.y *= *factor, sum.z *= *factor, sum.w *= *factor;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (column + j + k < columns) to[k] = narrow<T>(v[k]);
    }
}

// How many rows a segment has. Where a group has tiles for all `workers` (blocks, or pairs), its rows are not cut: what parts cost to write and to join is
// that of some 800 rows of a tile. Where all groups together have tiles for half of the workers at most, segments are such that there are no more pieces than workers, as a group
// leaves one that is not full (30 000 rows of 8 groups, 128 x 128 in f32: 25 us; of 1024 rows 45; 100 003 rows of 20: 45.6 and 50.3). In between they are such that,
// were all rows in one group, there would be one and a half pieces for each worker, but have 1024 rows at least (6000 rows of 24 groups, 1024 x 768 in bf16: 28 us; with three
// pieces and 256 rows 54).
inline int64_t outer_segment(int64_t rows, int64_t groups, int64_t tiles, int workers) {
    if (tiles >= workers) return std::max<int64_t>(rows, 1);
    const int64_t others = workers - groups * tiles; // that do not work on the last segment of a group
    if (2 * others >= workers) return std::max<int64_t>(ceil_div(rows * tiles, others * kBoxDepth) * kBoxDepth, 256);
    return std::max<int64_t>(ceil_div(2 * rows * tiles, int64_t(workers) * 3 * kBoxDepth) * kBoxDepth, 1024);
}
// Room for the parts: a group of r > segment rows leaves at most 2 r / segment of each tile.
inline int64_t most_outer_parts(int64_t rows, int64_t tiles, int64_t segment) { return tiles * (rows / segment * 2); }

// Launches a block, or a pair of them, for each piece of work.
template <typename L, typename... P, typename... A>
void launch_blocks(const Call& call, const std::string& op, void (*kernel)(P...), int64_t pieces, const A&... arguments) {
    allow_dynamic_smem(kernel, call.device, L::kBytes);
    fits_int32(static_cast<size_t>(2 * pieces), "the number of tiles", op);
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = L::kPair ? 2 : 1, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    config.gridDim = dim3(static_cast<unsigned>(pieces) * (L::kPair ? 2 : 1));
    config.blockDim = dim3(L::kThreads);
    config.dynamicSmemBytes = L::kBytes;
    config.stream = call.stream;
    MOPS_CUDA_OK(cudaLaunchKernelEx(&config, kernel, P(arguments)...));
}

template <typename T, int kRows, int kColumns>
void join_outer(const Call& call, const OuterProblem& p, const float* parts, int64_t most_parts, int64_t tiles, int64_t segment,
                const std::string& op) {
    const int64_t rows = p.X.shape[0], joins = tiles * std::min<int64_t>(p.groups, rows / segment);
    fits_int32(static_cast<size_t>(joins), "the number of tiles", op);
    // blocks to a tile: few where there are many tiles (most of which may be whole), up to one for each 1024 values
    const int64_t most = kRows * kColumns / 1024, shares = std::min(most, std::max(most / 8, ceil_div(int64_t(sm_count(call.device)) * 8, joins)));
    grouped_outer_join<T, kRows, kColumns><<<dim3(static_cast<unsigned>(joins), static_cast<unsigned>(shares)), 256, 0, call.stream>>>(
        static_cast<T*>(p.out.data), parts, most_parts, p.offsets, p.groups, rows, static_cast<int>(p.X.shape[1]),
        static_cast<int>(p.Y.shape[1]), segment, p.factor);
    MOPS_CUDA_OK(cudaGetLastError());
}

} // namespace mops_b200

#endif
