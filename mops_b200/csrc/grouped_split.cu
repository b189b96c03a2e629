// grouped_matrix_product on tensor cores for operands that the copy engine cannot bring in as they are: f32, and f16 or bf16 whose rows
// begin anywhere. Eight warps load the operands, turn them into what the tensor cores take and put that into the ring of
// stages; the rest is as in grouped_mma.cu.
//
// f32: a value is split into three bf16 parts of eight bits each, by cutting bits off, so that the parts add up to the value exactly:
// x = x0 + x1 + x2. Of the nine products of parts the six of up to 2^-16 of the largest are computed, the small ones first (the three left out are about 2^-24 of the
// result, as a rounding to f32 is). The tensor cores add to their f32 accumulators by cutting off what does not fit, an error of one sign
// that grows with the number of additions; so an accumulator takes one stage (64 values of depth) and is then added, rounded, to sums in
// registers. An infinite or NaN operand gives NaN.
#include "grouped_block.cuh"
#include "grouped_mma.hpp"

namespace mops_b200 {
namespace {

constexpr int kFillWarps = 8, kStoreWarps = 8;
constexpr int kThreads = (1 + kFillWarps + kStoreWarps) * 32;
constexpr int kFillThreads = kFillWarps * 32;
constexpr int kMultiplyWarp = kFillWarps;

template <int kColumns, int kParts> struct Layout {
    static constexpr int kA = kTileRows * kBoxRow, kB = kColumns * kBoxRow; // bytes of one part of a stage
    static constexpr int kStage = kParts * (kA + kB);
    static constexpr int kStages = kParts == 3 ? 2 : kColumns == 128 ? 6 : 8;
    static constexpr int kStagingAt = kStages * kStage;
    static constexpr int kStaging = 32 * 33 * 4; // bytes: 32 x 32 sums of one warp, rows one word apart in banks
    static constexpr int kBarriersAt = kStagingAt + kStoreWarps * kStaging;
    static constexpr int kBytes = kBarriersAt + 256 + 1024;
    static constexpr unsigned kTmem = 2 * kColumns;
    static constexpr unsigned kFillers = kFillWarps, kStorers = kStoreWarps;
};

// ------------------------------------------------------------------ bringing operands in
// A chunk is eight neighbouring values, 16 bytes of a row of a stage.
template <typename T> struct Chunk {
    static constexpr int kWords = 8 * sizeof(T) / 4;
    uint32_t w[kWords];
};

// n values (at most eight; none if n <= 0) from p, zeros behind them. [begin, end): the bytes that the array reaches over. Loads are of
// 16 bytes, at multiples of 16 and inside of the array; near its ends, value by value.
template <typename T>
__device__ __forceinline__ void load_chunk(Chunk<T>& c, const T* p, int n, const unsigned char* begin, const unsigned char* end) {
    constexpr int kWords = Chunk<T>::kWords;
    n = min(n, 8);
#pragma unroll
    for (int i = 0; i < kWords; i++) c.w[i] = 0;
    if (n <= 0) return;
    const unsigned char* at = reinterpret_cast<const unsigned char*>(p);
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
    const unsigned char* from = at - shift;
    const int vectors = (shift + n * static_cast<int>(sizeof(T)) + 15) / 16;
    if (from >= begin && from + 16 * vectors <= end) {
        uint32_t w[kWords + 4];
#pragma unroll
        for (int v = 0; v < kWords / 4 + 1; v++) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (v < vectors) u = __ldg(reinterpret_cast<const uint4*>(from) + v);
            w[4 * v] = u.x, w[4 * v + 1] = u.y, w[4 * v + 2] = u.z, w[4 * v + 3] = u.w;
        }
        // shift the words down by 8, 4 and 2 bytes as needed
        if (shift & 8) {
#pragma unroll
            for (int i = 0; i < kWords + 2; i++) w[i] = w[i + 2];
        }
        if (shift & 4) {
#pragma unroll
            for (int i = 0; i < kWords + 1; i++) w[i] = w[i + 1];
        }
        const int bits = (shift & 3) * 8;
#pragma unroll
        for (int i = 0; i < kWords; i++) c.w[i] = sizeof(T) == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], bits);
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < kWords; i++) {
                if constexpr (sizeof(T) == 4) {
                    if (i >= n) c.w[i] = 0;
                } else {
                    if (2 * i >= n) c.w[i] = 0;
                    else if (2 * i + 1 >= n) c.w[i] &= 0xffff;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i >= n) break;
            if constexpr (sizeof(T) == 4) c.w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
            else c.w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p) + i)) << (16 * (i & 1));
        }
    }
}

// Puts a chunk into its place in each part of a stage.
template <typename T>
__device__ __forceinline__ void store_chunk(const Chunk<T>& c, uint32_t address, uint32_t part_bytes) {
    if constexpr (sizeof(T) == 2) {
        smem_store16(address, make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]));
    } else {
        uint32_t part[3][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t x[2] = {c.w[2 * i], c.w[2 * i + 1]};
#pragma unroll
            for (int k = 0; k < 3; k++) {
                part[k][i] = __byte_perm(x[0], x[1], 0x7632); // the upper halves
#pragma unroll
                for (int j = 0; j < 2; j++)
                    x[j] = __float_as_uint(__uint_as_float(x[j]) - __uint_as_float(x[j] & 0xffff0000u));
            }
        }
#pragma unroll
        for (int k = 0; k < 3; k++) smem_store16(address + k * part_bytes, make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]));
    }
}

// One operand in memory. [begin, end): the bytes that it reaches over.
template <typename T> struct Matrix {
    const T* data;
    int64_t stride, slice; // in values, between rows and between groups
    const unsigned char *begin, *end;
};

// One operand of a stage: kRows rows of 64 values. K-major: the tile's rows, along the depth. MN-major: boxes of 64 rows, a row for
// each value of depth.
template <typename T, bool MN, int kRows> struct Source {
    const T* p;        // the tile's first value of the stage
    const Matrix<T>* m;
    int across, depth; // how much of it there is from there
    static constexpr int kChunks = kRows * 8 / kFillThreads; // of each thread

    __device__ __forceinline__ void begin(const Matrix<T>& of, const T* first, int64_t size_across, int64_t size_depth) {
        m = &of, p = first;
        across = static_cast<int>(min(size_across, int64_t(kRows))), depth = static_cast<int>(size_depth);
    }
    __device__ __forceinline__ void advance() {
        p += MN ? kBoxDepth * m->stride : kBoxDepth;
        depth -= kBoxDepth;
    }
    __device__ __forceinline__ void load(Chunk<T>& c, int k) const {
        const int task = k * kFillThreads + (threadIdx.x % kFillThreads), row = task / 8, value = task % 8 * 8;
        if constexpr (MN) {
            const int d = row % 64, i = row / 64 * 64 + value;
            load_chunk<T>(c, p + d * m->stride + i, d < depth ? across - i : 0, m->begin, m->end);
        } else {
            load_chunk<T>(c, p + row * m->stride + value, row < across ? depth - value : 0, m->begin, m->end);
        }
    }
    __device__ static __forceinline__ void store(const Chunk<T>& c, int k, uint32_t to) {
        const int task = k * kFillThreads + (threadIdx.x % kFillThreads), row = task / 8, chunk = task % 8;
        store_chunk<T>(c, to + row * kBoxRow + ((chunk ^ (row & 7)) << 4), kRows * kBoxRow);
    }
};

// ------------------------------------------------------------------ the work of a block
// What both kernels do with a tile once they know where its operands lie.
template <typename T, bool A_MN, bool B_MN, int kColumns> struct Tiles {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
    using L = Layout<kColumns, kParts>;
    using A = Source<T, A_MN, kTileRows>;
    using B = Source<T, B_MN, kColumns>;
    static constexpr bool kBf16 = !std::is_same<T, __half>::value;
    static constexpr int kOwn = kColumns / 2; // columns of a storing warp
    // stages that an accumulator takes before it is added to the sums in registers
    static constexpr int kRun = kParts == 3 ? 1 : INT32_MAX;

    Block<L>& block;
    int64_t step = 0, run = 0; // so far

    // A filling warp, through all of the block's tiles: next() finds one, at(tile, a, b) says where its operands begin and returns its number of
    // stages. The next stage's values are loaded into registers while this one's are put into place.
    template <typename Next, typename At> __device__ __forceinline__ void fill(Next next, At at, int lane) {
        Chunk<T> a[A::kChunks], b[B::kChunks];
        A from_a;
        B from_b;
        auto t = next();
        if (!t.found) return;
        int steps = at(t, from_a, from_b), s = 0;
#pragma unroll
        for (int k = 0; k < A::kChunks; k++) from_a.load(a[k], k);
#pragma unroll
        for (int k = 0; k < B::kChunks; k++) from_b.load(b[k], k);
        for (bool more = true; more; step++) {
            if (++s < steps) {
                from_a.advance();
                from_b.advance();
            } else {
                t = next();
                more = t.found;
                if (more) steps = at(t, from_a, from_b), s = 0;
            }
            bool ok = true;
            if (lane == 0) ok = block.wait_empty(step);
            if (!__shfl_sync(kFullMask, ok, 0)) return;
            const uint32_t to = block.stage(step);
#pragma unroll
            for (int k = 0; k < A::kChunks; k++) {
                A::store(a[k], k, to);
                if (more) from_a.load(a[k], k);
            }
#pragma unroll
            for (int k = 0; k < B::kChunks; k++) {
                B::store(b[k], k, to + kParts * L::kA);
                if (more) from_b.load(b[k], k);
            }
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbarrier_arrive(&block.b->full[step % L::kStages]);
        }
    }

    // One thread.
    __device__ __forceinline__ bool multiply(int steps) {
        constexpr uint32_t instruction = instruction_descriptor(kBf16, A_MN, B_MN, kColumns);
        for (int s = 0; s < steps; s++, step++) {
            if (s % kRun == 0) {
                if (!block.wait_free(run)) return false;
            }
            if (!block.wait_full(step)) return false;
            tmem_fence_after_sync();
            const uint64_t da = operand_descriptor(block.stage(step), kBoxBytes);
            const uint64_t db = operand_descriptor(block.stage(step) + kParts * L::kA, kBoxBytes);
            constexpr int kProducts = kParts == 3 ? 6 : 1;
            constexpr int part_a[6] = {0, 2, 1, 0, 1, 0}, part_b[6] = {2, 0, 1, 1, 0, 0}; // small products first
            bool add = s % kRun != 0;
#pragma unroll
            for (int i = 0; i < kProducts; i++) {
                const uint64_t pa = da + (kParts == 3 ? part_a[i] * (L::kA >> 4) : 0), pb = db + (kParts == 3 ? part_b[i] * (L::kB >> 4) : 0);
#pragma unroll
                for (int k = 0; k < kBoxDepth / 16; k++, add = true)
                    umma(block.accumulator(run), pa + k * kDepthStep<A_MN>, pb + k * kDepthStep<B_MN>, instruction, add);
            }
            umma_arrive(&block.b->empty[step % L::kStages]);
            if ((s + 1) % kRun == 0 || s + 1 == steps) umma_arrive(&block.b->done[run & 1]), run++;
        }
        return true;
    }

    // A storing warp: the tile's sums of its 32 rows and kOwn columns.
    __device__ __forceinline__ bool collect(float (&sum)[kOwn], int steps, int quadrant, int half, int lane) {
        const int runs = kRun == 1 ? steps : steps > 0 ? 1 : 0;
#pragma unroll
        for (int i = 0; i < kOwn; i++) sum[i] = 0;
        for (int i = 0; i < runs; i++, run++) {
            if (!block.wait_done(run)) return false;
            tmem_fence_after_sync();
            const uint32_t from = tmem_quadrant(block.accumulator(run), quadrant) + half * kOwn;
#pragma unroll
            for (int c = 0; c < kOwn; c += 32) {
                uint32_t r[32];
                tmem_load(from + c, r);
                tmem_wait_load();
                tmem_pin(r);
#pragma unroll
                for (int j = 0; j < 32; j++) sum[c + j] += __uint_as_float(r[j]);
            }
            tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbarrier_arrive(&block.b->free[run & 1]);
        }
        return true;
    }

    // Writes them, 32 columns at a time through shared memory, a row after the other.
    __device__ __forceinline__ void store(const float (&sum)[kOwn], int warp, T* out, int64_t stride, int64_t here, int64_t wide, int lane) {
        float* staging = reinterpret_cast<float*>(block.smem + L::kStagingAt + warp * L::kStaging);
#pragma unroll
        for (int c = 0; c < kOwn; c += 32) {
            if (c >= wide) break;
#pragma unroll
            for (int j = 0; j < 32; j++) staging[lane * 33 + j] = sum[c + j];
            __syncwarp();
            if (c + lane < wide) {
                const int rows = static_cast<int>(min(here, int64_t(32)));
#pragma unroll 8
                for (int r = 0; r < rows; r++) out[r * stride + c + lane] = narrow<T>(staging[r * 33 + lane]);
            }
            __syncwarp();
        }
    }
};

// ---------------------------------------------------------------------------------- rows
template <typename T, bool M_MN, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_split(T* __restrict__ out, const __grid_constant__ Matrix<T> x, const __grid_constant__ Matrix<T> m, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
                   int64_t depth, int64_t columns, Status st) {
    extern __shared__ unsigned char raw[];
    using Work = Tiles<T, false, M_MN, kColumns>;
    using L = typename Work::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    const int64_t column_tiles = (columns + kColumns - 1) / kColumns;
    const int steps = static_cast<int>((depth + kBoxDepth - 1) / kBoxDepth);
    Work work{block};
    GroupWalk<RowTiles> walk(offsets, groups, rows, -1, groups, RowTiles{kTileRows, column_tiles});
    struct Tile {
        bool found, in_group;
        int64_t row, hi, group, column;
    };
    int64_t want = static_cast<int64_t>(blockIdx.x) - gridDim.x;
    auto next = [&](bool only_groups) { // the block's next tile
        Tile t;
        do {
            want += gridDim.x;
            const GroupPiece piece = walk.find(want, lane);
            t.found = piece.found;
            int64_t tile_row, tile_column;
            banded(piece.within, max((piece.hi - piece.lo + kTileRows - 1) / kTileRows, int64_t(1)), column_tiles, tile_row, tile_column);
            t.row = piece.lo + tile_row * kTileRows, t.hi = piece.hi, t.group = piece.group, t.column = tile_column * kColumns;
            t.in_group = piece.group >= 0 && piece.group < groups;
        } while (t.found && only_groups && !t.in_group);
        return t;
    };
    if (warp < kFillWarps) {
        work.fill([&] { return next(true); },
                  [&](const Tile& t, typename Work::A& a, typename Work::B& b) {
                      a.begin(x, x.data + t.row * x.stride, t.hi - t.row, depth);
                      b.begin(m, m.data + t.group * m.slice + t.column * (M_MN ? 1 : m.stride), columns - t.column, depth);
                      return steps;
                  },
                  lane);
    } else if (warp == kMultiplyWarp) {
        for (Tile t = next(true); t.found; t = next(true)) {
            bool ok = true;
            if (lane == 0) ok = work.multiply(steps);
            if (!__shfl_sync(kFullMask, ok, 0)) break;
        }
    } else {
        const int quadrant = warp & 3, half = (warp - kMultiplyWarp - 1) / 4;
        for (Tile t = next(false); t.found; t = next(false)) {
            float sum[Work::kOwn];
            if (!work.collect(sum, t.in_group ? steps : 0, quadrant, half, lane)) break;
            const int64_t row = t.row + quadrant * 32, column = t.column + half * Work::kOwn;
            work.store(sum, warp - kMultiplyWarp - 1, out + row * columns + column, columns, t.hi - row, columns - column, lane);
        }
    }
    __syncwarp();
    block.end(warp);
}

// ------------------------------------------------------------------------- outer products
template <typename T, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_outer_split(T* __restrict__ out, const __grid_constant__ Matrix<T> x, const __grid_constant__ Matrix<T> y, float* __restrict__ parts, int64_t most_parts,
                    const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int64_t height, int64_t columns, int64_t segment,
                    Status st) {
    extern __shared__ unsigned char raw[];
    using Work = Tiles<T, true, true, kColumns>;
    using L = typename Work::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    const int64_t row_tiles = (height + kTileRows - 1) / kTileRows, column_tiles = (columns + kColumns - 1) / kColumns;
    const int64_t tiles = row_tiles * column_tiles;
    Work work{block};
    GroupWalk<OuterPieces> walk(offsets, groups, rows, 0, groups - 1, OuterPieces{segment, tiles});
    struct Piece {
        bool found, part;
        int64_t row, column, lo, hi, group, within;
        int steps;
    };
    int64_t want = static_cast<int64_t>(blockIdx.x) - gridDim.x;
    auto next = [&](bool only_full) {
        Piece t;
        do {
            want += gridDim.x;
            const GroupPiece piece = walk.find(want, lane);
            t.found = piece.found, t.group = piece.group, t.within = piece.within, t.part = piece.hi - piece.lo > segment;
            const int64_t part = piece.within / tiles;
            int64_t tile_row, tile_column;
            banded(piece.within - part * tiles, row_tiles, column_tiles, tile_row, tile_column);
            t.row = tile_row * kTileRows, t.column = tile_column * kColumns;
            t.lo = piece.lo + part * segment, t.hi = min(t.lo + segment, piece.hi);
            t.steps = static_cast<int>((t.hi - t.lo + kBoxDepth - 1) / kBoxDepth);
        } while (t.found && only_full && t.steps == 0);
        return t;
    };
    if (warp < kFillWarps) {
        work.fill([&] { return next(true); },
                  [&](const Piece& t, typename Work::A& a, typename Work::B& b) {
                      a.begin(x, x.data + t.lo * x.stride + t.row, height - t.row, t.hi - t.lo);
                      b.begin(y, y.data + t.lo * y.stride + t.column, columns - t.column, t.hi - t.lo);
                      return t.steps;
                  },
                  lane);
    } else if (warp == kMultiplyWarp) {
        for (Piece t = next(true); t.found; t = next(true)) {
            bool ok = true;
            if (lane == 0) ok = work.multiply(t.steps);
            if (!__shfl_sync(kFullMask, ok, 0)) break;
        }
    } else {
        const int quadrant = warp & 3, half = (warp - kMultiplyWarp - 1) / 4;
        for (Piece t = next(false); t.found; t = next(false)) {
            float sum[Work::kOwn];
            if (!work.collect(sum, t.steps, quadrant, half, lane)) break;
            if (t.part) {
                const int64_t slot = parts_before(offsets, groups, rows, t.group, OuterParts{segment, tiles}, lane) + t.within;
                // (there are more parts than there is room for only where offsets descend, which is reported)
                if (slot >= most_parts) continue;
                float* to = parts + (slot * kTileRows + quadrant * 32 + lane) * kColumns + half * Work::kOwn;
#pragma unroll
                for (int i = 0; i < Work::kOwn; i += 4)
                    *reinterpret_cast<float4*>(to + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
            } else {
                const int64_t row = t.row + quadrant * 32, column = t.column + half * Work::kOwn;
                work.store(sum, warp - kMultiplyWarp - 1, out + (t.group * height + row) * columns + column, columns, height - row, columns - column,
                           lane);
            }
        }
    }
    __syncwarp();
    block.end(warp);
}

template <typename T> Matrix<T> matrix(const Array& a, int64_t rows, int64_t stride, int64_t row_values, int64_t slices, int64_t slice) {
    const unsigned char* begin = static_cast<const unsigned char*>(a.data);
    return {static_cast<const T*>(a.data), stride, slice, begin,
            begin + ((slices - 1) * slice + (rows - 1) * stride + row_values) * static_cast<int64_t>(sizeof(T))};
}

template <typename F> void for_split_type(int32_t type, F&& f) {
    if (type == MOPS_B200_F32) f(float());
    else if (type == MOPS_B200_F16) f(__half());
    else f(__nv_bfloat16());
}

} // namespace

bool multiply_rows_split(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.X.type == MOPS_B200_F64 || p.depth == 0 || p.groups == 0) return false;
    const bool mn = p.column_stride == 1;
    const int64_t stride = mn ? p.depth_stride : p.column_stride; // of M
    const int sms = sm_count(call.device);
    for_split_type(p.X.type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto major, auto width) {
            constexpr bool M_MN = decltype(major)::value;
            constexpr int kColumns = decltype(width)::value;
            using L = typename Tiles<T, false, M_MN, kColumns>::L;
            const Matrix<T> x = matrix<T>(p.X, p.rows, p.X.stride[0], p.depth, 1, 0);
            const Matrix<T> m = matrix<T>(p.M, mn ? p.depth : p.columns, stride, mn ? p.columns : p.depth, p.groups, p.M.stride[0]);
            const int64_t tiles = most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, kColumns);
            auto kernel = grouped_rows_split<T, M_MN, kColumns>;
            allow_dynamic_smem(kernel, call.device, L::kBytes);
            kernel<<<static_cast<unsigned>(std::min<int64_t>(tiles, sms)), kThreads, L::kBytes, call.stream>>>(
                static_cast<T*>(p.out.data), x, m, p.offsets, p.groups, p.rows, p.depth, p.columns, call.status);
            note_kernel_f("grouped_rows_split<%s,%s,%d>", array_type_name<T>(), M_MN ? "columns" : "depth", kColumns);
        };
        auto by_width = [&](auto major) {
            if (p.columns > 64 && most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, 128) >= sms / 2)
                launch(major, std::integral_constant<int, 128>());
            else launch(major, std::integral_constant<int, 64>());
        };
        if (mn) by_width(std::true_type());
        else by_width(std::false_type());
    });
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

bool multiply_outer_split(const Call& call, const OuterProblem& p, const std::string& op) {
    const int64_t rows = p.X.shape[0], height = p.X.shape[1], columns = p.Y.shape[1];
    if (p.X.type == MOPS_B200_F64 || rows == 0) return false;
    const int sms = sm_count(call.device);
    for_split_type(p.X.type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto width) {
            constexpr int kColumns = decltype(width)::value;
            using L = typename Tiles<T, true, true, kColumns>::L;
            const int64_t tiles = ceil_div(height, kTileRows) * ceil_div(columns, kColumns);
            const int64_t segment = outer_segment(rows, tiles, sms), most_parts = most_outer_parts(rows, tiles, segment);
            float* parts = rows > segment ? static_cast<float*>(scratch_alloc(call, static_cast<size_t>(most_parts) * kTileRows * kColumns * sizeof(float)))
                                          : nullptr;
            auto kernel = grouped_outer_split<T, kColumns>;
            allow_dynamic_smem(kernel, call.device, L::kBytes);
            const int64_t pieces = tiles * (rows / segment + p.groups);
            kernel<<<static_cast<unsigned>(std::min<int64_t>(pieces, sms)), kThreads, L::kBytes, call.stream>>>(
                static_cast<T*>(p.out.data), matrix<T>(p.X, rows, p.X.stride[0], height, 1, 0), matrix<T>(p.Y, rows, p.Y.stride[0], columns, 1, 0),
                parts, most_parts, p.offsets, p.groups, rows, height, columns, segment, call.status);
            if (rows > segment) {
                join_outer<T, kColumns>(call, p, parts, most_parts, tiles, segment, op);
                scratch_free(call, parts);
            }
            note_kernel_f("grouped_outer_split<%s,%d>", array_type_name<T>(), kColumns);
        };
        if (columns > 64) launch(std::integral_constant<int, 128>());
        else launch(std::integral_constant<int, 64>());
    });
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
