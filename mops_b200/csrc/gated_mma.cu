// grouped_gated_product on tensor cores, for f16 and bf16.
//
// A tile's accumulators hold its columns of U and, behind them, the same columns of V, so the lane of a row makes the output, or dU and dV, of what it finds in its own row, and neither U nor V ever leaves
// the SM: f32 to the end, rounded once. The backward pass computes U and V again (a third more of its products; kept in 16 bits, their rounding would add to that of dU and dV), writes dU and dV side by
// side and leaves the rest to the grouped products.
//
// Bound by the tensor cores: 16 384 rows of 8 groups, 2048 x 2 x 2048 in bf16, 207 us (1.33 PFLOP/s), dU and dV 220, at 1965 MHz, which the GPU holds for some milliseconds; in steps without a pause 245 and 256, at
// the 1455 MHz that the power limit leaves. 8192 rows of 16 groups, 2048 x 2 x 1280, 82 us (1.05), by blocks that fetch their operands for themselves, in five rounds of tiles that are 4.9 full. Few rows by memory: 16 of 12 groups, 2048 x 2 x 1024 (101 MB), 20 us.
#include "activation.cuh"
#include "few_rows.cuh"
#include "gated_mma.hpp"
#include "tile_rows.cuh"

namespace mops_b200 {
namespace {

// Of a lane's row: N values of the output of those of U and V.
template <bool BF16, int kActivation>
__device__ __forceinline__ void gate_values(const uint32_t (&u)[32], const uint32_t (&v)[32], uint4* to) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; j++)
        w[j] = pack_pair<BF16>(FastGate<kActivation>(__uint_as_float(u[2 * j])).value * __uint_as_float(v[2 * j]),
                               FastGate<kActivation>(__uint_as_float(u[2 * j + 1])).value * __uint_as_float(v[2 * j + 1]));
#pragma unroll
    for (int j = 0; j < 4; j++) to[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

template <bool BF16, int kActivation, int kColumns> struct GateStore {
    static constexpr bool kHalves = true, kAllRows = false;
    static constexpr int kStoreWarps = kColumns == 256 ? 8 : 4, kStaging = BoxOut::kBytes;
    struct Args {
        CUtensorMap map;
        uint16_t* out;
        int64_t stride;
        int columns;
        bool loose;
    };
    BoxOut out;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0;
    __device__ GateStore(const Args& a, uint32_t staging, int lane) : out{a.map, a.out, a.stride, a.columns, a.loose}, staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int) { row = r, here = h, column = piece.column; }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
        if (column + part * 64 >= out.columns) return;
        uint4 values[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t u[32], v[32];
            tmem_load(accumulator + part * 64 + h * 32, u);
            tmem_load(accumulator + kColumns / 2 + part * 64 + h * 32, v);
            tmem_wait_load();
            tmem_pin(u);
            tmem_pin(v);
            gate_values<BF16, kActivation>(u, v, values + 4 * h);
        }
        out.put(values, staging, row, here, column + part * 64, lane);
    }
    __device__ __forceinline__ void clear() const { out.clear(row, here, column, kColumns / 2, lane); }
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

template <bool BF16, int kActivation, int kColumns> struct GateStoreVjp {
    static constexpr bool kHalves = true, kAllRows = false;
    static constexpr int kStoreWarps = kColumns == 256 ? 8 : 4, kStaging = BoxOut::kBytes;
    using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
    struct Args {
        CUtensorMap map_u, map_v;
        uint16_t* out;
        int columns; // of dU, a multiple of 8
        const T* grad;
        int64_t grad_stride;
        int grad_columns;
        bool grad_aligned; // rows begin on multiples of 16 bytes
    };
    const Args& a;
    BoxOut out_u, out_v;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0;
    bool fetched = false; // the gradient's rows are in the staging memory
    __device__ GateStoreVjp(const Args& a, uint32_t staging, int lane)
        : a(a), out_u{a.map_u, a.out, 2 * int64_t(a.columns), a.columns, false}, out_v{a.map_v, a.out + a.columns, 2 * int64_t(a.columns), a.columns, false},
          staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int part) {
        row = r, here = h, column = piece.column;
        const int first = column + part * 64;
        fetched = a.grad_aligned && piece.group >= 0 && here > 0 && first + 64 <= a.grad_columns;
        if (fetched) RowsIn::fetch(staging, a.grad + row * a.grad_stride + first, a.grad_stride * 2, here, lane);
    }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
        const int first = column + part * 64;
        if (first >= a.columns) return;
        uint4 grad_u[8], grad_v[8];
        const T* from = a.grad + (row + lane) * a.grad_stride + first;
        if (fetched) RowsIn::wait();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t u[32], v[32];
            tmem_load(accumulator + part * 64 + h * 32, u);
            tmem_load(accumulator + kColumns / 2 + part * 64 + h * 32, v);
            tmem_wait_load();
            tmem_pin(u);
            tmem_pin(v);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                Pack<T, 8> g;
                if (fetched) {
                    *reinterpret_cast<uint4*>(&g) = RowsIn::chunk(staging, h * 4 + j, lane);
                } else {
                    const int c = h * 32 + j * 8, n = lane < here ? a.grad_columns - first - c : 0; // values that there are
#pragma unroll
                    for (int k = 0; k < 8; k++) g.v[k] = k < n ? from[c + k] : T(0.f);
                }
                uint32_t du[4], dv[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float x[2], y[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int at = j * 8 + k * 2 + i;
                        const FastGate<kActivation> gate(__uint_as_float(u[at]));
                        const float d = widen(g.v[k * 2 + i]);
                        x[i] = d * __uint_as_float(v[at]) * gate.slope;
                        y[i] = d * gate.value;
                    }
                    du[k] = pack_pair<BF16>(x[0], x[1]);
                    dv[k] = pack_pair<BF16>(y[0], y[1]);
                }
                grad_u[h * 4 + j] = make_uint4(du[0], du[1], du[2], du[3]);
                grad_v[h * 4 + j] = make_uint4(dv[0], dv[1], dv[2], dv[3]);
            }
        }
        __syncwarp();
        out_u.put(grad_u, staging, row, here, first, lane);
        out_v.put(grad_v, staging, row, here, first, lane);
    }
    __device__ __forceinline__ void clear() const {} // (nothing reads those of rows of no group)
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

// ------------------------------------------------------------------------------ a few rows
// As few_rows_mma (grouped_few.cu): the matrices' columns are the 128 lanes of the accumulator, 64 of the gate and the same 64 of the values, the rows of A its columns.
template <typename T, bool M_MN, int kRows, int kActivation>
__global__ void __launch_bounds__(kTileThreads)
few_rows_gated(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_gate, const __grid_constant__ CUtensorMap map_value,
               T* __restrict__ out, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int depth, int columns, Status st) {
    extern __shared__ unsigned char raw[];
    using L = FewLayout<kRows>;
    constexpr int kHalf = kTileRows / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int column = static_cast<int>(blockIdx.x) / parts * kHalf;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(offsets, groups, rows, st);
    if (blockIdx.y == 0 && rank == 0) clear_others<T, kHalf, kTileThreads>(out, offsets, groups, rows, column, columns);
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
            const int group = static_cast<int>(piece.group), deep = s * kBoxDepth;
            mbarrier_arrive_expect(full, L::kStage);
            box_in(m, map_gate, M_MN ? column : deep, M_MN ? deep : column, group, full);
            box_in(m + kBoxBytes, map_value, M_MN ? column : deep, M_MN ? deep : column, group, full);
            box_in(m + L::kM, map_x, deep, static_cast<int>(row), 0, full);
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
    // The sums go through shared memory, where the stages were: U and V of a value are in different lanes, and those of the parts in different blocks; each block of a cluster joins every parts-th row.
    const uint32_t accumulator = tmem_quadrant(block.rings->tmem, warp);
    float* part = reinterpret_cast<float*>(block.smem) + threadIdx.x;
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 8) {
        if (r0 >= here) break;
        uint32_t v[8];
        tmem_load(accumulator + r0, v);
        tmem_wait_load();
        tmem_pin(v);
#pragma unroll
        for (int r = 0; r < 8; r++)
            part[(r0 + r) * kTileRows] = from < to ? __uint_as_float(v[r]) : 0.f; // (a part of no steps has left nothing in its accumulator)
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    const int mine = threadIdx.x % kHalf, side = threadIdx.x / kHalf;
    const float* parts_of[kMostParts];
#pragma unroll
    for (int b = 0; b < kMostParts; b++) {
        const float* own = reinterpret_cast<const float*>(block.smem) + mine;
        parts_of[b] = parts > 1 ? cluster.map_shared_rank(own, b < parts ? b : rank) : own;
    }
    for (int r = rank + side * parts; r < here; r += 2 * parts) {
        float u[kMostParts], v[kMostParts], sum_u = 0, sum_v = 0; // (side by side: the way to another SM and back takes its time)
#pragma unroll
        for (int b = 0; b < kMostParts; b++) {
            u[b] = b < parts ? parts_of[b][r * kTileRows] : 0.f;
            v[b] = b < parts ? parts_of[b][r * kTileRows + kHalf] : 0.f;
        }
#pragma unroll
        for (int b = 0; b < kMostParts; b++) sum_u += u[b], sum_v += v[b];
        if (column + mine < columns) out[(row + r) * columns + column + mine] = narrow<T>(FastGate<kActivation>(sum_u).value * sum_v);
    }
    if (parts > 1) cluster.sync(); // (nobody leaves while others read its sums)
    block.end(warp);
}

bool few_gated(const Call& call, const GatedProblem& p, const Array& output, const std::string& op) {
    // as in the plain product of few rows
    if (p.rows > 32 && (p.rows > 128 || p.depth < 2048)) return false;
    auto launch = [&](auto zero, auto major, auto high, auto activation) {
        using T = decltype(zero);
        constexpr bool M_MN = decltype(major)::value;
        constexpr int kRowsOf = decltype(high)::value;
        using L = FewLayout<kRowsOf>;
        const int64_t across = ceil_div(p.columns, kTileRows / 2), pieces = std::min<int64_t>(p.rows, p.groups + p.rows / kRowsOf);
        const int parts = parts_of_depth(across * pieces, sm_count(call.device), p.depth, kRowsOf == 16 ? 128 : 512);
        const CUtensorMap x = tensor_map(p.A.type, p.A.data, p.depth, p.rows, 1, p.A.stride[0], 0, kRowsOf);
        auto half = [&](int i) {
            return M_MN ? tensor_map(p.A.type, p.half(i), p.columns, p.depth, p.groups, p.W.stride[1], p.W.stride[0], 64)
                        : tensor_map(p.A.type, p.half(i), p.depth, p.columns, p.groups, p.W.stride[2], p.W.stride[0], 64);
        };
        auto kernel = few_rows_gated<T, M_MN, kRowsOf, decltype(activation)::value>;
        allow_dynamic_smem(kernel, call.device, L::kBytes);
        Clusters clusters(call, op, across, parts, pieces, kTileThreads, L::kBytes);
        MOPS_CUDA_OK(cudaLaunchKernelEx(&clusters.config, kernel, x, half(0), half(1), static_cast<T*>(output.data), p.offsets, p.groups, p.rows,
                                        static_cast<int>(p.depth), static_cast<int>(output.shape[1]), call.status));
        note_kernel_f("few_rows_gated<%s,%s,%d>, %d parts", array_type_name<T>(), M_MN ? "columns" : "depth", kRowsOf, parts);
    };
    auto by_activation = [&](auto zero, auto major, auto high) {
        for_activation(p.activation, [&](auto f) { launch(zero, major, high, f); });
    };
    auto by_rows = [&](auto zero, auto major) {
        if (p.rows > 32) by_activation(zero, major, std::integral_constant<int, 64>());
        else by_activation(zero, major, std::integral_constant<int, 16>());
    };
    auto by_major = [&](auto zero) {
        if (p.by_columns()) by_rows(zero, std::true_type());
        else by_rows(zero, std::false_type());
    };
    if (p.A.type == MOPS_B200_BF16) by_major(__nv_bfloat16());
    else by_major(__half());
    return true;
}

// Calls f(type, major, activation, columns, pair) with what fits the problem.
template <typename F> void choose_tiles(const Call& call, const GatedProblem& p, F&& f) {
    const int sms = sm_count(call.device);
    auto by_width = [&](auto type, auto major, auto activation) {
        using std::integral_constant;
        const int64_t across = ceil_div(p.columns, 128);
        // (half a tile of each group is rows that are not there; a pair takes some 0.9 of the time of two blocks: 8192 rows of 16 groups, 2048 x 1280: six rounds of pairs 87 us, five of blocks 80)
        const int64_t of_blocks = ceil_div((2 * p.rows / kTileRows + p.groups) * across, 2 * sms);
        const int64_t of_pairs = ceil_div((p.rows / kTileRows + p.groups) * across, sms);
        if (p.columns > 64 && most_row_tiles(p.rows, p.groups, kTileRows) * across >= sms) {
            if (10 * of_blocks >= 9 * of_pairs) f(type, major, activation, integral_constant<int, 256>(), std::true_type());
            else f(type, major, activation, integral_constant<int, 256>(), std::false_type());
        } else {
            f(type, major, activation, integral_constant<int, 128>(), std::false_type());
        }
    };
    auto by_activation = [&](auto type, auto major) {
        for_activation(p.activation, [&](auto activation) { by_width(type, major, activation); });
    };
    auto by_major = [&](auto type) {
        if (p.by_columns()) by_activation(type, std::true_type());
        else by_activation(type, std::false_type());
    };
    if (p.A.type == MOPS_B200_BF16) by_major(std::true_type());
    else by_major(std::false_type());
}

template <bool BF16, bool M_MN, int kColumns, bool kPair, typename E>
void launch_gated(const Call& call, const GatedProblem& p, const typename E::Args& args, const char* name, const std::string& op) {
    const TileProblem problem{p.A, p.offsets, p.groups, p.rows, p.depth, p.columns};
    const TileOperand halves[2] = {{p.half(0), p.W.stride[1], p.W.stride[2], p.W.stride[0]}, {p.half(1), p.W.stride[1], p.W.stride[2], p.W.stride[0]}};
    launch_tiles<BF16, M_MN, kColumns, kPair, E, DecodeRows>(call, op, problem, halves, args);
    note_kernel_f("%s<%s,%s,%d,%s>", name, BF16 ? "bf16" : "f16", M_MN ? "columns" : "depth", kColumns, kPair ? "pair" : "block");
    MOPS_CUDA_OK(cudaGetLastError());
}

} // namespace

void gated_rows_mma(const Call& call, const GatedProblem& p, const Array& output, const std::string& op) {
    if (few_gated(call, p, output, op)) return;
    choose_tiles(call, p, [&](auto type, auto major, auto activation, auto width, auto paired) {
        constexpr bool BF16 = decltype(type)::value;
        constexpr int kColumns = decltype(width)::value;
        using E = GateStore<BF16, decltype(activation)::value, kColumns>;
        const int64_t columns = output.shape[1];
        const bool loose = columns % 8 != 0 || reinterpret_cast<uintptr_t>(output.data) % 16 != 0;
        typename E::Args args{};
        if (!loose) args.map = tensor_map(p.A.type, output.data, columns, p.rows, 1, columns, 0, 32);
        args.out = static_cast<uint16_t*>(output.data), args.stride = columns, args.columns = static_cast<int>(columns), args.loose = loose;
        launch_gated<BF16, decltype(major)::value, kColumns, decltype(paired)::value, E>(call, p, args, "gated_rows_mma", op);
    });
}

void gated_rows_vjp_mma(const Call& call, const GatedProblem& p, void* to, const Array& grad, const std::string& op) {
    choose_tiles(call, p, [&](auto type, auto major, auto activation, auto width, auto paired) {
        constexpr bool BF16 = decltype(type)::value;
        constexpr int kColumns = decltype(width)::value;
        using E = GateStoreVjp<BF16, decltype(activation)::value, kColumns>;
        typename E::Args args{};
        uint16_t* out = static_cast<uint16_t*>(to);
        args.map_u = tensor_map(p.A.type, out, p.columns, p.rows, 1, 2 * p.columns, 0, 32);
        args.map_v = tensor_map(p.A.type, out + p.columns, p.columns, p.rows, 1, 2 * p.columns, 0, 32);
        args.out = out, args.columns = static_cast<int>(p.columns);
        args.grad = static_cast<const typename E::T*>(grad.data), args.grad_stride = grad.stride[0], args.grad_columns = static_cast<int>(grad.shape[1]);
        args.grad_aligned = reinterpret_cast<uintptr_t>(grad.data) % 16 == 0 && grad.stride[0] % 8 == 0;
        launch_gated<BF16, decltype(major)::value, kColumns, decltype(paired)::value, E>(call, p, args, "gated_rows_vjp_mma", op);
    });
}

} // namespace mops_b200
