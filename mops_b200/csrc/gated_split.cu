// grouped_gated_product on tensor cores, for f32: products in three bf16 parts (grouped_split.cu), whose sums of U and V are gated in registers.
// 100 003 rows of 20 groups, 128 x 2 x 128, gelu: 66 us (102 MB of rows take 16, six products 24), dU and dV 87. With a depth of two or four stages a tile, operands that are cut into parts, sums that leave
// tensor memory after each stage and what the stores do of them take turns on one SM.
#include "activation.cuh"
#include "gated_mma.hpp"
#include "split_rows.cuh"

namespace mops_b200 {
namespace {

template <int kActivation> struct GateStore32 {
    static constexpr bool kHalves = true;
    struct Args {
        CUtensorMap map;
        float* out;
        int columns;
        bool loose;
    };
    BoxOut32 out;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0;
    __device__ GateStore32(const Args& a, uint32_t staging, int lane) : out{a.map, a.out, a.columns, a.columns, a.loose}, staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) { row = r, here = h, column = piece.column + half * 32; }
    __device__ __forceinline__ void store(float (&sum)[64]) const {
        if (column >= out.columns) return;
#pragma unroll
        for (int j = 0; j < 32; j++) sum[j] = Gate<kActivation, float>(sum[j]).value * sum[32 + j];
        out.put(reinterpret_cast<const float(&)[32]>(sum[0]), staging, row, here, column, lane);
    }
    __device__ __forceinline__ void clear() const { out.clear(row, here, column, kSplitColumns / 2, lane); }
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

template <int kActivation> struct GateStoreVjp32 {
    static constexpr bool kHalves = true;
    struct Args {
        CUtensorMap map_u, map_v;
        float* out;
        int64_t stride;
        int columns; // of dU
        bool loose;
        const float* grad;
        int64_t grad_stride;
        bool grad_aligned; // rows begin on multiples of 16 bytes
    };
    const Args& a;
    BoxOut32 out_u, out_v;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0;
    __device__ GateStoreVjp32(const Args& a, uint32_t staging, int lane)
        : a(a), out_u{a.map_u, a.out, a.stride, a.columns, a.loose}, out_v{a.map_v, a.out + a.columns, a.stride, a.columns, a.loose}, staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int half) {
        row = r, here = h, column = piece.column + half * 32;
        if (lane < here && column < a.columns) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(a.grad + (row + lane) * a.grad_stride + column));
    }
    __device__ __forceinline__ void store(float (&sum)[64]) const { // (the sums become dU and dV where they are)
        if (column >= a.columns) return;
        const float* from = a.grad + (row + lane) * a.grad_stride + column;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int n = lane < here ? a.columns - column - 4 * j : 0; // values that there are
            alignas(16) float d[4];
            if (a.grad_aligned && n >= 4) {
                *reinterpret_cast<float4*>(d) = *reinterpret_cast<const float4*>(from + 4 * j);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) d[k] = k < n ? from[4 * j + k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float &u = sum[4 * j + k], &v = sum[32 + 4 * j + k];
                const Gate<kActivation, float> gate(u);
                u = d[k] * v * gate.slope;
                v = d[k] * gate.value;
            }
        }
        out_u.put(reinterpret_cast<const float(&)[32]>(sum[0]), staging, row, here, column, lane);
        out_v.put(reinterpret_cast<const float(&)[32]>(sum[32]), staging, row, here, column, lane);
    }
    __device__ __forceinline__ void clear() const {} // (nothing reads those of rows of no group)
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

template <typename E> void launch_gated(const Call& call, const GatedProblem& p, const typename E::Args& args, const char* name, const std::string& op) {
    const TileProblem problem{p.A, p.offsets, p.groups, p.rows, p.depth, p.columns};
    const TileOperand halves[2] = {{p.half(0), p.W.stride[1], p.W.stride[2], p.W.stride[0]}, {p.half(1), p.W.stride[1], p.W.stride[2], p.W.stride[0]}};
    if (p.by_columns()) launch_split<true, E, DecodeRows>(call, op, problem, halves, args);
    else launch_split<false, E, DecodeRows>(call, op, problem, halves, args);
    note_kernel_f("%s<%s>", name, p.by_columns() ? "columns" : "depth");
    MOPS_CUDA_OK(cudaGetLastError());
}

} // namespace

void gated_rows_split(const Call& call, const GatedProblem& p, const Array& output, const std::string& op) {
    for_activation(p.activation, [&](auto activation) {
        using E = GateStore32<decltype(activation)::value>;
        const int64_t columns = output.shape[1];
        typename E::Args args{};
        args.loose = columns % 4 != 0 || reinterpret_cast<uintptr_t>(output.data) % 16 != 0;
        if (!args.loose) args.map = tensor_map(MOPS_B200_F32, output.data, columns, p.rows, 1, columns, 0, 32);
        args.out = static_cast<float*>(output.data), args.columns = static_cast<int>(columns);
        launch_gated<E>(call, p, args, "gated_rows_split", op);
    });
}

void gated_rows_vjp_split(const Call& call, const GatedProblem& p, const Array& to, const Array& grad, const std::string& op) {
    for_activation(p.activation, [&](auto activation) {
        using E = GateStoreVjp32<decltype(activation)::value>;
        const int64_t columns = grad.shape[1];
        typename E::Args args{};
        float* out = static_cast<float*>(to.data);
        args.loose = columns % 4 != 0;
        if (!args.loose) {
            args.map_u = tensor_map(MOPS_B200_F32, out, columns, p.rows, 1, to.stride[0], 0, 32);
            args.map_v = tensor_map(MOPS_B200_F32, out + columns, columns, p.rows, 1, to.stride[0], 0, 32);
        }
        args.out = out, args.stride = to.stride[0], args.columns = static_cast<int>(columns);
        args.grad = static_cast<const float*>(grad.data), args.grad_stride = grad.stride[0];
        args.grad_aligned = reinterpret_cast<uintptr_t>(grad.data) % 16 == 0 && grad.stride[0] % 4 == 0;
        launch_gated<E>(call, p, args, "gated_rows_vjp_split", op);
    });
}

bool multiply_rows_sliced(const Call& call, const RowsProblem& p, int64_t least, const std::string& op) {
    const int64_t sms = sm_count(call.device), tiles = most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, kSplitColumns);
    const int64_t slices = best_slices(tiles, sms, ceil_div(p.depth, split::kDepth), 0.7, least, static_cast<double>(p.rows) * p.columns * 8);
    if (2 * tiles > sms || slices == 1) return false;
    const int64_t stride = (p.columns + 3) / 4 * 4;
    Scratch room(call, static_cast<size_t>(slices * p.rows * stride) * sizeof(float));
    const TileProblem problem{p.X, p.offsets, p.groups, p.rows, p.depth, p.columns, slices};
    const TileOperand m{p.M.data, p.depth_stride, p.column_stride, p.M.stride[0]}, operands[2] = {m, m};
    const SumStore32::Args args = sum_args(room.as<float>(), slices, p.rows, stride, p.columns, false);
    if (m.by_columns()) launch_split<true, SumStore32, DecodeRowSlices>(call, op, problem, operands, args);
    else launch_split<false, SumStore32, DecodeRowSlices>(call, op, problem, operands, args);
    const int64_t blocks = std::min<int64_t>(ceil_div(p.rows * stride / 4, 256), sms * 16);
    add_slices<<<static_cast<unsigned>(blocks), 256, 0, call.stream>>>(static_cast<float*>(p.out.data), room.as<float>(), static_cast<int>(slices), p.rows, stride,
                                                                        static_cast<int>(p.columns));
    MOPS_CUDA_OK(cudaGetLastError());
    note_kernel_f("split_rows, %d slices", static_cast<int>(slices));
    return true;
}

} // namespace mops_b200
