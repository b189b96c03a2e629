// grouped_gated_product: the gated feed-forward layer of groups of rows. W[g] holds the N columns of the gate and, behind them, those of the values.
//
//   U = A[r,:] W[g][:, :N], V = A[r,:] W[g][:, N:]       for offsets[g] <= r < offsets[g+1]
//   output[r,:] = f(U) V
//   dV = grad_output f(U), dU = grad_output V f'(U)
//   grad_A[r,:] = [dU dV] W[g]^T, grad_W[g] = A[rows of g]^T [dU dV]
//
// On tensor cores U and V are gated where they are summed (gated_mma.cu, gated_split.cu). Here: f64, and f32 in the forms that those leave to other kernels (few rows, halves that begin anywhere). U and V, side by
// side in scratch memory, are one grouped product; a pass over them makes the output of them, or, where they stood, dU and dV, of which the gradients are the grouped products that they are for a plain
// layer. f16 and bf16 are widened to f32 where there are few rows to differentiate.
#include "activation.cuh"
#include "block_ops.hpp"
#include "convert.cuh"
#include "gated_mma.hpp"
#include "grouped_mma.hpp"
#include "pack.hpp"

namespace mops_b200 {
namespace {

// out[r,j] = f(u) v
template <int kActivation, typename T, typename S>
__global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
gate_rows(T* __restrict__ out, const S* __restrict__ uv, int64_t rows, int64_t columns) {
    for (int64_t r = first_row(); r < rows; r += row_step())
        for (int64_t j = threadIdx.x; j < columns; j += kRowThreads) {
            const S u = uv[r * 2 * columns + j], v = uv[r * 2 * columns + columns + j];
            out[r * columns + j] = narrow<T>(Gate<kActivation, S>(u).value * v);
        }
}

// u, v become dU, dV
template <int kActivation, typename T, typename S>
__global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
gate_rows_vjp(S* __restrict__ uv, const T* __restrict__ grad, int64_t grad_stride, int64_t rows, int64_t columns) {
    for (int64_t r = first_row(); r < rows; r += row_step())
        for (int64_t j = threadIdx.x; j < columns; j += kRowThreads) {
            S *u = uv + r * 2 * columns + j, *v = u + columns;
            const Gate<kActivation, S> gate(*u);
            const S g = widen(grad[r * grad_stride + j]);
            *u = g * *v * gate.slope;
            *v = g * gate.value;
        }
}

const char* const kIndexNames[] = {"offsets"};

void check_gated(Array& A, Array& W, Array& offsets, Array& rows, const char* rows_name, int32_t activation, const std::string& op) {
    check_floating(A.type, "A", op);
    check_array(A, "A", 2, A.type, op);
    check_array(W, "W", 3, A.type, op);
    check_array(rows, rows_name, 2, A.type, op);
    check_array(offsets, "offsets", 1, MOPS_B200_I32, op);
    check_size(A.shape[1], "A", 1, W.shape[1], "W", 1, op);
    check_size(rows.shape[0], rows_name, 0, A.shape[0], "A", 0, op);
    if (W.shape[2] % 2 != 0) throw std::runtime_error("W must have as many columns for the gate as for the values, an even number in all, in " + op);
    check_size(rows.shape[1], rows_name, 1, W.shape[2] / 2, "one half of W", 2, op);
    check_size(offsets.shape[0], "offsets", 0, W.shape[0] + 1, "the groups of W (and one)", 0, op);
    check_rows(A, "A", op);
    check_matrices(W, "W", op);
    if (offsets.stride[0] != 1) throw std::runtime_error("offsets must be contiguous in " + op);
    for (int64_t n : {A.shape[0], A.shape[1], W.shape[0], W.shape[2]}) fits_int32(static_cast<size_t>(n), "a size", op);
    if (activation != MOPS_B200_SILU && activation != MOPS_B200_GELU)
        throw std::runtime_error("unknown activation " + std::to_string(activation) + " in " + op);
}

// In f32 (f64 for f64), what the products are made of: A and W, widened where they have 16 bits, and U and V, or dU and dV, side by side.
struct Widened {
    const Call& call;
    const std::string& op;
    Scratch room_A, room_W, room_uv;
    Packing packing;
    Array A, W, uv;
    int32_t type;
    bool fused = false; // gated where they are summed
    Widened(const Call& call, const Array& a, const Array& w, const std::string& op)
        : call(call), op(op), room_A(call), room_W(call), room_uv(call), packing(call), A(a), W(w), type(a.type == MOPS_B200_F64 ? MOPS_B200_F64 : MOPS_B200_F32) {
        if (type != a.type) {
            room_A.take(static_cast<size_t>(values_of(a)) * 4 + 16);
            room_W.take(static_cast<size_t>(values_of(w)) * 4 + 16);
            A = converted(call, a, room_A.as<float>(), type);
            W = converted(call, w, room_W.as<float>(), type);
        }
        if (type == MOPS_B200_F32 && W.shape[0] > 0 && W.shape[1] > 0 && !straight_rows(W, A.shape[0], W.stride[2] == 1)) {
            packing.add(A);
            packing.add(W);
            packing.run();
            fused = A.shape[0] > 0 && W.shape[2] > 0 && (W.stride[2] != 1 || W.shape[2] % 8 == 0);
        }
    }
    GatedProblem problem(const int32_t* offsets, int32_t activation) const {
        return {A, W, offsets, W.shape[0], A.shape[0], A.shape[1], W.shape[2] / 2, activation};
    }
    void take_uv() {
        room_uv.take(static_cast<size_t>(A.shape[0] * W.shape[2] * type_bytes(type)) + 16);
        uv = contiguous(room_uv.as<void>(), type, A.shape[0], W.shape[2]);
    }
    void multiply(const int32_t* offsets) {
        take_uv();
        multiply_rows(call, {uv, A, W, W.stride[1], W.stride[2], offsets, W.shape[0], A.shape[0], A.shape[1], W.shape[2]}, op);
    }
};

// ---- f16 and bf16 on tensor cores
// n values where there are m, zeros behind those, by kRowThreads threads: 16 bytes at a time, as the result lies.
__device__ __forceinline__ void copy_run(uint16_t* q, int n, const uint16_t* p, int m, const unsigned char* begin, const unsigned char* end) {
    const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(q) & 15)) & 15) / 2), packs = (n - head) / 8;
    for (int i = threadIdx.x; i < head; i += kRowThreads) q[i] = i < m ? p[i] : 0;
    for (int c = threadIdx.x; c < packs; c += kRowThreads) {
        const int at = head + c * 8;
        *reinterpret_cast<uint4*>(q + at) = at < m ? load_anywhere<__half>(reinterpret_cast<const __half*>(p + at), m - at, begin, end) : make_uint4(0, 0, 0, 0);
    }
    for (int i = head + packs * 8 + threadIdx.x; i < n; i += kRowThreads) q[i] = i < m ? p[i] : 0;
}
// The halves of matrices (of `from_columns` columns each) where those of others (of `to_columns`) are, both by columns or both by depth; zeros where there are none. A row of `to` to kRowThreads threads.
// Of groups without rows: zeros (kZeros), or nothing, as nobody reads their matrices. (43 groups of 464 x 2 x 802, 128 MB read and written: 27 us, value by value 42; 62 groups of 594 x 2 x 1405,
// three of which have rows: 11 and 120)
template <bool kByColumns, bool kZeros>
__global__ void __launch_bounds__(kRowThreads * kRowsAtATime)
copy_halves(uint16_t* __restrict__ to, int64_t to_group_stride, int64_t to_stride, int to_columns, const uint16_t* __restrict__ from, int64_t from_group_stride, int64_t from_stride,
            int from_columns, int64_t groups, int to_depth, int from_depth, const unsigned char* end, const int32_t* __restrict__ offsets) {
    const unsigned char* begin = reinterpret_cast<const unsigned char*>(from);
    const int64_t outer = kByColumns ? to_depth : 2 * to_columns;
    for (int64_t row = first_row(); row < groups * outer; row += row_step()) {
        const int64_t g = row / outer;
        const int o = static_cast<int>(row - g * outer);
        uint16_t* q = to + g * to_group_stride + o * to_stride;
        const uint16_t* p = from + g * from_group_stride;
        const bool empty = __ldg(offsets + g + 1) <= __ldg(offsets + g);
        if (empty && !kZeros) continue;
        if constexpr (kByColumns) { // depth o, both halves of its row
            for (int half = 0; half < 2; half++)
                copy_run(q + half * to_columns, to_columns, p + o * from_stride + half * from_columns, o < from_depth && !empty ? from_columns : 0, begin, end);
        } else {
            const int half = o >= to_columns, j = half ? o - to_columns : o;
            copy_run(q, to_depth, p + (half * from_columns + j) * from_stride, j < from_columns && !empty ? from_depth : 0, begin, end);
        }
    }
}
// A and W as the copy engine can fetch them, or copies: rows of A whole packs apart, and of W both halves, with zeros behind the columns of either up to a multiple of 8. `padded`: gradients
// are to be taken, too, whose products go along both halves at once.
struct Boxed {
    const Call& call;
    Packing packing;
    Scratch room;
    GatedProblem p;
    int64_t real_columns; // of a half
    Boxed(const Call& call, const Array& A, const Array& W, const int32_t* offsets, int32_t activation, bool gradients)
        : call(call), packing(call), room(call), p{A, W, offsets, W.shape[0], A.shape[0], A.shape[1], W.shape[2] / 2, activation}, real_columns(W.shape[2] / 2) {
        packing.add(p.A);
        const int64_t columns = real_columns;
        if (columns % 8 != 0 && (gradients || p.by_columns())) {
            const int64_t groups = p.groups, depth = p.depth, wide = (columns + 7) / 8 * 8, deep = (depth + 7) / 8 * 8;
            p.columns = wide;
            p.W = p.by_columns() ? contiguous(nullptr, A.type, groups, depth, 2 * wide) : contiguous(nullptr, A.type, groups, 2 * wide, deep);
            room.take(static_cast<size_t>(values_of(p.W)) * 2);
            p.W.data = room.as<void>();
            if (W.stride[2] != 1) std::swap(p.W.shape[1], p.W.shape[2]), std::swap(p.W.stride[1], p.W.stride[2]);
            move_halves<false>(p.W, wide, W, columns);
            p.W.shape[1] = depth;
        } else {
            packing.add(p.W);
        }
        packing.run();
    }
    // The halves of `from` (of `n` columns each) go where those of `to` (of `m`) are; both are stored the same way round.
    template <bool kZeros> void move_halves(const Array& to, int64_t m, const Array& from, int64_t n) {
        const bool by_columns = from.stride[2] == 1;
        const int64_t rows = to.shape[0] * (by_columns ? to.shape[1] : 2 * m);
        const int64_t outer = by_columns ? from.shape[1] : 2 * n, inner = by_columns ? 2 * n : from.shape[1], stride = by_columns ? from.stride[1] : from.stride[2];
        const unsigned char* end = static_cast<const unsigned char*>(from.data) + ((from.shape[0] - 1) * from.stride[0] + (outer - 1) * stride + inner) * 2;
        auto kernel = by_columns ? copy_halves<true, kZeros> : copy_halves<false, kZeros>;
        kernel<<<row_blocks(call, rows), row_threads(), 0, call.stream>>>(
            static_cast<uint16_t*>(to.data), to.stride[0], by_columns ? to.stride[1] : to.stride[2], static_cast<int>(m), static_cast<const uint16_t*>(from.data),
            from.stride[0], stride, static_cast<int>(n), to.shape[0], static_cast<int>(to.shape[1]), static_cast<int>(from.shape[1]), end, p.offsets);
        MOPS_CUDA_OK(cudaGetLastError());
    }
};

bool sixteen_bits(const Array& A, const Array& W) {
    return (A.type == MOPS_B200_F16 || A.type == MOPS_B200_BF16) && A.shape[0] > 0 && A.shape[1] > 0 && W.shape[0] > 0 && W.shape[2] > 0;
}

// Up to so many values of dU and dV gradients are computed in f32 throughout: the errors of so few, rounded to 16 bits, do not average out. (On average they add to the error of results that are rounded
// themselves as much as that is, 1.4 times in all.)
constexpr int64_t kFewGradients = 2048;

void gradients_16(const Call& call, const Array& grad_A, const Array& grad_W, bool turned, const Array& grad_output, const Array& A, const Array& W, const int32_t* offsets,
                  int32_t activation, const std::string& op) {
    Boxed boxed(call, A, W, offsets, activation, true);
    const GatedProblem& p = boxed.p;
    Scratch room(call, static_cast<size_t>(p.rows * 2 * p.columns) * 2);
    const Array duv = contiguous(room.as<void>(), A.type, p.rows, 2 * p.columns);
    gated_rows_vjp_mma(call, p, duv.data, grad_output, op);
    if (grad_A.data != nullptr)
        multiply_rows(call, {grad_A, duv, p.W, p.W.stride[2], p.W.stride[1], offsets, p.groups, p.rows, 2 * p.columns, p.depth}, op);
    if (grad_W.data == nullptr) return;
    Array to = grad_W;
    Scratch room_W(call);
    const bool padded = p.columns != boxed.real_columns;
    if (padded) { // the products of the columns that there are not, too
        to = turned ? contiguous(nullptr, A.type, p.groups, 2 * p.columns, p.depth) : contiguous(nullptr, A.type, p.groups, p.depth, 2 * p.columns);
        room_W.take(static_cast<size_t>(values_of(to)) * 2);
        to.data = room_W.as<void>();
    }
    if (turned) multiply_outer(call, {to, duv, p.A, offsets, p.groups}, op);
    else multiply_outer(call, {to, p.A, duv, offsets, p.groups}, op);
    if (padded) {
        Array result = grad_W;
        if (turned)
            for (Array* a : {&to, &result}) std::swap(a->shape[1], a->shape[2]), std::swap(a->stride[1], a->stride[2]);
        boxed.move_halves<true>(result, boxed.real_columns, to, p.columns);
    }
}

// f(T(), S()) with T the type and S that of sums
template <typename F> void for_types(int32_t type, F&& f) {
    for_type(type, [&](auto zero) { f(zero, Sum<decltype(zero)>()); });
}

} // namespace

void grouped_gated_product(Array output, Array A, Array W, Array offsets, int32_t activation) {
    const std::string op = "cuda_grouped_gated_product";
    check_gated(A, W, offsets, output, "output", activation, op);
    check_output(output, "output", op);
    if (output.shape[0] == 0 || output.shape[1] == 0) return;
    Call call = begin_call();
    const int32_t* starts = static_cast<const int32_t*>(offsets.data);
    if (sixteen_bits(A, W)) {
        Boxed boxed(call, A, W, starts, activation, false);
        gated_rows_mma(call, boxed.p, output, op);
        end_call(call, op.c_str(), kIndexNames, 1);
        return;
    }
    Widened wide(call, A, W, op);
    if (wide.fused && A.type == MOPS_B200_F32) {
        gated_rows_split(call, wide.problem(starts, activation), output, op);
        end_call(call, op.c_str(), kIndexNames, 1);
        return;
    }
    wide.multiply(starts);
    for_types(A.type, [&](auto zero, auto sum) {
        using T = decltype(zero);
        using S = decltype(sum);
        for_activation(activation, [&](auto f) {
            gate_rows<decltype(f)::value, T, S><<<row_blocks(call, output.shape[0]), row_threads(), 0, call.stream>>>(
                static_cast<T*>(output.data), static_cast<const S*>(wide.uv.data), output.shape[0], output.shape[1]);
        });
        note_kernel_f("gate_rows<%s>", array_type_name<T>());
    });
    MOPS_CUDA_OK(cudaGetLastError());
    end_call(call, op.c_str(), kIndexNames, 1);
}

void grouped_gated_product_vjp(Array grad_A, Array grad_W, Array grad_output, Array A, Array W, Array offsets, int32_t activation) {
    const std::string op = "cuda_grouped_gated_product_vjp";
    check_gated(A, W, offsets, grad_output, "grad_output", activation, op);
    check_rows(grad_output, "grad_output", op);
    const bool need_A = grad_A.data != nullptr, need_W = grad_W.data != nullptr;
    if (need_A) {
        check_array(grad_A, "grad_A", 2, A.type, op);
        for (int d = 0; d < 2; d++) check_size(grad_A.shape[d], "grad_A", d, A.shape[d], "A", d, op);
        check_output(grad_A, "grad_A", op);
    }
    bool turned = false; // grad_W[g] is stored column by column
    if (need_W) {
        check_array(grad_W, "grad_W", 3, A.type, op);
        for (int d = 0; d < 3; d++) check_size(grad_W.shape[d], "grad_W", d, W.shape[d], "W", d, op);
        turned = grad_W.stride[2] != 1;
        if (turned) std::swap(grad_W.shape[1], grad_W.shape[2]), std::swap(grad_W.stride[1], grad_W.stride[2]);
        check_output(grad_W, "grad_W", op);
    }
    if (!need_A && !need_W) return;
    Call call = begin_call();
    const int32_t* starts = static_cast<const int32_t*>(offsets.data);
    const int64_t rows = A.shape[0], columns = W.shape[2];
    if (sixteen_bits(A, W) && rows * columns > kFewGradients) {
        gradients_16(call, grad_A, grad_W, turned, grad_output, A, W, starts, activation, op);
        end_call(call, op.c_str(), kIndexNames, 1);
        return;
    }
    Widened wide(call, A, W, op);
    if (wide.fused) {
        Scratch room(call);
        Array grad = grad_output;
        if (A.type != wide.type) {
            room.take(static_cast<size_t>(values_of(grad)) * 4 + 16);
            grad = converted(call, grad_output, room.as<float>(), wide.type);
        }
        wide.take_uv();
        gated_rows_vjp_split(call, wide.problem(starts, activation), wide.uv, grad, op);
    } else {
        wide.multiply(starts);
    }
    if (!wide.fused && rows > 0 && columns > 0) {
        for_types(A.type, [&](auto zero, auto sum) {
            using T = decltype(zero);
            using S = decltype(sum);
            for_activation(activation, [&](auto f) {
                gate_rows_vjp<decltype(f)::value, T, S><<<row_blocks(call, rows), row_threads(), 0, call.stream>>>(
                    static_cast<S*>(wide.uv.data), static_cast<const T*>(grad_output.data), grad_output.stride[0], rows, columns / 2);
            });
            note_kernel_f("gate_rows_vjp<%s>", array_type_name<T>());
        });
        MOPS_CUDA_OK(cudaGetLastError());
    }
    // as of a plain layer whose output's gradient is dU and dV
    Packing packing(call);
    if (wide.type == MOPS_B200_F32 && rows > 0 && A.shape[1] > 0 && W.shape[0] > 0 && columns > 0) {
        const bool rows_packed = need_A && !straight_rows(wide.W, rows, wide.W.stride[1] == 1);
        const bool outer_packed = need_W && !straight_outer(rows, W.shape[0], W.shape[1], columns, wide.type);
        if (rows_packed || outer_packed) packing.add(wide.uv);
        if (rows_packed) packing.add(wide.W);
        if (outer_packed) packing.add(wide.A);
        packing.run();
    }
    const bool widened = wide.type != A.type;
    Scratch room(call);
    auto result = [&](Array& gradient, auto&& make) { // in the type of the products, and rounded where that is another one
        Array to = gradient;
        if (widened) {
            room.take(static_cast<size_t>(values_of(gradient)) * 4 + 16);
            to.data = room.as<void>();
            to.type = wide.type;
        }
        make(to);
        if (widened)
            for_type(A.type, [&](auto zero) {
                using T = decltype(zero);
                (void)converted(call, to, static_cast<T*>(gradient.data), A.type);
            });
    };
    if (need_A)
        result(grad_A, [&](const Array& to) {
            const RowsProblem problem{to, wide.uv, wide.W, wide.W.stride[2], wide.W.stride[1], starts, W.shape[0], rows, columns, A.shape[1]};
            if (!wide.fused || !multiply_rows_sliced(call, problem, 16, op)) multiply_rows(call, problem, op);
        });
    if (need_W)
        result(grad_W, [&](const Array& to) {
            if (turned) multiply_outer(call, {to, wide.uv, wide.A, starts, W.shape[0]}, op);
            else multiply_outer(call, {to, wide.A, wide.uv, starts, W.shape[0]}, op);
        });
    room.free();
    packing.release();
    end_call(call, op.c_str(), kIndexNames, 1);
}

} // namespace mops_b200
