// gated_residual_norm: the residual connection around a block, with the norm behind the block, its gate and scale, and the
// norm in front of the next block, in one pass over a row. With z = sigmoid(gate) (1 without a gate), q = 1 / rms(branch),
// n = q branch and r = 1 / rms(stream), rms(v)^2 = mean(v^2) + epsilon:
//
//   stream = residual + scale weight_branch z n,    normed = weight_output r stream
//
// and, with the gradients gs of stream and gh of normed, C columns:
//
//   ds = gs + r weight_output gh - stream r^3 / C sum(weight_output gh stream)     (over the row)
//   grad_residual = ds
//   grad_gate = ds scale weight_branch n z (1 - z)                                 (summed over the row for a gate per row)
//   dn = ds scale weight_branch z,    grad_branch = q (dn - n mean(dn n))
//   P = sum over rows of ds z n,    grad_scale = weight_branch P,    grad_weight_branch = scale P
//   grad_weight_output = sum over rows of gh stream r
//
// The backward pass computes the stream again from the inputs: it reads as many bytes as the stream has, and has it before it was
// rounded.
#include "arrays.hpp"
#include "block_ops.hpp"

namespace mops_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

enum Gate : int { kNoGate = 0, kRowGate = 1, kFullGate = 2 };

template <typename S> __device__ __forceinline__ S sigmoid(S v) { return S(1) / (S(1) + exp(-v)); }
template <> __device__ __forceinline__ float sigmoid<float>(float v) { return 1.0f / (1.0f + expf(-v)); }
template <typename S> __device__ __forceinline__ S inverse_root(S v) { return S(1) / sqrt(v); }

// The sums of K values over the block, for every thread.
template <int K, typename S> __device__ __forceinline__ void block_sums(S (&v)[K], S (*shared)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = warp_sum(v[k]);
    __syncthreads(); // (the previous sums have been read)
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; k++) shared[warp][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        v[k] = 0;
        for (int w = 0; w < kWarps; w++) v[k] += shared[w][k];
    }
}

template <typename T> struct Inputs {
    const T *residual, *branch, *gate, *scale, *weight_branch, *weight_output;
    int64_t residual_stride, branch_stride, gate_stride;
    int64_t rows, columns;
    double epsilon;
};

template <typename T, int GATE> __device__ __forceinline__ Sum<T> gate_of(const Inputs<T>& in, int64_t row, int64_t c) {
    if constexpr (GATE == kNoGate) return 1;
    else return sigmoid<Sum<T>>(widen(in.gate[row * in.gate_stride + (GATE == kFullGate ? c : 0)]));
}

template <typename T, int GATE>
__global__ void __launch_bounds__(kThreads)
residual_norm_plain(T* __restrict__ stream, T* __restrict__ normed, Inputs<T> in) {
    using S = Sum<T>;
    __shared__ S shared[kWarps][1];
    const S epsilon = static_cast<S>(in.epsilon);
    for (int64_t row = blockIdx.x; row < in.rows; row += gridDim.x) {
        const T *x = in.residual + row * in.residual_stride, *b = in.branch + row * in.branch_stride;
        S sum[1] = {0};
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) sum[0] += widen(b[c]) * widen(b[c]);
        block_sums(sum, shared);
        const S q = inverse_root<S>(sum[0] / static_cast<S>(in.columns) + epsilon);
        auto value = [&](int64_t c) {
            return widen(x[c]) +
                   widen(in.scale[c]) * widen(in.weight_branch[c]) * gate_of<T, GATE>(in, row, c) * (widen(b[c]) * q);
        };
        sum[0] = 0;
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) {
            const S y = value(c);
            sum[0] += y * y;
            stream[row * in.columns + c] = narrow<T>(y);
        }
        block_sums(sum, shared);
        const S r = inverse_root<S>(sum[0] / static_cast<S>(in.columns) + epsilon);
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads)
            normed[row * in.columns + c] = narrow<T>(widen(in.weight_output[c]) * value(c) * r);
    }
}

template <typename T> struct Gradients {
    T *residual, *branch, *gate;     // nullptr: not asked for
    const T *stream, *normed;        // of the outputs
    int64_t stream_stride, normed_stride;
    Sum<T>* columns;                 // [blocks][2][columns]: sums over a block's rows of ds z n and of gh stream r
};

template <typename T, int GATE>
__global__ void __launch_bounds__(kThreads)
residual_norm_vjp_plain(Gradients<T> g, Inputs<T> in) {
    using S = Sum<T>;
    __shared__ S shared[kWarps][2];
    const S epsilon = static_cast<S>(in.epsilon), C = static_cast<S>(in.columns);
    S* own = g.columns + static_cast<int64_t>(blockIdx.x) * 2 * in.columns;
    for (int64_t c = threadIdx.x; c < 2 * in.columns; c += kThreads) own[c] = 0;
    __syncthreads();
    for (int64_t row = blockIdx.x; row < in.rows; row += gridDim.x) {
        const T *x = in.residual + row * in.residual_stride, *b = in.branch + row * in.branch_stride;
        const T *gs = g.stream + row * g.stream_stride, *gh = g.normed + row * g.normed_stride;
        S sum[2] = {0, 0};
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) sum[0] += widen(b[c]) * widen(b[c]);
        block_sums(sum, shared);
        const S q = inverse_root<S>(sum[0] / C + epsilon);
        auto stream = [&](int64_t c, S z) {
            return widen(x[c]) + widen(in.scale[c]) * widen(in.weight_branch[c]) * z * (widen(b[c]) * q);
        };
        sum[0] = sum[1] = 0;
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) {
            const S y = stream(c, gate_of<T, GATE>(in, row, c));
            sum[0] += y * y;
            sum[1] += widen(in.weight_output[c]) * widen(gh[c]) * y;
        }
        block_sums(sum, shared);
        const S r = inverse_root<S>(sum[0] / C + epsilon), back = sum[1] * r * r * r / C;
        auto ds_of = [&](int64_t c, S y) { return widen(gs[c]) + r * widen(in.weight_output[c]) * widen(gh[c]) - y * back; };
        sum[0] = sum[1] = 0;
        for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) {
            const S z = gate_of<T, GATE>(in, row, c), y = stream(c, z), ds = ds_of(c, y), n = widen(b[c]) * q;
            const S full = ds * widen(in.scale[c]) * widen(in.weight_branch[c]) * n;
            sum[0] += full * z;
            if (g.residual != nullptr) g.residual[row * in.columns + c] = narrow<T>(ds);
            if constexpr (GATE == kFullGate)
                if (g.gate != nullptr) g.gate[row * in.columns + c] = narrow<T>(full * z * (1 - z));
            if constexpr (GATE == kRowGate) sum[1] += full * z * (1 - z);
            own[c] += ds * z * n;
            own[in.columns + c] += widen(gh[c]) * y * r;
        }
        block_sums(sum, shared);
        if constexpr (GATE == kRowGate)
            if (g.gate != nullptr && threadIdx.x == 0) g.gate[row] = narrow<T>(sum[1]);
        const S mean = sum[0] / C;
        if (g.branch != nullptr)
            for (int64_t c = threadIdx.x; c < in.columns; c += kThreads) {
                const S z = gate_of<T, GATE>(in, row, c), y = stream(c, z), ds = ds_of(c, y), n = widen(b[c]) * q;
                const S dn = ds * widen(in.scale[c]) * widen(in.weight_branch[c]) * z;
                g.branch[row * in.columns + c] = narrow<T>(q * (dn - n * mean));
            }
    }
}

// The sums over rows from those of the blocks: a warp for 32 columns... a block adds up kWarps ranges of blocks, then those.
template <typename T>
__global__ void __launch_bounds__(kThreads)
residual_norm_columns(T* __restrict__ grad_scale, T* __restrict__ grad_weight_branch, T* __restrict__ grad_weight_output,
                      const T* __restrict__ scale, const T* __restrict__ weight_branch, const Sum<T>* __restrict__ sums,
                      int64_t blocks, int64_t columns) {
    using S = Sum<T>;
    __shared__ S shared[kWarps][2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    S sum[2] = {0, 0};
    if (c < columns)
        for (int64_t b = warp; b < blocks; b += kWarps) {
            sum[0] += sums[2 * b * columns + c];
            sum[1] += sums[(2 * b + 1) * columns + c];
        }
    shared[warp][0][lane] = sum[0];
    shared[warp][1][lane] = sum[1];
    __syncthreads();
    if (warp != 0 || c >= columns) return;
    sum[0] = sum[1] = 0;
    for (int w = 0; w < kWarps; w++) sum[0] += shared[w][0][lane], sum[1] += shared[w][1][lane];
    if (grad_scale != nullptr) grad_scale[c] = narrow<T>(widen(weight_branch[c]) * sum[0]);
    if (grad_weight_branch != nullptr) grad_weight_branch[c] = narrow<T>(widen(scale[c]) * sum[0]);
    if (grad_weight_output != nullptr) grad_weight_output[c] = narrow<T>(sum[1]);
}

// Checks the inputs; returns which gate there is.
Gate check_inputs(Array& residual, Array& branch, Array& gate, Array& scale, Array& weight_branch, Array& weight_output,
                  double epsilon, const std::string& op) {
    check_floating(residual.type, "residual", op);
    const int32_t type = residual.type;
    check_array(residual, "residual", 2, type, op);
    check_array(branch, "branch", 2, type, op);
    for (int d = 0; d < 2; d++) check_size(branch.shape[d], "branch", d, residual.shape[d], "residual", d, op);
    check_rows(residual, "residual", op);
    check_rows(branch, "branch", op);
    const struct { Array& a; const char* name; } vectors[] = {
        {scale, "scale"}, {weight_branch, "weight_branch"}, {weight_output, "weight_output"}};
    for (const auto& v : vectors) {
        check_array(v.a, v.name, 1, type, op);
        check_size(v.a.shape[0], v.name, 0, residual.shape[1], "residual", 1, op);
        check_rows(v.a, v.name, op);
    }
    fits_int32(static_cast<size_t>(residual.shape[0]), "residual.shape[0]", op);
    fits_int32(static_cast<size_t>(residual.shape[1]), "residual.shape[1]", op);
    if (!(epsilon >= 0)) throw std::runtime_error("epsilon must not be negative in " + op);
    if (gate.dimensions == 0) return kNoGate;
    check_array(gate, "gate", 2, type, op);
    check_size(gate.shape[0], "gate", 0, residual.shape[0], "residual", 0, op);
    check_rows(gate, "gate", op);
    if (gate.shape[1] == residual.shape[1]) return kFullGate;
    if (gate.shape[1] != 1)
        throw std::runtime_error("gate must have as many columns as residual, or one, in " + op);
    return kRowGate;
}

template <typename T>
Inputs<T> inputs_of(const Array& residual, const Array& branch, const Array& gate, const Array& scale, const Array& weight_branch,
                    const Array& weight_output, double epsilon) {
    auto data = [](const Array& a) { return static_cast<const T*>(a.data); };
    return {data(residual), data(branch), data(gate), data(scale), data(weight_branch), data(weight_output),
            residual.stride[0], branch.stride[0], gate.stride[0], residual.shape[0], residual.shape[1], epsilon};
}

template <typename F> void for_gate(Gate gate, F&& f) {
    if (gate == kNoGate) f(std::integral_constant<int, kNoGate>());
    else if (gate == kRowGate) f(std::integral_constant<int, kRowGate>());
    else f(std::integral_constant<int, kFullGate>());
}

} // namespace

void gated_residual_norm(Array stream, Array normed, Array residual, Array branch, Array gate, Array scale,
                         Array weight_branch, Array weight_output, double epsilon) {
    const std::string op = "cuda_gated_residual_norm";
    const Gate kind = check_inputs(residual, branch, gate, scale, weight_branch, weight_output, epsilon, op);
    const struct { Array& a; const char* name; } outputs[] = {{stream, "stream"}, {normed, "normed"}};
    for (const auto& o : outputs) {
        check_array(o.a, o.name, 2, residual.type, op);
        for (int d = 0; d < 2; d++) check_size(o.a.shape[d], o.name, d, residual.shape[d], "residual", d, op);
        check_output(o.a, o.name, op);
    }
    if (residual.shape[0] == 0 || residual.shape[1] == 0) return;
    Call call = begin_call();
    for_type(residual.type, [&](auto zero) {
        using T = decltype(zero);
        for_gate(kind, [&](auto g) {
            constexpr int GATE = decltype(g)::value;
            const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(residual.shape[0], int64_t(sm_count(call.device)) * 8));
            residual_norm_plain<T, GATE><<<blocks, kThreads, 0, call.stream>>>(
                static_cast<T*>(stream.data), static_cast<T*>(normed.data),
                inputs_of<T>(residual, branch, gate, scale, weight_branch, weight_output, epsilon));
            note_kernel_f("residual_norm_plain<%s,%d>", array_type_name<T>(), GATE);
        });
    });
    end_call(call, op.c_str(), nullptr, 0);
}

void gated_residual_norm_vjp(Array grad_residual, Array grad_branch, Array grad_gate, Array grad_scale,
                             Array grad_weight_branch, Array grad_weight_output, Array grad_stream, Array grad_normed,
                             Array residual, Array branch, Array gate, Array scale, Array weight_branch,
                             Array weight_output, double epsilon) {
    const std::string op = "cuda_gated_residual_norm_vjp";
    const Gate kind = check_inputs(residual, branch, gate, scale, weight_branch, weight_output, epsilon, op);
    const struct { Array& a; const char* name; } given[] = {{grad_stream, "grad_stream"}, {grad_normed, "grad_normed"}};
    for (const auto& o : given) {
        check_array(o.a, o.name, 2, residual.type, op);
        for (int d = 0; d < 2; d++) check_size(o.a.shape[d], o.name, d, residual.shape[d], "residual", d, op);
        check_rows(o.a, o.name, op);
    }
    if (kind == kNoGate && grad_gate.data != nullptr)
        throw std::runtime_error("there is no gate to compute grad_gate for in " + op);
    const struct { Array& a; const char* name; const Array& like; const char* like_name; } outputs[] = {
        {grad_residual, "grad_residual", residual, "residual"}, {grad_branch, "grad_branch", branch, "branch"},
        {grad_gate, "grad_gate", gate, "gate"}, {grad_scale, "grad_scale", scale, "scale"},
        {grad_weight_branch, "grad_weight_branch", weight_branch, "weight_branch"},
        {grad_weight_output, "grad_weight_output", weight_output, "weight_output"}};
    for (const auto& o : outputs) {
        if (o.a.data == nullptr) continue;
        check_array(o.a, o.name, o.like.dimensions, residual.type, op);
        for (int d = 0; d < o.like.dimensions; d++) check_size(o.a.shape[d], o.name, d, o.like.shape[d], o.like_name, d, op);
        check_output(o.a, o.name, op);
    }
    const int64_t rows = residual.shape[0], columns = residual.shape[1];
    if (columns == 0 && (rows == 0 || grad_gate.data == nullptr)) return;
    Call call = begin_call();
    if (columns == 0) { // nothing goes through the gates
        MOPS_CUDA_OK(cudaMemsetAsync(grad_gate.data, 0, static_cast<size_t>(rows * grad_gate.shape[1] * type_bytes(grad_gate.type)),
                                     call.stream));
        return end_call(call, op.c_str(), nullptr, 0);
    }
    for_type(residual.type, [&](auto zero) {
        using T = decltype(zero);
        auto data = [](const Array& a) { return static_cast<T*>(a.data); };
        const int64_t blocks = std::min<int64_t>(rows, int64_t(sm_count(call.device)) * 4);
        Sum<T>* sums = static_cast<Sum<T>*>(scratch_alloc(call, static_cast<size_t>(2 * blocks * columns) * sizeof(Sum<T>)));
        for_gate(kind, [&](auto g) {
            constexpr int GATE = decltype(g)::value;
            if (rows > 0)
                residual_norm_vjp_plain<T, GATE><<<static_cast<unsigned>(blocks), kThreads, 0, call.stream>>>(
                    Gradients<T>{data(grad_residual), data(grad_branch), data(grad_gate), data(grad_stream), data(grad_normed),
                                 grad_stream.stride[0], grad_normed.stride[0], sums},
                    inputs_of<T>(residual, branch, gate, scale, weight_branch, weight_output, epsilon));
            note_kernel_f("residual_norm_vjp_plain<%s,%d>", array_type_name<T>(), GATE);
        });
        if (grad_scale.data != nullptr || grad_weight_branch.data != nullptr || grad_weight_output.data != nullptr)
            residual_norm_columns<T><<<static_cast<unsigned>(ceil_div(columns, 32)), kThreads, 0, call.stream>>>(
                data(grad_scale), data(grad_weight_branch), data(grad_weight_output), data(scale), data(weight_branch), sums,
                blocks, columns);
        scratch_free(call, sums);
    });
    end_call(call, op.c_str(), nullptr, 0);
}

} // namespace mops_b200
