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
#include <initializer_list>

#include "arrays.hpp"
#include "block_ops.hpp"

namespace mops_b200 {
namespace {

// ---------------------------------------------------------------------------- rows of any length
// A block takes a row after another and reads it as often as it needs it.
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

// ---------------------------------------------------------------- rows that fit into registers
// A team of threads (a warp, or a block) takes one row after another, each thread kPacks packs of N values: kPacks * N values of each
// array. The next row's values are on their way while this one is worked on. Blocks stay for the whole call, so that scales and weights are read
// once and the sums over rows stay in registers until the end.
constexpr int kTeamThreads = 512; // at most

// The sums of K values over the team, for every thread of it. `shared`: two of these are used in turn, so that one barrier does.
template <typename S> struct TeamSums {
    S (*shared)[kTeamThreads / 32][2];
    int warps, turn = 0;
    template <int K> __device__ __forceinline__ void add_up(S (&v)[K]) {
#pragma unroll
        for (int k = 0; k < K; k++) v[k] = warp_sum(v[k]);
        if (warps == 1) return;
        S(*to)[2] = shared[turn];
        turn ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) to[threadIdx.x >> 5][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) v[k] = 0;
        for (int w = 0; w < warps; w++)
#pragma unroll
            for (int k = 0; k < K; k++) v[k] += to[w][k];
    }
};

// A thread's values of a row.
template <typename T, int N, int kPacks> struct Values {
    Pack<T, N> p[kPacks];
    __device__ __forceinline__ Sum<T> operator[](int i) const { return widen(p[i / N].v[i % N]); }
    // `row` begins the row; packs behind the row's end are zeros
    __device__ __forceinline__ void load(const T* __restrict__ row, int member, int team, int packs) {
#pragma unroll
        for (int k = 0; k < kPacks; k++) {
            const int at = k * team + member;
            if (at < packs) p[k] = *reinterpret_cast<const Pack<T, N>*>(row + static_cast<int64_t>(at) * N);
            else
#pragma unroll
                for (int i = 0; i < N; i++) p[k].v[i] = narrow<T>(0);
        }
    }
};
template <int N, int kPacks, typename T>
__device__ __forceinline__ void store_values(T* __restrict__ row, const Sum<T> (&v)[N * kPacks], int member, int team, int packs) {
#pragma unroll
    for (int k = 0; k < kPacks; k++) {
        const int at = k * team + member;
        Pack<T, N> p;
#pragma unroll
        for (int i = 0; i < N; i++) p.v[i] = narrow<T>(v[k * N + i]);
        if (at < packs) *reinterpret_cast<Pack<T, N>*>(row + static_cast<int64_t>(at) * N) = p;
    }
}

// The gate of 16-bit values needs fewer bits than that of f32.
template <typename T> __device__ __forceinline__ Sum<T> gate_value(Sum<T> v) {
    if constexpr (sizeof(T) == 2) return __fdividef(1.0f, 1.0f + __expf(-v));
    else return sigmoid<Sum<T>>(v);
}

template <typename T, int GATE, int N, int kPacks>
__global__ void __launch_bounds__(kTeamThreads)
residual_norm_rows(T* __restrict__ stream, T* __restrict__ normed, const __grid_constant__ Inputs<T> in, int team) {
    using S = Sum<T>;
    constexpr int kValues = N * kPacks;
    using V = Values<T, N, kPacks>;
    __shared__ S shared[2][kTeamThreads / 32][2];
    const int member = threadIdx.x % team, teams = blockDim.x / team, packs = static_cast<int>(in.columns / N);
    const S epsilon = static_cast<S>(in.epsilon), C = static_cast<S>(in.columns);
    TeamSums<S> sums{shared, team / 32};
    V s, w, p;
    s.load(in.scale, member, team, packs);
    w.load(in.weight_branch, member, team, packs);
    p.load(in.weight_output, member, team, packs);
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + threadIdx.x / team;
    V next_x, next_b, next_g;
    T next_gate{};
    auto fetch = [&](int64_t r) {
        if (r >= in.rows) return;
        next_b.load(in.branch + r * in.branch_stride, member, team, packs);
        next_x.load(in.residual + r * in.residual_stride, member, team, packs);
        if constexpr (GATE == kFullGate) next_g.load(in.gate + r * in.gate_stride, member, team, packs);
        if constexpr (GATE == kRowGate) next_gate = in.gate[r * in.gate_stride];
    };
    fetch(row);
    for (; row < in.rows; row += step) { // (all teams of a block of several are warps, which do not wait for one another)
        const V x = next_x, b = next_b, g = next_g;
        const T gate = next_gate;
        fetch(row + step);
        S sum[1] = {0};
#pragma unroll
        for (int i = 0; i < kValues; i++) sum[0] += b[i] * b[i];
        sums.add_up(sum);
        const S q = inverse_root<S>(sum[0] / C + epsilon);
        const S z_row = GATE == kRowGate ? gate_value<T>(widen(gate)) : S(1);
        S y[kValues];
        sum[0] = 0;
#pragma unroll
        for (int i = 0; i < kValues; i++) {
            const S z = GATE == kFullGate ? gate_value<T>(g[i]) : z_row;
            y[i] = x[i] + s[i] * w[i] * z * (b[i] * q);
            sum[0] += y[i] * y[i];
        }
        store_values<N, kPacks>(stream + row * in.columns, y, member, team, packs);
        sums.add_up(sum);
        const S r = inverse_root<S>(sum[0] / C + epsilon);
#pragma unroll
        for (int i = 0; i < kValues; i++) y[i] = p[i] * y[i] * r;
        store_values<N, kPacks>(normed + row * in.columns, y, member, team, packs);
    }
}

template <typename T, int GATE, int N, int kPacks>
__global__ void __launch_bounds__(kTeamThreads)
residual_norm_vjp_rows(const __grid_constant__ Gradients<T> grad, const __grid_constant__ Inputs<T> in, int team) {
    using S = Sum<T>;
    constexpr int kValues = N * kPacks;
    using V = Values<T, N, kPacks>;
    __shared__ S shared[2][kTeamThreads / 32][2];
    const int member = threadIdx.x % team, teams = blockDim.x / team, packs = static_cast<int>(in.columns / N);
    const S epsilon = static_cast<S>(in.epsilon), C = static_cast<S>(in.columns);
    TeamSums<S> sums{shared, team / 32};
    V s, w, p;
    s.load(in.scale, member, team, packs);
    w.load(in.weight_branch, member, team, packs);
    p.load(in.weight_output, member, team, packs);
    S of_branch[kValues], of_output[kValues]; // sums over the team's rows
#pragma unroll
    for (int i = 0; i < kValues; i++) of_branch[i] = of_output[i] = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + threadIdx.x / team;
    V next_x, next_b, next_g, next_gs, next_gh;
    T next_gate{};
    auto fetch = [&](int64_t r) {
        if (r >= in.rows) return;
        next_b.load(in.branch + r * in.branch_stride, member, team, packs);
        next_x.load(in.residual + r * in.residual_stride, member, team, packs);
        if constexpr (GATE == kFullGate) next_g.load(in.gate + r * in.gate_stride, member, team, packs);
        if constexpr (GATE == kRowGate) next_gate = in.gate[r * in.gate_stride];
        next_gh.load(grad.normed + r * grad.normed_stride, member, team, packs);
        next_gs.load(grad.stream + r * grad.stream_stride, member, team, packs);
    };
    fetch(row);
    for (; row < in.rows; row += step) {
        const V x = next_x, b = next_b, g = next_g, gs = next_gs, gh = next_gh;
        const T gate = next_gate;
        fetch(row + step);
        S sum[2] = {0, 0};
        S one[1] = {0};
#pragma unroll
        for (int i = 0; i < kValues; i++) one[0] += b[i] * b[i];
        sums.add_up(one);
        const S q = inverse_root<S>(one[0] / C + epsilon);
        const S z_row = GATE == kRowGate ? gate_value<T>(widen(gate)) : S(1);
        S z[kValues], y[kValues];
#pragma unroll
        for (int i = 0; i < kValues; i++) {
            z[i] = GATE == kFullGate ? gate_value<T>(g[i]) : z_row;
            y[i] = x[i] + s[i] * w[i] * z[i] * (b[i] * q);
            sum[0] += y[i] * y[i];
            sum[1] += p[i] * gh[i] * y[i];
        }
        sums.add_up(sum);
        const S r = inverse_root<S>(sum[0] / C + epsilon), back = sum[1] * r * r * r / C;
        sum[0] = sum[1] = 0;
#pragma unroll
        for (int i = 0; i < kValues; i++) {
            const S zn = z[i] * (b[i] * q);
            of_output[i] += gh[i] * y[i] * r;
            y[i] = gs[i] + r * (p[i] * gh[i]) - y[i] * back; // from here on the stream's gradient
            of_branch[i] += y[i] * zn;
            const S full = y[i] * s[i] * w[i] * zn;
            sum[0] += full;
            if constexpr (GATE == kRowGate) sum[1] += full * (1 - z[i]);
        }
        if (grad.residual != nullptr) store_values<N, kPacks>(grad.residual + row * in.columns, y, member, team, packs);
        if constexpr (GATE == kFullGate)
            if (grad.gate != nullptr) {
                S v[kValues];
#pragma unroll
                for (int i = 0; i < kValues; i++) v[i] = y[i] * s[i] * w[i] * z[i] * (b[i] * q) * (1 - z[i]);
                store_values<N, kPacks>(grad.gate + row * in.columns, v, member, team, packs);
            }
        if constexpr (GATE == kRowGate) {
            sums.add_up(sum);
            if (grad.gate != nullptr && member == 0) grad.gate[row] = narrow<T>(sum[1]);
        } else {
            one[0] = sum[0];
            sums.add_up(one);
            sum[0] = one[0];
        }
        const S mean = sum[0] / C;
#pragma unroll
        for (int i = 0; i < kValues; i++) y[i] = q * (y[i] * s[i] * w[i] * z[i] - b[i] * q * mean);
        if (grad.branch != nullptr) store_values<N, kPacks>(grad.branch + row * in.columns, y, member, team, packs);
    }
    if (grad.columns == nullptr) return;
    // the teams of a block add to its sums one after the other
    S* own = grad.columns + static_cast<int64_t>(blockIdx.x) * 2 * in.columns;
    for (int t = 0; t < teams; t++) {
        if (t > 0) __syncthreads();
        if (static_cast<int>(threadIdx.x) / team != t) continue;
#pragma unroll
        for (int i = 0; i < kValues; i++) {
            const int pack = i / N * team + member;
            if (pack >= packs) continue;
            const int64_t c = static_cast<int64_t>(pack) * N + i % N;
            own[c] = (t > 0 ? own[c] : S(0)) + of_branch[i];
            own[in.columns + c] = (t > 0 ? own[in.columns + c] : S(0)) + of_output[i];
        }
    }
}

// The sums over rows from those of the blocks: 32 warps add up a range of blocks each, for 32 columns, then those.
constexpr int kColumnThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kColumnThreads)
residual_norm_columns(T* __restrict__ grad_scale, T* __restrict__ grad_weight_branch, T* __restrict__ grad_weight_output,
                      const T* __restrict__ scale, const T* __restrict__ weight_branch, const Sum<T>* __restrict__ sums,
                      int64_t blocks, int64_t columns) {
    using S = Sum<T>;
    __shared__ S shared[kColumnThreads / 32][2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    S sum[2] = {0, 0};
    if (c < columns) {
#pragma unroll 4
        for (int64_t b = warp; b < blocks; b += kColumnThreads / 32) {
            sum[0] += sums[2 * b * columns + c];
            sum[1] += sums[(2 * b + 1) * columns + c];
        }
    }
    shared[warp][0][lane] = sum[0];
    shared[warp][1][lane] = sum[1];
    __syncthreads();
    if (warp != 0 || c >= columns) return;
    sum[0] = sum[1] = 0;
#pragma unroll
    for (int v = 0; v < kColumnThreads / 32; v++) sum[0] += shared[v][0][lane], sum[1] += shared[v][1][lane];
    if (grad_scale != nullptr) grad_scale[c] = narrow<T>(widen(weight_branch[c]) * sum[0]);
    if (grad_weight_branch != nullptr) grad_weight_branch[c] = narrow<T>(widen(scale[c]) * sum[0]);
    if (grad_weight_output != nullptr) grad_weight_output[c] = narrow<T>(sum[1]);
}

// How a call's rows are shared out: threads to a row, and to a block. threads == 0: rows are too long for the registers of a block.
struct Teams {
    int team, threads;
    int64_t blocks(int64_t rows, int resident) const {
        return std::min<int64_t>(ceil_div(rows, threads / team), resident);
    }
};
inline Teams teams_of(int64_t columns, int values) {
    const int64_t needed = ceil_div(columns, values);
    if (needed > kTeamThreads) return {0, 0};
    if (needed <= 32) return {32, 256};
    const int team = static_cast<int>(ceil_div(needed, 32) * 32);
    return {team, team};
}
// Values of a thread, in 16-byte packs or one by one: eight of them (f64: four), or twice as many for long rows.
template <typename T> constexpr int kFewValues = sizeof(T) == 8 ? 4 : 8;

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

bool all_aligned(std::initializer_list<const Array*> arrays) {
    for (const Array* a : arrays)
        if (!aligned16(*a)) return false;
    return true;
}

// Calls f(values of a pack, values of a thread) for the widths that a row may fit, until it says that it did.
template <typename T, typename F> bool by_values(bool whole, F&& f) {
    constexpr int few = kFewValues<T>;
    if (whole)
        return f(std::integral_constant<int, kPack<T>>(), std::integral_constant<int, few>()) ||
               f(std::integral_constant<int, kPack<T>>(), std::integral_constant<int, 2 * few>());
    return f(std::integral_constant<int, 1>(), std::integral_constant<int, few>()) ||
           f(std::integral_constant<int, 1>(), std::integral_constant<int, 2 * few>());
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
            const auto in = inputs_of<T>(residual, branch, gate, scale, weight_branch, weight_output, epsilon);
            auto in_registers = [&](auto width, auto count) {
                constexpr int N = decltype(width)::value, kPacks = decltype(count)::value / N;
                const Teams t = teams_of(in.columns, N * kPacks);
                if (t.threads == 0) return false;
                auto kernel = residual_norm_rows<T, GATE, N, kPacks>;
                const int resident = resident_blocks(kernel, call.device, t.threads, 0) * sm_count(call.device);
                kernel<<<static_cast<unsigned>(t.blocks(in.rows, resident)), t.threads, 0, call.stream>>>(
                    static_cast<T*>(stream.data), static_cast<T*>(normed.data), in, t.team);
                note_kernel_f("residual_norm_rows<%s,%d,%d,%d>", array_type_name<T>(), GATE, N, kPacks);
                return true;
            };
            const bool whole = all_aligned({&stream, &normed, &residual, &branch, &scale, &weight_branch, &weight_output}) &&
                               (GATE != kFullGate || aligned16(gate));
            if (by_values<T>(whole, in_registers)) return;
            const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(residual.shape[0], int64_t(sm_count(call.device)) * 8));
            residual_norm_plain<T, GATE><<<blocks, kThreads, 0, call.stream>>>(
                static_cast<T*>(stream.data), static_cast<T*>(normed.data), in);
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
        const bool of_columns = grad_scale.data != nullptr || grad_weight_branch.data != nullptr || grad_weight_output.data != nullptr;
        int64_t blocks = 0;
        Sum<T>* sums = nullptr;
        auto room = [&](int64_t for_blocks) {
            blocks = for_blocks;
            sums = static_cast<Sum<T>*>(scratch_alloc(call, static_cast<size_t>(2 * blocks * columns) * sizeof(Sum<T>)));
            return Gradients<T>{data(grad_residual), data(grad_branch), data(grad_gate), data(grad_stream), data(grad_normed),
                                grad_stream.stride[0], grad_normed.stride[0], sums};
        };
        for_gate(kind, [&](auto g) {
            constexpr int GATE = decltype(g)::value;
            if (rows == 0) return;
            const auto in = inputs_of<T>(residual, branch, gate, scale, weight_branch, weight_output, epsilon);
            auto in_registers = [&](auto width, auto count) {
                constexpr int N = decltype(width)::value, kPacks = decltype(count)::value / N;
                const Teams t = teams_of(columns, N * kPacks);
                if (t.threads == 0) return false;
                auto kernel = residual_norm_vjp_rows<T, GATE, N, kPacks>;
                const int resident = resident_blocks(kernel, call.device, t.threads, 0) * sm_count(call.device);
                const Gradients<T> grad = room(t.blocks(rows, resident));
                kernel<<<static_cast<unsigned>(blocks), t.threads, 0, call.stream>>>(grad, in, t.team);
                note_kernel_f("residual_norm_vjp_rows<%s,%d,%d,%d>", array_type_name<T>(), GATE, N, kPacks);
                return true;
            };
            const bool whole = all_aligned({&grad_residual, &grad_branch, &grad_stream, &grad_normed, &residual, &branch, &scale,
                                            &weight_branch, &weight_output}) &&
                               (GATE != kFullGate || (aligned16(gate) && aligned16(grad_gate)));
            if (by_values<T>(whole, in_registers)) return;
            const Gradients<T> grad = room(std::min<int64_t>(rows, int64_t(sm_count(call.device)) * 4));
            residual_norm_vjp_plain<T, GATE><<<static_cast<unsigned>(blocks), kThreads, 0, call.stream>>>(grad, in);
            note_kernel_f("residual_norm_vjp_plain<%s,%d>", array_type_name<T>(), GATE);
        });
        MOPS_CUDA_OK(cudaGetLastError());
        if (of_columns)
            residual_norm_columns<T><<<static_cast<unsigned>(ceil_div(columns, 32)), kColumnThreads, 0, call.stream>>>(
                data(grad_scale), data(grad_weight_branch), data(grad_weight_output), data(scale), data(weight_branch), sums,
                blocks, columns);
        if (sums != nullptr) scratch_free(call, sums);
    });
    end_call(call, op.c_str(), nullptr, 0);
}

} // namespace mops_b200
