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
#include "bulk.cuh"
#include "pairs.cuh"

namespace mops_b200 {
namespace {

// ---------------------------------------------------------------------------- rows of any length
// A block takes a row after another and reads it as often as it needs it. 500 rows of 100 000 columns in bf16: 880 us, backward 1.94 ms; bounded by the latency of
// one load after the other.
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

enum Gate : int { kNoGate = 0, kRowGate = 1, kFullGate = 2 };

__device__ __forceinline__ float exponential(float v) { return expf(v); }
__device__ __forceinline__ double exponential(double v) { return exp(v); }

// z = sigmoid(v) = 1 / (1 + e) with e = exp(-v), and 1 - z as e z: 1 - z itself would be what z was rounded by for large v (in f32 nothing is left of it from v = 17 on).
// Where e is infinite z is 0, and so is everything that 1 - z is multiplied with.
__device__ __forceinline__ float complement(float e, float z) { return fminf(e, 3.402823466e38f) * z; }
__device__ __forceinline__ double complement(double e, double z) {
    return __hiloint2double(min(__double2hiint(e), 0x7fefffff), __double2loint(e)) * z; // (the largest finite power of e: e is not negative)
}
template <typename S> __device__ __forceinline__ S sigmoid(S v, S& one_minus) {
    const S e = exponential(-v), z = S(1) / (S(1) + e);
    one_minus = complement(e, z);
    return z;
}
template <typename S> __device__ __forceinline__ S inverse_root(S v) { return S(1) / sqrt(v); }
template <> __device__ __forceinline__ float inverse_root<float>(float v) { return rsqrtf(v); }

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

template <typename T, int GATE> __device__ __forceinline__ Sum<T> gate_of(const Inputs<T>& in, int64_t row, int64_t c, Sum<T>& one_minus) {
    if constexpr (GATE == kNoGate) return one_minus = 0, Sum<T>(1);
    else return sigmoid<Sum<T>>(widen(in.gate[row * in.gate_stride + (GATE == kFullGate ? c : 0)]), one_minus);
}
template <typename T, int GATE> __device__ __forceinline__ Sum<T> gate_of(const Inputs<T>& in, int64_t row, int64_t c) {
    Sum<T> one_minus;
    return gate_of<T, GATE>(in, row, c, one_minus);
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
            S one_minus;
            const S z = gate_of<T, GATE>(in, row, c, one_minus), y = stream(c, z), ds = ds_of(c, y), n = widen(b[c]) * q;
            const S full = ds * widen(in.scale[c]) * widen(in.weight_branch[c]) * n;
            sum[0] += full * z;
            if (g.residual != nullptr) g.residual[row * in.columns + c] = narrow<T>(ds);
            if constexpr (GATE == kFullGate)
                if (g.gate != nullptr) g.gate[row * in.columns + c] = narrow<T>(full * z * one_minus);
            if constexpr (GATE == kRowGate) sum[1] += full * z * one_minus;
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
// once and the sums over rows stay in registers until the end. Where rows are not whole packs: 20 000 rows of 250 columns in f32 23.8 us (4.2 TB/s), backward 59 us.
constexpr int kTeamThreads = 512; // at most (so a thread has 128 registers)
// Values of a thread, in 16-byte packs or one by one: eight of them (f64: four), or twice as many for long rows.
template <typename T> constexpr int kFewValues = sizeof(T) == 8 ? 4 : 8;

// Sums over the team, of one value or of two, for every thread of it. The warps' sums go through shared memory, in two places that are used in
// turn, so that one barrier does. Two values are added up together: half of the lanes for each.
template <typename S> struct TeamSums {
    static constexpr int kMost = kTeamThreads / 32; // warps
    static_assert(kMost == 16, "half a warp adds up the warps' sums");
    struct Place {
        S of_warp[2 * kMost]; // of the first value, then of the second
    };
    Place* places;
    bool one_warp;
    int turn = 0;
    __device__ TeamSums(Place (&shared)[2], int team) : places(shared), one_warp(team == 32) {
        if (one_warp) return;
        for (int i = threadIdx.x; i < 4 * kMost; i += blockDim.x) shared[i / (2 * kMost)].of_warp[i % (2 * kMost)] = 0; // (of warps that there are none of)
        __syncthreads();
    }
    __device__ __forceinline__ static S half_sum(S v) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
        return v;
    }
    __device__ __forceinline__ void add_up(S& a) {
        a = warp_sum(a);
        if (one_warp) return;
        Place& place = places[turn];
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) place.of_warp[threadIdx.x >> 5] = a;
        __syncthreads();
        a = half_sum(place.of_warp[threadIdx.x & (kMost - 1)]);
    }
    __device__ __forceinline__ void add_up(S& a, S& b) {
        const bool upper = threadIdx.x & 16;
        S v = half_sum((upper ? b : a) + __shfl_xor_sync(kFullMask, upper ? a : b, 16));
        if (!one_warp) {
            Place& place = places[turn];
            turn ^= 1;
            if ((threadIdx.x & 15) == 0) place.of_warp[(upper ? kMost : 0) + (threadIdx.x >> 5)] = v;
            __syncthreads();
            v = half_sum(place.of_warp[threadIdx.x & 31]);
        }
        const S other = __shfl_xor_sync(kFullMask, v, 16);
        a = upper ? other : v;
        b = upper ? v : other;
    }
};

// A thread's values of a row, kPacks packs of N; where a pack lies behind the row's end, zeros (which stay in `p` from one row to the next).
template <typename T, int N, int kPacks> struct alignas(16) Values {
    static constexpr int kPairs = N * kPacks / 2;
    T v[N * kPacks];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N * kPacks; i++) v[i] = narrow<T>(0);
    }
    // first: the thread's first pack of the row
    __device__ __forceinline__ void load(const T* __restrict__ first, int member, int team, int packs) {
#pragma unroll
        for (int k = 0; k < kPacks; k++)
            if (k * team + member < packs)
                *reinterpret_cast<Pack<T, N>*>(&v[k * N]) = *reinterpret_cast<const Pack<T, N>*>(first + k * team * N);
    }
    __device__ __forceinline__ void store(T* __restrict__ first, int member, int team, int packs) const {
#pragma unroll
        for (int k = 0; k < kPacks; k++)
            if (k * team + member < packs)
                *reinterpret_cast<Pack<T, N>*>(first + k * team * N) = *reinterpret_cast<const Pack<T, N>*>(&v[k * N]);
    }
    // What is computed from the values behind this is computed anew, not kept from before.
    __device__ __forceinline__ void forget() {
        uint32_t* w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
        for (int i = 0; i < static_cast<int>(N * kPacks * sizeof(T) / 4); i++) asm volatile("" : "+r"(w[i]));
    }
    __device__ __forceinline__ Pair<Sum<T>> operator[](int i) const { return widen2(&v[2 * i]); }
    __device__ __forceinline__ void set(int i, Pair<Sum<T>> value) { narrow2(&v[2 * i], value); }
};

// sigmoid(v), and 1 - sigmoid(v). In f32 and f64 with the functions of the mathematical library; of 16-bit gates, whose results are rounded to as many bits, by
// the approximate instructions (2^v within 2 units of the 22nd bit, 1 / v within 1 of the 23rd), so that e^-v is off by some 2^-21 + |v| 2^-23 of itself, and 1 - sigmoid(v), which is made
// without a difference that cancels, as well.
template <typename T> __device__ __forceinline__ Pair<Sum<T>> gates(Pair<Sum<T>> v, Pair<Sum<T>>& one_minus) {
    if constexpr (sizeof(T) == 2) {
        Pair<float> e = v * -1.44269504f, z;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
        z = e + both(1.0f);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(z.x) : "f"(z.x));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(z.y) : "f"(z.y));
        one_minus = Pair<float>{fminf(e.x, 3.402823466e38f), fminf(e.y, 3.402823466e38f)} * z;
        return z;
    } else {
        const Sum<T> x = sigmoid<Sum<T>>(v.x, one_minus.x);
        return {x, sigmoid<Sum<T>>(v.y, one_minus.y)};
    }
}
template <typename T> __device__ __forceinline__ Pair<Sum<T>> gates(Pair<Sum<T>> v) {
    Pair<Sum<T>> one_minus;
    return gates<T>(v, one_minus);
}

// A thread's own weights: scale * weight_branch, where registers are short in shared memory, and weight_output.
template <typename T, int N, int kPacks, bool kShared> struct Weights {
    using S = Sum<T>;
    using V = Values<T, N, kPacks>;
    struct alignas(16) Two { // pairs
        Pair<S> v[2];
    };
    Pair<S> own[kShared ? 1 : V::kPairs];
    const Two* place; // what a thread has is `threads` apart
    int threads;
    V p;
    // room: of the block's threads, 2 kPairs values each
    __device__ __forceinline__ void load(const Inputs<T>& in, int member, int team, int packs, S* room) {
        V s, w;
        s.clear(), w.clear(), p.clear();
        s.load(in.scale + member * N, member, team, packs);
        w.load(in.weight_branch + member * N, member, team, packs);
        p.load(in.weight_output + member * N, member, team, packs);
        Two* to = reinterpret_cast<Two*>(room) + threadIdx.x;
        threads = blockDim.x;
        place = to;
#pragma unroll
        for (int i = 0; i < V::kPairs; i++) {
            if constexpr (kShared) to[i / 2 * threads].v[i % 2] = s[i] * w[i];
            else own[i] = s[i] * w[i];
        }
    }
    __device__ __forceinline__ Pair<S> sw(int i) const {
        if constexpr (kShared) return place[i / 2 * threads].v[i % 2];
        else return own[i];
    }
};

// A row forward, in two steps, with what is held in between.
template <typename T, int GATE, int N, int kPacks> struct RowForward {
    using S = Sum<T>;
    using V = Values<T, N, kPacks>;
    Pair<S> y[V::kPairs];
    S per_column, epsilon;
    __device__ RowForward(const Inputs<T>& in) : per_column(S(1) / static_cast<S>(in.columns)), epsilon(static_cast<S>(in.epsilon)) {}

    __device__ __forceinline__ S inverse_rms(const V& b, TeamSums<S>& sums) const {
        Pair<S> square = both(S(0));
#pragma unroll
        for (int i = 0; i < V::kPairs; i++) square = fma2(b[i], b[i], square);
        S sum = total(square);
        sums.add_up(sum);
        return inverse_root<S>(sum * per_column + epsilon);
    }
    template <typename W> // returns the sum of squares of the thread's values
    __device__ __forceinline__ S stream(V& out, const W& weights, const V& x, const V& b, const V& g, T gate, S q) {
        const Pair<S> z_row = GATE == kRowGate ? gates<T>(both(widen(gate))) : both(S(1));
        Pair<S> square = both(S(0));
#pragma unroll
        for (int i = 0; i < V::kPairs; i++) {
            const Pair<S> z = GATE == kFullGate ? gates<T>(g[i]) : z_row;
            y[i] = fma2(weights.sw(i) * z, b[i] * q, x[i]);
            square = fma2(y[i], y[i], square);
            out.set(i, y[i]);
        }
        return total(square);
    }
    __device__ __forceinline__ void normed(V& out, const V& p, S sum_of_squares) const {
        const S r = inverse_root<S>(sum_of_squares * per_column + epsilon);
#pragma unroll
        for (int i = 0; i < V::kPairs; i++) out.set(i, p[i] * (y[i] * r));
    }
};

template <typename T, int GATE, int N, int kPacks>
__global__ void __launch_bounds__(kTeamThreads)
residual_norm_rows(T* __restrict__ stream, T* __restrict__ normed, const __grid_constant__ Inputs<T> in, int team) {
    using S = Sum<T>;
    using V = Values<T, N, kPacks>;
    __shared__ typename TeamSums<S>::Place shared[2];
    const int member = threadIdx.x % team, teams = blockDim.x / team, packs = static_cast<int>(in.columns / N);
    TeamSums<S> sums(shared, team);
    Weights<T, N, kPacks, false> weights;
    weights.load(in, member, team, packs, nullptr);
    RowForward<T, GATE, N, kPacks> work(in);
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + threadIdx.x / team;
    V next_x, next_b, next_g, out;
    T next_gate{};
    next_x.clear(), next_b.clear(), next_g.clear();
    auto fetch = [&](int64_t r) {
        if (r >= in.rows) return;
        next_b.load(in.branch + r * in.branch_stride + member * N, member, team, packs);
        next_x.load(in.residual + r * in.residual_stride + member * N, member, team, packs);
        if constexpr (GATE == kFullGate) next_g.load(in.gate + r * in.gate_stride + member * N, member, team, packs);
        if constexpr (GATE == kRowGate) next_gate = in.gate[r * in.gate_stride];
    };
    fetch(row);
    for (; row < in.rows; row += step) { // (teams of a block of several are warps, which do not wait for one another)
        const V x = next_x, b = next_b, g = next_g;
        const T gate = next_gate;
        fetch(row + step);
        const S q = work.inverse_rms(b, sums);
        S sum = work.stream(out, weights, x, b, g, gate, q);
        const int64_t at = row * in.columns + member * N;
        out.store(stream + at, member, team, packs);
        sums.add_up(sum);
        work.normed(out, weights.p, sum);
        out.store(normed + at, member, team, packs);
    }
}

// Rows that a block shares and whose packs are whole: the rows of the inputs come into shared memory by bulk copies, kRing rows ahead, which
// leaves registers for two blocks on an SM: while one waits at a barrier the other works. Bounded by memory: 16 384 rows of 4096 columns in bf16 take 110 to 119 us (670 MB, 5.6 to 6.1 TB/s),
// backward 206 us (1.07 GB, 5.2 TB/s); 20 011 of 1000 in f32, a gate for each row, 55 and 82 to 86 us (5.8 and 5.6 to 5.9 TB/s). In registers alone the first took 287 and 438 us.
template <typename T, int kInputs, int kRing> struct RowRing {
    unsigned char* places;
    uint64_t* full;
    int row_bytes, at = 0;
    unsigned round = 0;

    __device__ RowRing(unsigned char* places, uint64_t (&full)[kRing], int64_t columns)
        : places(places), full(full), row_bytes(static_cast<int>(columns * sizeof(T))) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < kRing; i++) mbarrier_init(&full[i], 1);
            mbarrier_init_fence();
        }
    }
    // one thread; rows: where each input's row begins
    __device__ __forceinline__ void fetch(int place, const T* const (&rows)[kInputs]) {
        unsigned char* to = places + place * kInputs * row_bytes;
        mbarrier_arrive_expect(&full[place], static_cast<unsigned>(kInputs * row_bytes));
#pragma unroll
        for (int i = 0; i < kInputs; i++) bulk_copy_in(to + i * row_bytes, rows[i], row_bytes, &full[place]);
    }
    __device__ __forceinline__ bool wait() { return mbarrier_wait(&full[at], round); }
    __device__ __forceinline__ const T* row() const { return reinterpret_cast<const T*>(places + at * kInputs * row_bytes); }
    __device__ __forceinline__ void next() {
        if (++at == kRing) at = 0, round ^= 1;
    }
    // A wait ran out: reports that, and the copying thread stays until the copies that may be under way, to this place and the next ones, are there (or another wait runs
    // out), as the block's shared memory is another one's afterwards. rows: that are left, from the one waited for on; places: that are filled at most.
    __device__ void give_up(const Status& st, int64_t rows, int places) {
        report_stalled(st);
        if (threadIdx.x != 0) return;
        for (int i = 0; i < places && i < rows; i++, next()) (void)wait();
    }
};
constexpr int kForwardRing = 3, kBackwardRing = 2;

template <typename T, int GATE, int kPacks>
__global__ void __launch_bounds__(kTeamThreads)
residual_norm_staged(T* __restrict__ stream, T* __restrict__ normed, const __grid_constant__ Inputs<T> in, Status st) {
    using S = Sum<T>;
    constexpr int N = kPack<T>, kInputs = GATE == kFullGate ? 3 : 2;
    using V = Values<T, N, kPacks>;
    extern __shared__ __align__(128) unsigned char stages[];
    __shared__ typename TeamSums<S>::Place shared[2];
    __shared__ uint64_t full[kForwardRing];
    const int member = threadIdx.x, team = blockDim.x, packs = static_cast<int>(in.columns / N), columns = static_cast<int>(in.columns);
    RowRing<T, kInputs, kForwardRing> ring(stages, full, in.columns);
    TeamSums<S> sums(shared, team); // (ends with a barrier: a team of one warp does not come here)
    const int64_t step = gridDim.x;
    auto fetch = [&](int64_t r, int place) {
        if (threadIdx.x != 0 || r >= in.rows) return;
        const T* b = in.branch + r * in.branch_stride;
        const T* x = in.residual + r * in.residual_stride;
        if constexpr (GATE == kFullGate) ring.fetch(place, {b, x, in.gate + r * in.gate_stride});
        else ring.fetch(place, {b, x});
    };
    int64_t row = blockIdx.x;
    for (int i = 0; i < kForwardRing; i++) fetch(row + i * step, i);
    Weights<T, N, kPacks, false> weights;
    weights.load(in, member, team, packs, nullptr);
    RowForward<T, GATE, N, kPacks> work(in);
    for (; row < in.rows; row += step, ring.next()) {
        const T gate = GATE == kRowGate ? in.gate[row * in.gate_stride] : T{};
        if (!ring.wait()) return ring.give_up(st, (in.rows - row + step - 1) / step, kForwardRing);
        const T* first = ring.row() + member * N;
        V x, b, g, out;
        x.clear(), b.clear(), g.clear();
        b.load(first, member, team, packs);
        const S q = work.inverse_rms(b, sums);
        x.load(first + columns, member, team, packs);
        if constexpr (GATE == kFullGate) g.load(first + 2 * columns, member, team, packs);
        S sum = work.stream(out, weights, x, b, g, gate, q);
        const int64_t at = row * in.columns + member * N;
        out.store(stream + at, member, team, packs);
        sums.add_up(sum); // (and everybody is done with the row's place)
        fetch(row + kForwardRing * step, ring.at);
        work.normed(out, weights.p, sum);
        out.store(normed + at, member, team, packs);
    }
}

// The backward pass of a row, in steps, with what is held from one to the next. The gates are computed twice, which takes fewer instructions than
// to hold them in registers that there are not.
template <typename T, int GATE, int N, int kPacks, bool kShared> struct RowBackward {
    using S = Sum<T>;
    using V = Values<T, N, kPacks>;
    static constexpr int kPairs = V::kPairs;
    const Weights<T, N, kPacks, kShared>& weights;
    S per_column, epsilon;
    Pair<S> y[kPairs];                            // the stream, then the gradient of n
    Pair<S> of_branch[kPairs], of_output[kPairs]; // sums over rows

    __device__ RowBackward(const Weights<T, N, kPacks, kShared>& weights, const Inputs<T>& in)
        : weights(weights), per_column(S(1) / static_cast<S>(in.columns)), epsilon(static_cast<S>(in.epsilon)) {
#pragma unroll
        for (int i = 0; i < kPairs; i++) of_branch[i] = of_output[i] = both(S(0));
    }
    __device__ __forceinline__ static S squares_of(const V& b) {
        Pair<S> square = both(S(0));
#pragma unroll
        for (int i = 0; i < kPairs; i++) square = fma2(b[i], b[i], square);
        return total(square);
    }
    __device__ __forceinline__ S inverse_rms(S sum_of_squares) const { return inverse_root<S>(sum_of_squares * per_column + epsilon); }
    // sums of squares of the stream, and of its products with the gradient of its norm
    __device__ __forceinline__ void forward(const V& x, const V& b, const V& g, S z_row, const V& gh, S q, S& squares, S& products) {
        Pair<S> square = both(S(0)), along = both(S(0));
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const Pair<S> z = GATE == kFullGate ? gates<T>(g[i]) : both(z_row);
            y[i] = fma2(weights.sw(i) * z, b[i] * q, x[i]);
            square = fma2(y[i], y[i], square);
            along = fma2(weights.p[i] * gh[i], y[i], along);
        }
        squares = total(square), products = total(along);
    }
    // The gradients of the stream and of full gates; returns the sum of dn n. (That of a gate for a row is 1 - z times it.)
    __device__ __forceinline__ S backward(V& out_stream, V& out_gate, const V& b, const V& g, S z_row, const V& gs, const V& gh, S q, S squares,
                                          S products) {
        const S r = inverse_rms(squares), back = -products * r * r * r * per_column;
        Pair<S> sum = both(S(0));
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            Pair<S> one_minus;
            const Pair<S> z = GATE == kFullGate ? gates<T>(g[i], one_minus) : both(z_row);
            const Pair<S> n = b[i] * q, h = gh[i] * r;
            of_output[i] = fma2(h, y[i], of_output[i]);
            const Pair<S> ds = fma2(weights.p[i], h, fma2(y[i], both(back), gs[i]));
            out_stream.set(i, ds);
            const Pair<S> dz = ds * z;
            of_branch[i] = fma2(dz, n, of_branch[i]);
            y[i] = dz * weights.sw(i);
            const Pair<S> all = y[i] * n;
            sum = sum + all;
            if constexpr (GATE == kFullGate) out_gate.set(i, all * one_minus);
        }
        return total(sum);
    }
    __device__ __forceinline__ void branch(V& out, const V& b, S q, S sum) const {
        const S lost = -q * sum * per_column;
#pragma unroll
        for (int i = 0; i < kPairs; i++) out.set(i, fma2(b[i], both(lost), y[i]) * q);
    }
    // the sums over the rows of this thread; `add`: on top of what is there
    __device__ __forceinline__ void leave(S* own, const Inputs<T>& in, int member, int team, int packs, bool add) const {
#pragma unroll
        for (int i = 0; i < 2 * kPairs; i++) {
            const int pack = i / N * team + member;
            if (pack >= packs) continue;
            const int64_t c = static_cast<int64_t>(pack) * N + i % N;
            own[c] = (add ? own[c] : S(0)) + (i & 1 ? of_branch[i / 2].y : of_branch[i / 2].x);
            own[in.columns + c] = (add ? own[in.columns + c] : S(0)) + (i & 1 ? of_output[i / 2].y : of_output[i / 2].x);
        }
    }
};
// The gate of a row. 1 minus it, which only one thread of the team needs, later, it leaves in shared memory: registers are short.
template <typename T, int GATE> __device__ __forceinline__ Sum<T> row_gate(const Inputs<T>& in, int64_t row, int member, Sum<T>& one_minus) {
    if constexpr (GATE == kRowGate) {
        Pair<Sum<T>> other;
        const Sum<T> z = gates<T>(both(widen(in.gate[row * in.gate_stride])), other).x;
        if (member == 0) one_minus = other.x;
        return z;
    } else {
        return 1;
    }
}

template <typename T, int GATE, int N, int kPacks>
__global__ void __launch_bounds__(kTeamThreads, 1)
residual_norm_vjp_rows(const __grid_constant__ Gradients<T> grad, const __grid_constant__ Inputs<T> in, int team) {
    using S = Sum<T>;
    using V = Values<T, N, kPacks>;
    __shared__ typename TeamSums<S>::Place shared[2];
    __shared__ S one_minus[kTeamThreads / 32];
    const int member = threadIdx.x % team, teams = blockDim.x / team, packs = static_cast<int>(in.columns / N);
    TeamSums<S> sums(shared, team);
    Weights<T, N, kPacks, false> weights;
    weights.load(in, member, team, packs, nullptr);
    RowBackward<T, GATE, N, kPacks, false> work(weights, in);
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    V x, b, g, gs, gh, out, out_gate;
    x.clear(), b.clear(), g.clear(), gs.clear(), gh.clear();
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * teams + threadIdx.x / team; row < in.rows; row += step) {
        b.load(in.branch + row * in.branch_stride + member * N, member, team, packs);
        x.load(in.residual + row * in.residual_stride + member * N, member, team, packs);
        gh.load(grad.normed + row * grad.normed_stride + member * N, member, team, packs);
        if constexpr (GATE == kFullGate) g.load(in.gate + row * in.gate_stride + member * N, member, team, packs);
        gs.load(grad.stream + row * grad.stream_stride + member * N, member, team, packs);
        const S z_row = row_gate<T, GATE>(in, row, member, one_minus[threadIdx.x / 32]);
        S of_b = work.squares_of(b), squares, products;
        sums.add_up(of_b);
        const S q = work.inverse_rms(of_b);
        work.forward(x, b, g, z_row, gh, q, squares, products);
        sums.add_up(squares, products);
        if constexpr (GATE == kFullGate) g.forget(); // (else gates and their exponentials stay in registers that there are not)
        S sum = work.backward(out, out_gate, b, g, z_row, gs, gh, q, squares, products);
        const int64_t at = row * in.columns + member * N;
        if (grad.residual != nullptr) out.store(grad.residual + at, member, team, packs);
        if (GATE == kFullGate && grad.gate != nullptr) out_gate.store(grad.gate + at, member, team, packs);
        sums.add_up(sum);
        if (GATE == kRowGate && grad.gate != nullptr && member == 0) grad.gate[row] = narrow<T>(sum * one_minus[threadIdx.x / 32]);
        work.branch(out, b, q, sum);
        if (grad.branch != nullptr) out.store(grad.branch + at, member, team, packs);
    }
    // the teams of a block add to its sums one after the other
    S* own = grad.columns + static_cast<int64_t>(blockIdx.x) * 2 * in.columns;
    for (int t = 0; t < teams; t++) {
        if (t > 0) __syncthreads();
        if (static_cast<int>(threadIdx.x) / team == t) work.leave(own, in, member, team, packs, t > 0);
    }
}

// (The sum of squares of the next row's branch is added up together with the last sum of this one.)
template <typename T, int GATE, int kPacks>
__global__ void __launch_bounds__(kTeamThreads)
residual_norm_vjp_staged(const __grid_constant__ Gradients<T> grad, const __grid_constant__ Inputs<T> in, Status st) {
    using S = Sum<T>;
    constexpr int N = kPack<T>, kInputs = GATE == kFullGate ? 5 : 4;
    using V = Values<T, N, kPacks>;
    extern __shared__ __align__(128) unsigned char stages[];
    __shared__ typename TeamSums<S>::Place shared[2];
    __shared__ uint64_t full[kBackwardRing];
    __shared__ S one_minus;
    const int member = threadIdx.x, team = blockDim.x, packs = static_cast<int>(in.columns / N), columns = static_cast<int>(in.columns);
    RowRing<T, kInputs, kBackwardRing> ring(stages, full, in.columns);
    TeamSums<S> sums(shared, team); // (ends with a barrier: a team of one warp does not come here)
    const int64_t step = gridDim.x;
    auto fetch = [&](int64_t r, int place) {
        if (threadIdx.x != 0 || r >= in.rows) return;
        const T *b = in.branch + r * in.branch_stride, *x = in.residual + r * in.residual_stride;
        const T *gh = grad.normed + r * grad.normed_stride, *gs = grad.stream + r * grad.stream_stride;
        if constexpr (GATE == kFullGate) ring.fetch(place, {b, x, gh, gs, in.gate + r * in.gate_stride});
        else ring.fetch(place, {b, x, gh, gs});
    };
    int64_t row = blockIdx.x;
    for (int i = 0; i < kBackwardRing; i++) fetch(row + i * step, i);
    Weights<T, N, kPacks, true> weights;
    weights.load(in, member, team, packs, reinterpret_cast<S*>(stages + kBackwardRing * kInputs * ring.row_bytes));
    RowBackward<T, GATE, N, kPacks, true> work(weights, in);
    if (!ring.wait()) return ring.give_up(st, (in.rows - row + step - 1) / step, kBackwardRing); // (a block has at least one row)
    V b;
    b.clear();
    b.load(ring.row() + member * N, member, team, packs);
    S of_b = work.squares_of(b);
    sums.add_up(of_b);
    while (row < in.rows) {
        const S z_row = row_gate<T, GATE>(in, row, member, one_minus), q = work.inverse_rms(of_b);
        const T* first = ring.row() + member * N;
        const int place = ring.at;
        V out;
        S squares, products;
        {
            V x, g, gh;
            x.clear(), g.clear(), gh.clear();
            x.load(first + columns, member, team, packs);
            gh.load(first + 2 * columns, member, team, packs);
            if constexpr (GATE == kFullGate) g.load(first + 4 * columns, member, team, packs);
            work.forward(x, b, g, z_row, gh, q, squares, products);
        }
        sums.add_up(squares, products);
        const int64_t at = row * in.columns + member * N;
        S sum;
        {
            V g, gs, gh, out_gate;
            g.clear(), gs.clear(), gh.clear();
            gh.load(first + 2 * columns, member, team, packs);
            gs.load(first + 3 * columns, member, team, packs);
            if constexpr (GATE == kFullGate) g.load(first + 4 * columns, member, team, packs);
            sum = work.backward(out, out_gate, b, g, z_row, gs, gh, q, squares, products);
            if (grad.residual != nullptr) out.store(grad.residual + at, member, team, packs);
            if (GATE == kFullGate && grad.gate != nullptr) out_gate.store(grad.gate + at, member, team, packs);
        }
        ring.next();
        V next_b;
        next_b.clear();
        if (row + step < in.rows) {
            if (!ring.wait()) return ring.give_up(st, 1, 1);
            next_b.load(ring.row() + member * N, member, team, packs);
        }
        of_b = work.squares_of(next_b);
        sums.add_up(sum, of_b);
        fetch(row + kBackwardRing * step, place); // (everybody is done with it)
        if (GATE == kRowGate && grad.gate != nullptr && member == 0) grad.gate[row] = narrow<T>(sum * one_minus);
        work.branch(out, b, q, sum);
        if (grad.branch != nullptr) out.store(grad.branch + at, member, team, packs);
        b = next_b;
        row += step;
    }
    work.leave(grad.columns + static_cast<int64_t>(blockIdx.x) * 2 * in.columns, in, member, team, packs, false);
}

// The sums over rows from those of the blocks. A block takes eight columns: each eight lanes add up a part of the blocks (a sector of 32 bytes of f32 at a time), then
// the parts are added up. (With 32 columns to a block, 1000 columns of 888 blocks took 17 us: too few blocks, each with too many loads in a row.)
constexpr int kColumnThreads = 1024, kColumnsAtOnce = 8, kColumnParts = kColumnThreads / kColumnsAtOnce;
template <typename T>
__global__ void __launch_bounds__(kColumnThreads)
residual_norm_columns(T* __restrict__ grad_scale, T* __restrict__ grad_weight_branch, T* __restrict__ grad_weight_output,
                      const T* __restrict__ scale, const T* __restrict__ weight_branch, const Sum<T>* __restrict__ sums,
                      int64_t blocks, int64_t columns) {
    using S = Sum<T>;
    __shared__ S shared[kColumnThreads / 32][2][kColumnsAtOnce];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = threadIdx.x / kColumnsAtOnce;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kColumnsAtOnce + threadIdx.x % kColumnsAtOnce;
    S sum[2] = {0, 0};
    if (c < columns) {
#pragma unroll 4
        for (int64_t b = part; b < blocks; b += kColumnParts) {
            sum[0] += sums[2 * b * columns + c];
            sum[1] += sums[(2 * b + 1) * columns + c];
        }
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        sum[k] += __shfl_xor_sync(kFullMask, sum[k], 8);
        sum[k] += __shfl_xor_sync(kFullMask, sum[k], 16);
        if (lane < kColumnsAtOnce) shared[warp][k][lane] = sum[k];
    }
    __syncthreads();
    if (threadIdx.x >= kColumnsAtOnce || c >= columns) return;
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

// Whether a block may have so much dynamic shared memory beside its own.
bool fits_block(const Call& call, size_t bytes) { return bytes + 4096 <= static_cast<size_t>(max_optin_smem(call.device)); }

bool all_aligned(std::initializer_list<const Array*> arrays) {
    for (const Array* a : arrays)
        if (!aligned16(*a)) return false;
    return true;
}

// Calls f(values of a pack, values of a thread) for the widths that a row may fit, until it says that it did: few values where they fit a
// warp, else twice as many: half as many threads have the registers for that, and what is done once for a thread is done half as often
// (16384 x 4096 in bf16, backward: 207 us, with few 271 us).
template <typename T, typename F> bool by_values(bool whole, int64_t columns, F&& f) {
    constexpr int few = kFewValues<T>;
    auto with = [&](auto width) {
        if (columns <= 32 * few) return f(width, std::integral_constant<int, few>());
        return f(width, std::integral_constant<int, 2 * few>());
    };
    return whole ? with(std::integral_constant<int, kPack<T>>()) : with(std::integral_constant<int, 1>());
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
                if constexpr (N > 1 && N * kPacks > kFewValues<T>) {
                    const size_t stages = static_cast<size_t>(kForwardRing) * (GATE == kFullGate ? 3 : 2) * in.columns * sizeof(T);
                    if (t.team > 32 && fits_block(call, stages)) {
                        auto kernel = residual_norm_staged<T, GATE, kPacks>;
                        const int resident = resident_blocks(kernel, call.device, t.threads, stages) * sm_count(call.device);
                        kernel<<<static_cast<unsigned>(t.blocks(in.rows, resident)), t.threads, stages, call.stream>>>(
                            static_cast<T*>(stream.data), static_cast<T*>(normed.data), in, call.status);
                        note_kernel_f("residual_norm_staged<%s,%d,%d>", array_type_name<T>(), GATE, kPacks);
                        return true;
                    }
                }
                auto kernel = residual_norm_rows<T, GATE, N, kPacks>;
                const int resident = resident_blocks(kernel, call.device, t.threads, 0) * sm_count(call.device);
                kernel<<<static_cast<unsigned>(t.blocks(in.rows, resident)), t.threads, 0, call.stream>>>(
                    static_cast<T*>(stream.data), static_cast<T*>(normed.data), in, t.team);
                note_kernel_f("residual_norm_rows<%s,%d,%d,%d>", array_type_name<T>(), GATE, N, kPacks);
                return true;
            };
            const bool whole = all_aligned({&stream, &normed, &residual, &branch, &scale, &weight_branch, &weight_output}) &&
                               (GATE != kFullGate || aligned16(gate));
            if (by_values<T>(whole, residual.shape[1], in_registers)) return;
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
        Scratch of_blocks(call);
        auto room = [&](int64_t for_blocks) {
            blocks = for_blocks;
            of_blocks.take(static_cast<size_t>(2 * blocks * columns) * sizeof(Sum<T>));
            return Gradients<T>{data(grad_residual), data(grad_branch), data(grad_gate), data(grad_stream), data(grad_normed),
                                grad_stream.stride[0], grad_normed.stride[0], of_blocks.as<Sum<T>>()};
        };
        for_gate(kind, [&](auto g) {
            constexpr int GATE = decltype(g)::value;
            if (rows == 0) return;
            const auto in = inputs_of<T>(residual, branch, gate, scale, weight_branch, weight_output, epsilon);
            auto in_registers = [&](auto width, auto count) {
                constexpr int N = decltype(width)::value, kPacks = decltype(count)::value / N;
                const Teams t = teams_of(columns, N * kPacks);
                if (t.threads == 0) return false;
                if constexpr (N > 1 && N * kPacks > kFewValues<T>) {
                    const size_t stages = static_cast<size_t>(kBackwardRing) * (GATE == kFullGate ? 5 : 4) * columns * sizeof(T) +
                                          static_cast<size_t>(t.threads) * N * kPacks * sizeof(Sum<T>);
                    if (t.team > 32 && fits_block(call, stages)) {
                        auto kernel = residual_norm_vjp_staged<T, GATE, kPacks>;
                        const int resident = resident_blocks(kernel, call.device, t.threads, stages) * sm_count(call.device);
                        const Gradients<T> grad = room(t.blocks(rows, resident));
                        kernel<<<static_cast<unsigned>(blocks), t.threads, stages, call.stream>>>(grad, in, call.status);
                        note_kernel_f("residual_norm_vjp_staged<%s,%d,%d>", array_type_name<T>(), GATE, kPacks);
                        return true;
                    }
                }
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
            if (by_values<T>(whole, residual.shape[1], in_registers)) return;
            const Gradients<T> grad = room(std::min<int64_t>(rows, int64_t(sm_count(call.device)) * 4));
            residual_norm_vjp_plain<T, GATE><<<static_cast<unsigned>(blocks), kThreads, 0, call.stream>>>(grad, in);
            note_kernel_f("residual_norm_vjp_plain<%s,%d>", array_type_name<T>(), GATE);
        });
        MOPS_CUDA_OK(cudaGetLastError());
        if (of_columns)
            residual_norm_columns<T><<<static_cast<unsigned>(ceil_div(columns, kColumnsAtOnce)), kColumnThreads, 0, call.stream>>>(
                data(grad_scale), data(grad_weight_branch), data(grad_weight_output), data(scale), data(weight_branch), of_blocks.as<Sum<T>>(),
                blocks, columns);
        of_blocks.free();
    });
    end_call(call, op.c_str(), nullptr, 0);
}

} // namespace mops_b200
