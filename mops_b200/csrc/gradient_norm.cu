// gradient_norm, clip_gradient_norm: the norm of all gradients of a model together, and their scaling to a largest norm.
//
//   norm = sqrt(sum over all tensors of x^2), output = x min(1, max_norm / norm)
//
// Bounded by memory: 2 bytes a value for the norm of bf16, and 4 for its scaling, which has to read again what the norm was taken of. All tensors go in one launch, as a table among the kernel's
// arguments (so a captured graph keeps it): their values are cut into chunks, of which a block takes every so many-th, and the second kernel goes through them backwards, so that it
// finds what was read last in L2. 60 tensors in bf16, 852 MB: the squares 142 us (6.0 TB/s), scaling 279 (6.1 TB/s read and written); the two read everything twice but for some 20 MB.
#include <vector>

#include "block_ops.hpp"
#include "convert.cuh"

namespace mops_b200 {
namespace {

constexpr int kThreads = 256;
// Packs of 16 bytes that a thread has under way, and blocks of an SM: while squares are added up, and while values are scaled.
constexpr int kSumPacks = 8, kSumBlocks = 4, kScalePacks = 4, kScaleBlocks = 6;
constexpr int kMostTensors = 448; // of a launch, whose arguments have 32 KB

struct Entry {
    const void* from;
    void* to;
    int64_t values;
    int64_t first; // chunk
    int32_t type;
};
template <int kMost> struct Table {
    int n, chunk; // bytes
    int64_t chunks;
    Entry entry[kMost];
};

// The chunk's tensor, and its values [lo, hi).
struct Chunk {
    const Entry* entry;
    int64_t lo, hi;
};
template <int kMost> __device__ __forceinline__ Chunk find_chunk(const Table<kMost>& table, int64_t chunk) {
    int lo = 0, hi = table.n - 1; // the last entry whose first chunk is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (table.entry[mid].first <= chunk) lo = mid;
        else hi = mid - 1;
    }
    Chunk c;
    c.entry = &table.entry[lo];
    const int64_t size = table.chunk / (c.entry->type == MOPS_B200_F64 ? 8 : c.entry->type == MOPS_B200_F32 ? 4 : 2);
    c.lo = (chunk - c.entry->first) * size;
    c.hi = min(c.lo + size, c.entry->values);
    return c;
}

// N values from or to anywhere; `aligned`: to multiples of 16 bytes.
template <int N, typename T> __device__ __forceinline__ Pack<T, N> load_pack(const T* p, bool aligned) {
    if (aligned) return *reinterpret_cast<const Pack<T, N>*>(p);
    Pack<T, N> v;
#pragma unroll
    for (int k = 0; k < N; k++) v.v[k] = p[k];
    return v;
}
template <int N, typename T> __device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v, bool aligned) {
    if (aligned) {
        store_through(p, v);
        return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) p[k] = v.v[k];
}

// Calls body(where, pack) for packs of a chunk's n values, kInFlight of which a thread loads before it goes on with the first, and for single values where they do not fill one; the same threads take the
// same values wherever a tensor begins.
template <int kInFlight, typename T, typename F> __device__ __forceinline__ void for_packs(const T* __restrict__ p, int n, bool aligned, F&& body) {
    constexpr int N = kPack<T>;
    const int whole = n / N * N;
    int i = threadIdx.x * N;
    if (aligned)
        for (; i + (kInFlight - 1) * kThreads * N < whole; i += kInFlight * kThreads * N) {
            Pack<T, N> v[kInFlight];
#pragma unroll
            for (int k = 0; k < kInFlight; k++) v[k] = *reinterpret_cast<const Pack<T, N>*>(p + i + k * kThreads * N);
#pragma unroll
            for (int k = 0; k < kInFlight; k++) body(i + k * kThreads * N, v[k]);
        }
#pragma unroll 1
    for (; i < whole; i += kThreads * N) body(i, load_pack<N>(p + i, aligned));
    for (i = whole + threadIdx.x; i < n; i += kThreads) body(i, load_pack<1>(p + i, true));
}

template <typename F> __device__ __forceinline__ void with_type(int32_t type, F&& f) {
    if (type == MOPS_B200_BF16) f(__nv_bfloat16());
    else if (type == MOPS_B200_F32) f(float());
    else if (type == MOPS_B200_F16) f(__half());
    else f(double());
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double of_warp[kThreads / 32];
    v = warp_sum(v);
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = v;
    __syncthreads();
    double all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++) all += of_warp[w];
    __syncthreads();
    return all;
}

template <int kMost>
__global__ void __launch_bounds__(kThreads, kSumBlocks)
sum_squares(double* __restrict__ sums, const __grid_constant__ Table<kMost> table) {
    double sum = 0;
    for (int64_t chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const Chunk c = find_chunk(table, chunk);
        with_type(c.entry->type, [&](auto zero) {
            using T = decltype(zero);
            using S = Sum<T>;
            const T* p = static_cast<const T*>(c.entry->from) + c.lo;
            S part[kPack<T>] = {};
            const bool aligned = reinterpret_cast<uintptr_t>(p) % 16 == 0;
            for_packs<kSumPacks>(p, static_cast<int>(c.hi - c.lo), aligned, [&](int, const auto& v) {
                constexpr int N = sizeof(v) / sizeof(T);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const S x = widen(v.v[k]);
                    part[k] += x * x;
                }
            });
#pragma unroll
            for (int k = 0; k < kPack<T>; k++) sum += part[k];
        });
    }
    const double all = block_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

// By a block, in an order that depends on n alone.
__device__ __forceinline__ double join_sums(const double* __restrict__ sums, int n) {
    double sum = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += sums[i];
    return sqrt(block_sum(sum));
}
__device__ __forceinline__ void write_norm(void* to, bool wide, double norm) {
    if (wide) *static_cast<double*>(to) = norm;
    else *static_cast<float*>(to) = static_cast<float>(norm);
}

__global__ void __launch_bounds__(kThreads)
join_norm(void* __restrict__ norm, bool wide, const double* __restrict__ sums, int n) {
    after_others();
    const double value = join_sums(sums, n);
    if (threadIdx.x == 0) write_norm(norm, wide, value);
}

template <int kMost>
__global__ void __launch_bounds__(kThreads, kScaleBlocks)
scale_values(void* norm, bool wide, const double* __restrict__ sums, int n, double max_norm, const __grid_constant__ Table<kMost> table) {
    after_others();
    const double value = join_sums(sums, n);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) write_norm(norm, wide, value);
    const double factor = isfinite(value) && value > max_norm ? max_norm / value : 1.0;
    for (int64_t chunk = table.chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        const Chunk c = find_chunk(table, chunk);
        if (factor == 1.0 && c.entry->from == c.entry->to) continue;
        with_type(c.entry->type, [&](auto zero) {
            using T = decltype(zero);
            using S = Sum<T>;
            const T* p = static_cast<const T*>(c.entry->from) + c.lo;
            T* q = static_cast<T*>(c.entry->to) + c.lo;
            const S f = static_cast<S>(factor);
            const bool as_it_is = factor == 1.0;
            const bool from_aligned = reinterpret_cast<uintptr_t>(p) % 16 == 0, to_aligned = reinterpret_cast<uintptr_t>(q) % 16 == 0;
            for_packs<kScalePacks>(p, static_cast<int>(c.hi - c.lo), from_aligned, [&](int i, auto v) {
                constexpr int N = sizeof(v) / sizeof(T);
                if (!as_it_is) {
#pragma unroll
                    for (int k = 0; k < N; k++) v.v[k] = narrow<T>(widen(v.v[k]) * f);
                }
                store_pack(q + i, v, to_aligned || N == 1);
            });
        });
    }
}

// The tensors' tables, and how many chunks all have.
struct Tensors {
    std::vector<Entry> entries; // of those that have values; `first` counts from the start of its launch
};

Tensors check_tensors(Array& norm, const Array* outputs, const Array* gradients, int64_t n, const std::string& op) {
    if (n < 0 || (n > 0 && gradients == nullptr)) throw std::runtime_error("no gradients in " + op);
    bool wide = false;
    Tensors t;
    for (int64_t i = 0; i < n; i++) {
        Array g = gradients[i];
        check_floating(g.type, "a gradient", op);
        check_array(g, "a gradient", std::min(std::max(g.dimensions, 1), 3), g.type, op);
        check_output(g, "a gradient", op);
        wide |= g.type == MOPS_B200_F64;
        void* to = nullptr;
        if (outputs != nullptr) {
            Array o = outputs[i];
            check_array(o, "an output", g.dimensions, g.type, op);
            for (int d = 0; d < g.dimensions; d++) check_size(o.shape[d], "an output", d, g.shape[d], "its gradient", d, op);
            check_output(o, "an output", op);
            to = o.data;
        }
        if (values_of(g) > 0) t.entries.push_back(Entry{g.data, to, values_of(g), 0, g.type});
    }
    check_array(norm, "norm", 1, wide ? MOPS_B200_F64 : MOPS_B200_F32, op);
    if (norm.shape[0] != 1) throw std::runtime_error("norm must have one value in " + op);
    // no two of them overlap, but an output and its gradient where they are the same (and gradients of which only the norm is asked for)
    using Place = std::pair<uintptr_t, uintptr_t>;
    auto place = [](const void* p, int64_t bytes) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(p);
        return Place{from, from + static_cast<uintptr_t>(bytes)};
    };
    const Place result = place(norm.data, type_bytes(norm.type));
    std::vector<Place> places;
    places.reserve(2 * t.entries.size());
    for (const Entry& e : t.entries) {
        const int64_t bytes = e.values * type_bytes(e.type);
        places.push_back(place(e.from, bytes));
        if (outputs != nullptr && e.to != e.from) places.push_back(place(e.to, bytes));
    }
    bool apart = true;
    for (const Place& p : places) apart = apart && (p.second <= result.first || result.second <= p.first);
    if (outputs != nullptr) {
        std::sort(places.begin(), places.end());
        for (size_t i = 1; i < places.size(); i++) apart = apart && places[i - 1].second <= places[i].first;
    }
    if (!apart) throw std::runtime_error("gradients and " + std::string(outputs != nullptr ? "outputs" : "norm") + " overlap in " + op);
    return t;
}

// Chunks of 8 KB where that leaves no block without one, up to 128 KB where there are several for each: a block that goes on to another chunk has nothing under way meanwhile.
template <typename F> void for_tables(const Tensors& t, int64_t blocks, F&& f) {
    int64_t bytes = 0;
    for (const Entry& e : t.entries) bytes += e.values * type_bytes(e.type);
    int chunk = 8192;
    while (chunk < 131072 && bytes / chunk > 4 * blocks) chunk *= 2;
    auto go = [&](auto most) {
        constexpr int kMost = decltype(most)::value;
        for (size_t at = 0; at < t.entries.size(); at += kMost) {
            Table<kMost> table;
            table.n = static_cast<int>(std::min<size_t>(kMost, t.entries.size() - at));
            table.chunk = chunk;
            table.chunks = 0;
            for (int i = 0; i < table.n; i++) {
                table.entry[i] = t.entries[at + i];
                table.entry[i].first = table.chunks;
                table.chunks += ceil_div(table.entry[i].values * type_bytes(table.entry[i].type), chunk);
            }
            f(table, most);
        }
    };
    if (t.entries.size() <= 32) go(std::integral_constant<int, 32>());
    else go(std::integral_constant<int, kMostTensors>());
}

void norm_of(Array norm, const Array* outputs, const Array* gradients, int64_t n, double max_norm, const std::string& op) {
    const Tensors t = check_tensors(norm, outputs, gradients, n, op);
    if (outputs != nullptr && !(max_norm >= 0)) throw std::runtime_error("max_norm must not be negative in " + op);
    Call call = begin_call();
    const int64_t most = int64_t(sm_count(call.device)) * kSumBlocks, most_scaling = int64_t(sm_count(call.device)) * kScaleBlocks, launches = ceil_div(static_cast<int64_t>(t.entries.size()), 32);
    Scratch room(call, static_cast<size_t>(most * std::max<int64_t>(launches, 1)) * sizeof(double));
    double* sums = room.as<double>();
    const bool wide = norm.type == MOPS_B200_F64;
    int64_t parts = 0;
    for_tables(t, most, [&](const auto& table, auto most_tensors) {
        const int64_t blocks = std::min(table.chunks, most);
        sum_squares<decltype(most_tensors)::value><<<static_cast<unsigned>(blocks), kThreads, 0, call.stream>>>(sums + parts, table);
        parts += blocks;
    });
    MOPS_CUDA_OK(cudaGetLastError());
    bool written = false;
    if (outputs != nullptr)
        for_tables(t, most, [&](const auto& table, auto most_tensors) {
            const int64_t blocks = std::min(table.chunks, most_scaling);
            launch_early(call, scale_values<decltype(most_tensors)::value>, static_cast<unsigned>(blocks), kThreads, written ? nullptr : norm.data, wide, sums,
                         static_cast<int>(parts), max_norm, table);
            written = true;
        });
    if (!written) launch_early(call, join_norm, 1, kThreads, norm.data, wide, sums, static_cast<int>(parts));
    MOPS_CUDA_OK(cudaGetLastError());
    note_kernel_f("sum_squares, %d tensors", static_cast<int>(t.entries.size()));
    end_call(call, op.c_str(), nullptr, 0);
}

} // namespace

void gradient_norm(Array norm, const Array* gradients, int64_t n) {
    norm_of(norm, nullptr, gradients, n, 0, "cuda_gradient_norm");
}

void clip_gradient_norm(Array norm, const Array* outputs, const Array* gradients, int64_t n, double max_norm) {
    if (n > 0 && outputs == nullptr) throw std::runtime_error("no outputs in cuda_clip_gradient_norm");
    static const Array none{};
    norm_of(norm, outputs != nullptr ? outputs : &none, gradients, n, max_norm, "cuda_clip_gradient_norm");
}

} // namespace mops_b200
