// embedding_lookup: rows of a table, scaled, and the gradient of the table.
//
//   output[t,:] = scale W[indices[t],:]
//   grad_W[v,:] = scale sum_{t: indices[t] = v} grad_output[t,:]
//
// Both move bytes and little else. The gradient is a segmented reduction over the sorted tokens, as the scatter
// operations are: no atomics, so that the same call gives the same bits, and every row of grad_W is written once.
#include "arrays.hpp"
#include "block_ops.hpp"
#include "sort.hpp"

namespace mops_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// x / d for x < 2^32, by a multiplication: d times the rounded-up quotient 2^(32 + s) / d exceeds 2^(32 + s) by less than 2^s
// when 2^s >= d.
struct Divider {
    uint32_t d, shift;
    uint64_t factor;
    explicit Divider(uint32_t divisor) : d(divisor), shift(0) {
        while ((uint64_t(1) << shift) < d) shift++;
        factor = ((uint64_t(1) << (32 + shift)) + d - 1) / d;
    }
    __device__ __forceinline__ uint32_t divide(uint32_t x) const {
        return static_cast<uint32_t>((__umul64hi(factor << (31 - shift), uint64_t(x) << 1)));
    }
};

// ------------------------------------------------------------------------------ forward
// The output is cut into packs of N values, rows one after the other, and a block takes 1024 packs in a row; so blocks have the same
// work whatever the width of a row, and a single token still uses many SMs.
constexpr int kPacksPerThread = 4;

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_rows(T* __restrict__ output, const T* __restrict__ W, int64_t stride, const int32_t* __restrict__ indices,
               int64_t index_stride, int64_t tokens, int64_t rows, uint32_t packs, Divider by_packs, Sum<T> scale, Status st) {
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * kPacksPerThread);
    const int64_t t0 = first / packs;
    const uint32_t p0 = static_cast<uint32_t>(first - t0 * packs);
    Pack<T, N> value[kPacksPerThread];
    int64_t token[kPacksPerThread];
    uint32_t pack[kPacksPerThread];
#pragma unroll
    for (int k = 0; k < kPacksPerThread; k++) {
        const uint32_t at = p0 + k * kThreads + threadIdx.x;
        const uint32_t t = by_packs.divide(at);
        token[k] = t0 + t;
        pack[k] = at - t * packs;
        if (token[k] >= tokens) continue;
        const int32_t row = __ldg(indices + token[k] * index_stride);
        if (static_cast<uint32_t>(row) < static_cast<uint64_t>(rows)) {
            value[k] = *reinterpret_cast<const Pack<T, N>*>(W + row * stride + static_cast<int64_t>(pack[k]) * N);
        } else {
            if (pack[k] == 0) report_bad_index(st, 0);
#pragma unroll
            for (int i = 0; i < N; i++) value[k].v[i] = narrow<T>(0);
        }
    }
#pragma unroll
    for (int k = 0; k < kPacksPerThread; k++) {
        if (token[k] >= tokens) continue;
#pragma unroll
        for (int i = 0; i < N; i++) value[k].v[i] = narrow<T>(widen(value[k].v[i]) * scale);
        *reinterpret_cast<Pack<T, N>*>(output + (token[k] * packs + pack[k]) * N) = value[k];
    }
}

// ------------------------------------------------------------------------------ gradient
// The sorted tokens are cut into chunks. A warp takes a chunk and a slab of 32 N columns and adds up the rows of grad_output, token
// by token. A run of equal tokens that lies inside a chunk goes to its row of grad_W at once; of one
// that a chunk's end cuts, each chunk leaves a partial sum (place 0: the run had begun before the chunk;
// place 1: it begins in it and goes on after it), and embedding_join adds those up.
constexpr int kRowsInFlight = 8; // loads of a warp under way

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_sums(T* __restrict__ grad_W, const T* __restrict__ grad_output, int64_t stride,
               const int32_t* __restrict__ sorted, const int32_t* __restrict__ permutation, int64_t tokens, int64_t rows,
               int64_t columns, int chunk, int64_t chunks, int64_t slabs, Sum<T> scale, Sum<T>* __restrict__ partial) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (unit >= chunks * slabs) return;
    const int64_t c = unit / slabs;
    const int64_t column = ((unit - c * slabs) * 32 + lane) * N;
    const bool mine = column < columns;
    const int64_t lo = c * chunk, hi = min(lo + chunk, tokens);
    int32_t before = lo > 0 ? __ldg(sorted + lo - 1) : -1; // the key in front of the next entry
    bool begun_before = true;                               // the run at hand began before the chunk
    Sum<T> sum[N];
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] = 0;
    for (int64_t base = lo; base < hi; base += 32) {
        const int n = static_cast<int>(min(hi - base, int64_t(32)));
        // the keys of 32 entries, and of the one behind them
        const int32_t key = base + lane < tokens ? __ldg(sorted + base + lane) : -1;
        const int32_t from = lane < n ? __ldg(permutation + base + lane) : 0;
        const int32_t beyond = base + 32 < tokens ? __ldg(sorted + base + 32) : -1;
        for (int j0 = 0; j0 < n; j0 += kRowsInFlight) {
            Pack<T, N> value[kRowsInFlight];
#pragma unroll
            for (int u = 0; u < kRowsInFlight; u++) {
                const int64_t t = __shfl_sync(kFullMask, from, (j0 + u) & 31);
                if (mine && j0 + u < n)
                    value[u] = *reinterpret_cast<const Pack<T, N>*>(grad_output + t * stride + column);
            }
#pragma unroll
            for (int u = 0; u < kRowsInFlight; u++) {
                const int j = j0 + u;
                if (j >= n) break;
                const int32_t k = __shfl_sync(kFullMask, key, j);
                const int32_t next = j == 31 ? beyond : __shfl_sync(kFullMask, key, (j + 1) & 31);
                if (k >= rows) return; // (sorted behind all others) tokens that give no gradient
                if (k != before) {
                    begun_before = false;
#pragma unroll
                    for (int i = 0; i < N; i++) sum[i] = 0;
                }
                before = k;
                if (mine) {
#pragma unroll
                    for (int i = 0; i < N; i++) sum[i] += widen(value[u].v[i]);
                }
                const bool ends = next != k, cut = base + j == hi - 1 && !ends;
                if (!ends && !cut) continue;
                if (!mine) continue;
                if (begun_before || cut) {
                    Sum<T>* to = partial + (2 * c + (begun_before ? 0 : 1)) * columns + column;
#pragma unroll
                    for (int i = 0; i < N; i++) to[i] = sum[i];
                } else {
                    Pack<T, N> out;
#pragma unroll
                    for (int i = 0; i < N; i++) out.v[i] = narrow<T>(sum[i] * scale);
                    *reinterpret_cast<Pack<T, N>*>(grad_W + k * columns + column) = out;
                }
            }
        }
    }
}

// Adds up the partial sums of the run that begins in chunk blockIdx.x and goes on after it, if there is one: each warp
// those of a range of chunks, then one after the other.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_join(T* __restrict__ grad_W, const int32_t* __restrict__ sorted, int64_t tokens, int64_t rows, int64_t columns,
               int chunk, Sum<T> scale, const Sum<T>* __restrict__ partial) {
    __shared__ Sum<T> joined[kWarps][32 * N];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = blockIdx.x, lo = c * chunk, last = lo + chunk - 1;
    if (last + 1 >= tokens) return;
    const int32_t k = __ldg(sorted + last);
    if (k >= rows || __ldg(sorted + last + 1) != k) return;
    if (lo > 0 && __ldg(sorted + lo - 1) == k) return;
    const int64_t end = warp_lower_bound(sorted, last + 1, tokens, k + 1, lane); // (k < rows <= 2^31 - 1)
    const int64_t n = (end - 1) / chunk - c + 1;                              // chunks of the run
    const int64_t per = (n + kWarps - 1) / kWarps;
    const int64_t from = min(warp * per, n), to = min(from + per, n);
    for (int64_t slab = blockIdx.y; slab * 32 * N < columns; slab += gridDim.y) {
        const int64_t column = (slab * 32 + lane) * N;
        const bool mine = column < columns;
        Sum<T> sum[N];
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] = 0;
        if (mine) {
#pragma unroll 8
            for (int64_t i = from; i < to; i++) {
                const Sum<T>* p = partial + (2 * (c + i) + (i == 0 ? 1 : 0)) * columns + column;
#pragma unroll
                for (int v = 0; v < N; v++) sum[v] += p[v];
            }
        }
#pragma unroll
        for (int v = 0; v < N; v++) joined[warp][lane * N + v] = sum[v];
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * N; i += kThreads) {
            const int64_t to_column = slab * 32 * N + i;
            if (to_column >= columns) break;
            Sum<T> all = 0;
            for (int w = 0; w < kWarps; w++) all += joined[w][i];
            grad_W[k * columns + to_column] = narrow<T>(all * scale);
        }
        __syncthreads();
    }
}

// Zeros for the rows that no token asks for: a block looks 64 rows up in the sorted tokens, a thread each, and clears those
// that are not there.
constexpr int kClearRows = 64;

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_clear(T* __restrict__ grad_W, const int32_t* __restrict__ sorted, int64_t tokens, int64_t rows,
                uint32_t packs, Divider by_packs) {
    __shared__ bool empty[kClearRows];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kClearRows;
    const int here = static_cast<int>(min(rows - row0, int64_t(kClearRows)));
    if (threadIdx.x < here) {
        const int32_t v = static_cast<int32_t>(row0 + threadIdx.x);
        int64_t lo = 0, hi = tokens;
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (__ldg(sorted + mid) < v) lo = mid + 1;
            else hi = mid;
        }
        empty[threadIdx.x] = lo >= tokens || __ldg(sorted + lo) != v;
    }
    __syncthreads();
    Pack<T, N> zero;
#pragma unroll
    for (int i = 0; i < N; i++) zero.v[i] = narrow<T>(0);
    for (int r = 0; r < here; r++) {
        if (!empty[r]) continue;
        for (uint32_t p = threadIdx.x; p < packs; p += kThreads)
            *reinterpret_cast<Pack<T, N>*>(grad_W + ((row0 + r) * packs + p) * N) = zero;
    }
}

const char* const kIndexNames[] = {"indices"};

void check_common(Array& table, const char* table_name, Array& rows, const char* rows_name, Array& indices,
                  const std::string& op) {
    check_floating(table.type, table_name, op);
    check_array(table, table_name, 2, table.type, op);
    check_array(rows, rows_name, 2, table.type, op);
    check_array(indices, "indices", 1, MOPS_B200_I32, op);
    check_size(rows.shape[0], rows_name, 0, indices.shape[0], "indices", 0, op);
    check_size(rows.shape[1], rows_name, 1, table.shape[1], table_name, 1, op);
    fits_int32(static_cast<size_t>(table.shape[0]), "the number of rows", op);
    fits_int32(static_cast<size_t>(table.shape[1]), "the number of columns", op);
    fits_int32(static_cast<size_t>(indices.shape[0]), "indices.shape[0]", op);
}

unsigned grid_of(int64_t blocks, const std::string& op) {
    fits_int32(static_cast<size_t>(blocks), "the number of blocks", op);
    return static_cast<unsigned>(blocks);
}

} // namespace

void embedding_lookup(Array output, Array W, Array indices, double scale) {
    const std::string op = "cuda_embedding_lookup";
    check_common(W, "W", output, "output", indices, op);
    check_rows(W, "W", op);
    check_output(output, "output", op);
    const int64_t tokens = indices.shape[0], columns = W.shape[1];
    if (tokens == 0 || columns == 0) return;
    Call call = begin_call();
    for_type(W.type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto width) {
            constexpr int N = decltype(width)::value;
            const int64_t packs = columns / N;
            const int64_t blocks = ceil_div(tokens * packs, kThreads * kPacksPerThread);
            embedding_rows<T, N><<<grid_of(blocks, op), kThreads, 0, call.stream>>>(
                static_cast<T*>(output.data), static_cast<const T*>(W.data), W.stride[0],
                static_cast<const int32_t*>(indices.data), indices.stride[0], tokens, W.shape[0],
                static_cast<uint32_t>(packs), Divider(static_cast<uint32_t>(packs)), static_cast<Sum<T>>(scale),
                call.status);
            note_kernel_f("embedding_rows<%s,%d>", array_type_name<T>(), N);
        };
        if (aligned16(W) && aligned16(output)) launch(std::integral_constant<int, kPack<T>>());
        else launch(std::integral_constant<int, 1>());
    });
    end_call(call, op.c_str(), kIndexNames, 1);
}

void embedding_lookup_vjp(Array grad_W, Array grad_output, Array indices, double scale, int64_t padding_index) {
    const std::string op = "cuda_embedding_lookup_vjp";
    if (grad_W.data == nullptr) return; // not asked for, or empty
    check_common(grad_W, "grad_W", grad_output, "grad_output", indices, op);
    check_rows(grad_output, "grad_output", op);
    check_output(grad_W, "grad_W", op);
    const int64_t tokens = indices.shape[0], rows = grad_W.shape[0], columns = grad_W.shape[1];
    if (padding_index < -1 || padding_index >= rows)
        throw std::runtime_error("padding_index " + std::to_string(padding_index) + " is not a row of W in " + op);
    if (indices.stride[0] != 1) throw std::runtime_error("indices must be contiguous in " + op);
    if (rows == 0 || columns == 0) return;
    Call call = begin_call();
    const size_t index_room = (static_cast<size_t>(tokens) * sizeof(int32_t) + 255) / 256 * 256;
    unsigned char* order = static_cast<unsigned char*>(scratch_alloc(call, 2 * index_room + 256));
    int32_t* sorted = reinterpret_cast<int32_t*>(order);
    int32_t* permutation = reinterpret_cast<int32_t*>(order + index_room);
    // tokens outside of the table and those of the padding row sort behind all others
    if (tokens > 0)
        sort_keys(call, sorted, permutation, static_cast<const int32_t*>(indices.data), tokens, rows,
                  static_cast<int32_t>(rows), static_cast<int32_t>(padding_index));
    for_type(grad_W.type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto width) {
            constexpr int N = decltype(width)::value;
            const int64_t packs = columns / N, slabs = ceil_div(columns, 32 * N);
            // Chunks as long as they can be while there are some 30 warps for each SM.
            int chunk = 256;
            while (chunk > 32 && ceil_div(tokens, chunk) * slabs < int64_t(sm_count(call.device)) * 32) chunk /= 2;
            const int64_t chunks = ceil_div(tokens, chunk);
            T* out = static_cast<T*>(grad_W.data);
            embedding_clear<T, N><<<grid_of(ceil_div(rows, kClearRows), op), kThreads, 0, call.stream>>>(
                out, sorted, tokens, rows, static_cast<uint32_t>(packs), Divider(static_cast<uint32_t>(packs)));
            if (tokens > 0) {
                Sum<T>* partial = static_cast<Sum<T>*>(
                    scratch_alloc(call, static_cast<size_t>(2 * chunks * columns) * sizeof(Sum<T>)));
                embedding_sums<T, N><<<grid_of(ceil_div(chunks * slabs, kWarps), op), kThreads, 0, call.stream>>>(
                    out, static_cast<const T*>(grad_output.data), grad_output.stride[0], sorted, permutation, tokens, rows,
                    columns, chunk, chunks, slabs, static_cast<Sum<T>>(scale), partial);
                if (chunks > 1)
                    embedding_join<T, N>
                        <<<dim3(grid_of(chunks, op), static_cast<unsigned>(std::min<int64_t>(slabs, 65535))), kThreads, 0,
                           call.stream>>>(out, sorted, tokens, rows, columns, chunk, static_cast<Sum<T>>(scale), partial);
                scratch_free(call, partial);
            }
            note_kernel_f("embedding_sums<%s,%d>", array_type_name<T>(), N);
        };
        if (aligned16(grad_W) && aligned16(grad_output)) launch(std::integral_constant<int, kPack<T>>());
        else launch(std::integral_constant<int, 1>());
    });
    scratch_free(call, order);
    end_call(call, op.c_str(), kIndexNames, 1);
}

} // namespace mops_b200
