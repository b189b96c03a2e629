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

// ------------------------------------------------------------------------------ forward
// The output is cut into packs of N values, rows one after the other, and a block takes 1024 packs in a row; so blocks have the same
// work whatever the width of a row. Bounded by memory: 65 536 tokens of 2048 columns in bf16 take 66 us, in which 93 MB
// are read and 268 MB written (5.4 TB/s); with a thread's loads one after the other and ordinary stores 95 us.
constexpr int kPacksPerThread = 4;

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_rows(T* __restrict__ output, const T* __restrict__ W, int64_t stride, const int32_t* __restrict__ indices,
               int64_t index_stride, int64_t tokens, int64_t rows, uint32_t packs, Divider by_packs, Sum<T> scale, Status st) {
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * kPacksPerThread);
    const int64_t t0 = first >> 32 ? first / packs : by_packs.divide(static_cast<uint32_t>(first));
    const uint32_t p0 = static_cast<uint32_t>(first - t0 * packs);
    // all indices, then all values: each load of a thread is on its way before the first is waited for
    int64_t token[kPacksPerThread];
    uint32_t pack[kPacksPerThread];
    int32_t row[kPacksPerThread];
#pragma unroll
    for (int k = 0; k < kPacksPerThread; k++) {
        const uint32_t at = p0 + k * kThreads + threadIdx.x;
        const uint32_t t = by_packs.divide(at);
        token[k] = t0 + t;
        pack[k] = at - t * packs;
        row[k] = __ldg(indices + min(token[k], tokens - 1) * index_stride);
    }
    Pack<T, N> value[kPacksPerThread];
#pragma unroll
    for (int k = 0; k < kPacksPerThread; k++) {
#pragma unroll
        for (int i = 0; i < N; i++) value[k].v[i] = narrow<T>(0);
        if (static_cast<uint32_t>(row[k]) < static_cast<uint64_t>(rows))
            value[k] = *reinterpret_cast<const Pack<T, N>*>(W + row[k] * stride + static_cast<int64_t>(pack[k]) * N);
    }
#pragma unroll
    for (int k = 0; k < kPacksPerThread; k++) {
        if (token[k] >= tokens) continue;
        if (static_cast<uint32_t>(row[k]) >= static_cast<uint64_t>(rows) && pack[k] == 0) report_bad_index(st, 0);
#pragma unroll
        for (int i = 0; i < N; i++) value[k].v[i] = narrow<T>(widen(value[k].v[i]) * scale);
        store_through(output + (token[k] * packs + pack[k]) * N, value[k]);
    }
}

// ------------------------------------------------------------------------------ gradient
// Few tokens: one block sorts them, in shared memory, while the others clear the rows of grad_W that no token asks for, which takes
// longer. Digits of up to nine bits (so that 2^18 rows take two passes), lowest first, every pass stable: a warp's keys in order, warps in order.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32, kOrderItems = 16;
constexpr int kFewTokens = kOrderThreads * kOrderItems;
struct OrderMemory {
    int32_t keys[kFewTokens];
    uint16_t values[kFewTokens];
    uint16_t counts[kOrderWarps][kDigits]; // then: how many of a digit earlier warps have
    int32_t of_warp[kDigits / 32], first[kDigits]; // of each digit
};
constexpr int kFlags = sizeof(OrderMemory); // rows that a block looks at together, a byte each

// The lanes whose digit is the caller's (of those that have one), by a ballot for each bit: a few instructions each, where __match_any_sync
// takes hundreds of clocks with all warps of an SM at it.
__device__ __forceinline__ unsigned lanes_with(int digit, bool in) {
    unsigned peers = __ballot_sync(kFullMask, in);
#pragma unroll
    for (int bit = 0; bit < kDigitBits; bit++) {
        const unsigned set = __ballot_sync(kFullMask, digit >> bit & 1);
        peers &= digit >> bit & 1 ? set : ~set;
    }
    return peers;
}

__device__ __forceinline__ void sort_few(OrderMemory& m, int32_t* __restrict__ sorted, int32_t* __restrict__ permutation,
                                         const int32_t* __restrict__ indices, int tokens, int32_t rows, int32_t dropped, int passes, int digit_bits, const Status& st) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rounds = (tokens + kOrderThreads - 1) / kOrderThreads, first = warp * rounds * 32 + lane;
    int32_t key[kOrderItems];
    uint32_t value[kOrderItems]; // where the key was; above that, the place among the warp's keys of its digit
#pragma unroll
    for (int r = 0; r < kOrderItems; r++) {
        const int at = first + r * 32;
        value[r] = at;
        key[r] = r < rounds && at < tokens ? __ldg(indices + at) : 0;
    }
    bool bad = false;
#pragma unroll
    for (int r = 0; r < kOrderItems; r++) {
        const bool outside = static_cast<uint32_t>(key[r]) >= static_cast<uint32_t>(rows);
        bad |= outside;
        if (outside || key[r] == dropped) key[r] = rows;
    }
    if (bad && rows > 0) report_bad_index(st, 0);
    const int mask = (1 << digit_bits) - 1;
    for (int pass = 0; pass < passes; pass++) {
        const int shift = digit_bits * pass;
        for (int i = tid; i < kOrderWarps * kDigits / 2; i += kOrderThreads) reinterpret_cast<uint32_t*>(m.counts)[i] = 0;
        __syncthreads();
        // each warp counts its digits
        constexpr int kSide = 2; // side by side
#pragma unroll
        for (int r0 = 0; r0 < kOrderItems; r0 += kSide) {
            if (r0 >= rounds) break;
            unsigned peers[kSide];
#pragma unroll
            for (int u = 0; u < kSide; u++) peers[u] = lanes_with(key[r0 + u] >> shift & mask, r0 + u < rounds && first + (r0 + u) * 32 < tokens);
#pragma unroll
            for (int u = 0; u < kSide; u++) {
                const int r = r0 + u, digit = key[r] >> shift & mask;
                const bool in = peers[u] >> lane & 1;
                const int rank = __popc(peers[u] & ((1u << lane) - 1));
                if (in) value[r] |= static_cast<uint32_t>(m.counts[warp][digit] + rank) << 16;
                __syncwarp();
                if (in && rank == 0) m.counts[warp][digit] += __popc(peers[u]);
                __syncwarp();
            }
        }
        __syncthreads();
        // where each warp's keys of a digit go: behind smaller digits, and behind earlier warps
        int total = 0, up_to = 0;
        if (tid < kDigits) {
#pragma unroll
            for (int w0 = 0; w0 < kOrderWarps; w0 += 16) {
                int n[16];
#pragma unroll
                for (int w = 0; w < 16; w++) n[w] = m.counts[w0 + w][tid];
#pragma unroll
                for (int w = 0; w < 16; w++) {
                    m.counts[w0 + w][tid] = static_cast<uint16_t>(total);
                    total += n[w];
                }
            }
            up_to = total;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(kFullMask, up_to, d);
                if (lane >= d) up_to += v;
            }
            if (lane == 31) m.of_warp[warp] = up_to;
        }
        __syncthreads();
        if (tid < kDigits) {
            int base = up_to - total;
            for (int w = 0; w < warp; w++) base += m.of_warp[w];
            m.first[tid] = base;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOrderItems; r++) {
            if (r >= rounds || first + r * 32 >= tokens) break;
            const int digit = key[r] >> shift & mask;
            const int to = m.first[digit] + m.counts[warp][digit] + (value[r] >> 16);
            m.keys[to] = key[r];
            m.values[to] = static_cast<uint16_t>(value[r]);
        }
        __syncthreads();
        if (pass == passes - 1) break;
#pragma unroll
        for (int r = 0; r < kOrderItems; r++) {
            const int at = first + r * 32;
            if (r < rounds && at < tokens) key[r] = m.keys[at], value[r] = m.values[at];
        }
    }
    for (int i = tid; i < tokens; i += kOrderThreads) sorted[i] = m.keys[i], permutation[i] = m.values[i];
}

// (16 384 tokens among 100 003 rows of 1024 columns in bf16: 35 us. The sort's two passes take 34, bound by the instructions and shared-memory accesses of one SM; the
// clearing of 170 MB, beside it, some 30.)
// Clears the rows [lo, hi) that no token asks for. A block marks in shared memory which ones are, kFlags rows at a time.
// It writes 16 bytes at a time wherever rows begin: what lies in several rows in one piece if all of them are empty. (487 tokens among 53 826 rows of 1586 columns in f32: 64 us; value
// by value 103.)
template <typename T>
__device__ __forceinline__ void clear_rows(unsigned char* flags, T* __restrict__ grad_W, const int32_t* __restrict__ indices, int tokens,
                                           int64_t lo, int64_t hi, int32_t dropped, uint32_t columns, const Divider& by_columns) {
    constexpr int N = kPack<T>;
    Pack<T, N> zero;
#pragma unroll
    for (int i = 0; i < N; i++) zero.v[i] = narrow<T>(0);
    for (int64_t row0 = lo; row0 < hi; row0 += kFlags) {
        const int here = static_cast<int>(min(hi - row0, int64_t(kFlags)));
        __syncthreads();
        for (int i = threadIdx.x; i < (here + 3) / 4; i += kOrderThreads) reinterpret_cast<uint32_t*>(flags)[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (int t = threadIdx.x; t < tokens; t += kOrderThreads) {
            const int32_t row = __ldg(indices + t);
            if (row >= row0 && row < row0 + here && row != dropped) flags[row - row0] = 1;
        }
        __syncthreads();
        // as many rows at a time as 32 bits do for
        const int group = max(1, static_cast<int>((1u << 30) / columns));
        for (int r0 = 0; r0 < here; r0 += group) {
            T* const to = grad_W + (row0 + r0) * columns;
            const uint32_t head = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to) % 16 / sizeof(T)); // values behind a multiple of 16 bytes
            const uint32_t end = head + static_cast<uint32_t>(min(group, here - r0)) * columns;
            for (uint32_t at = threadIdx.x * N; at < end; at += kOrderThreads * N) {
                const uint32_t first = max(at, head) - head, n = min(at + N, end) - head - first;
                uint32_t r = by_columns.divide(first), c = first - r * columns;
                bool empty = !flags[r0 + r];
                for (uint32_t next = r + 1, reach = columns - c; reach < n; reach += columns) empty = empty && !flags[r0 + next++];
                if (empty && n == N) {
                    store_through(to + first, zero);
                    continue;
                }
                for (uint32_t v = first; v < first + n; v++) {
                    if (!flags[r0 + r]) to[v] = zero.v[0];
                    if (++c == columns) c = 0, r++;
                }
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kOrderThreads, 1)
embedding_order(T* __restrict__ grad_W, int32_t* __restrict__ sorted, int32_t* __restrict__ permutation, const int32_t* __restrict__ indices,
                int tokens, int32_t rows, int32_t dropped, int passes, int digit_bits, uint32_t columns, Divider by_columns, Status st) {
    extern __shared__ __align__(16) unsigned char memory[];
    if (blockIdx.x == 0) {
        sort_few(*reinterpret_cast<OrderMemory*>(memory), sorted, permutation, indices, tokens, rows, dropped, passes, digit_bits, st);
    } else {
        const int64_t blocks = gridDim.x - 1, b = blockIdx.x - 1;
        clear_rows(memory, grad_W, indices, tokens, rows * b / blocks, rows * (b + 1) / blocks, dropped, columns, by_columns);
    }
}

// Many tokens are sorted by kernels of their own (sort.cu). Then a block looks 64 rows up in the sorted tokens, a thread each, and clears those
// that are not there.
constexpr int kClearRows = 64;
template <typename T>
__device__ __forceinline__ void clear_some_rows(int64_t row0, T* __restrict__ grad_W, const int32_t* __restrict__ sorted, int64_t tokens, int64_t rows,
                                                uint32_t columns) {
    __shared__ bool empty[kClearRows];
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
    constexpr int N = kPack<T>;
    Pack<T, N> zero;
#pragma unroll
    for (int i = 0; i < N; i++) zero.v[i] = narrow<T>(0);
    const uint32_t lane = threadIdx.x % 32;
    for (int r = threadIdx.x / 32; r < here; r += kWarps) {
        if (!empty[r]) continue;
        // up to the first multiple of 16 bytes, whole ones, and the rest
        T* const row = grad_W + (row0 + r) * columns;
        const uint32_t before = min(static_cast<uint32_t>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)), columns);
        const uint32_t whole = (columns - before) / N * N;
        if (lane < before) row[lane] = zero.v[0];
        for (uint32_t c = lane * N; c < whole; c += 32 * N) store_through(row + before + c, zero);
        for (uint32_t c = before + whole + lane; c < columns; c += 32) row[c] = zero.v[0];
    }
}

// The sorted tokens are cut into chunks. A warp takes a chunk and a slab of 32 N columns and adds up the rows of grad_output, token
// by token. A run of equal tokens that lies inside a chunk goes to its row of grad_W at once; of one
// that a chunk's end cuts, each chunk leaves a partial sum (place 0: the run had begun before the chunk;
// place 1: it begins in it and goes on after it), and embedding_join adds those up. Bounded by memory: 200 003 tokens of 256 columns in f32 43.5 us, 4.7 TB/s.
// The first clear_blocks blocks clear rows instead.
constexpr int kRowsInFlight = 8; // loads of a warp under way

// (Partial sums are vectors of whole packs: slabs * 32 N columns.)
template <typename S, int N> struct alignas(N * sizeof(S) < 16 ? N * sizeof(S) : 16) Sums {
    S v[N];
};

// Keeps loaded packs as they are up to here.
template <typename T, int N, int M> __device__ __forceinline__ void keep_packed(Pack<T, N> (&v)[M]) {
    if constexpr (N * sizeof(T) % 4 == 0) {
#pragma unroll
        for (int u = 0; u < M; u++) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&v[u]);
#pragma unroll
            for (int i = 0; i < static_cast<int>(N * sizeof(T) / 4); i++) asm volatile("" : "+r"(w[i]));
        }
    } else {
#pragma unroll
        for (int u = 0; u < M; u++) asm volatile("" : "+h"(*reinterpret_cast<uint16_t*>(&v[u])));
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 4)
embedding_sums(T* __restrict__ grad_W, const T* __restrict__ grad_output, int64_t stride,
               const int32_t* __restrict__ sorted, const int32_t* __restrict__ permutation, int64_t tokens, int64_t rows,
               int64_t columns, int chunk, int64_t chunks, int64_t slabs, Sum<T> scale, Sums<Sum<T>, N>* __restrict__ partial,
               int64_t clear_blocks) {
    if (blockIdx.x < clear_blocks) {
        clear_some_rows(blockIdx.x * int64_t(kClearRows), grad_W, sorted, tokens, rows, static_cast<uint32_t>(columns));
        return;
    }
    const int lane = threadIdx.x & 31;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) - clear_blocks) * kWarps + (threadIdx.x >> 5);
    if (unit >= chunks * slabs) return;
    const int64_t c = unit / slabs, slab = unit - c * slabs;
    const int64_t column = (slab * 32 + lane) * N;
    const bool mine = column < columns;
    const T* from_column = grad_output + (mine ? column : 0);
    const int64_t lo = c * chunk, hi = min(lo + chunk, tokens);
    bool begun_before = true; // the run at hand began before the chunk
    Sums<Sum<T>, N> sum;
#pragma unroll
    for (int i = 0; i < N; i++) sum.v[i] = 0;
    for (int64_t base = lo; base < hi; base += 32) {
        const int n = static_cast<int>(min(hi - base, int64_t(32)));
        // the keys of 32 entries, of the one in front of them and of the one behind them
        const int32_t key = base + lane < tokens ? __ldg(sorted + base + lane) : -1;
        const int32_t from = lane < n ? __ldg(permutation + base + lane) : 0;
        int32_t before = __shfl_up_sync(kFullMask, key, 1), after = __shfl_down_sync(kFullMask, key, 1);
        if (lane == 0) before = base > 0 ? __ldg(sorted + base - 1) : -1;
        if (lane == 31) after = base + 32 < tokens ? __ldg(sorted + base + 32) : -1;
        // entries that begin a run and that end one, and those that give no gradient (sorted behind all others)
        const unsigned begins = __ballot_sync(kFullMask, before != key), ends = __ballot_sync(kFullMask, after != key);
        const int valid = __popc(__ballot_sync(kFullMask, lane < n && key < rows));
        const int64_t offset = from * stride; // (of lane's entry)
        const uint32_t offset_lo = static_cast<uint32_t>(offset), offset_hi = static_cast<uint32_t>(offset >> 32);
        auto leave = [&](int j) { // the run ends with entry j, or the chunk does
            if (begun_before || !(ends >> j & 1)) {
                partial[((2 * c + (begun_before ? 0 : 1)) * slabs + slab) * 32 + lane] = sum;
                return;
            }
            const int64_t k = __shfl_sync(kFullMask, key, j);
            Pack<T, N> out;
#pragma unroll
            for (int i = 0; i < N; i++) out.v[i] = narrow<T>(sum.v[i] * scale);
            if (mine) *reinterpret_cast<Pack<T, N>*>(grad_W + k * columns + column) = out;
        };
        auto restart = [&] {
            begun_before = false;
#pragma unroll
            for (int i = 0; i < N; i++) sum.v[i] = 0;
        };
        for (int j0 = 0; j0 < valid; j0 += kRowsInFlight) {
            Pack<T, N> value[kRowsInFlight];
#pragma unroll
            for (int u = 0; u < kRowsInFlight; u++) { // (the last entry again where there are no more, and the first column)
                const int j = min(j0 + u, valid - 1);
                const int64_t at = static_cast<int64_t>(static_cast<uint64_t>(__shfl_sync(kFullMask, offset_hi, j)) << 32 |
                                                        __shfl_sync(kFullMask, offset_lo, j));
                value[u] = *reinterpret_cast<const Pack<T, N>*>(from_column + at);
            }
            keep_packed(value); // (else each load is waited for, to be widened, before the next)
            const unsigned group = (1u << kRowsInFlight) - 1;
            if (j0 + kRowsInFlight <= valid && !((begins >> j0 >> 1 | ends >> j0) & group >> 1)) { // one run
                if (begins >> j0 & 1) restart();
#pragma unroll
                for (int u = 0; u < kRowsInFlight; u++)
#pragma unroll
                    for (int i = 0; i < N; i++) sum.v[i] += widen(value[u].v[i]);
                const int j = j0 + kRowsInFlight - 1;
                if (ends >> j & 1 || base + j == hi - 1) leave(j);
                continue;
            }
#pragma unroll
            for (int u = 0; u < kRowsInFlight; u++) {
                const int j = j0 + u;
                if (j >= valid) break;
                if (begins >> j & 1) restart();
#pragma unroll
                for (int i = 0; i < N; i++) sum.v[i] += widen(value[u].v[i]);
                if (ends >> j & 1 || base + j == hi - 1) leave(j);
            }
        }
        if (valid < n) return;
    }
}

// Adds up the partial sums of the runs that begin in a chunk and go on after it. A warp looks at a chunk; a run of a few chunks it adds up by itself, one of
// more than kWarps chunks the warps of the block do together, each a range of them (there is one at most: it ends behind the block's chunks).
// (With a block for each chunk it was the blocks that cost time: 14 us for the 95 runs of 200 003 tokens, 256 columns in f32; 9.7 us so.)
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
embedding_join(T* __restrict__ grad_W, const int32_t* __restrict__ sorted, int64_t tokens, int64_t rows, int64_t columns,
               int chunk, int64_t chunks, int64_t slabs, Sum<T> scale, const Sums<Sum<T>, N>* __restrict__ partial) {
    __shared__ Sums<Sum<T>, N> joined[kWarps][32];
    __shared__ int64_t long_run[2]; // its first chunk (-1: there is none), and how many chunks it has
    __shared__ int32_t long_key;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) long_run[0] = -1;
    __syncthreads();
    // the sum over chunks from <= i < to of the run that begins in chunk c
    auto add = [&](int64_t c, int64_t slab, int64_t from, int64_t to) {
        Sums<Sum<T>, N> sum;
#pragma unroll
        for (int i = 0; i < N; i++) sum.v[i] = 0;
        auto part = [&](int64_t i) { return partial[((2 * (c + i) + (i == 0 ? 1 : 0)) * slabs + slab) * 32 + lane]; };
        int64_t i = from;
        constexpr int kAtOnce = 64 / N < 16 ? 64 / N : 16; // (a long run is a chain of these loads)
        for (; i + kAtOnce <= to; i += kAtOnce) {
            Sums<Sum<T>, N> v[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) v[u] = part(i + u);
#pragma unroll
            for (int u = 0; u < kAtOnce; u++)
#pragma unroll
                for (int x = 0; x < N; x++) sum.v[x] += v[u].v[x];
        }
        for (; i < to; i++) {
            const Sums<Sum<T>, N> v = part(i);
#pragma unroll
            for (int x = 0; x < N; x++) sum.v[x] += v.v[x];
        }
        return sum;
    };
    auto store = [&](int64_t k, int64_t slab, const Sums<Sum<T>, N>& sum) {
        const int64_t column = (slab * 32 + lane) * N;
        Pack<T, N> out;
#pragma unroll
        for (int i = 0; i < N; i++) out.v[i] = narrow<T>(sum.v[i] * scale);
        if (column < columns) *reinterpret_cast<Pack<T, N>*>(grad_W + k * columns + column) = out;
    };
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kWarps + warp, lo = c * chunk, last = lo + chunk - 1;
    if (c < chunks && last + 1 < tokens) {
        const int32_t k = __ldg(sorted + last), next = __ldg(sorted + last + 1), before = lo > 0 ? __ldg(sorted + lo - 1) : -1;
        if (k < rows && next == k && before != k) {
            // its end: mostly in the next chunk
            const int64_t near = min(last + 1 + 32, tokens);
            const bool same = last + 1 + lane < near && __ldg(sorted + last + 1 + lane) == k;
            const unsigned run = __ballot_sync(kFullMask, same);
            const int64_t end = run == kFullMask ? warp_lower_bound(sorted, near, tokens, k + 1, lane) // (k < rows <= 2^31 - 1)
                                                 : last + 1 + __popc(run);
            const int64_t n = (end - 1) / chunk - c + 1; // chunks of the run
            if (n <= kWarps)
                for (int64_t slab = blockIdx.y; slab < slabs; slab += gridDim.y) store(k, slab, add(c, slab, 0, n));
            else if (lane == 0)
                long_run[0] = c, long_run[1] = n, long_key = k;
        }
    }
    __syncthreads();
    if (long_run[0] < 0) return;
    const int64_t n = long_run[1], per = (n + kWarps - 1) / kWarps;
    for (int64_t slab = blockIdx.y; slab < slabs; slab += gridDim.y) {
        joined[warp][lane] = add(long_run[0], slab, min(warp * per, n), min((warp + 1) * per, n));
        __syncthreads();
        if (warp == 0) {
            Sums<Sum<T>, N> sum = joined[0][lane];
#pragma unroll
            for (int w = 1; w < kWarps; w++)
#pragma unroll
                for (int x = 0; x < N; x++) sum.v[x] += joined[w][lane].v[x]; // (zeros of those that had none)
            store(long_key, slab, sum);
        }
        __syncthreads();
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

// Calls `launch` with the number of values, 16 bytes at most, that rows of both arrays are made of (150 517 tokens, 460 columns in bf16, a step: 123 us in packs of
// four values, 268 one by one).
template <typename T, typename F> void widest(const Array& a, const Array& b, F&& launch) {
    auto in_packs = [&](int bytes) { return aligned(a, bytes) && aligned(b, bytes); };
    if (in_packs(16)) return launch(std::integral_constant<int, kPack<T>>());
    if constexpr (kPack<T> > 2)
        if (in_packs(8)) return launch(std::integral_constant<int, kPack<T> / 2>());
    if constexpr (kPack<T> > 4)
        if (in_packs(4)) return launch(std::integral_constant<int, kPack<T> / 4>());
    launch(std::integral_constant<int, 1>());
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
        widest<T>(W, output, launch);
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
    Scratch order(call, 2 * index_room + 256);
    int32_t* sorted = order.as<int32_t>();
    int32_t* permutation = reinterpret_cast<int32_t*>(order.as<unsigned char>() + index_room);
    const int32_t* given = static_cast<const int32_t*>(indices.data);
    for_type(grad_W.type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto width) {
            constexpr int N = decltype(width)::value;
            const int64_t packs = columns / N, slabs = ceil_div(columns, 32 * N);
            T* out = static_cast<T*>(grad_W.data);
            // tokens outside of the table and those of the padding row sort behind all others
            int64_t clear_blocks = ceil_div(rows, kClearRows);
            if (tokens <= kFewTokens) {
                int bits = 1;
                while ((int64_t(1) << bits) < rows + 1) bits++;
                const int passes = (bits + kDigitBits - 1) / kDigitBits;
                auto kernel = embedding_order<T>;
                allow_dynamic_smem(kernel, call.device, sizeof(OrderMemory));
                const int64_t blocks = std::min<int64_t>(ceil_div(rows * columns, 4 * kOrderThreads * kPack<T>), sm_count(call.device) - 1);
                kernel<<<grid_of(1 + blocks, op), kOrderThreads, sizeof(OrderMemory), call.stream>>>(
                    out, sorted, permutation, given, static_cast<int>(tokens), static_cast<int32_t>(rows), static_cast<int32_t>(padding_index),
                    passes, (bits + passes - 1) / passes, static_cast<uint32_t>(columns), Divider(static_cast<uint32_t>(columns)), call.status);
                note_kernel_f("embedding_order<%s>", array_type_name<T>());
                clear_blocks = 0;
                if (tokens == 0) return;
            } else {
                sort_keys(call, sorted, permutation, given, tokens, rows, static_cast<int32_t>(rows), static_cast<int32_t>(padding_index));
            }
            // Chunks such that all warps are resident at once, 32 on each SM (200 003 tokens, 256 columns in f32: chunks of 96, 43.5 us; of 64, of which a third of an SM's
            // warps wait for the others to end, 45); no longer than 256, for many columns, and no shorter than 16.
            const int64_t of_warp = ceil_div(tokens * slabs, int64_t(sm_count(call.device)) * 32);
            const int chunk = static_cast<int>(std::min<int64_t>(ceil_div(of_warp, 16) * 16, 256));
            const int64_t chunks = ceil_div(tokens, chunk);
            using P = Sums<Sum<T>, N>;
            Scratch sums(call, static_cast<size_t>(2 * chunks * slabs * 32) * sizeof(P));
            P* partial = sums.as<P>();
            embedding_sums<T, N><<<grid_of(clear_blocks + ceil_div(chunks * slabs, kWarps), op), kThreads, 0, call.stream>>>(
                out, static_cast<const T*>(grad_output.data), grad_output.stride[0], sorted, permutation, tokens, rows,
                columns, chunk, chunks, slabs, static_cast<Sum<T>>(scale), partial, clear_blocks);
            if (chunks > 1)
                embedding_join<T, N>
                    <<<dim3(grid_of(ceil_div(chunks, kWarps), op), static_cast<unsigned>(std::min<int64_t>(slabs, 65535))), kThreads, 0, call.stream>>>(
                        out, sorted, tokens, rows, columns, chunk, chunks, slabs, static_cast<Sum<T>>(scale), partial);
            sums.free();
            note_kernel_f("embedding_sums<%s,%d>", array_type_name<T>(), N);
        };
        widest<T>(grad_W, grad_output, launch);
    });
    order.free();
    end_call(call, op.c_str(), kIndexNames, 1);
}

} // namespace mops_b200
