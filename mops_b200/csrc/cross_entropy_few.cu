// linear_cross_entropy of a few rows in f16, bf16 and f32: how likely the tokens in flight were.
//
// The table is all that is moved, once. A warp takes 16 of its rows at a time, whose values go from memory straight to the operands of matrix instructions (16 of the table's rows by 8 of A's): a lane has 8
// neighbours of each row, and as the order of a sum's terms is free, A is read from shared memory in the order that this gives. No row of the table passes through shared memory, none has to begin
// anywhere near the others. Sums of exponentials are kept by the lanes from one unit of 16 rows to the next, as in cross_entropy_mma.cu, and joined for the block at the end.
//
// Bound by memory: 8 rows of 50 021 x 1024 (102 MB, 16 us) take 20 us, of 400 003 x 1024 129 us (6.3 TB/s); a kernel that fetched tiles of 128 rows of the table for tcgen05.mma 26 and 154, as each tile's
// rows were read 128 bytes at a time and a third round of tiles did not fill the SMs.
#include "block_ops.hpp"
#include "loss_rows.cuh"
#include "pack.hpp"

namespace mops_b200 {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kFewThreads = 512, kFewWarps = kFewThreads / 32;
constexpr int kUnitRows = 16, kFewDepth = 32; // of the table; of a step
constexpr int kMostFewBytes = 200 * 1024;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF16> __device__ __forceinline__ void multiply16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

struct FewOperand { // rows of 16 bits, and where they begin and end
    const uint16_t* data;
    int64_t stride, rows;
    const unsigned char *begin, *end;
};

// kTiles: of 8 rows of A. The table's rows begin on multiples of 16 bytes. split: so many warps of a block have a part of a unit's depth each (a power of 2; more than 1 only where every unit has such warps).
template <bool BF16, int kTiles>
__global__ void __launch_bounds__(kFewThreads, 1)
loss_few(PartSum<float>* __restrict__ parts, float* __restrict__ at_target, const FewOperand A, const FewOperand W, int depth, const int32_t* __restrict__ targets, float scale,
         float scale2, int row_bytes, int split) {
    extern __shared__ __align__(16) unsigned char rows_of_A[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int chunks = (depth + kFewDepth - 1) / kFewDepth, own_chunks = (chunks + split - 1) / split, part = warp & (split - 1);
    const int chunk0 = min(part * own_chunks, chunks), chunk1 = min(chunk0 + own_chunks, chunks);
    // (neighbouring units go to different blocks: the last ones are spread over all)
    const int64_t first = static_cast<int64_t>(warp / split) * gridDim.x + blockIdx.x;
    if (first * kUnitRows < W.rows) // (under way while A is read)
        for (int i = 0; i < kUnitRows; i++)
            for (int c = chunk0 * kFewDepth + lane * 64; c < min(chunk1 * kFewDepth, depth); c += 32 * 64)
                asm volatile("prefetch.global.L2 [%0];\n" ::"l"(W.data + min(first * kUnitRows + i, W.rows - 1) * W.stride + c));
    for (int i = warp; i < kTiles * 8; i += kFewWarps) // zeros where there is nothing
        for (int c = lane; c < chunks * 4; c += 32) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (i < A.rows && c * 8 < depth) v = load_anywhere<__half>(reinterpret_cast<const __half*>(A.data) + i * A.stride + c * 8, depth - c * 8, A.begin, A.end);
            *reinterpret_cast<uint4*>(rows_of_A + i * row_bytes + c * 16) = v;
        }
    float4* const of_parts = reinterpret_cast<float4*>(rows_of_A + kTiles * 8 * row_bytes); // (if there are parts)
    int target[kTiles][2];
    float top[kTiles][2], sum[kTiles][2]; // of x log2(e)
#pragma unroll
    for (int j = 0; j < kTiles; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = j * 8 + 2 * t + e;
            target[j][e] = i < A.rows ? targets[i] : -1;
            top[j][e] = -INFINITY, sum[j][e] = 0;
        }
    __syncthreads();
    const unsigned char* const own = rows_of_A + g * row_bytes + t * 16;

    for (int64_t unit = first;; unit += static_cast<int64_t>(kFewWarps) * gridDim.x) {
        const bool there = unit * kUnitRows < W.rows;
        if (!there && split == 1) break;
        const int64_t v[2] = {unit * kUnitRows + g, unit * kUnitRows + g + 8};
        const uint16_t* const p[2] = {W.data + min(v[0], W.rows - 1) * W.stride + t * 8, W.data + min(v[1], W.rows - 1) * W.stride + t * 8};
        float x[kTiles][4] = {};
        auto steps = [&](int c, auto many, auto whole) {
            constexpr int kMany = decltype(many)::value;
            uint4 w[kMany][2];
#pragma unroll
            for (int k = 0; k < kMany; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int d = (c + k) * kFewDepth;
                    if constexpr (decltype(whole)::value) w[k][h] = load_once(p[h] + d);
                    else if (d + t * 8 < depth) w[k][h] = load_anywhere<__half>(reinterpret_cast<const __half*>(p[h]) + d, depth - d - t * 8, W.begin, W.end);
                    else w[k][h] = make_uint4(0, 0, 0, 0);
                }
#pragma unroll
            for (int k = 0; k < kMany; k++)
#pragma unroll
                for (int j = 0; j < kTiles; j++) {
                    const uint4 q = *reinterpret_cast<const uint4*>(own + j * 8 * row_bytes + (c + k) * kFewDepth * 2);
                    multiply16<BF16>(x[j], w[k][0].x, w[k][1].x, w[k][0].y, w[k][1].y, q.x, q.y);
                    multiply16<BF16>(x[j], w[k][0].z, w[k][1].z, w[k][0].w, w[k][1].w, q.z, q.w);
                }
        };
        if (there) {
            const int whole = min(chunk1, depth / kFewDepth);
            int c = chunk0;
            for (; c + 8 <= whole; c += 8) steps(c, std::integral_constant<int, 8>(), std::true_type());
            for (; c + 2 <= whole; c += 2) steps(c, std::integral_constant<int, 2>(), std::true_type());
            for (; c < chunk1; c++) steps(c, std::integral_constant<int, 1>(), std::false_type());
        }
        if (split > 1) { // the only unit
            float4* const to = of_parts + warp * kTiles * 32 + lane;
#pragma unroll
            for (int j = 0; j < kTiles; j++) to[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
            __syncthreads();
            if (!there || part > 0) break;
#pragma unroll 1
            for (int q = 1; q < split; q++)
#pragma unroll
                for (int j = 0; j < kTiles; j++) {
                    const float4 more = to[(q * kTiles + j) * 32];
                    x[j][0] += more.x, x[j][1] += more.y, x[j][2] += more.z, x[j][3] += more.w;
                }
        }
#pragma unroll
        for (int j = 0; j < kTiles; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float own_x[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    own_x[h] = v[h] < W.rows ? x[j][2 * h + e] : -INFINITY;
                    if (v[h] < W.rows && v[h] == target[j][e]) at_target[j * 8 + 2 * t + e] = own_x[h] * scale;
                }
                const float now = fmaxf(top[j][e], fmaxf(own_x[0], own_x[1]) * scale2), base = PartSum<float>::from(now);
                const float before = top[j][e] == -INFINITY ? sum[j][e] : sum[j][e] * exp2_fast(PartSum<float>::from(top[j][e]) - base);
                sum[j][e] = before + (exp2_fast(fmaf(own_x[0], scale2, -base)) + exp2_fast(fmaf(own_x[1], scale2, -base)));
                top[j][e] = now;
            }
        if (split > 1) break;
    }
    __shared__ PartSum<float> of_warp[kFewWarps][kTiles * 8];
#pragma unroll
    for (int j = 0; j < kTiles; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            PartSum<float> all{top[j][e] * kLn2, sum[j][e]};
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                const PartSum<float> other{__shfl_xor_sync(kFullMask, all.top, d), __shfl_xor_sync(kFullMask, all.sum, d)};
                all.join(other);
            }
            if (g == 0) of_warp[warp][j * 8 + 2 * t + e] = all;
        }
    __syncthreads();
    if (threadIdx.x < A.rows) {
        PartSum<float> all = of_warp[0][threadIdx.x];
#pragma unroll 1
        for (int w = 1; w < kFewWarps; w++) all.join(of_warp[w][threadIdx.x]);
        parts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = all;
    }
}

// ---- f32, by the ordinary units: a warp takes 16 of the table's rows, eight lanes to four of them, kVector neighbours to a lane at a time. 8 rows of A with 50 021 x 1024
// (205 MB, 31 us): 49 us, on tensor cores in three parts 94; 16 rows 87 and 94; 5 with 104 534 x 146 19 us, by a product into memory and a pass over it 72. Reading A from shared memory takes as long as the
// products, which wait for memory in between: fetching a warp's next rows ahead to L2 costs more (54 us) than it gives.
template <int kVector> struct FewVector {
    float v[kVector];
    __device__ __forceinline__ void load(const float* p) {
        if constexpr (kVector == 4) {
            const uint4 w = load_once(reinterpret_cast<const uint16_t*>(p));
            v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
        } else if constexpr (kVector == 2) {
            const float2 w = __ldg(reinterpret_cast<const float2*>(p));
            v[0] = w.x, v[1] = w.y;
        } else {
            v[0] = __ldg(p);
        }
    }
    __device__ __forceinline__ void load_shared(const float* p) {
        if constexpr (kVector == 4) {
            const float4 w = *reinterpret_cast<const float4*>(p);
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else if constexpr (kVector == 2) {
            const float2 w = *reinterpret_cast<const float2*>(p);
            v[0] = w.x, v[1] = w.y;
        } else {
            v[0] = *p;
        }
    }
};
struct FewOperand32 {
    const float* data;
    int64_t stride, rows;
};

// kTiles: of 8 rows of A. split: as in loss_few.
template <int kTiles, int kVector>
__global__ void __launch_bounds__(kFewThreads, 1)
loss_few32(PartSum<float>* __restrict__ parts, float* __restrict__ at_target, const FewOperand32 A, const FewOperand32 W, int depth, const int32_t* __restrict__ targets, float scale,
           int row_values, int split) {
    constexpr int kRows = kTiles * 8, kStep = 8 * kVector, kMany = kVector == 4 ? (kTiles == 1 ? 4 : 2) : 4;
    extern __shared__ __align__(16) float values_of_A[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 3, t = lane & 7;
    const int chunks = (depth + kStep - 1) / kStep, own_chunks = (chunks + split - 1) / split, part = warp & (split - 1);
    const int chunk0 = min(part * own_chunks, chunks), chunk1 = min(chunk0 + own_chunks, chunks);
    const int64_t first = static_cast<int64_t>(warp / split) * gridDim.x + blockIdx.x;
    for (int i = warp; i < kRows; i += kFewWarps)
        for (int c = lane; c < row_values; c += 32) values_of_A[i * row_values + c] = i < A.rows && c < depth ? A.data[i * A.stride + c] : 0.f;
    float* const of_parts = values_of_A + kRows * row_values; // (if there are parts)
    int target[kTiles];
    PartSum<float> all[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; j++) target[j] = j * 8 + t < A.rows ? targets[j * 8 + t] : -1, all[j] = PartSum<float>::none();
    __syncthreads();
    const float* const own = values_of_A + t * kVector;

    for (int64_t unit = first;; unit += static_cast<int64_t>(kFewWarps) * gridDim.x) {
        const bool there = unit * kUnitRows < W.rows;
        if (!there && split == 1) break;
        const float* p[4];
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = W.data + min(unit * kUnitRows + g + 4 * k, W.rows - 1) * W.stride + t * kVector;
        float sum[4][kRows] = {};
        auto steps = [&](int c, auto many, bool whole) {
            constexpr int kNow = decltype(many)::value;
            FewVector<kVector> w[kNow][4];
#pragma unroll
            for (int q = 0; q < kNow; q++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int d = (c + q) * kStep;
                    if (whole) {
                        w[q][k].load(p[k] + d);
                    } else {
#pragma unroll
                        for (int e = 0; e < kVector; e++) w[q][k].v[e] = d + t * kVector + e < depth ? __ldg(p[k] + d + e) : 0.f;
                    }
                }
#pragma unroll
            for (int q = 0; q < kNow; q++)
#pragma unroll
                for (int i = 0; i < kRows; i++) {
                    FewVector<kVector> a;
                    a.load_shared(own + i * row_values + (c + q) * kStep);
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int e = 0; e < kVector; e++) sum[k][i] = fmaf(w[q][k].v[e], a.v[e], sum[k][i]);
                }
        };
        if (there) {
            const int whole = min(chunk1, depth / kStep);
            int c = chunk0;
            for (; c + kMany <= whole; c += kMany) steps(c, std::integral_constant<int, kMany>(), true);
            for (; c < chunk1; c++) steps(c, std::integral_constant<int, 1>(), c < whole);
        }
        // of each row of A the sums of eight lanes, to the lane of that number
        float x[kTiles][4];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < kTiles; j++) {
                float four[4], two[2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float low = sum[k][j * 8 + i], high = sum[k][j * 8 + i + 4];
                    four[i] = (t & 4 ? high : low) + __shfl_xor_sync(kFullMask, t & 4 ? low : high, 4);
                }
#pragma unroll
                for (int i = 0; i < 2; i++) two[i] = (t & 2 ? four[i + 2] : four[i]) + __shfl_xor_sync(kFullMask, t & 2 ? four[i] : four[i + 2], 2);
                x[j][k] = (t & 1 ? two[1] : two[0]) + __shfl_xor_sync(kFullMask, t & 1 ? two[0] : two[1], 1);
            }
        if (split > 1) { // the only unit
            float* const to = of_parts + warp * kTiles * 4 * 32 + lane;
#pragma unroll
            for (int j = 0; j < kTiles; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) to[(j * 4 + k) * 32] = x[j][k];
            __syncthreads();
            if (!there || part > 0) break;
#pragma unroll 1
            for (int q = 1; q < split; q++)
#pragma unroll
                for (int j = 0; j < kTiles; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) x[j][k] += to[((q * kTiles + j) * 4 + k) * 32];
        }
#pragma unroll
        for (int j = 0; j < kTiles; j++) {
            PartSum<float> now{-INFINITY, 0.f};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int64_t v = unit * kUnitRows + g + 4 * k;
                if (v < W.rows && v == target[j]) at_target[j * 8 + t] = x[j][k] * scale;
                x[j][k] = v < W.rows ? x[j][k] : -INFINITY;
                now.top = fmaxf(now.top, x[j][k] * scale);
            }
            const float base = PartSum<float>::from(now.top);
#pragma unroll
            for (int k = 0; k < 4; k++) now.sum += expf(fmaf(x[j][k], scale, -base));
            all[j].join(now);
        }
        if (split > 1) break;
    }
    __shared__ PartSum<float> of_warp[kFewWarps][kRows];
#pragma unroll
    for (int j = 0; j < kTiles; j++) {
#pragma unroll
        for (int d = 8; d < 32; d <<= 1) {
            const PartSum<float> other{__shfl_xor_sync(kFullMask, all[j].top, d), __shfl_xor_sync(kFullMask, all[j].sum, d)};
            all[j].join(other);
        }
        if (g == 0) of_warp[warp][j * 8 + t] = all[j];
    }
    __syncthreads();
    if (threadIdx.x < A.rows) {
        PartSum<float> whole = of_warp[0][threadIdx.x];
#pragma unroll 1
        for (int w = 1; w < kFewWarps; w++) whole.join(of_warp[w][threadIdx.x]);
        parts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = whole;
    }
}

int few_row_values(int64_t depth) { return static_cast<int>(ceil_div(depth, 32) * 32); }

FewOperand operand_of(const Array& a) {
    const unsigned char* begin = static_cast<const unsigned char*>(a.data);
    return {static_cast<const uint16_t*>(a.data), a.stride[0], a.shape[0], begin, begin + ((a.shape[0] - 1) * a.stride[0] + a.shape[1]) * 2};
}

// bytes of a row of A in shared memory: eight lanes that read 16 bytes each, of two rows, find them in different banks
int few_row_bytes(int64_t depth) {
    const int64_t bytes = ceil_div(depth, kFewDepth) * kFewDepth * 2;
    return static_cast<int>(bytes % 128 == 0 ? bytes + 64 : bytes);
}

} // namespace

// (with more than 16 rows what is read from shared memory is the bound: 24 rows of 50 021 x 4096 138 us, 91 by the kernel of cross_entropy_mma.cu; 16 of them 90 and 90, 16 rows of 50 021 x 1024 23 and 26)
bool few_loss_rows(const LossProblem& p) {
    const int64_t n = p.A.shape[0];
    if (p.A.type == MOPS_B200_F32) return n <= 16 && p.A.shape[1] > 0 && p.A.shape[1] <= kMostFewBytes / 32 && ceil_div(n, 8) * 32 * few_row_values(p.A.shape[1]) <= kMostFewBytes;
    return n <= 16 && p.A.shape[1] <= kMostFewBytes / 16 && ceil_div(n, 8) * 8 * few_row_bytes(p.A.shape[1]) <= kMostFewBytes && p.W.stride[0] % 8 == 0 &&
           reinterpret_cast<uintptr_t>(p.W.data) % 16 == 0;
}

static void launch_few(const Call& call, const LossProblem& p, unsigned blocks, PartSum<float>* parts, float* at_target) {
    const int tiles = static_cast<int>(ceil_div(p.A.shape[0], 8));
    int split = 1; // (8 rows of 3000 x 4096: 14.0 us, 18.8 with a warp to a unit)
    while (split < kFewWarps && ceil_div(p.W.shape[0], kUnitRows) * 2 * split <= int64_t(blocks) * kFewWarps && p.A.shape[1] >= 2 * split * 4 * kFewDepth) split *= 2;
    if (p.A.type == MOPS_B200_F32) {
        const FewOperand32 A{static_cast<const float*>(p.A.data), p.A.stride[0], p.A.shape[0]}, W{static_cast<const float*>(p.W.data), p.W.stride[0], p.W.shape[0]};
        const int values = few_row_values(p.A.shape[1]);
        const size_t shared = (static_cast<size_t>(tiles * 8 * values) + (split > 1 ? static_cast<size_t>(tiles) * 4 * kFewThreads : 0)) * sizeof(float);
        auto launch = [&](auto most, auto vector) {
            auto kernel = loss_few32<decltype(most)::value, decltype(vector)::value>;
            allow_dynamic_smem(reinterpret_cast<const void*>(kernel), call.device, shared);
            kernel<<<blocks, kFewThreads, shared, call.stream>>>(parts, at_target, A, W, static_cast<int>(p.A.shape[1]), static_cast<const int32_t*>(p.targets.data),
                                                                 static_cast<float>(p.scale), values, split);
            note_kernel_f("loss_few<f32,%d,%d>", tiles, static_cast<int>(vector));
        };
        auto by_rows = [&](auto vector) {
            if (tiles == 1) launch(std::integral_constant<int, 1>(), vector);
            else launch(std::integral_constant<int, 2>(), vector);
        };
        const uintptr_t place = reinterpret_cast<uintptr_t>(W.data) | static_cast<uintptr_t>(W.stride * 4);
        if (place % 16 == 0) by_rows(std::integral_constant<int, 4>());
        else if (place % 8 == 0) by_rows(std::integral_constant<int, 2>());
        else by_rows(std::integral_constant<int, 1>());
        MOPS_CUDA_OK(cudaGetLastError());
        return;
    }
    const int bytes = few_row_bytes(p.A.shape[1]);
    const FewOperand A = operand_of(p.A), W = operand_of(p.W);
    auto launch = [&](auto type, auto most) {
        constexpr bool BF16 = decltype(type)::value;
        auto kernel = loss_few<BF16, decltype(most)::value>;
        const size_t shared = static_cast<size_t>(tiles * 8 * bytes) + (split > 1 ? static_cast<size_t>(tiles) * kFewThreads * sizeof(float4) : 0);
        allow_dynamic_smem(reinterpret_cast<const void*>(kernel), call.device, shared);
        kernel<<<blocks, kFewThreads, shared, call.stream>>>(parts, at_target, A, W, static_cast<int>(p.A.shape[1]), static_cast<const int32_t*>(p.targets.data),
                                                                        static_cast<float>(p.scale), static_cast<float>(p.scale * 1.4426950408889634), bytes, split);
        note_kernel_f("loss_few<%s,%d>", BF16 ? "bf16" : "f16", tiles);
    };
    auto by_rows = [&](auto type) {
        if (tiles == 1) launch(type, std::integral_constant<int, 1>());
        else launch(type, std::integral_constant<int, 2>());
    };
    if (p.A.type == MOPS_B200_BF16) by_rows(std::true_type());
    else by_rows(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
}

void loss_forward_few(const Call& call, const LossProblem& p, const Array& loss, const Array& log_sum) {
    const int64_t n = p.A.shape[0], parts = std::min<int64_t>(ceil_div(p.W.shape[0], kUnitRows), sm_count(call.device)); // of a row: a block to each
    Scratch room(call, static_cast<size_t>(n * parts) * sizeof(PartSum<float>) + static_cast<size_t>(n) * sizeof(float));
    PartSum<float>* sums = room.as<PartSum<float>>();
    float* at_target = reinterpret_cast<float*>(sums + n * parts);
    launch_few(call, p, static_cast<unsigned>(parts), sums, at_target);
    join_rows<float>(call, loss, log_sum, sums, parts, at_target, LossRows{}, p.targets, p.W.shape[0], p.ignored);
}

} // namespace mops_b200
