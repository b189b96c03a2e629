// grouped_matrix_product on tensor cores, for f32.
//
// A value is split into three bf16 parts of eight bits each, by cutting bits off, so that the parts add up to the value: x = x0 + x1 +
// x2 (of values below some 2^-110 the bits under 2^-133, the smallest bf16, are lost). Of the nine products of parts the six of up to 2^-16 of the largest are computed, the small ones first; the three left out are about
// 2^-24 of the result, as a rounding to f32 is. The tensor cores add to their f32 accumulators by cutting off what does not fit, an error of one sign that
// grows with the number of additions; so an accumulator takes kRun stages (64 values of depth) and is then added, rounded, to sums in
// registers. That is the choice here: f32 results whose error is about twice that of f32 products and sums rounded one by one (K = 128, normal values: 4.0e-7 and 2.0e-7 of the norm), at two to
// three times the rate that the ordinary units could reach (74 TFLOP/s). Calls of few rows (grouped_few.cu) go to those. Sums that come out as NaN, as they do wherever an operand is infinite, are computed again by the ordinary units (repair()), so
// infinities come out as f32 arithmetic has them.
//
// The copy engine fetches boxes of f32 into one ring of stages; eight warps split them, the parts of the rows' operand go to tensor memory and those of the other to
// a second ring; one thread issues the products; eight warps add up what the accumulators hold and store the tiles. Bounded by shared memory: of a stage of 64 values of
// depth, 128 x 128, it moves 64 KB in, 64 KB out, 48 KB of parts in and 96 KB of them to the tensor cores. (With the parts of both operands in shared memory
// it was 416 KB, and 2.0 us for such a stage.) 16 384 rows of 8 groups, 1024 x 1024: 209 us (164 TFLOP/s, 0.99 P of bf16), gradients 204 and 269. Shallow products are bounded by memory and by the
// number of tiles: 100 003 rows of 20 groups, 128 x 128: 34 us, of which a tile on every SM takes 4.1 (4.5 TB/s) and beginning and end 6.5.
#include <mutex>
#include <set>

#include "grouped_block.cuh"
#include "grouped_mma.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {
namespace {

constexpr int kSplitWarps = 8, kStoreWarps = 8;
constexpr int kMultiplyWarp = kSplitWarps + kStoreWarps, kCopyWarp = kMultiplyWarp + 1, kPieceWarp = kMultiplyWarp + 2;
constexpr int kThreads = (kMultiplyWarp + 4) * 32; // (registers are dealt out to four warps at a time)
constexpr int kSplitThreads = kSplitWarps * 32;
constexpr int kDepth = 32; // values of depth in a stage: a row of 128 bytes in f32
constexpr int kRun = 2;    // stages that an accumulator takes
constexpr int kParts = 3;

// Registers per thread: those who store hold a tile's sums, the others need few. What the parts take adds up to what the block is launched
// with (check_registers).
constexpr int kLaunchRegisters = 96, kSplitRegisters = 80, kStoreRegisters = 120, kMultiplyRegisters = 64;
static_assert(kSplitWarps * kSplitRegisters + kStoreWarps * kStoreRegisters + 4 * kMultiplyRegisters <= kThreads / 32 * kLaunchRegisters,
              "a block cannot have more registers than it is launched with");
template <int kRegisters> __device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegisters));
}
template <int kRegisters> __device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegisters));
}

template <int kColumns> struct Layout {
    static constexpr int kRawA = kTileRows * kDepth * 4, kRawB = kColumns * kDepth * 4; // bytes of a stage of f32
    static constexpr int kB = kRawB / 2;                                                // of one part
    static constexpr int kRaw = kRawA + kRawB, kStage = kParts * kB;
    static constexpr int kRaws = kColumns == 128 ? 4 : 6, kStages = 2;
    static constexpr int kPartColumns = kDepth / 2; // of tensor memory, of a part of the rows' operand
    static constexpr int kStagesAt = kRaws * kRaw;
    static constexpr int kStaging = 32 * 32 * 4; // bytes: 32 x 32 sums of a warp
    static constexpr int kStagingAt = kStagesAt + kStages * kStage;
    static constexpr int kRingsAt = kStagingAt + kStoreWarps * kStaging;
    static constexpr int kBytes = kRingsAt + 512 + 1024;
    static constexpr unsigned kSums = 2 * kColumns; // columns of tensor memory of the accumulators; the parts come behind them
    static constexpr unsigned kTmem = kColumns == 128 ? 512 : 256;
    static_assert(kSums + kStages * kParts * kPartColumns <= kTmem, "room for the parts");
    static constexpr bool kPair = false, kRepairs = true;
    static constexpr int kPieces = 3; // known ahead
    static constexpr int kThreads = mops_b200::kThreads;
    struct Rings {
        Pieces<kPieces> pieces;
        Ring<kRaws> raws;
        Ring<kStages> stages;
        Ring<2> accumulators;
        int valid[kRaws]; // rows of depth that a raw stage has (MN-major); -1: there are no more
        uint32_t tmem;
        int gave_up;
        long long patience;
        __device__ void begin() {
            patience = kPatience;
            raws.begin(1, kSplitWarps);
            stages.begin(kSplitWarps, 1);
            accumulators.begin(1, kStoreWarps);
            pieces.begin(kStoreWarps + 2, false); // (those who store, copy and multiply)
        }
    };
    static_assert(sizeof(Rings) <= 512, "room for the rings");
};

// Cuts the top eight bits off each of two values and returns them side by side.
__device__ __forceinline__ uint32_t cut_part(uint32_t& x, uint32_t& y) {
    const uint32_t part = __byte_perm(x, y, 0x7632); // the upper halves
    x = __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffff0000u));
    y = __float_as_uint(__uint_as_float(y) - __uint_as_float(y & 0xffff0000u));
    return part;
}

// Operands of a stage in f32: boxes of rows of 128 bytes, swizzled; K-major one of a row for each row or column of the operand, MN-major one for each 32 of
// them, 32 rows of depth high.
//
// The rows' operand, by its lanes of tensor memory: warps w and w + 4 take 32 rows, half of the depth each.
template <bool MN> struct RowOperand {
    static constexpr int kBoxHeight = MN ? kDepth : kTileRows, kBoxes = MN ? kTileRows / 32 : 1, kHalf = kDepth / 2;
    // (Eight neighbouring lanes read from different banks.)
    __device__ static __forceinline__ void load(uint32_t (&x)[kHalf], uint32_t raw, int quadrant, int half, int lane) {
        if constexpr (MN) {
            const uint32_t box = raw + quadrant * (kDepth * 128) + lane % 4 * 4;
#pragma unroll
            for (int i = 0; i < kHalf; i++) {
                const int d = half * kHalf + i;
                x[i] = smem_load4(box + d * 128 + ((lane / 4 ^ (d & 7)) << 4));
            }
        } else {
            const uint32_t row = raw + (quadrant * 32 + lane) * 128;
#pragma unroll
            for (int c = 0; c < kHalf / 4; c++) {
                const uint4 v = smem_load16(row + (((half * (kHalf / 4) + c) ^ (lane & 7)) << 4));
                x[4 * c] = v.x, x[4 * c + 1] = v.y, x[4 * c + 2] = v.z, x[4 * c + 3] = v.w;
            }
        }
    }
    // to: the stage's first column, in the warp's lanes
    __device__ static __forceinline__ void store(uint32_t (&x)[kHalf], uint32_t to, int half, int valid) {
        if constexpr (MN) { // rows of depth of another group
#pragma unroll
            for (int i = 0; i < kHalf; i++)
                if (half * kHalf + i >= valid) x[i] = 0;
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            uint32_t w[kHalf / 2];
#pragma unroll
            for (int j = 0; j < kHalf / 2; j++) w[j] = cut_part(x[2 * j], x[2 * j + 1]);
            tmem_store(to + p * (kDepth / 2) + half * (kHalf / 2), w);
        }
    }
};

// The columns' operand. In parts: K-major kRows rows of 64 bytes, MN-major boxes of 64 columns, 32 rows of 128 bytes.
template <bool MN, int kRows> struct ColumnOperand {
    static constexpr int kChunks = kRows * kDepth / 8 / kSplitThreads; // of eight values, of a thread
    static constexpr int kPart = kRows * kDepth * 2;
    static constexpr int kBoxHeight = MN ? kDepth : kRows, kBoxes = MN ? kRows / 32 : 1;
    static constexpr int kPartRow = MN ? 128 : 64;
    static constexpr uint64_t kStep = (MN ? 16 * 128 : 32) >> 4; // 16 values of depth, in a descriptor

    // (Neighbouring lanes read from different banks: eight of them two rows of four chunks, or one row of two boxes.)
    __device__ static __forceinline__ void load(uint4 (&v)[2], uint32_t raw, int k) {
        const int task = k * kSplitThreads + (threadIdx.x % kSplitThreads);
        if constexpr (MN) {
            const int i = task % (kRows / 8), d = task / (kRows / 8), box = i / 4, odd = box & 1;
            const uint32_t row = raw + box * (kDepth * 128) + d * 128;
            const int first = 2 * (i % 4) + odd;
            const uint4 a = smem_load16(row + ((first ^ (d & 7)) << 4)), b = smem_load16(row + ((first ^ 1 ^ (d & 7)) << 4));
            v[0] = odd ? b : a;
            v[1] = odd ? a : b;
        } else {
            const int c = task % 4, r = task / 4;
#pragma unroll
            for (int h = 0; h < 2; h++) v[h] = smem_load16(raw + r * 128 + (((2 * c + h) ^ (r & 7)) << 4));
        }
    }
    __device__ static __forceinline__ void store(const uint4 (&v)[2], uint32_t to, int k, int valid) {
        const int task = k * kSplitThreads + (threadIdx.x % kSplitThreads);
        uint32_t x[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
        if constexpr (MN) {
            const int i = task % (kRows / 8), d = task / (kRows / 8);
            to += i / 8 * (kDepth * 128) + d * 128 + ((i % 8 ^ (d & 7)) << 4);
            if (d >= valid) { // a row of another group
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = 0;
            }
        } else {
            const int c = task % 4, r = task / 4;
            to += r * 64 + ((c ^ (r >> 1 & 3)) << 4);
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = cut_part(x[2 * j], x[2 * j + 1]);
            smem_store16(to + p * kPart, make_uint4(w[0], w[1], w[2], w[3]));
        }
    }
    __device__ static __forceinline__ uint64_t descriptor(uint32_t at) { return operand_descriptor<kPartRow>(at, kDepth * 128); }
};

// The operands in global memory: value (i, j) of a product is the sum of a[i * a_row + d * a_step] * b[j * b_column + d * b_step] over d < depth.
struct Terms {
    const float *a, *b;
    int64_t a_row, a_step, b_column, b_step;
    int depth;
    int rows, columns; // that there are from the warp's first ones on

    // By the warp: lanes take every 32nd value of depth. (The sum's order is another one than that of a thread by itself; this is for sums that are infinite or NaN.)
    __device__ __forceinline__ float product(int i, int j, int lane) const {
        const float *x = a + i * a_row, *y = b + j * b_column;
        constexpr int kInFlight = 8;
        float sum = 0;
        for (int d0 = 0; d0 < depth; d0 += 32 * kInFlight) {
            float u[kInFlight], v[kInFlight];
#pragma unroll
            for (int k = 0; k < kInFlight; k++) {
                const int d = d0 + k * 32 + lane;
                u[k] = d < depth ? x[d * a_step] : 0.f;
                v[k] = d < depth ? y[d * b_step] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kInFlight; k++) sum += u[k] * v[k];
            if (__any_sync(kFullMask, sum != sum)) break; // it stays so
        }
        return warp_sum(sum);
    }
    // Whether the first few terms already say that value (i, j) is NaN, as where nothing else is left.
    __device__ __forceinline__ bool nan_at_once(int i, int j) const {
        float sum = 0;
#pragma unroll
        for (int d = 0; d < 4; d++)
            if (d < depth) sum += a[i * a_row + d * a_step] * b[j * b_column + d * b_step];
        return sum != sum;
    }
};

// What the parts of a block do, of both kernels.
template <bool A_MN, bool B_MN, int kColumns> struct Work {
    using L = Layout<kColumns>;
    using A = RowOperand<A_MN>;
    using B = ColumnOperand<B_MN, kColumns>;
    static constexpr int kOwn = kColumns / 2; // columns of a storing warp

    Block<L>& block;
    Turn<L::kRaws> raw;
    Turn<L::kStages> stage;
    Turn<2> run;
    int64_t fetched = 0;

    // The copying thread: a stage of both operands; boxes of A at (a_inner, a_outer), of B at (b_inner, b_outer, slice). valid < 0: no more will come.
    __device__ __forceinline__ bool fetch(const CUtensorMap& map_a, const CUtensorMap& map_b, int a_inner, int a_outer, int b_inner,
                                          int b_outer, int slice, int valid) {
        if (!block.wait_empty(block.rings->raws, raw)) return false;
        uint64_t* full = &block.rings->raws.full[raw.at];
        *static_cast<volatile int*>(&block.rings->valid[raw.at]) = valid;
        if (valid < 0) {
            mbarrier_arrive(full);
            return true;
        }
        const uint32_t a = block.base + static_cast<uint32_t>(raw.at) * L::kRaw, b = a + L::kRawA;
        mbarrier_arrive_expect(full, L::kRaw);
#pragma unroll
        for (int i = 0; i < A::kBoxes; i++) box_in(a + i * A::kBoxHeight * 128, map_a, a_inner + 32 * i, a_outer, 0, full);
#pragma unroll
        for (int i = 0; i < B::kBoxes; i++) box_in(b + i * B::kBoxHeight * 128, map_b, b_inner + 32 * i, b_outer, slice, full);
        raw.next();
        fetched++;
        return true;
    }

    // A splitting warp, until no more stages come.
    __device__ __forceinline__ uint32_t parts_at() const {
        return block.rings->tmem + L::kSums + static_cast<uint32_t>(stage.at) * (kParts * L::kPartColumns);
    }
    __device__ __forceinline__ uint32_t stage_at() const { return block.base + L::kStagesAt + static_cast<uint32_t>(stage.at) * L::kStage; }

    __device__ __forceinline__ void split(int warp, int lane) {
        for (;;) {
            bool ok = true;
            if (lane == 0) ok = block.wait_full(block.rings->raws, raw);
            if (!__shfl_sync(kFullMask, ok, 0)) return;
            if (lane != 0) ok = block.wait_full(block.rings->raws, raw); // (so that every lane has seen it)
            const int valid = *static_cast<volatile int*>(&block.rings->valid[raw.at]);
            if (valid < 0) return;
            const uint32_t from = block.base + static_cast<uint32_t>(raw.at) * L::kRaw;
            uint32_t a[A::kHalf];
            uint4 b[B::kChunks][2];
            A::load(a, from, warp & 3, warp / 4, lane);
#pragma unroll
            for (int k = 0; k < B::kChunks; k++) B::load(b[k], from + L::kRawA, k);
            if (lane == 0) ok = block.wait_empty(block.rings->stages, stage);
            if (!__shfl_sync(kFullMask, ok, 0)) return;
            tmem_fence_after_sync();
            A::store(a, tmem_quadrant(parts_at(), warp), warp / 4, valid);
#pragma unroll
            for (int k = 0; k < B::kChunks; k++) B::store(b[k], stage_at(), k, valid);
            tmem_wait_store();
            tmem_fence_before_sync();
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) {
                mbarrier_arrive(&block.rings->stages.full[stage.at]);
                // Not before what was loaded has been used: an arrival overtakes loads that are still queued, and the copy engine would write
                // over what they are to read.
                mbarrier_arrive(&block.rings->raws.empty[raw.at]);
            }
            stage.next();
            raw.next();
        }
    }

    // The multiplying thread: a tile.
    __device__ __forceinline__ bool multiply(int steps) {
        constexpr uint32_t instruction = instruction_descriptor(true, false, B_MN, kColumns);
        constexpr int part_a[6] = {0, 2, 1, 0, 1, 0}, part_b[6] = {2, 0, 1, 1, 0, 0}; // small products first
        for (int s = 0; s < steps; s++) {
            if (s % kRun == 0 && !block.wait_empty(block.rings->accumulators, run)) return false;
            if (!block.wait_full(block.rings->stages, stage)) return false;
            tmem_fence_after_sync();
            const uint32_t a = parts_at(), accumulator = block.rings->tmem + static_cast<uint32_t>(run.at) * kColumns;
            const uint64_t b = B::descriptor(stage_at());
#pragma unroll
            for (int i = 0; i < 6; i++)
#pragma unroll
                for (int k = 0; k < kDepth / 16; k++)
                    umma_from_tmem(accumulator, a + part_a[i] * L::kPartColumns + k * 8, b + (part_b[i] * (L::kB >> 4) + k * B::kStep), instruction,
                                   s % kRun + i + k > 0);
            umma_arrive(&block.rings->stages.empty[stage.at]);
            stage.next();
            if ((s + 1) % kRun == 0 || s + 1 == steps) {
                umma_arrive(&block.rings->accumulators.full[run.at]);
                run.next();
            }
        }
        return true;
    }

    // A storing warp: the tile's sums of its 32 rows and kOwn columns.
    __device__ __forceinline__ bool collect(float (&sum)[kOwn], int steps, int quadrant, int half, int lane) {
#pragma unroll
        for (int i = 0; i < kOwn; i++) sum[i] = 0;
        for (int s = 0; s < steps; s += kRun) {
            if (!block.wait_full(block.rings->accumulators, run)) return false;
            tmem_fence_after_sync();
            const uint32_t from = tmem_quadrant(block.rings->tmem + static_cast<uint32_t>(run.at) * kColumns, quadrant) + half * kOwn;
#pragma unroll
            for (int c = 0; c < kOwn; c += 32) {
                uint32_t r[32];
                tmem_load(from + c, r);
                tmem_wait_load();
                tmem_pin(r);
#pragma unroll
                for (int j = 0; j < 32; j++) sum[c + j] += __uint_as_float(r[j]);
            }
            tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbarrier_arrive(&block.rings->accumulators.empty[run.at]);
            run.next();
        }
        return true;
    }

    // An infinite value has no second and third part (inf - inf), so that all sums of its row, or of its column, come out as NaN. Those are computed again, as the
    // ordinary units do it, and written over what has been stored. out: the warp's first value. (All of it in one place, behind the stores: a look at every sum in front of them, and a copy
    // of this for each of them, took 2 of 33 us of a product of 128 values in depth.)
    template <typename MakeTerms> __device__ __forceinline__ void repair(const float (&sum)[kOwn], int warp, int lane, float* out, int64_t stride, MakeTerms make) {
        long long start = clock64();
        const Terms terms = make();
        float* const staging = reinterpret_cast<float*>(block.smem + L::kStagingAt + warp * L::kStaging) + lane * 32;
        if (lane == 0) boxes_written();
        __syncwarp();
#pragma unroll 1
        for (int c = 0; c < kOwn; c += 32) {
#pragma unroll
            for (int j = 0; j < 32; j++) staging[j ^ lane] = c == 0 ? sum[j] : sum[kOwn - 32 + j]; // (each lane another bank)
#pragma unroll 1
            for (int j = 0; j < 32 && c + j < terms.columns; j++) {
                const float value = staging[j ^ lane];
                unsigned bad = __ballot_sync(kFullMask, lane < terms.rows && value != value && !terms.nan_at_once(lane, c + j));
                for (; bad != 0; bad &= bad - 1) {
                    const int i = __ffs(bad) - 1;
                    const float again = terms.product(i, c + j, lane);
                    if (lane == i) out[i * stride + c + j] = again;
                }
                const long long now = clock64(); // (so long others wait longer for this warp)
                if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long*>(&block.rings->patience), static_cast<unsigned long long>(now - start));
                start = now;
            }
        }
        __syncwarp();
    }

    // Writes them, 32 columns at a time through shared memory: by the copy engine, box by box, or where there are not all 32 rows of a box (`here`), or rows of the
    // output begin anywhere (loose), a row after the other. out: the first value. Returns whether there are sums to repair: some are NaN in the lane's first column, or in the
    // first row.
    __device__ __forceinline__ bool store(const float (&sum)[kOwn], int warp, const CUtensorMap& map, int column, int row, int slice, float* out,
                                          int64_t stride, int64_t here, int64_t wide, bool loose, int lane) {
        unsigned char* place = block.smem + L::kStagingAt + warp * L::kStaging;
        const int rows = static_cast<int>(min(here, int64_t(32)));
        const bool box = !loose && rows == 32;
        bool odd = sum[0] != sum[0];
#pragma unroll
        for (int c = 0; c < kOwn; c += 32) {
            if (c >= wide || rows <= 0) break;
            if (lane == 0) boxes_left<0>();
            __syncwarp();
            if (box) {
                const uint32_t to = smem_address(place);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    smem_store16(to + lane * 128 + ((j ^ (lane & 7)) << 4),
                                 make_uint4(__float_as_uint(sum[c + 4 * j]), __float_as_uint(sum[c + 4 * j + 1]),
                                            __float_as_uint(sum[c + 4 * j + 2]), __float_as_uint(sum[c + 4 * j + 3])));
                async_proxy_fence();
                __syncwarp();
                odd |= isnan(*reinterpret_cast<const float*>(place + lane * 4));
                if (lane == 0) box_out(map, column + c, row, slice, to);
            } else {
                float* staging = reinterpret_cast<float*>(place);
#pragma unroll
                for (int j = 0; j < 32; j++) staging[lane * 32 + (j ^ lane)] = sum[c + j]; // (each lane another bank)
                __syncwarp();
                odd |= isnan(staging[lane]);
                if (c + lane < wide) {
#pragma unroll 8
                    for (int r = 0; r < rows; r++) out[r * stride + c + lane] = staging[r * 32 + (lane ^ r)];
                }
                __syncwarp();
            }
        }
        return __any_sync(kFullMask, odd && rows > 0);
    }
    // The same of sums that go elsewhere.
    __device__ __forceinline__ static bool any_nan(const float (&sum)[kOwn]) {
        float check[8] = {}; // (side by side)
#pragma unroll
        for (int i = 0; i < kOwn; i++) check[i % 8] = fmaf(sum[i], 0.f, check[i % 8]);
        const float all = (check[0] + check[1] + (check[2] + check[3])) + (check[4] + check[5] + (check[6] + check[7]));
        return __any_sync(kFullMask, isnan(all));
    }
};

// ---------------------------------------------------------------------------------- rows
// out[r,:] = X[r,:] M[group of r]. M_MN: the columns of M are neighbours in memory, else its depth is.
struct RowOperands {
    const float *x, *m;
    int64_t x_stride, group_stride, depth_stride, column_stride; // of m the last three
};
template <bool M_MN, int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_split(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_out,
                   float* __restrict__ out, const __grid_constant__ RowOperands from, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int depth,
                   int columns, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using W = Work<false, M_MN, kColumns>;
    using L = typename W::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    W work{block};
    Supply<L> supply{block};
    Piece piece;
    if (warp < kSplitWarps) {
        fewer_registers<kSplitRegisters>();
        work.split(warp, lane);
    } else if (warp < kMultiplyWarp) {
        more_registers<kStoreRegisters>();
        const int quadrant = warp & 3, half = (warp - kSplitWarps) / 4;
        while (supply.next(piece, lane)) {
            float sum[W::kOwn];
            if (!work.collect(sum, piece.steps, quadrant, half, lane)) break;
            const int64_t row = piece.lo + quadrant * 32, column = piece.column + half * W::kOwn;
            if (work.store(sum, warp - kSplitWarps, map_out, column, static_cast<int>(row), 0, out + row * columns + column, columns, piece.hi - row,
                           columns - column, loose, lane))
                work.repair(sum, warp - kSplitWarps, lane, out + row * columns + column, columns, [&] {
                    return Terms{from.x + row * from.x_stride, from.m + piece.group * from.group_stride + column * from.column_stride, from.x_stride, 1, from.column_stride,
                                 from.depth_stride, depth, static_cast<int>(min(piece.hi - row, int64_t(32))), static_cast<int>(columns - column)};
                });
        }
    } else {
        fewer_registers<kMultiplyRegisters>();
        bool ok = true;
        if (warp == kMultiplyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0) ok = work.multiply(piece.steps);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
        } else if (warp == kPieceWarp) {
            hand_out(block, 0, lane, DecodeRows<kTileRows, kColumns>(offsets, groups, rows, columns, (depth + kDepth - 1) / kDepth, lane));
        } else if (warp == kCopyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0)
                    for (int s = 0; s < piece.steps && ok; s++)
                        ok = work.fetch(map_x, map_m, s * kDepth, static_cast<int>(piece.lo), M_MN ? piece.column : s * kDepth,
                                        M_MN ? s * kDepth : piece.column, piece.group, kDepth);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
            if (lane == 0) {
                if (ok) (void)work.fetch(map_x, map_m, 0, 0, 0, 0, 0, -1);
                block.drain(block.rings->raws, work.raw, work.fetched);
            }
        }
    }
    if (lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

// ------------------------------------------------------------------------- outer products
// out[g] = X[rows of g]^T Y[rows of g].
struct OuterOperands {
    const float *x, *y;
    int64_t x_stride, y_stride;
};
template <int kColumns>
__global__ void __launch_bounds__(kThreads, 1)
grouped_outer_split(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                    const __grid_constant__ CUtensorMap map_out, float* __restrict__ out, float* __restrict__ parts, int64_t most_parts, const __grid_constant__ OuterOperands from,
                    const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int height, int columns, int64_t segment, bool loose, Status st) {
    extern __shared__ unsigned char raw[];
    using W = Work<true, true, kColumns>;
    using L = typename W::L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Block<L> block(raw, st);
    block.begin(warp);
    if (blockIdx.x == 0) check_offsets(offsets, groups, rows, st);

    W work{block};
    Supply<L> supply{block};
    Piece piece;
    if (warp < kSplitWarps) {
        fewer_registers<kSplitRegisters>();
        work.split(warp, lane);
    } else if (warp < kMultiplyWarp) {
        more_registers<kStoreRegisters>();
        const int quadrant = warp & 3, half = (warp - kSplitWarps) / 4;
        while (supply.next(piece, lane)) {
            float sum[W::kOwn];
            if (!work.collect(sum, piece.steps, quadrant, half, lane)) break;
            const int64_t row = piece.row + quadrant * 32, column = piece.column + half * W::kOwn;
            float* to = out + (static_cast<int64_t>(piece.group) * height + row) * columns + column;
            int64_t stride = columns;
            bool odd;
            if (piece.slot >= 0) {
                // (there are more parts than there is room for only where offsets descend, which is reported)
                if (piece.slot >= most_parts) continue;
                to = parts + (piece.slot * kTileRows + quadrant * 32) * kColumns + half * W::kOwn;
                stride = kColumns;
#pragma unroll
                for (int i = 0; i < W::kOwn; i += 4)
                    *reinterpret_cast<float4*>(to + lane * kColumns + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
                odd = W::any_nan(sum);
            } else {
                // (the copy engine leaves out what lies behind the output's last row)
                odd = work.store(sum, warp - kSplitWarps, map_out, column, static_cast<int>(row), piece.group, to, columns,
                                 loose || row >= height ? height - row : 32, columns - column, loose, lane);
            }
            if (odd)
                work.repair(sum, warp - kSplitWarps, lane, to, stride, [&] {
                    return Terms{from.x + piece.lo * from.x_stride + row, from.y + piece.lo * from.y_stride + column, 1, from.x_stride, 1, from.y_stride,
                                 static_cast<int>(piece.hi - piece.lo), static_cast<int>(height - row), static_cast<int>(columns - column)};
                });
        }
    } else {
        fewer_registers<kMultiplyRegisters>();
        bool ok = true;
        if (warp == kMultiplyWarp) {
            while (ok && supply.next(piece, lane)) {
                if (lane == 0) ok = work.multiply(piece.steps);
                ok = __shfl_sync(kFullMask, ok, 0);
            }
        } else if (warp == kPieceWarp) {
            hand_out(block, 0, lane, DecodeOuter<kTileRows, kColumns, kDepth>(offsets, groups, rows, height, columns, segment, lane));
        } else if (warp == kCopyWarp) {
            while (ok && supply.next(piece, lane)) {
                const int lo = static_cast<int>(piece.lo), hi = static_cast<int>(piece.hi);
                if (lane == 0)
                    for (int s = 0; s < piece.steps && ok; s++)
                        ok = work.fetch(map_x, map_y, piece.row, lo + s * kDepth, piece.column, lo + s * kDepth, 0, min(hi - lo - s * kDepth, kDepth));
                ok = __shfl_sync(kFullMask, ok, 0);
            }
            if (lane == 0) {
                if (ok) (void)work.fetch(map_x, map_y, 0, 0, 0, 0, 0, -1);
                block.drain(block.rings->raws, work.raw, work.fetched);
            }
        }
    }
    if (lane == 0) boxes_left<0>();
    __syncwarp();
    block.end(warp);
}

// That the compiler gave the kernel the registers that its parts deal out among themselves (with fewer they would wait for good).
void check_registers(const void* kernel, const std::string& op) {
    static std::mutex mutex;
    static std::set<const void*> good;
    std::lock_guard<std::mutex> lock(mutex);
    if (good.count(kernel)) return;
    cudaFuncAttributes attributes;
    MOPS_CUDA_OK(cudaFuncGetAttributes(&attributes, kernel));
    if (attributes.numRegs != kLaunchRegisters)
        throw std::runtime_error("internal error in operation " + op + ": a kernel was built with " +
                                 std::to_string(attributes.numRegs) + " registers");
    good.insert(kernel);
}

} // namespace

bool multiply_rows_split(const Call& call, const RowsProblem& p, const std::string& op) {
    if (p.X.type != MOPS_B200_F32 || p.depth == 0 || p.groups == 0) return false;
    const bool mn = p.column_stride == 1;
    const int64_t stride = mn ? p.depth_stride : p.column_stride; // of M
    const int sms = sm_count(call.device);
    auto launch = [&](auto major, auto width) {
        constexpr bool M_MN = decltype(major)::value;
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, p.depth, p.rows, 1, p.X.stride[0], 0, kTileRows);
        const CUtensorMap m = M_MN ? tensor_map(p.X.type, p.M.data, p.columns, p.depth, p.groups, stride, p.M.stride[0], kDepth)
                                   : tensor_map(p.X.type, p.M.data, p.depth, p.columns, p.groups, stride, p.M.stride[0], kColumns);
        const bool loose = p.columns % 4 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, p.columns, p.rows, 1, p.columns, 0, 32);
        const int64_t tiles = most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, kColumns);
        auto kernel = grouped_rows_split<M_MN, kColumns>;
        check_registers(reinterpret_cast<const void*>(kernel), op);
        const RowOperands from{static_cast<const float*>(p.X.data), static_cast<const float*>(p.M.data), p.X.stride[0], p.M.stride[0], p.depth_stride, p.column_stride};
        launch_blocks<L>(call, op, kernel, tiles, x, m, out, static_cast<float*>(p.out.data), from, p.offsets, p.groups, p.rows,
                         static_cast<int>(p.depth), static_cast<int>(p.columns), loose, call.status);
        note_kernel_f("grouped_rows_split<%s,%d>", M_MN ? "columns" : "depth", kColumns);
    };
    auto by_width = [&](auto major) {
        if (p.columns > 64 && most_row_tiles(p.rows, p.groups, kTileRows) * ceil_div(p.columns, 128) >= sms / 2)
            launch(major, std::integral_constant<int, 128>());
        else launch(major, std::integral_constant<int, 64>());
    };
    if (mn) by_width(std::true_type());
    else by_width(std::false_type());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

bool multiply_outer_split(const Call& call, const OuterProblem& p, const std::string& op) {
    const int64_t rows = p.X.shape[0], height = p.X.shape[1], columns = p.Y.shape[1];
    if (p.X.type != MOPS_B200_F32 || rows == 0) return false;
    const int sms = sm_count(call.device);
    auto launch = [&](auto width) {
        constexpr int kColumns = decltype(width)::value;
        using L = Layout<kColumns>;
        const CUtensorMap x = tensor_map(p.X.type, p.X.data, height, rows, 1, p.X.stride[0], 0, kDepth);
        const CUtensorMap y = tensor_map(p.X.type, p.Y.data, columns, rows, 1, p.Y.stride[0], 0, kDepth);
        const int64_t tiles = ceil_div(height, kTileRows) * ceil_div(columns, kColumns);
        const int64_t segment = outer_segment(rows, p.groups, tiles, sms), most_parts = most_outer_parts(rows, tiles, segment);
        Scratch room(call);
        if (rows > segment) room.take(static_cast<size_t>(most_parts) * kTileRows * kColumns * sizeof(float));
        float* parts = room.as<float>();
        auto kernel = grouped_outer_split<kColumns>;
        check_registers(reinterpret_cast<const void*>(kernel), op);
        const bool loose = columns % 4 != 0 || reinterpret_cast<uintptr_t>(p.out.data) % 16 != 0;
        const CUtensorMap out = loose ? x : tensor_map(p.X.type, p.out.data, columns, height, p.groups, columns, height * columns, 32);
        const OuterOperands from{static_cast<const float*>(p.X.data), static_cast<const float*>(p.Y.data), p.X.stride[0], p.Y.stride[0]};
        launch_blocks<L>(call, op, kernel, tiles * (rows / segment + p.groups), x, y, out, static_cast<float*>(p.out.data), parts, most_parts, from, p.offsets,
                         p.groups, rows, static_cast<int>(height), static_cast<int>(columns), segment, loose, call.status);
        if (rows > segment) {
            join_outer<float, kTileRows, kColumns>(call, p, parts, most_parts, tiles, segment, op);
            room.free();
        }
        note_kernel_f("grouped_outer_split<%d>", kColumns);
    };
    if (columns > 64) launch(std::integral_constant<int, 128>());
    else launch(std::integral_constant<int, 64>());
    MOPS_CUDA_OK(cudaGetLastError());
    return true;
}

} // namespace mops_b200
