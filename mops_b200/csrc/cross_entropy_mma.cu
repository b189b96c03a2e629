// linear_cross_entropy on tensor cores, for f16 and bf16.
//
// Forward: the logits of a tile stay in tensor memory; a lane takes the largest of its row and the sum of exponentials, 32 columns at a time, and what is left of a tile is one such pair for each row
// and half, which loss_join adds up. Backward, a piece of the vocabulary at a time: the same product, from whose tiles come dx in 16 bits (rows x piece, in scratch memory); grad_W of the piece is its outer
// product with A, and its product with the piece's rows of W is added to f32 sums for grad_A.
//
// dx is rounded to 16 bits in units of the largest gradient of a loss (f16: of 2^-14 of it, so that probabilities down to 2^-28 are normal numbers), which
// multiplies the results: so the gradient of a mean, which is the same for all rows, leaves -1 at the targets as it is. A row's value there is 1 - exp(-loss), not the difference of rounded numbers.
// A row's gradient is for the most part that of its target, whose rounding is an error of the row as a whole; where there are too few rows for such errors to average out, dx is kept in two parts of
// 16 bits (a row of what the first leaves under it, and rows of A twice): the products are bounded by memory there.
//
// Bound by the tensor cores: 8192 rows (7782 that count) of 100 003 x 1024 in bf16, 1.59 TFLOP for each product: the loss 1151 us (1.38 PFLOP/s), in four pieces dx 1243, grad_A 1287, grad_W 1311, at up to
// 1965 MHz, which the GPU holds for some milliseconds. In steps without a pause, at the 1455 MHz that the power limit leaves: 1340, 1480, 1500, 1570. Some 45 us each way are the numbering and gathering of rows and
// the joins.
//
// The tensor cores' sums are truncated, not rounded: losses and sums are off by some 2.5e-10 of themselves for each value of depth (1024: 2e-7, 4096: 1e-6).
#include <numeric>

#include "block_ops.hpp"
#include "grouped_mma.hpp"
#include "loss_rows.cuh"
#include "pack.hpp"
#include "tile_rows.cuh"

namespace mops_b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kGatherThreads = 256;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------- forward
template <int kColumns> struct LossStore {
    static constexpr bool kHalves = false, kAllRows = false;
    static constexpr int kStoreWarps = 8, kStaging = 0, kOwn = kColumns / 2;
    struct Args {
        PartSum<float>* parts; // row by row
        int64_t n;             // of a row
        float* at_target;
        const int32_t* target;
        int columns;
        float scale, scale2;   // scale2: times log2(e)
    };
    const Args& a;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0, target = -1;
    __device__ LossStore(const Args& a, uint32_t, int lane) : a(a), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int) {
        row = r + lane, here = h, column = piece.column;
        target = lane < here && piece.group >= 0 ? a.target[row] : -1;
    }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
        const int first = column + part * kOwn, wide = min(a.columns - first, kOwn);
        if (wide <= 0) return;
        float top = -INFINITY, sum = 0; // of x log2(e)
#pragma unroll 1
        for (int c = 0; c < wide; c += 32) {
            uint32_t r[32];
            tmem_load(accumulator + part * kOwn + c, r);
            tmem_wait_load();
            tmem_pin(r);
            if (c + 32 > wide) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (c + j >= wide) r[j] = __float_as_uint(-INFINITY);
            }
            const int at = target - first - c;
            if (__any_sync(kFullMask, at >= 0 && at < 32)) {
                float x = 0;
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j == at) x = __uint_as_float(r[j]);
                if (at >= 0 && at < 32 && c + at < wide) a.at_target[row] = x * a.scale;
            }
            float most[4];
#pragma unroll
            for (int j = 0; j < 4; j++) most[j] = __uint_as_float(r[j]);
#pragma unroll
            for (int j = 4; j < 32; j++) most[j % 4] = fmaxf(most[j % 4], __uint_as_float(r[j]));
            const float now = fmaxf(top, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * a.scale2), base = PartSum<float>::from(now);
            sum *= top == -INFINITY ? 1.f : exp2_fast(PartSum<float>::from(top) - base);
            top = now;
            float more[4] = {};
#pragma unroll
            for (int j = 0; j < 32; j++) more[j % 4] += exp2_fast(fmaf(__uint_as_float(r[j]), a.scale2, -base));
            sum += (more[0] + more[1]) + (more[2] + more[3]);
        }
        if (lane < here) a.parts[row * a.n + first / kOwn] = PartSum<float>{top * kLn2, sum};
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {}
};

// ------------------------------------------------------------------------------ backward
// What dx takes of a row: dx = exp2(acc scale2 - base) factor, and its value at the target.
struct alignas(16) RowFactors {
    float base, factor, at_target;
    int32_t target;
};

template <bool BF16, int kColumns, bool kTwoParts> struct GradientStore {
    static constexpr bool kHalves = false, kAllRows = true; // (zeros behind the last row, up to the end of the tile: products over the rows take whole stages of 64)
    static constexpr int kStoreWarps = 8, kStaging = BoxOut::kBytes, kOwn = kColumns / 2;
    struct Args {
        CUtensorMap map, map_rest;
        uint16_t *out, *rest;
        int64_t stride;
        int columns, first_column; // of the piece
        float scale2;
        const RowFactors* factors;
    };
    const Args& a;
    BoxOut out, rest;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0;
    RowFactors f{};
    __device__ GradientStore(const Args& a, uint32_t staging, int lane)
        : a(a), out{a.map, a.out, a.stride, a.columns, false}, rest{a.map_rest, a.rest, a.stride, a.columns, false}, staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int) {
        row = r, here = h, column = piece.column;
        if (lane < here && piece.group >= 0) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(a.factors + row + lane));
            f = RowFactors{__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), static_cast<int32_t>(v.w) - a.first_column};
        }
    }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
#pragma unroll 1
        for (int c = part * kOwn; c < part * kOwn + kOwn; c += 64) {
            if (column + c >= a.columns) return;
            uint4 v[8], w[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t r[32];
                tmem_load(accumulator + c + h * 32, r);
                tmem_wait_load();
                tmem_pin(r);
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = exp2_fast(fmaf(__uint_as_float(r[j]), a.scale2, -f.base)) * f.factor;
                const int at = f.target - column - c - h * 32;
                if (__any_sync(kFullMask, at >= 0 && at < 32)) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (j == at) x[j] = f.at_target;
                }
                if (here < 32) {
#pragma unroll
                    for (int j = 0; j < 32; j++) x[j] = lane < here ? x[j] : 0.f;
                }
                auto packs = [&](uint4* to) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        to[h * 4 + j] = make_uint4(pack_pair<BF16>(x[8 * j], x[8 * j + 1]), pack_pair<BF16>(x[8 * j + 2], x[8 * j + 3]),
                                                   pack_pair<BF16>(x[8 * j + 4], x[8 * j + 5]), pack_pair<BF16>(x[8 * j + 6], x[8 * j + 7]));
                };
                packs(v);
                if constexpr (kTwoParts) {
                    using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
#pragma unroll
                    for (int j = 0; j < 32; j++) x[j] -= widen(narrow<T>(x[j]));
                    packs(w);
                }
            }
            out.put(v, staging, row, 32, column + c, lane); // (there is room up to the end of the tile)
            if constexpr (kTwoParts) rest.put(w, staging, row, 32, column + c, lane);
        }
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

// Sums in f32: of the first piece of the vocabulary they are written, those of others are added to what is there. Each slice of the depth has sums of its own, so that no two
// blocks add to one place, and the order of the additions is that of the pieces. The last piece may have fewer stages than there are slices: a slice without any has summed nothing, and its accumulator has what
// another tile left there.
template <int kColumns> struct SumStore {
    static constexpr bool kHalves = false, kAllRows = false;
    static constexpr int kStoreWarps = 8, kStaging = 32 * kBoxRow, kOwn = kColumns / 2;
    struct Args {
        CUtensorMap map;
        float* out;
        int64_t rows, stride; // of a slice; stride: a multiple of 4
        int columns;
        bool add;
    };
    const Args& a;
    uint32_t staging;
    int lane;
    int64_t row = 0;
    int here = 0, column = 0, slice = 0;
    bool empty = false;
    __device__ SumStore(const Args& a, uint32_t staging, int lane) : a(a), staging(staging), lane(lane) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int) {
        row = r, here = h, column = piece.column, slice = piece.row, empty = piece.steps == 0;
    }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
        if (empty && a.add) return;
#pragma unroll 1
        for (int c = part * kOwn; c < part * kOwn + kOwn; c += 32) {
            if (column + c >= a.columns) return;
            uint32_t r[32];
            tmem_load(accumulator + c, r);
            tmem_wait_load();
            tmem_pin(r);
            if (empty) {
#pragma unroll
                for (int j = 0; j < 32; j++) r[j] = 0;
            }
            if (here == 32) {
                if (lane == 0) boxes_left<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++)
                    smem_store16(staging + lane * kBoxRow + ((j ^ (lane & 7)) << 4), make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]));
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    if (a.add) box_add(a.map, column + c, static_cast<int>(row), slice, staging);
                    else box_out(a.map, column + c, static_cast<int>(row), slice, staging);
                }
            } else if (lane < here) {
                float* to = a.out + (slice * a.rows + row + lane) * a.stride + column + c;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (column + c + 4 * j < a.columns) { // (there is room up to a multiple of 4)
                        float4 v = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
                        if (a.add) {
                            const float4 w = *reinterpret_cast<const float4*>(to + 4 * j);
                            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
                        }
                        *reinterpret_cast<float4*>(to + 4 * j) = v;
                    }
            }
        }
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

// grad_W = factor dx^T A in 16 bits (DecodeDepth); zeros where there are no rows.
template <bool BF16> struct ScaledStore {
    static constexpr bool kHalves = false, kAllRows = false;
    static constexpr int kStoreWarps = 8, kStaging = BoxOut::kBytes, kOwn = 128;
    struct Args {
        CUtensorMap map;
        uint16_t* out;
        int columns;
        bool loose;
        const float* factor;
    };
    BoxOut out;
    uint32_t staging;
    int lane;
    float factor;
    int64_t row = 0;
    int here = 0, column = 0;
    bool empty = false;
    __device__ ScaledStore(const Args& a, uint32_t staging, int lane)
        : out{a.map, a.out, a.columns, a.columns, a.loose}, staging(staging), lane(lane), factor(__ldg(a.factor)) {}
    __device__ __forceinline__ void begin(const Piece& piece, int64_t r, int h, int) { row = r, here = h, column = piece.column, empty = piece.steps == 0; }
    __device__ __forceinline__ void store(uint32_t accumulator, int part) {
#pragma unroll 1
        for (int c = part * kOwn; c < part * kOwn + kOwn; c += 64) {
            if (column + c >= out.columns) return;
            uint4 v[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t r[32];
                tmem_load(accumulator + c + h * 32, r);
                tmem_wait_load();
                tmem_pin(r);
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = empty ? 0.f : __uint_as_float(r[j]) * factor;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[h * 4 + j] = make_uint4(pack_pair<BF16>(x[8 * j], x[8 * j + 1]), pack_pair<BF16>(x[8 * j + 2], x[8 * j + 3]),
                                              pack_pair<BF16>(x[8 * j + 4], x[8 * j + 5]), pack_pair<BF16>(x[8 * j + 6], x[8 * j + 7]));
            }
            out.put(v, staging, row, here, column + c, lane);
        }
    }
    __device__ __forceinline__ void clear() const {}
    __device__ __forceinline__ void end() const {
        if (lane == 0) boxes_left<0>();
    }
};

// to[i,:] = from[order[i],:], or rows 2i and 2i + 1, a warp to a row; and what dx takes of the row, if that is asked for.
struct FactorArgs {
    RowFactors* factors; // none: a forward pass
    float* factor;       // of the results
    const float *grad_loss, *grad_log_sum, *loss, *log_sum;
    float scale, units; // units: that are 1, 2^14 for f16
};
__global__ void __launch_bounds__(kGatherThreads)
gather_rows(uint16_t* __restrict__ to, int64_t to_stride, const __half* __restrict__ from, int64_t stride, bool aligned, const unsigned char* begin,
            const unsigned char* end, const LossRows rows, int64_t columns, bool twice,
            const FactorArgs f) {
    const int64_t kept = rows.offsets[1];
    const int lane = threadIdx.x & 31;
    if (f.factors != nullptr) { // zeros behind the last row, up to a whole stage (there is room for them)
        const int64_t packs = to_stride / 8, first = (twice ? 2 * kept : kept) * packs, last = ((twice ? 2 * kept : kept) + 63) / 64 * 64 * packs;
        for (int64_t c = first + static_cast<int64_t>(blockIdx.x) * kGatherThreads + threadIdx.x; c < last; c += static_cast<int64_t>(gridDim.x) * kGatherThreads)
            reinterpret_cast<uint4*>(to)[c] = make_uint4(0, 0, 0, 0);
    }
    const float unit = f.factors != nullptr ? *rows.unit : 0.f;
    if (f.factors != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *f.factor = unit * f.scale / f.units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kGatherThreads / 32) + threadIdx.x / 32; i < kept; i += static_cast<int64_t>(gridDim.x) * (kGatherThreads / 32)) {
        const int64_t r = rows.order[i];
        const __half* p = from + r * stride;
        const int64_t packs = to_stride / 8;
        uint4* q = reinterpret_cast<uint4*>(to) + (twice ? 2 * i : i) * packs;
        if (twice) {
            for (int64_t c = lane; c < packs; c += 32) q[c] = q[c + packs] = load_anywhere<__half>(p + c * 8, columns - c * 8, begin, end);
        } else if (aligned) {
#pragma unroll 4
            for (int64_t c = lane; c < packs; c += 32) q[c] = __ldg(reinterpret_cast<const uint4*>(p) + c);
        } else {
#pragma unroll 2
            for (int64_t c = lane; c < packs; c += 32) q[c] = load_anywhere<__half>(p + c * 8, columns - c * 8, begin, end);
        }
        if (f.factors != nullptr && lane == 0) {
            const float of_loss = f.grad_loss != nullptr ? f.grad_loss[r] : 0.f, of_sum = f.grad_log_sum != nullptr ? f.grad_log_sum[r] : 0.f;
            // (a gradient of which the largest is nothing is nothing, or infinite)
            const float g = unit > 0.f ? of_loss / unit * f.units : of_loss, both = unit > 0.f ? (of_loss + of_sum) / unit * f.units : of_loss + of_sum;
            f.factors[i] = RowFactors{f.log_sum[r] * kLog2e, both, fmaf(both, expf(-f.loss[r]), -g), rows.target[i]};
        }
    }
}

unsigned warps_for(const Call& call, int64_t rows) {
    return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(rows, kGatherThreads / 32), 1), int64_t(sm_count(call.device)) * 16));
}

int64_t whole_packs(int64_t n) { return (n + 7) / 8 * 8; }

// The kept rows of A, one after the other (or each twice), as the copy engine can fetch them.
Array gathered(const Call& call, Scratch& room, const Array& A, const LossRows& rows, bool twice, const FactorArgs& factors) {
    const int64_t stride = whole_packs(A.shape[1]), copies = twice ? 2 : 1;
    room.take(static_cast<size_t>((copies * A.shape[0] + 63) / 64 * 64 * stride) * 2);
    Array to = contiguous(room.as<void>(), A.type, copies * A.shape[0], A.shape[1]);
    to.stride[0] = stride;
    const bool aligned = A.shape[1] % 8 == 0 && A.stride[0] % 8 == 0 && reinterpret_cast<uintptr_t>(A.data) % 16 == 0;
    const unsigned char* begin = static_cast<const unsigned char*>(A.data);
    gather_rows<<<warps_for(call, A.shape[0]), kGatherThreads, 0, call.stream>>>(static_cast<uint16_t*>(to.data), stride, static_cast<const __half*>(A.data), A.stride[0],
                                                                                  aligned, begin, begin + ((A.shape[0] - 1) * A.stride[0] + A.shape[1]) * 2, rows,
                                                                                  A.shape[1], twice, factors);
    MOPS_CUDA_OK(cudaGetLastError());
    return to;
}

template <typename F> void for_sixteen(int32_t type, F&& f) {
    if (type == MOPS_B200_BF16) f(std::true_type());
    else f(std::false_type());
}

// Up to so many rows dx is kept in two parts.
constexpr int64_t kTwoPartsTo = 256;

} // namespace

void loss_forward_mma(const Call& call, const LossProblem& p, const Array& loss, const Array& log_sum, const std::string& op) {
    using std::integral_constant;
    const int64_t n = p.A.shape[0], vocabulary = p.W.shape[0];
    Scratch room_rows(call), room_A(call);
    Packing packing(call);
    Array A = p.A, W = p.W;
    LossRows rows{};
    if (few_loss_rows(p)) return loss_forward_few(call, p, loss, log_sum);
    const int32_t* targets = static_cast<const int32_t*>(p.targets.data);
    const bool gather = worth_gathering(A.type, n, vocabulary, p.A.shape[1]);
    if (gather) {
        rows = take_rows(room_rows, n);
        prepare_rows<float>(call, rows, static_cast<float*>(loss.data), static_cast<float*>(log_sum.data), p.targets, vocabulary, p.ignored, nullptr, nullptr);
        A = gathered(call, room_A, p.A, rows, false, {});
    } else {
        packing.add(A);
    }
    packing.add(W);
    packing.run();
    // (where rows are a quarter of a box at most, which is fetched for each tile, tiles of 128 columns leave no SM with twice the work of others: 32 rows of 50 021 x 1024 26 us; with more, wider ones are
    // faster: 66 rows of 88288 x 736 41 us in tiles of 128, 36 in tiles of 256)
    const bool narrow_tiles = n <= kTileRows / 4;
    const int64_t own = narrow_tiles ? 64 : 128, parts = ceil_div(vocabulary, own);
    Scratch room(call, static_cast<size_t>(n * parts) * sizeof(PartSum<float>) + static_cast<size_t>(n) * sizeof(float));
    PartSum<float>* sums = room.as<PartSum<float>>();
    float* at_target = reinterpret_cast<float*>(sums + n * parts);
    const float scale = static_cast<float>(p.scale), scale2 = static_cast<float>(p.scale * 1.4426950408889634);
    const TileProblem problem{A, rows.offsets, 1, n, A.shape[1], vocabulary};
    const TileOperand operands[2] = {{W.data, 1, W.stride[0], 0}, {W.data, 1, W.stride[0], 0}};
    for_sixteen(A.type, [&](auto type) {
        auto launch = [&](auto width, auto paired) {
            using E = LossStore<decltype(width)::value>;
            const typename E::Args args{sums, parts, at_target, gather ? rows.target : targets, static_cast<int>(vocabulary), scale, scale2};
            if (gather) launch_tiles<decltype(type)::value, false, decltype(width)::value, decltype(paired)::value, E, DecodeRows>(call, op, problem, operands, args);
            else launch_tiles<decltype(type)::value, false, decltype(width)::value, decltype(paired)::value, E, DecodeTable>(call, op, problem, operands, args);
            note_kernel_f("loss_rows_mma<%s,%d,%s>", type ? "bf16" : "f16", static_cast<int>(width), paired ? "pair" : "block");
        };
        if (narrow_tiles) launch(integral_constant<int, 128>(), std::false_type());
        else if (n <= kTileRows) launch(integral_constant<int, 256>(), std::false_type());
        else launch(integral_constant<int, 256>(), std::true_type());
    });
    MOPS_CUDA_OK(cudaGetLastError());
    join_rows<float>(call, loss, log_sum, sums, parts, at_target, rows, p.targets, vocabulary, p.ignored);
}

void loss_backward_mma(const Call& call, const LossProblem& p, const Array& grad_A, const Array& grad_W, const Array& grad_loss, const Array& grad_log_sum, const Array& loss,
                       const Array& log_sum, const std::string& op) {
    using std::integral_constant;
    const int64_t n = p.A.shape[0], vocabulary = p.W.shape[0], columns = p.A.shape[1];
    const int sms = sm_count(call.device);
    const bool need_A = grad_A.data != nullptr, need_W = grad_W.data != nullptr;
    Scratch room_rows(call), room_A(call), room_factors(call, static_cast<size_t>(n) * sizeof(RowFactors) + 16);
    const LossRows rows = take_rows(room_rows, n);
    const float* of_loss = static_cast<const float*>(grad_loss.data);
    const float* of_sum = static_cast<const float*>(grad_log_sum.data);
    prepare_rows<float>(call, rows, nullptr, nullptr, p.targets, vocabulary, p.ignored, of_loss, of_sum);
    RowFactors* factors = room_factors.as<RowFactors>();
    float* factor = reinterpret_cast<float*>(factors + n);
    const float scale2 = static_cast<float>(p.scale * 1.4426950408889634);
    const bool twice = n <= kTwoPartsTo;
    const int64_t copies = twice ? 2 : 1, all = copies * n; // rows of dx
    const int64_t height = n <= kTileRows ? kTileRows : 2 * kTileRows, whole = ceil_div(n, height) * height; // of a tile, and rows up to the end of one
    const int32_t* all_rows = twice ? rows.doubled : rows.offsets;
    const Array A = gathered(call, room_A, p.A, rows, twice,
                             {factors, factor, of_loss, of_sum, static_cast<const float*>(loss.data), static_cast<const float*>(log_sum.data), static_cast<float>(p.scale),
                              p.A.type == MOPS_B200_F16 ? 16384.f : 1.f});
    Array first = A; // of the two rows of each
    first.shape[0] = n, first.stride[0] = copies * A.stride[0];
    Packing packing(call);
    Array W = p.W;
    packing.add(W);
    packing.run();
    // Pieces of the vocabulary: as wide as there is room for dx, by steps whose tiles of grad_W are whole rounds of pairs (8192 rows of 100 003 x 1024: seven equal pieces, whose last rounds were a twelfth
    // full, took 1666 us for grad_W, some 1300 in these).
    constexpr int64_t kMostValues = int64_t(1) << 28; // of dx, with those behind the last row
    const int64_t most = std::max<int64_t>(kMostValues / (copies * whole) / 256 * 256, 256), across = ceil_div(columns, 256), unit = sms / 2 / std::gcd<int64_t>(sms / 2, across) * 256;
    const int64_t width = std::min(unit <= most ? most / unit * unit : most, whole_packs(vocabulary)), pieces = ceil_div(vocabulary, width);
    Scratch room_dx(call, static_cast<size_t>(copies * whole * width) * 2);
    // Slices of the piece for the products with W.
    const int64_t steps = ceil_div(std::min(width, vocabulary), kBoxDepth);
    const int64_t slices = best_slices(ceil_div(all, 2 * kTileRows) * ceil_div(columns, 256), sms / 2, steps, 0.42, 16, static_cast<double>(all) * columns * 8);
    const int64_t stride = (columns + 3) / 4 * 4;
    Scratch room_sums(call);
    if (need_A) room_sums.take(static_cast<size_t>(slices * all * stride) * sizeof(float));
    float* sums = room_sums.as<float>();
    for (int64_t v0 = 0; v0 < vocabulary; v0 += width) {
        const int64_t here = std::min(width, vocabulary - v0);
        uint16_t* w = static_cast<uint16_t*>(W.data) + v0 * W.stride[0];
        Array dx = contiguous(room_dx.as<void>(), A.type, all, here);
        dx.stride[0] = width;
        for_sixteen(A.type, [&](auto type) {
            constexpr bool BF16 = decltype(type)::value;
            auto launch = [&](auto parts) {
                using E = GradientStore<BF16, 256, decltype(parts)::value>;
                typename E::Args args{};
                args.out = static_cast<uint16_t*>(dx.data), args.rest = args.out + width, args.stride = copies * width;
                args.map = tensor_map(A.type, args.out, here, whole, 1, args.stride, 0, 32);
                if (twice) args.map_rest = tensor_map(A.type, args.rest, here, whole, 1, args.stride, 0, 32);
                args.columns = static_cast<int>(here), args.first_column = static_cast<int>(v0);
                args.scale2 = scale2, args.factors = factors;
                const TileProblem problem{first, rows.offsets, 1, n, columns, here};
                const TileOperand operands[2] = {{w, 1, W.stride[0], 0}, {w, 1, W.stride[0], 0}};
                if (n <= kTileRows) launch_tiles<BF16, false, 256, false, E, DecodeRows>(call, op, problem, operands, args);
                else launch_tiles<BF16, false, 256, true, E, DecodeRows>(call, op, problem, operands, args);
            };
            if (twice) launch(std::true_type());
            else launch(std::false_type());
            if (need_A) {
                const TileProblem sum_problem{dx, all_rows, 1, all, here, columns, slices};
                const TileOperand by_rows[2] = {{w, W.stride[0], 1, 0}, {w, W.stride[0], 1, 0}};
                using Sums = SumStore<256>;
                typename Sums::Args to{};
                to.map = tensor_map(MOPS_B200_F32, sums, columns, all, slices, stride, all * stride, 32);
                to.out = sums, to.rows = all, to.stride = stride, to.columns = static_cast<int>(columns), to.add = v0 > 0;
                launch_tiles<BF16, true, 256, true, Sums, DecodeRowSlices>(call, op, sum_problem, by_rows, to);
            }
        });
        MOPS_CUDA_OK(cudaGetLastError());
        uint16_t* const to_W = need_W ? static_cast<uint16_t*>(grad_W.data) + v0 * columns : nullptr;
        // (whole tiles of the gradient, or rows cut into slices and joined. Where the tiles are more than half of the pairs, or rows few, the first: 16384 rows of 9000 x 512 118 us against 151, of
        // 5000 x 512 108 and 114, of 2048 x 512 105 and 52; 1500 rows of 1000 x 256 16 and 18; 8192 rows of 26 112 x 1024 333 and 350)
        if (need_W && (ceil_div(here, 2 * kTileRows) * across >= sms / 4 || all <= 2048)) {
            for_sixteen(A.type, [&](auto type) {
                using E = ScaledStore<decltype(type)::value>;
                typename E::Args to{};
                to.loose = columns % 8 != 0 || reinterpret_cast<uintptr_t>(to_W) % 16 != 0;
                if (!to.loose) to.map = tensor_map(A.type, to_W, columns, here, 1, columns, 0, 32);
                to.out = to_W, to.columns = static_cast<int>(columns), to.factor = factor;
                // (the rows up to a whole stage are zeros)
                const TileProblem outer{dx, all_rows, 1, here, (all + 63) / 64 * 64, columns};
                const TileOperand a{A.data, A.stride[0], 1, 0}, operands[2] = {a, a};
                launch_tiles<decltype(type)::value, true, 256, true, E, DecodeDepth>(call, op, outer, operands, to);
            });
        } else if (need_W)
            multiply_outer(call, {contiguous(static_cast<uint16_t*>(grad_W.data) + v0 * columns, A.type, 1, here, columns), dx, A, all_rows, 1, factor}, op);
    }
    if (need_A)
        for_sixteen(A.type, [&](auto type) {
            using T = std::conditional_t<decltype(type)::value, __nv_bfloat16, __half>;
            scatter_sums(call, static_cast<T*>(grad_A.data), sums, slices, stride, rows, n, columns, twice, factor);
        });
    MOPS_CUDA_OK(cudaGetLastError());
    note_kernel_f("loss_gradient_mma<%s>, %d pieces, %d slices", A.type == MOPS_B200_BF16 ? "bf16" : "f16", static_cast<int>(pieces), static_cast<int>(slices));
}

} // namespace mops_b200
