#include "pack.hpp"

#include "checks.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kBlocks = 8;     // that an SM has threads for
constexpr int64_t kLeastOfRun = 2; // copies of a thread

struct Jobs {
    Packing::Job job[Packing::kMost];
};

// Arrays whose rows begin anywhere, as a user's odd widths are, cannot be fetched by the copy engine; a copy of them costs less than tiles put together value by value
// (3001 rows of 7 groups, 509 x 771 in bf16, forward and gradients: 200 us so, 89 with copies; the copies of A and W, 7 MB, take some 5 us of it).
// A thread copies 16 bytes at a time; 2 to 32 threads side by side, as many as a row may need, take a row, so that where it lies is worked out once for all of them (32 003 rows of 771 in
// f16: 18.5 us; worked out for every 16 bytes 29).
template <typename T>
__global__ void __launch_bounds__(kThreads)
pack_rows(const __grid_constant__ Jobs jobs) {
    const Packing::Job& j = jobs.job[blockIdx.y];
    const int64_t rows = j.slices * j.outer, step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < rows; row += step) {
        const int64_t slice = j.slices == 1 ? 0 : row / j.outer;
        const T* p = static_cast<const T*>(j.from) + slice * j.slice_stride + (row - slice * j.outer) * j.outer_stride;
        uint4* to = static_cast<uint4*>(j.to) + row * j.packs;
#pragma unroll 4
        for (int64_t pack = threadIdx.x; pack < j.packs; pack += blockDim.x)
            to[pack] = load_anywhere<T>(p + pack * kPack<T>, j.inner - pack * kPack<T>, j.begin, j.end);
    }
}

// The same where there are so few rows that SMs would be without work: each is cut into runs, which such groups of threads take one after the other. (A matrix of 3 x 500 001 in bf16 with 300 rows, products and
// all: 313 us for 1375, 16 x 100 003 74 for 287. As a kernel of its own, since this one has 40 registers, with which 20 000 rows of 1001 take 54 us for 48.)
struct Runs {
    int64_t of_a_row[Packing::kMost], packs[Packing::kMost]; // packs: of a run
};
template <typename T>
__global__ void __launch_bounds__(kThreads)
pack_runs(const __grid_constant__ Jobs jobs, const __grid_constant__ Runs runs) {
    const Packing::Job& j = jobs.job[blockIdx.y];
    const int64_t of_a_row = runs.of_a_row[blockIdx.y], all = j.slices * j.outer * of_a_row, step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    for (int64_t run = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; run < all; run += step) {
        const int64_t row = run / of_a_row, slice = row / j.outer;
        const int64_t first = (run - row * of_a_row) * runs.packs[blockIdx.y], end = min(first + runs.packs[blockIdx.y], j.packs);
        const T* p = static_cast<const T*>(j.from) + slice * j.slice_stride + (row - slice * j.outer) * j.outer_stride;
        uint4* to = static_cast<uint4*>(j.to) + row * j.packs;
#pragma unroll 4
        for (int64_t pack = first + threadIdx.x; pack < end; pack += blockDim.x)
            to[pack] = load_anywhere<T>(p + pack * kPack<T>, j.inner - pack * kPack<T>, j.begin, j.end);
    }
}

} // namespace

void Packing::add(Array& a) {
    const int last = a.dimensions - 1;
    const int inner = a.dimensions == 3 && a.stride[last] != 1 ? last - 1 : last, outer = a.dimensions == 3 && inner == last - 1 ? last : last - 1;
    const int64_t slices = a.dimensions == 3 ? a.shape[0] : 1, slice_stride = a.dimensions == 3 ? a.stride[0] : 0;
    if (slices == 0 || a.shape[inner] == 0 || a.shape[outer] == 0 ||
        boxable(a.type, a.data, a.shape[inner], a.shape[outer], slices, a.stride[outer], slice_stride))
        return;
    const int64_t bytes = type_bytes(a.type), values = 16 / bytes, packs = ceil_div(a.shape[inner], values);
    Job& j = jobs_[n_];
    type_ = a.type;
    j.from = a.data;
    j.to = scratch_alloc(call_, static_cast<size_t>(slices * a.shape[outer] * packs) * 16);
    n_++;
    j.outer = a.shape[outer], j.outer_stride = a.stride[outer], j.slices = slices, j.slice_stride = slice_stride;
    j.inner = a.shape[inner], j.packs = packs;
    j.begin = static_cast<const unsigned char*>(a.data);
    j.end = j.begin + ((slices - 1) * slice_stride + (j.outer - 1) * j.outer_stride + j.inner) * bytes;
    a.data = j.to;
    a.stride[outer] = packs * values;
    if (a.dimensions == 3) a.stride[0] = a.shape[outer] * packs * values;
}

void Packing::run() {
    if (n_ == 0) return;
    Jobs jobs{};
    int64_t most = 0, packs = 1;
    for (int i = 0; i < n_; i++) {
        jobs.job[i] = jobs_[i];
        most = std::max(most, jobs_[i].slices * jobs_[i].outer);
        packs = std::max(packs, jobs_[i].packs);
    }
    unsigned across = 2;
    while (across < 32 && across < packs) across *= 2;
    const dim3 block(across, kThreads / across);
    const int64_t sms = sm_count(call_.device), most_blocks = sms * 16;
    auto launch = [&](auto zero) {
        using T = decltype(zero);
        const int64_t blocks = ceil_div(most, block.y);
        if (blocks >= kBlocks * sms || packs < 2 * kLeastOfRun * across) {
            pack_rows<T><<<dim3(static_cast<unsigned>(std::min(blocks, most_blocks)), static_cast<unsigned>(n_)), block, 0, call_.stream>>>(jobs);
            return;
        }
        Runs runs{};
        most = 0;
        for (int i = 0; i < n_; i++) {
            const int64_t rows = jobs_[i].slices * jobs_[i].outer, steps = ceil_div(jobs_[i].packs, int64_t(across));
            runs.packs[i] = std::max(ceil_div(steps, ceil_div(kBlocks * sms * block.y, rows)), kLeastOfRun) * across;
            runs.of_a_row[i] = ceil_div(jobs_[i].packs, runs.packs[i]);
            most = std::max(most, rows * runs.of_a_row[i]);
        }
        pack_runs<T><<<dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(most, block.y), most_blocks)), static_cast<unsigned>(n_)), block, 0, call_.stream>>>(jobs, runs);
    };
    if (type_ == MOPS_B200_F32) launch(float());
    else launch(__half());
    note_kernel_f("pack_rows, %d arrays", n_);
    MOPS_CUDA_OK(cudaGetLastError());
}

void Packing::release() {
    while (n_ > 0) scratch_free(call_, jobs_[--n_].to);
}

} // namespace mops_b200
