#include "pack.hpp"

#include "checks.hpp"
#include "tensor_map.hpp"

namespace mops_b200 {
namespace {

constexpr int kThreads = 256;

struct Jobs {
    Packing::Job job[Packing::kMost];
};

// Arrays whose rows begin anywhere, as a user's odd widths are, cannot be fetched by the copy engine; a copy of them costs less than tiles put together value by value
// (3001 rows of 7 groups, 509 x 771 in bf16, forward and gradients: 200 us so, 89 with copies; the copies of A and W, 7 MB, take some 5 us of it).
// A thread copies 16 bytes: from the two vectors that they lie in (16-bit values: they begin at any multiple of 2 bytes) where both are inside of the
// array, else value by value.
template <typename T>
__global__ void __launch_bounds__(kThreads)
pack_rows(const __grid_constant__ Jobs jobs) {
    const Packing::Job& j = jobs.job[blockIdx.y];
    constexpr int kValues = kPack<T>;
    const int64_t pieces = j.slices * j.outer * j.packs;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; at < pieces; at += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t row = at / j.packs, pack = at - row * j.packs, slice = row / j.outer;
        const T* p = static_cast<const T*>(j.from) + slice * j.slice_stride + (row - slice * j.outer) * j.outer_stride + pack * kValues;
        const int64_t n = j.inner - pack * kValues;
        uint32_t w[8] = {};
        const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15;
        const unsigned char* from = reinterpret_cast<const unsigned char*>(p) - shift;
        if (sizeof(T) == 2 && n >= kValues && from >= j.begin && from + 32 <= j.end) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(from)), v = __ldg(reinterpret_cast<const uint4*>(from) + 1);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
            // down by 8, 4 and 2 bytes as needed
            if (shift & 8) {
#pragma unroll
                for (int i = 0; i < 6; i++) w[i] = w[i + 2];
            }
            if (shift & 4) {
#pragma unroll
                for (int i = 0; i < 5; i++) w[i] = w[i + 1];
            }
            if (shift & 2) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kValues; i++) {
                if (i >= n) continue;
                if constexpr (sizeof(T) == 2) w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p) + i)) << (16 * (i & 1));
                else w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
            }
        }
        reinterpret_cast<uint4*>(j.to)[at] = make_uint4(w[0], w[1], w[2], w[3]);
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
    int64_t most = 0;
    for (int i = 0; i < n_; i++) {
        jobs.job[i] = jobs_[i];
        most = std::max(most, jobs_[i].slices * jobs_[i].outer * jobs_[i].packs);
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(most, kThreads), int64_t(sm_count(call_.device)) * 16)), static_cast<unsigned>(n_));
    if (type_ == MOPS_B200_F32) pack_rows<float><<<grid, kThreads, 0, call_.stream>>>(jobs);
    else pack_rows<__half><<<grid, kThreads, 0, call_.stream>>>(jobs);
    note_kernel_f("pack_rows, %d arrays", n_);
    MOPS_CUDA_OK(cudaGetLastError());
}

void Packing::release() {
    while (n_ > 0) scratch_free(call_, jobs_[--n_].to);
}

} // namespace mops_b200
