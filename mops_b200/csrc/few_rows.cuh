// What the kernels for a few rows in all share: pieces of a few rows, clusters of blocks that have a part of the depth each, and
// how the blocks that multiply on tensor cores with the operands the other way round lay out shared memory.
#ifndef MOPS_B200_FEW_ROWS_CUH
#define MOPS_B200_FEW_ROWS_CUH

#include <cooperative_groups.h>

#include "group_tiles.cuh"
#include "grouped_block.cuh"

namespace mops_b200 {

namespace cg = cooperative_groups;

constexpr int kMostParts = 8;    // of the depth: blocks of a cluster

struct FewRows { // pieces: up to `most` rows of a group
    int most;
    __device__ int64_t operator()(int64_t rows) const { return (rows + most - 1) / most; }
};

// The rows of no group: zeros in kColumns columns.
template <typename T, int kColumns, int kThreads>
__device__ __forceinline__ void clear_others(T* __restrict__ out, const int32_t* __restrict__ offsets, int64_t groups, int64_t rows, int column, int columns) {
    for_rows_of_no_group(__ldg(offsets), __ldg(offsets + groups), rows, [&](int64_t r) {
        for (int c = threadIdx.x; c < kColumns && column + c < columns; c += kThreads) out[r * columns + column + c] = T(0);
    });
}

// How many parts the depth is cut into: until there are `enough` blocks, of `least` values of depth at least.
inline int parts_of_depth(int64_t tiles, int64_t enough, int64_t depth, int64_t least) {
    int parts = 1;
    while (parts < kMostParts && tiles * parts < enough && depth / (2 * parts) >= least) parts *= 2;
    return parts;
}

// Clusters of `parts` blocks along x.
struct Clusters {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute cluster{};
    Clusters(const Call& call, const std::string& op, int64_t tiles, int parts, int64_t pieces, int threads, int bytes) {
        fits_int32(static_cast<size_t>(tiles * parts), "the number of columns", op);
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = static_cast<unsigned>(parts), cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = 1;
        config.gridDim = dim3(static_cast<unsigned>(tiles * parts), static_cast<unsigned>(pieces));
        config.blockDim = dim3(static_cast<unsigned>(threads));
        config.dynamicSmemBytes = static_cast<size_t>(bytes);
        config.stream = call.stream;
    }
};

constexpr int kTileThreads = 128;
template <int kRows_> struct FewLayout {
    static constexpr bool kPair = false, kRepairs = false;
    static constexpr int kM = kTileRows * kBoxRow, kX = kRows_ * kBoxRow, kStage = kM + kX;
    static constexpr int kStages = 5 * (kTileRows + 16) / (kTileRows + kRows_); // some 90 KB, for two blocks on an SM
    static constexpr int kRingsAt = kStages * kStage;
    static constexpr int kBytes = kRingsAt + 256 + 1024;
    static constexpr unsigned kTmem = kRows_ < 32 ? 32 : kRows_;
    struct Rings {
        Ring<kStages> stages;
        uint64_t done;
        uint32_t tmem;
        int gave_up;
        __device__ void begin() {
            stages.begin(1, 1);
            mbarrier_init(&done, 1);
        }
    };
    static_assert(sizeof(Rings) <= 256, "room for the rings");
};

} // namespace mops_b200

#endif
