// Tiles of rows that belong to one group, for kernels over arrays whose rows are sorted by group.
//
// The offsets of the groups are in device memory, so the host does not know how many tiles there are. It launches for the
// most there can be (one partial tile for each group on top of the full ones), and each tile looks up which group it is
// in, a warp at a time: 32 groups per step, whose tiles a prefix sum over the lanes counts.
#ifndef MOPS_B200_GROUP_TILES_CUH
#define MOPS_B200_GROUP_TILES_CUH

#include "device.cuh"

namespace mops_b200 {

// Rows [row, row + rows) of `group`; group == -1: rows of no group. rows == 0: there is no such tile.
struct GroupTile {
    int64_t group, row;
    int rows;
};

// Where group g's rows lie, kept inside of [0, rows) whatever the offsets say. g == -1: the rows in front of the
// first group; g == groups: those behind the last one.
__device__ __forceinline__ void group_bounds(const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
                                             int64_t g, int64_t& lo, int64_t& hi) {
    lo = g < 0 ? 0 : min(max(int64_t(__ldg(offsets + g)), int64_t(0)), rows);
    hi = g >= groups ? rows : min(max(int64_t(__ldg(offsets + g + 1)), int64_t(0)), rows);
    hi = max(lo, hi);
}

inline int64_t most_tiles(int64_t rows, int64_t groups, int tile_rows) {
    return rows / tile_rows + std::min(rows, groups + 2);
}

// Walks the tiles of all groups in order. All lanes of a warp call it together and get the same answers; `want` must
// not decrease from call to call.
struct TileWalk {
    const int32_t* offsets;
    int64_t groups, rows;
    int tile_rows;
    int64_t base = -1, before = 0; // first group of the step at hand, tiles in front of it
    int64_t mine = -1;             // tiles of group base + lane (-1: not read yet)

    __device__ TileWalk(const int32_t* offsets, int64_t groups, int64_t rows, int tile_rows)
        : offsets(offsets), groups(groups), rows(rows), tile_rows(tile_rows) {}

    __device__ GroupTile find(int64_t want, int lane) {
        while (base <= groups) {
            if (mine < 0) {
                mine = 0;
                if (base + lane <= groups) {
                    int64_t lo, hi;
                    group_bounds(offsets, groups, rows, base + lane, lo, hi);
                    mine = ceil_div_device(hi - lo, tile_rows);
                }
            }
            int64_t up_to = mine; // tiles of groups base .. base + lane
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t v = __shfl_up_sync(kFullMask, up_to, d);
                if (lane >= d) up_to += v;
            }
            const unsigned reached = __ballot_sync(kFullMask, before + up_to > want);
            if (reached) {
                const int at = __ffs(reached) - 1;
                const int64_t within = want - before - __shfl_sync(kFullMask, up_to - mine, at);
                GroupTile t;
                t.group = base + at;
                int64_t lo, hi;
                group_bounds(offsets, groups, rows, t.group, lo, hi);
                t.row = lo + within * tile_rows;
                t.rows = static_cast<int>(min(hi - t.row, int64_t(tile_rows)));
                if (t.group >= groups) t.group = -1;
                return t;
            }
            before += __shfl_sync(kFullMask, up_to, 31);
            base += 32;
            mine = -1;
        }
        return GroupTile{-1, 0, 0};
    }

    __device__ static int64_t ceil_div_device(int64_t a, int64_t b) { return (a + b - 1) / b; }
};

// Reports offsets that are not ascending within [0, rows] (index array 0); any block may do it.
__device__ __forceinline__ void check_offsets(const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
                                              const Status& st) {
    bool bad = false;
    for (int64_t g = threadIdx.x; g <= groups; g += blockDim.x) {
        const int64_t v = __ldg(offsets + g);
        bad |= v < 0 || v > rows || (g < groups && __ldg(offsets + g + 1) < v);
    }
    if (bad) report_bad_index(st, 0);
}

} // namespace mops_b200

#endif
