// Pieces of work on arrays whose rows are sorted by group, found on the device.
//
// The offsets of the groups are in device memory, so the host does not know how many tiles of rows there are. Each worker (a
// warp) counts through the groups, 32 per step with a prefix sum over the lanes, to the piece that it is to do.
#ifndef MOPS_B200_GROUP_TILES_CUH
#define MOPS_B200_GROUP_TILES_CUH

#include "device.cuh"
#include "group_ranges.hpp"

namespace mops_b200 {

// Where group g's rows lie, kept inside of [0, rows) whatever the offsets say. g == -1: the rows in front of the
// first group; g == groups: those behind the last one.
__device__ __forceinline__ void group_bounds(const int32_t* __restrict__ offsets, int64_t groups, int64_t rows,
                                             int64_t g, int64_t& lo, int64_t& hi) {
    const RowRange r = rows_between(g < 0 ? 0 : int64_t(__ldg(offsets + g)), g >= groups ? rows : int64_t(__ldg(offsets + g + 1)), rows);
    lo = r.lo, hi = r.hi;
}

// The rows [lo, hi) of a group and which of its pieces is meant; found == false: there is no such piece.
struct GroupPiece {
    bool found;
    int64_t group, lo, hi, within;
};

// Walks the pieces of groups first .. last in order, where pieces(rows of the group) says how many a group has. All
// lanes of a warp call it together and get the same answers. It goes on from where the last call found its piece (and begins anew where a
// piece in front of that is asked for).
template <typename Pieces> struct GroupWalk {
    const int32_t* offsets;
    int64_t groups, rows, first, last;
    Pieces pieces;
    int64_t base, before = 0;  // first group of the step at hand, pieces in front of it
    int64_t up_to = 0;         // pieces of groups base .. base + lane
    bool counted = false;

    __device__ GroupWalk(const int32_t* offsets, int64_t groups, int64_t rows, int64_t first, int64_t last, Pieces pieces)
        : offsets(offsets), groups(groups), rows(rows), first(first), last(last), pieces(pieces), base(first) {}

    __device__ GroupPiece find(int64_t want, int lane) {
        if (want < before) base = first, before = 0, counted = false;
        while (base <= last) {
            if (!counted) {
                up_to = 0;
                if (base + lane <= last) {
                    int64_t lo, hi;
                    group_bounds(offsets, groups, rows, base + lane, lo, hi);
                    up_to = pieces(hi - lo);
                }
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int64_t v = __shfl_up_sync(kFullMask, up_to, d);
                    if (lane >= d) up_to += v;
                }
                counted = true;
            }
            const unsigned reached = __ballot_sync(kFullMask, before + up_to > want);
            if (reached) {
                const int at = __ffs(reached) - 1;
                const int64_t in_front = __shfl_sync(kFullMask, up_to, at > 0 ? at - 1 : 0);
                GroupPiece p;
                p.found = true;
                p.group = base + at;
                p.within = want - before - (at > 0 ? in_front : 0);
                group_bounds(offsets, groups, rows, p.group, p.lo, p.hi);
                return p;
            }
            before += __shfl_sync(kFullMask, up_to, 31);
            base += 32;
            counted = false;
        }
        return GroupPiece{false, 0, 0, 0, 0};
    }
};

// Tiles of `tile_rows` rows by `columns` tiles.
struct RowTiles {
    int tile_rows;
    int64_t columns;
    __device__ int64_t operator()(int64_t rows) const { return (rows + tile_rows - 1) / tile_rows * columns; }
};
inline int64_t most_row_tiles(int64_t rows, int64_t groups, int tile_rows) {
    return rows / tile_rows + std::min(rows, groups + 2);
}

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
