// Which rows belong to which expert: the group tables of the expert-layer operators.
//
// A group table is `groups + 1` int32 offsets in device memory, rows [offsets[g], offsets[g + 1]) of the row operand
// belonging to group g. The host never sees it, so a launch is sized by an upper bound and every workgroup finds its
// own tile here. What is read from the table is cut to [0, rows] before it becomes an address: a table with other
// contents gives wrong results, not accesses out of range.
#pragma once

#include "common.h"

namespace prism {

struct GroupTile {
    int group;    // -1: there is no such tile
    int row0;     // the tile's first row
    int row_end;  // one past the group's last row
};

__device__ __forceinline__ int clamp_offset(int v, int rows) { return v < 0 ? 0 : (v > rows ? rows : v); }

__device__ __forceinline__ int wave_inclusive_sum(int v, int lane) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Tile number `tile` of the row tiles of all groups, in group order, each group cut into tiles of `tile_rows` rows.
// Called by whole wavefronts; the result is wave-uniform. The sums stay below 2^31 whatever the table holds: a launch has at
// most 2^24 row tiles, no group has more tiles than that, and the search ends in the 64 groups that pass `tile`.
__device__ __forceinline__ GroupTile find_group_tile(const int32_t* offsets, int groups, int rows, int tile, int tile_rows) {
    const int lane = threadIdx.x & (kWave - 1);
    int before = 0;
    for (int base = 0; base < groups; base += kWave) {
        const int g = base + lane;
        int lo = 0, hi = 0;
        if (g < groups) {
            lo = clamp_offset(offsets[g], rows);
            hi = clamp_offset(offsets[g + 1], rows);
        }
        const int tiles = hi > lo ? (hi - lo - 1) / tile_rows + 1 : 0;
        const int upto = before + wave_inclusive_sum(tiles, lane);
        const unsigned long long mask = __ballot(upto > tile);
        if (mask) {
            const int src = __builtin_ctzll(mask);
            GroupTile t;
            t.group = __builtin_amdgcn_readfirstlane(base + src);
            const int index = tile - (__builtin_amdgcn_readlane(upto, src) - __builtin_amdgcn_readlane(tiles, src));  // within the group
            t.row0 = __builtin_amdgcn_readlane(lo, src) + index * tile_rows;
            t.row_end = __builtin_amdgcn_readlane(hi, src);
            return t;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return GroupTile{-1, 0, 0};
}

// The most row tiles that groups of together `rows` rows can have: a group wastes less than one tile, and a tile has
// at least one row.
inline long long most_row_tiles(long long rows, int groups, int tile_rows) {
    const long long cut = rows / tile_rows + groups;
    return cut < rows ? cut : rows;
}

}  // namespace prism
