// Products of a few rows on 16 x 16 x 32 matrix instructions, shared by the bf16 and the 4-bit weights.
//
// With up to 16 rows the weights bound the product: they go from memory into the registers of the wavefront that
// multiplies them, 16 columns to a tile, and the rows of x (padded to 16 with whatever is at hand: a row of the
// instruction's operand only enters its own row of the result) come with them.
#pragma once

#include <cmath>

#include "common.h"

namespace prism {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The x of instruction C of a round, from the round's loads. A load brings an instruction's x with 16 rows; with 4 rows (1
// row) it brings that of 4 (16) instructions, the 16 lanes holding rows 0 .. ROWS - 1 of one after the other, and a rotation
// within 16 lanes moves an instruction's rows to the lanes that count, 0 .. ROWS - 1.
template <int ROWS, int C, int LOADS>
__device__ __forceinline__ void instruction_x(const bf16x8 (&x)[LOADS], bf16x8& mine) {
    constexpr int BRINGS = 16 / ROWS, FROM = (C % BRINGS) * ROWS;
    mine = x[C / BRINGS];
    if constexpr (FROM != 0) {
        u32x4 v = __builtin_bit_cast(u32x4, mine);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_update_dpp(0, v[i], 0x120 + (16 - FROM), 0xf, 0xf, true);  // row_ror
        mine = __builtin_bit_cast(bf16x8, v);
    }
}

// The row tiles of a group table that exist, about: with fewer rows than groups, the groups that so many rows hit at random. Taken as one a
// row, 32 rows of 64 matrices of 1536 x 2048 in 4 bits, G = 128, take 15.1 us instead of 13.3 with weights that the memory-side
// cache holds and 16.1 instead of 15.1 with weights from memory (G = 32 with zero points: 17.3 and 16.5, 19.1 and 18.5).
inline long long busy_row_tiles(long long rows, int groups, long long most) {
    if (rows >= groups) return most;
    return static_cast<long long>(groups * -std::expm1(-static_cast<double>(rows) / groups) + 0.5);
}

// How a column tile's K is shared: by as few wavefronts as give every CU per_cu of them (each has a fixed cost, and their
// parts meet at the end), not more than there are steps of step_k. `busy`: the row tiles that exist, about.
inline int few_rows_k_parts(long long busy, int N, int K, int step_k, int most, int per_cu) {
    int parts = 1;
    while (parts < most && busy * ceil_div(N, 16) * parts < static_cast<long long>(per_cu) * cu_count() && parts * step_k < K) parts *= 2;
    return parts;
}

}  // namespace prism
