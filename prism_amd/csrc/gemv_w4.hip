// Few rows times weights held in 4 bits: y[r][n] = sum_k x[r][k] s[n][k / G] (q[n][k] - z[n][k / G]), one weight
// matrix, or one per group of rows (expert_groups.h). q: two weights to a byte, the even k in the low nibble; s: bf16;
// z: uint8, 8 where absent; x: bf16; sums in fp32.
//
// Reading q bounds it: N K / 2 bytes for 2 r N K flop. The weights go from memory straight into registers, become bf16
// there and are multiplied on the matrix cores (v_mfma_f32_16x16x32_bf16: 16 rows of x, padded with zeros, by 16
// columns n, 32 k at a time), so that 16 rows share one unpacking. Three things keep the vector ALU out of the way:
//   * the order of k inside an instruction is free as long as both operands have the same: a lane takes 16 consecutive
//     bytes of its row (32 weights; where groups are shorter than the 128 of a row's four lanes, the lanes exchange dwords
//     so that an instruction stays inside a group), and the values of a dword in the order 0 4 1 5 2 6 3 7, in which
//     `(w >> c) & 0x00780078 | 0x39803980` yields two of them;
//   * that pattern is the bf16 number 2^-16 (16 + q), exactly: what it adds is taken off per group of G, as
//     (16 + z) * (sum of 2^-16 x over the group), whose sums come from the same instruction on a matrix of 2^-16. With that
//     factor, taken back off the result, neither part overflows for any finite x (128 * 271 < 2^16) though x (q - z) does not,
//     and products keep all their bits down to the smallest x (2^-133 2^-16 is fp32's smallest number);
//   * the scale is applied to a group's fp32 sum, not to the weights. Nothing is rounded below 32 bits but the result.
// Calls back to back with the same weights every time, which the memory-side cache then holds, / with weights from memory: 8192 x
// 8192, G = 128, 1 row: 10.0 / 12.0 us (34.6 MB, 2.9 TB/s); 16384 x 16384: 26.6 / 32 to 38 us (139 MB, 3.7 to 4.3 TB/s); 32 rows of 64
// matrices 1536 x 2048, 26 of them used: 13.3 / 15.1 us with G = 128, 16.5 / 18.5 with G = 32, zero points and fp32 results. What is
// left is latency: two rounds of loads in flight a wavefront, three to six rounds a slice, and some 4 us in which the first weights
// arrive and the parts meet; 8 to 11 wavefronts a CU are there on average, of the 12 that the registers allow at G = 32 with zero
// points (16 elsewhere, 8 to 12 at group sizes that are looked up). x in LDS (+2 to 5 us), sixteen wavefronts a workgroup,
// all of K up front and non-temporal loads (+1.4 us) were slower.
// Beyond four rows x counts: a tile of 16 columns reads 8 bytes of weights and 2 bytes a row of x for a k, x from the L2.
// 8192 x 8192, G = 128, kernels by themselves: 1, 2, 4, 5, 8, 16 rows 11.7, 12.8, 14.1, 16.6, 18.8, 42.0 us; 64, 256, 2048 rows 94, 331, 2456 us,
// since every 16 rows unpack all weights again.
#include <type_traits>

#include "common.h"
#include "expert_groups.h"
#include "few_rows.h"
#include "tile_map.h"

namespace prism {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Waves = 8, kW4Few = 2, kW4Block = 128;  // most and fewest wavefronts of a workgroup; k per step: 16 B of weights a lane

struct W4Problem {
    const uint16_t* x;
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;
    const int32_t* offsets;  // null: one group of all rows
    void* y;
    long long ldx, ldq, ldy, q_stride, s_stride;  // q_stride, s_stride: between the groups' matrices
    int groups, rows, N, K, G, n_groups;          // n_groups: scales per row
    int tiles_n, row_tiles;  // workgroups along N, tiles of 16 rows
    int k_parts, n_parts; // wavefronts that share a column tile's K, column tiles of a workgroup
    int slice;            // steps of such a wavefront
};

__device__ __forceinline__ void store_y(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_y(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }

// The results' factor of 2^-16 is taken off at the end.
constexpr float kUnit = 65536.0f;

// Eight weights of a dword as bf16 2^-16 (16 + q), in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ bf16x8 weights_of(uint32_t w) {
    constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x39803980u;
    u32x4 r;
    r[0] = ((w << 3) & kMask) | kSixteen;
    r[1] = ((w >> 1) & kMask) | kSixteen;
    r[2] = ((w >> 5) & kMask) | kSixteen;
    r[3] = ((w >> 9) & kMask) | kSixteen;
    return __builtin_bit_cast(bf16x8, r);
}
// Eight consecutive values of x in that order.
__device__ __forceinline__ bf16x8 ordered(u32x4 v) {
    u32x4 r;
    r[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100u);
    r[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302u);
    r[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100u);
    r[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302u);
    return __builtin_bit_cast(bf16x8, r);
}

// A dword's four from each of a row's lanes, turned: dword j of the lane with l / 16 == i becomes dword i of the lane with
// l / 16 == j. Four swaps of halves and of rows of 16 lanes between registers, no LDS.
__device__ __forceinline__ u32x4 turned(u32x4 w) {
    auto swap32 = [](uint32_t& a, uint32_t& b) {
        const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    auto swap16 = [](uint32_t& a, uint32_t& b) {
        const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    uint32_t r0 = w[0], r1 = w[1], r2 = w[2], r3 = w[3];
    swap32(r0, r2);
    swap32(r1, r3);
    swap16(r0, r1);
    swap16(r2, r3);
    return u32x4{r0, r1, r2, r3};
}

// Scales of a step: kOne: a step is a group (G = 128); kTwo, kFour: it is two or four (64, 32); kAny: looked up.
enum class StepScales { kOne, kTwo, kFour, kAny };

constexpr int parts_of(StepScales s) { return s == StepScales::kOne ? 1 : (s == StepScales::kTwo ? 2 : 4); }

// What a wavefront works on: its lane's row of weights and scales, its steps (first .. first + slice - 1 of `steps`, of
// which `whole` are complete), and the tile's rows of x.
struct W4Slice {
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;
    const uint16_t* x;
    long long ldx;
    int rows, first, slice, whole, steps, K, G;
};

// The 16 x 16 result of a slice, 4 rows and a column to a lane, for up to ROWS rows of x (1, 4 or 16; see instruction_x).
template <StepScales SCALES, bool ZEROS, int ROWS>
__device__ __forceinline__ f32x4 multiply_slice(const W4Slice& p) {
    constexpr bool TURN = SCALES != StepScales::kOne;  // G below 128: an instruction's 32 k are consecutive
    constexpr int PARTS = parts_of(SCALES), PER = 4 / PARTS;  // parts of a step with a scale each, instructions of a part
    constexpr int U = ROWS == 16 ? 2 : 4;                     // steps of a round
    constexpr int BRINGS = 16 / ROWS, X_LOADS = U * 4 / BRINGS;
    const int lane = threadIdx.x % kWave, l16 = lane % 16, lq = lane / 16;
    const uint16_t* x_row = p.x + (l16 % ROWS < p.rows ? l16 % ROWS : p.rows - 1) * p.ldx + (TURN ? 8 : 32) * lq;
    // A round: the weights, scales and zero points of U steps and the x they meet, fetched two rounds ahead. Loads are
    // waited for in order: x is not asked for later than its weights, and nothing is fetched under a condition (where two
    // paths with different loads meet, the wait has to assume the shorter one and waits for the rounds ahead as well).
    struct Round {
        u32x4 w[U], x[X_LOADS];
        uint16_t s[U * PARTS];
        uint8_t z[U * PARTS];
    };
    // FULL: all U steps from `first` on are complete ones; else those that are not fetch the last complete one again.
    auto fetch = [&](auto full, Round& r, int first) {
        constexpr bool FULL = decltype(full)::value;
        auto step_of = [&](int u) { return FULL || first + u < p.whole ? first + u : p.whole - 1; };
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r.w[u], p.q + static_cast<long long>(step_of(u)) * (kW4Block / 2), 16);
#pragma unroll
        for (int j = 0; j < X_LOADS; ++j) {
            const int c = j * BRINGS + l16 / ROWS;  // the lane's instruction of the round
            __builtin_memcpy(&r.x[j], x_row + step_of(c / 4) * kW4Block + (TURN ? 32 : 8) * (c % 4), 16);
        }
        if constexpr (FULL && SCALES != StepScales::kAny) {
            __builtin_memcpy(r.s, p.scales + first * PARTS, U * PARTS * 2);
            if constexpr (ZEROS) __builtin_memcpy(r.z, p.zeros + first * PARTS, U * PARTS);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < PARTS; ++i) {
                    const int gi = SCALES != StepScales::kAny ? step_of(u) * PARTS + i : (step_of(u) * kW4Block + i * 32) / p.G;
                    r.s[u * PARTS + i] = p.scales[gi];
                    if constexpr (ZEROS) r.z[u * PARTS + i] = p.zeros[gi];
                }
        }
    };
    f32x4 total = {0.0f, 0.0f, 0.0f, 0.0f};
    const u32x4 one = {0x37803780u, 0x37803780u, 0x37803780u, 0x37803780u};  // 2^-16
    const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
    auto multiply = [&](u32x4 w, const bf16x8 (&x)[4], const uint16_t* s, const uint8_t* z) {
        if constexpr (TURN) w = turned(w);
        f32x4 dot[PARTS], sum[PARTS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i % PER == 0) dot[i / PER] = sum[i / PER] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            dot[i / PER] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], weights_of(w[i]), dot[i / PER], 0, 0, 0);
            sum[i / PER] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], ones, sum[i / PER], 0, 0, 0);
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const float scale = __builtin_bit_cast(float, static_cast<uint32_t>(s[part]) << 16), zero = ZEROS ? 16.0f + z[part] : 24.0f;
#pragma unroll
            for (int v = 0; v < (ROWS == 1 ? 1 : 4); ++v) total[v] = __builtin_fmaf(scale, __builtin_fmaf(-zero, sum[part][v], dot[part][v]), total[v]);
        }
    };
    auto compute = [&](const Round& r, int count) {
        bf16x8 x[X_LOADS];
#pragma unroll
        for (int j = 0; j < X_LOADS; ++j) x[j] = ordered(r.x[j]);
        auto step = [&](auto u_c) {
            constexpr int u = decltype(u_c)::value;
            if (u >= count) return;
            bf16x8 mine[4];
            instruction_x<ROWS, u * 4 + 0>(x, mine[0]);
            instruction_x<ROWS, u * 4 + 1>(x, mine[1]);
            instruction_x<ROWS, u * 4 + 2>(x, mine[2]);
            instruction_x<ROWS, u * 4 + 3>(x, mine[3]);
            multiply(r.w[u], mine, &r.s[u * PARTS], &r.z[u * PARTS]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        if constexpr (U == 4) {
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        }
    };
    using yes = std::integral_constant<bool, true>;
    using no = std::integral_constant<bool, false>;
    const int end = p.first + p.slice < p.whole ? p.first + p.slice : p.whole, rounds = end > p.first ? (end - p.first) / U : 0;
    if (rounds > 0) {
        auto round_at = [&](int r) { return p.first + (r < rounds ? r : rounds - 1) * U; };
        Round a, b;
        fetch(yes{}, a, p.first);
        fetch(yes{}, b, round_at(1));
        for (int r = 0;; r += 2) {
            compute(a, U);
            if (r + 2 >= rounds) {
                if (r + 1 < rounds) compute(b, U);
                break;
            }
            fetch(yes{}, a, round_at(r + 2));
            compute(b, U);
            fetch(yes{}, b, round_at(r + 3));
        }
    }
    const int behind = p.first + rounds * U;
    if (behind < end) {  // fewer than U complete steps are left
        Round a;
        fetch(no{}, a, behind);
        compute(a, end - behind);
    }
    if (p.whole < p.steps && p.first <= p.whole && p.whole < p.first + p.slice) {  // the partial last step: nothing is read beyond the rows
        const int bytes = (p.K + 1) / 2 - p.whole * (kW4Block / 2) - lq * 16;
        u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < bytes) w[i / 4] |= static_cast<uint32_t>(p.q[static_cast<long long>(p.whole) * (kW4Block / 2) + i]) << (8 * (i % 4));
        bf16x8 x[4];
        const uint16_t* own = p.x + (l16 < p.rows ? l16 : p.rows - 1) * p.ldx + p.whole * kW4Block + (TURN ? 8 : 32) * lq;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = p.K - p.whole * kW4Block - (TURN ? 8 : 32) * lq - (TURN ? 32 : 8) * i;
            u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) v[e / 2] |= static_cast<uint32_t>(own[(TURN ? 32 : 8) * i + e]) << (16 * (e % 2));
            x[i] = ordered(v);
        }
        uint16_t s[PARTS];
        uint8_t z[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int k = p.whole * kW4Block + i * (kW4Block / PARTS), gi = (k < p.K ? k : p.K - 1) / p.G;
            s[i] = p.scales[gi];
            z[i] = ZEROS ? p.zeros[gi] : 0;
        }
        multiply(w, x, s, z);
    }
    return total;
}

// Up to 16 rows by n_parts column tiles of 16, each by k_parts wavefronts (two to eight in all) that take consecutive steps,
// a slice each.
template <StepScales SCALES, bool ZEROS, typename OutT>
__global__ __launch_bounds__(kW4Waves * kWave) void gemv_w4_kernel(W4Problem p) {
    __shared__ f32x4 parts[kW4Waves * kWave];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane % 16, lq = lane / 16;
    const int k_part = wave % p.k_parts, n_part = wave / p.k_parts;
    // Workgroups 8 apart run on one XCD: the row tiles of a column tile follow each other there, so that its L2 has the
    // weights when the second one asks for them.
    const int xcd = blockIdx.x % kXcds, local = blockIdx.x / kXcds;
    const int tile = local % p.row_tiles, column = (local / p.row_tiles) * kXcds + xcd;
    if (column >= p.tiles_n) return;
    const int n0 = (column * p.n_parts + n_part) * 16;
    int row0, row_end, group = 0;
    if (p.offsets != nullptr) {
        const GroupTile t = find_group_tile(p.offsets, p.groups, p.rows, tile, 16);
        if (t.group < 0) return;
        row0 = t.row0;
        row_end = t.row_end;
        group = t.group;
    } else {
        row0 = tile * 16;
        row_end = p.rows;
    }
    const int n = n0 + l16 < p.N ? n0 + l16 : p.N - 1;  // columns beyond the last repeat it and are not written
    const long long scale_row = group * p.s_stride + static_cast<long long>(n) * p.n_groups;
    W4Slice s;
    s.q = p.q + group * p.q_stride + n * p.ldq + lq * 16;
    s.scales = p.scales + scale_row;
    s.zeros = ZEROS ? p.zeros + scale_row : nullptr;
    s.x = p.x + row0 * p.ldx;
    s.ldx = p.ldx;
    s.rows = row_end - row0 < 16 ? row_end - row0 : 16;
    s.whole = p.K / kW4Block;
    s.steps = (p.K + kW4Block - 1) / kW4Block;
    s.slice = p.slice;
    s.first = k_part * s.slice;
    s.K = p.K;
    s.G = p.G;
    f32x4 total;
    if (s.rows == 1) total = multiply_slice<SCALES, ZEROS, 1>(s);
    else if (s.rows <= 4) total = multiply_slice<SCALES, ZEROS, 4>(s);
    else total = multiply_slice<SCALES, ZEROS, 16>(s);
    // The parts of a column tile, added in their order.
    if (p.k_parts > 1) {
        parts[wave * kWave + lane] = total;
        __syncthreads();
        if (k_part != 0) return;
        for (int o = 1; o < p.k_parts; ++o) total += parts[(wave + o) * kWave + lane];
    }
    if (n0 + l16 >= p.N) return;
    OutT* y = static_cast<OutT*>(p.y);
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (4 * lq + v < s.rows) store_y(y + (row0 + 4 * lq + v) * p.ldy + n0 + l16, kUnit * total[v]);
}

template <StepScales SCALES>
int go(const W4Problem& p, int out_type, dim3 grid, hipStream_t s) {
    const dim3 block(static_cast<unsigned>(p.k_parts * p.n_parts * kWave));
    if (p.zeros != nullptr) {
        if (out_type == kTypeF32) gemv_w4_kernel<SCALES, true, float><<<grid, block, 0, s>>>(p);
        else gemv_w4_kernel<SCALES, true, uint16_t><<<grid, block, 0, s>>>(p);
    } else {
        if (out_type == kTypeF32) gemv_w4_kernel<SCALES, false, float><<<grid, block, 0, s>>>(p);
        else gemv_w4_kernel<SCALES, false, uint16_t><<<grid, block, 0, s>>>(p);
    }
    return check_launch("gemv_w4_kernel");
}

}  // namespace

int launch_gemv_w4(int groups, long long rows, int N, int K, const uint16_t* x, long long ldx, const uint8_t* q, long long ldq, long long q_stride,
                   const uint16_t* scales, const uint8_t* zeros, int group_size, const int32_t* offsets, void* y, long long ldy, int out_type, hipStream_t s) {
    const char* who = "prism_gemv_w4";
    if (groups < 0 || rows < 0 || N < 0 || K < 0) return fail(1, "%s: negative dimension (%d groups, %lld rows, N=%d, K=%d)", who, groups, rows, N, K);
    if (out_type != kTypeF32 && out_type != kTypeBf16) return fail(1, "%s: unknown output type %d", who, out_type);
    if (group_size < 32 || group_size % 32 != 0) return fail(1, "%s: group size %d, multiples of 32 are supported", who, group_size);
    if (rows > 0x7fffffffll - 256) return fail(1, "%s: %lld rows, at most 2^31 - 257 are supported", who, rows);
    if (groups > 0x7fffffff - 4096 || N > 0x7fffffff - 4096 || K > 0x7fffffff - 4096)
        return fail(1, "%s: %d groups, N=%d, K=%d: at most 2^31 - 4097 are supported", who, groups, N, K);
    if (offsets == nullptr && groups > 1) return fail(1, "%s: %d weight matrices need offsets", who, groups);
    if (groups == 0 || rows == 0 || N == 0) return 0;
    if (ldx < K || ldy < N || ldq < (static_cast<long long>(K) + 1) / 2) return fail(1, "%s: a row stride is shorter than its row", who);
    if (groups > 1 && q_stride < static_cast<long long>(N - 1) * ldq + (static_cast<long long>(K) + 1) / 2)
        return fail(1, "%s: the stride between weight matrices is shorter than a matrix", who);
    if (y == nullptr || (K > 0 && (x == nullptr || q == nullptr || scales == nullptr))) return fail(1, "%s: null pointer", who);
    const int size = out_type == kTypeF32 ? 4 : 2;
    if (!aligned2(x) || !aligned2(scales) || !aligned4(offsets) || !(size == 4 ? aligned4(y) : aligned2(y))) return fail(1, "%s: misaligned pointer", who);
    W4Problem p{};
    p.x = x; p.q = q; p.scales = scales; p.zeros = zeros; p.offsets = offsets; p.y = y;
    p.ldx = ldx; p.ldq = ldq; p.ldy = ldy; p.q_stride = q_stride;
    p.groups = groups; p.rows = static_cast<int>(rows); p.N = N; p.K = K; p.G = group_size;
    p.n_groups = ceil_div(K, group_size);
    p.s_stride = static_cast<long long>(N) * p.n_groups;
    Span matrices = matrix_span(q, N, (K + 1) / 2, ldq, 1);
    if (matrices.bytes != 0) matrices.bytes += static_cast<uintptr_t>(groups - 1) * q_stride;
    const uintptr_t scale_count = static_cast<uintptr_t>(groups) * p.s_stride;
    if (outputs_overlap({matrix_span(y, rows, N, ldy, size)}, {matrix_span(x, rows, K, ldx, 2), matrices, Span{scales, scale_count * 2}, Span{zeros, scale_count},
                                                               entries_span(offsets, groups + 1ll)}))
        return fail(1, "%s: the output overlaps an input", who);
    const long long row_tiles = offsets != nullptr ? most_row_tiles(rows, groups, 16) : ceil_div(rows, 16ll);
    const long long busy = offsets != nullptr ? busy_row_tiles(rows, groups, row_tiles) : row_tiles;
    // Twelve wavefronts a CU, none with less than a round of few rows (512 k: shorter slices only have the loop's last,
    // unpipelined part). Kernels by themselves with the same weights every time, against eight and single steps: 16384 x 16384 by 1 row 35.6 -> 30.2 us, 8192 x 1024 by 16 rows 7.1 -> 5.3,
    // 2048 x 1024 by 4 rows 5.0 -> 3.7, none of sixteen sizes slower by 1 %; sixteen wavefronts lose 40 % on
    // 14336 x 4096 by 1 row (9.1 -> 13.0 us) and 19 % on 8 matrices of 2048 x 2048 by 64 rows.
    p.k_parts = few_rows_k_parts(busy, N, K, 4 * kW4Block, kW4Waves, 12);
    // Whole rounds: only the last slice has steps outside the pipeline (5120 x 5120 by 4 rows, groups of 128: 13.3 -> 8.4 us).
    p.slice = ceil_div(ceil_div(ceil_div(K, kW4Block), p.k_parts), 4) * 4;
    p.n_parts = p.k_parts < kW4Few ? kW4Few / p.k_parts : 1;
    p.tiles_n = ceil_div(N, 16 * p.n_parts);
    const long long blocks = row_tiles * ceil_div(p.tiles_n, kXcds) * kXcds;
    if (!launchable(blocks, kW4Waves * kWave)) return fail(1, "%s: too many tiles", who);
    p.row_tiles = static_cast<int>(row_tiles);
    const dim3 grid(static_cast<unsigned>(blocks));
    if (group_size == 128) return go<StepScales::kOne>(p, out_type, grid, s);
    if (group_size == 64) return go<StepScales::kTwo>(p, out_type, grid, s);
    if (group_size == 32) return go<StepScales::kFour>(p, out_type, grid, s);
    return go<StepScales::kAny>(p, out_type, grid, s);
}

}  // namespace prism
