// Few rows times weights held in 4 bits: y[r][n] = sum_k x[r][k] s[n][k / G] (q[n][k] - z[n][k / G]), one weight
// matrix, or one per group of rows (expert_groups.h). q: two weights to a byte, the even k in the low nibble; s: bf16;
// z: uint8, 8 where absent; x: bf16; sums in fp32.
//
// Reading q bounds it: N K / 2 bytes for 2 r N K flop. The weights go from memory straight into registers, become bf16
// there and are multiplied on the matrix cores (v_mfma_f32_16x16x32_bf16: 16 rows of x, padded with zeros, by 16
// columns n, 32 k at a time), so that up to 16 rows cost what one costs. Three things keep the vector ALU out of the
// way:
//   * the order of k inside an instruction is free as long as both operands have the same: a lane takes 16 consecutive
//     bytes of its row (32 weights; where groups are shorter than the 128 of a row's four lanes, the lanes exchange dwords
//     so that an instruction stays inside a group), and the values of a dword in the order 0 4 1 5 2 6 3 7, in which
//     `(w >> c) & 0x00780078 | 0x41804180` yields two of them;
//   * that pattern is the bf16 number 16 + q, exactly: what it adds is taken off per group of G, as
//     (16 + z) * (sum of x over the group), whose sums come from the same instruction on a matrix of ones;
//   * the scale is applied to a group's fp32 sum, not to the weights. Nothing is rounded below 32 bits but the result.
#include <type_traits>

#include "common.h"
#include "expert_groups.h"

namespace prism {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Waves = 8, kW4Block = 128;  // wavefronts of a workgroup; k per step: 16 B of weights a lane
constexpr int round_steps(int mt) { return mt == 4 ? 2 : 4; }  // steps fetched together, a round ahead of their use
constexpr int kW4Lds = 60 * 1024;            // for the rows of x: two workgroups to a CU

struct W4Problem {
    const uint16_t* x;
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;
    const int32_t* offsets;  // null: one group of all rows
    void* y;
    long long ldx, ldq, ldy, q_stride, s_stride;  // q_stride, s_stride: between the groups' matrices
    int groups, rows, N, K, G, n_groups;          // n_groups: scales per row
    int tiles_n;          // workgroups along N
    int k_parts, chunk_k; // wavefronts that share a column tile's K; k of x in LDS at a time
};

__device__ __forceinline__ void store_y(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_y(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }

// Eight weights of a dword as bf16 16 + q, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ bf16x8 weights_of(uint32_t w) {
    constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u;
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

// MT: tiles of 16 rows. Eight wavefronts: 8 / k_parts column tiles of 16, each by k_parts wavefronts that take every
// k_parts-th step. The rows of x pass through LDS in chunks of chunk_k, in the order of `ordered`.
template <StepScales SCALES, int MT, bool ZEROS, typename OutT>
__global__ __launch_bounds__(kW4Waves * kWave) void gemv_w4_kernel(W4Problem p) {
    constexpr bool TURN = SCALES != StepScales::kOne;  // G below 128: an instruction's 32 k are consecutive
    constexpr int U = round_steps(MT);
    extern __shared__ __attribute__((aligned(16))) uint16_t xs[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane % 16, lq = lane / 16;
    const int k_part = wave % p.k_parts, n_part = wave / p.k_parts;
    const int tile = blockIdx.x / p.tiles_n, n0 = ((blockIdx.x % p.tiles_n) * (kW4Waves / p.k_parts) + n_part) * 16;
    int row0, row_end, group = 0;
    if (p.offsets != nullptr) {
        const GroupTile t = find_group_tile(p.offsets, p.groups, p.rows, tile, 16 * MT);
        if (t.group < 0) return;
        row0 = t.row0;
        row_end = t.row_end;
        group = t.group;
    } else {
        row0 = tile * 16 * MT;
        row_end = p.rows;
    }
    const int rows = row_end - row0 < 16 * MT ? row_end - row0 : 16 * MT;
    const int n = n0 + l16 < p.N ? n0 + l16 : p.N - 1;  // columns beyond the last repeat it and are not written
    const uint8_t* q = p.q + group * p.q_stride + n * p.ldq;
    const uint16_t* scales = p.scales + group * p.s_stride + static_cast<long long>(n) * p.n_groups;
    const uint8_t* zeros = ZEROS ? p.zeros + group * p.s_stride + static_cast<long long>(n) * p.n_groups : nullptr;

    // A round: the weights, scales and zero points of U steps, fetched a round ahead.
    constexpr int PARTS = SCALES == StepScales::kOne ? 1 : (SCALES == StepScales::kTwo ? 2 : 4);
    struct Round {
        u32x4 w[U];
        uint16_t s[U][PARTS];
        uint8_t z[U][PARTS];
    };
    const int whole = p.K / kW4Block, steps = (p.K + kW4Block - 1) / kW4Block;
    auto fetch = [&](Round& r, int round) {
        if (whole == 0) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = k_part + (round * U + u) * p.k_parts, step = at < whole ? at : whole - 1;
            __builtin_memcpy(&r.w[u], q + static_cast<long long>(step) * (kW4Block / 2) + lq * 16, 16);
            if constexpr (SCALES != StepScales::kAny) {
                __builtin_memcpy(r.s[u], scales + step * PARTS, PARTS * 2);
                if constexpr (ZEROS) __builtin_memcpy(r.z[u], zeros + step * PARTS, PARTS);
            } else {
#pragma unroll
                for (int i = 0; i < PARTS; ++i) {
                    const int gi = (step * kW4Block + i * 32) / p.G;
                    r.s[u][i] = scales[gi];
                    if constexpr (ZEROS) r.z[u][i] = zeros[gi];
                }
            }
        }
    };
    f32x4 total[MT] = {};
    const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
    const int stride = p.chunk_k + 8;  // of a row in LDS: padded by one packet
    const uint16_t* x_lane[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x_lane[m] = xs + (m * 16 + l16 < rows ? m * 16 + l16 : rows - 1) * stride + (TURN ? 8 : 32) * lq;
    // The instructions of one step, whose first k is at element `at` of the chunk.
    auto step = [&](u32x4 w, const uint16_t (&s)[PARTS], const uint8_t (&z)[PARTS], int at) {
        if constexpr (TURN) w = turned(w);
        f32x4 dot[MT], sum[MT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            constexpr int PER = 4 / PARTS;
            const bf16x8 wv = weights_of(w[i]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (i % PER == 0) dot[m] = sum[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const bf16x8 a = *reinterpret_cast<const bf16x8*>(x_lane[m] + at + (TURN ? 32 : 8) * i);
                dot[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, wv, dot[m], 0, 0, 0);
                sum[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ones, sum[m], 0, 0, 0);
            }
            if (i % PER == PER - 1) {
                const float scale = __builtin_bit_cast(float, static_cast<uint32_t>(s[i / PER]) << 16), zero = ZEROS ? 16.0f + z[i / PER] : 24.0f;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int v = 0; v < 4; ++v) total[m][v] = __builtin_fmaf(scale, __builtin_fmaf(-zero, sum[m][v], dot[m][v]), total[m][v]);
            }
        }
    };
    // Chunk of x from k = first on, zeros beyond K.
    auto stage = [&](int first) {
        const int left = (steps * kW4Block - first) / 8, packets = left < p.chunk_k / 8 ? left : p.chunk_k / 8;
        for (int i = threadIdx.x; i < rows * packets; i += kW4Waves * kWave) {
            const int row = i / packets, c = (i - row * packets) * 8, k = first + c;
            const uint16_t* x = p.x + (row0 + row) * p.ldx + k;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (k + 8 <= p.K) {
                __builtin_memcpy(&v, x, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + e < p.K) v[e / 2] |= static_cast<uint32_t>(x[e]) << (16 * (e % 2));
            }
            *reinterpret_cast<bf16x8*>(xs + row * stride + c) = ordered(v);
        }
    };
    const int per_round = p.k_parts * U, rounds = (steps + per_round - 1) / per_round, per_chunk = p.chunk_k / (per_round * kW4Block);
    Round now, ahead;
    fetch(now, 0);
    for (int r = 0; r < rounds; ++r) {
        const int chunk0 = r / per_chunk * per_chunk * per_round;  // the chunk's first step
        if (r % per_chunk == 0) {
            if (r > 0) __syncthreads();
            stage(chunk0 * kW4Block);
            __syncthreads();
        }
        if (r + 1 < rounds) fetch(ahead, r + 1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = k_part + (r * U + u) * p.k_parts;
            if (at < whole) step(now.w[u], now.s[u], now.z[u], (at - chunk0) * kW4Block);
        }
        now = ahead;
    }
    if (whole < steps && whole % p.k_parts == k_part) {  // the partial last step: nothing is read beyond the row
        const int chunk0 = (rounds - 1) / per_chunk * per_chunk * per_round, bytes = (p.K + 1) / 2;
        u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const int at = whole * (kW4Block / 2) + lq * 16 + b;
            if (at < bytes) w[b / 4] |= static_cast<uint32_t>(q[at]) << (8 * (b % 4));
        }
        uint16_t s[PARTS];
        uint8_t z[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int k = whole * kW4Block + i * (kW4Block / PARTS), gi = (k < p.K ? k : p.K - 1) / p.G;
            s[i] = scales[gi];
            z[i] = ZEROS ? zeros[gi] : 0;
        }
        step(w, s, z, (whole - chunk0) * kW4Block);
    }
    // The parts of a column tile, added in their order.
    f32x4* part = reinterpret_cast<f32x4*>(xs);  // [wave][MT][64]
    if (p.k_parts > 1) {
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; ++m) part[(wave * MT + m) * kWave + lane] = total[m];
        __syncthreads();
        if (k_part != 0) return;
        for (int o = 1; o < p.k_parts; ++o)
#pragma unroll
            for (int m = 0; m < MT; ++m) total[m] += part[((wave + o) * MT + m) * kWave + lane];
    }
    if (n0 + l16 >= p.N) return;
    OutT* y = static_cast<OutT*>(p.y);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = m * 16 + 4 * lq + v;
            if (row < rows) store_y(y + (row0 + row) * p.ldy + n0 + l16, total[m][v]);
        }
}

template <StepScales SCALES, int MT>
int go(const W4Problem& p, int out_type, dim3 grid, size_t lds, hipStream_t s) {
    const dim3 block(kW4Waves * kWave);
    if (p.zeros != nullptr) {
        if (out_type == kTypeF32) gemv_w4_kernel<SCALES, MT, true, float><<<grid, block, lds, s>>>(p);
        else gemv_w4_kernel<SCALES, MT, true, uint16_t><<<grid, block, lds, s>>>(p);
    } else {
        if (out_type == kTypeF32) gemv_w4_kernel<SCALES, MT, false, float><<<grid, block, lds, s>>>(p);
        else gemv_w4_kernel<SCALES, MT, false, uint16_t><<<grid, block, lds, s>>>(p);
    }
    return check_launch("gemv_w4_kernel");
}

template <StepScales SCALES>
int go_tiles(const W4Problem& p, int mt, int out_type, dim3 grid, size_t lds, hipStream_t s) {
    if (mt == 1) return go<SCALES, 1>(p, out_type, grid, lds, s);
    if (mt == 2) return go<SCALES, 2>(p, out_type, grid, lds, s);
    return go<SCALES, 4>(p, out_type, grid, lds, s);
}

}  // namespace

int launch_gemv_w4(int groups, long long rows, int N, int K, const uint16_t* x, long long ldx, const uint8_t* q, long long ldq, long long q_stride,
                   const uint16_t* scales, const uint8_t* zeros, int group_size, const int32_t* offsets, void* y, long long ldy, int out_type, hipStream_t s) {
    const char* who = "prism_gemv_w4";
    if (groups < 0 || rows < 0 || N < 0 || K < 0) return fail(1, "%s: negative dimension (%d groups, %lld rows, N=%d, K=%d)", who, groups, rows, N, K);
    if (out_type != kTypeF32 && out_type != kTypeBf16) return fail(1, "%s: unknown output type %d", who, out_type);
    if (group_size < 32 || group_size % 32 != 0) return fail(1, "%s: group size %d, multiples of 32 are supported", who, group_size);
    if (rows > 0x7fffffffll - 256) return fail(1, "%s: %lld rows, at most 2^31 - 257 are supported", who, rows);
    if (K > 0x7fffffff - 4096) return fail(1, "%s: K=%d is too large", who, K);
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
    const uintptr_t yb = reinterpret_cast<uintptr_t>(y), ye = yb + static_cast<uintptr_t>((rows - 1) * ldy + N) * size;
    auto meets = [&](const void* a, uintptr_t bytes) { const uintptr_t b = reinterpret_cast<uintptr_t>(a); return a != nullptr && b < ye && yb < b + bytes; };
    if (meets(x, static_cast<uintptr_t>((rows - 1) * ldx + K) * 2) ||
        meets(q, static_cast<uintptr_t>(groups - 1) * q_stride + static_cast<uintptr_t>(N - 1) * ldq + (K + 1) / 2) ||
        meets(scales, static_cast<uintptr_t>(groups) * p.s_stride * 2) || meets(zeros, static_cast<uintptr_t>(groups) * p.s_stride) ||
        meets(offsets, (static_cast<uintptr_t>(groups) + 1) * 4))
        return fail(1, "%s: the output overlaps an input", who);
    // Rows a tile: 16 cost what one costs; more are worth it when a group fills them, since every tile reads the group's
    // weights again.
    const long long per_group = ceil_div(rows, static_cast<long long>(groups));
    const int mt = per_group <= 16 ? 1 : (per_group <= 32 ? 2 : 4);
    const long long tiles = offsets != nullptr ? most_row_tiles(rows, groups, 16 * mt) : ceil_div(rows, static_cast<long long>(16 * mt));
    // Rows of x in LDS at a time: a chunk is a whole number of rounds, so many wavefronts to a column tile need few rows.
    const int most_rows = offsets == nullptr && rows < 16 * mt ? static_cast<int>(rows) : (rows < 16 * mt ? static_cast<int>(rows) : 16 * mt);
    const int fits = kW4Lds / (2 * most_rows) - 8;
    p.k_parts = kW4Waves;
    const int part_k = round_steps(mt) * kW4Block;  // of a wavefront's round
    while (p.k_parts > 1 && (p.k_parts * part_k > fits || p.k_parts * part_k / 2 >= K)) p.k_parts /= 2;
    const int round_k = p.k_parts * part_k;
    const int wanted = ceil_div(K > 0 ? K : 1, round_k);
    p.chunk_k = round_k * (fits / round_k < wanted ? fits / round_k : wanted);
    const size_t x_bytes = static_cast<size_t>(most_rows) * (p.chunk_k + 8) * 2, part_bytes = static_cast<size_t>(kW4Waves) * mt * kWave * 16;
    const size_t lds = x_bytes > part_bytes ? x_bytes : part_bytes;
    p.tiles_n = ceil_div(N, 16 * (kW4Waves / p.k_parts));
    if (tiles * p.tiles_n > 0x7fffffffll) return fail(1, "%s: too many tiles", who);
    const dim3 grid(static_cast<unsigned>(tiles * p.tiles_n));
    if (group_size == 128) return go_tiles<StepScales::kOne>(p, mt, out_type, grid, lds, s);
    if (group_size == 64) return go_tiles<StepScales::kTwo>(p, mt, out_type, grid, lds, s);
    if (group_size == 32) return go_tiles<StepScales::kFour>(p, mt, out_type, grid, lds, s);
    return go_tiles<StepScales::kAny>(p, mt, out_type, grid, lds, s);
}

}  // namespace prism
