// Few rows times weights held in 4 bits: y[r][n] = sum_k x[r][k] s[n][k / G] (q[n][k] - z[n][k / G]), one weight
// matrix, or one per group of rows (expert_groups.h). q: two weights to a byte, the even k in the low nibble; s: bf16;
// z: uint8, 8 where absent; x: bf16; sums in fp32.
//
// Reading q bounds it: N K / 2 bytes for 2 r N K flop. The weights go from memory straight into registers, become bf16
// there and are multiplied on the matrix cores (v_mfma_f32_16x16x32_bf16: 16 rows of x, padded with zeros, by 16
// columns n, 32 k at a time), so that up to 16 rows cost what one costs. Three things keep the vector ALU out of the
// way:
//   * the order of k inside an instruction is free as long as both operands have the same: a lane takes consecutive
//     weights of its row (16, 8 or 4 bytes, so that the four lanes of a row stay inside one group of G), and the values
//     of a dword in the order 0 4 1 5 2 6 3 7, in which `(w >> c) & 0x00780078 | 0x41804180` yields two of them;
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

constexpr int kW4Waves = 8, kW4Block = 128;  // wavefronts of a workgroup (they split K); k per step

struct W4Problem {
    const uint16_t* x;
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;
    const int32_t* offsets;  // null: one group of all rows
    void* y;
    long long ldx, ldq, ldy, q_stride, s_stride;  // q_stride, s_stride: between the groups' matrices
    int groups, rows, N, K, G, n_groups;          // n_groups: scales per row
    int tiles_n;
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

// RUN: consecutive weights of a lane (32, 16 or 8), G a multiple of 4 RUN. MT: tiles of 16 rows.
template <int RUN, int MT, bool ZEROS, typename OutT>
__global__ __launch_bounds__(kW4Waves * kWave) void gemv_w4_kernel(W4Problem p) {
    constexpr int LOADS = 32 / RUN;       // of RUN / 2 bytes a step
    constexpr int PER = 4 / LOADS;        // instructions a load feeds
    constexpr int U = MT == 1 ? 4 : (MT == 2 ? 2 : 1);  // steps in flight
    __shared__ f32x4 part[kW4Waves][MT][kWave];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane % 16, lq = lane / 16;
    const int tile = blockIdx.x / p.tiles_n, n0 = (blockIdx.x % p.tiles_n) * 16;
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
    const int n = n0 + l16 < p.N ? n0 + l16 : p.N - 1;
    const uint8_t* q = p.q + group * p.q_stride + n * p.ldq;
    const uint16_t* scales = p.scales + group * p.s_stride + static_cast<long long>(n) * p.n_groups;
    const uint8_t* zeros = ZEROS ? p.zeros + group * p.s_stride + static_cast<long long>(n) * p.n_groups : nullptr;

    f32x4 total[MT] = {};
    // k of instruction i of the step at kb, this lane's eight.
    auto k_of = [&](int kb, int i) { return kb + (i / PER) * (4 * RUN) + lq * RUN + (i % PER) * 8; };
    auto step = [&](auto guarded, auto count, const int (&kbs)[U]) {
        constexpr bool EDGE = decltype(guarded)::value;
        constexpr int C = decltype(count)::value;
        uint32_t w[C][4];
        u32x4 xv[C][MT][4];
        float s[C][LOADS], z[C][LOADS];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int kb = kbs[c];
            if constexpr (!EDGE) {
#pragma unroll
                for (int h = 0; h < LOADS; ++h) __builtin_memcpy(&w[c][h * PER], q + k_of(kb, h * PER) / 2, RUN / 2);
            } else {
                const int bytes = (p.K + 1) / 2;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = k_of(kb, i) / 2;
                    w[c][i] = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (at + b < bytes) w[c][i] |= static_cast<uint32_t>(q[at + b]) << (8 * b);
                }
            }
#pragma unroll
            for (int h = 0; h < LOADS; ++h) {
                const int at = kb + h * 4 * RUN, gi = (EDGE && at >= p.K ? p.K - 1 : at) / p.G;
                s[c][h] = __builtin_bit_cast(float, static_cast<uint32_t>(scales[gi]) << 16);
                z[c][h] = ZEROS ? 16.0f + zeros[gi] : 24.0f;
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int row = row0 + m * 16 + l16;
                const uint16_t* x = p.x + row * p.ldx;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = k_of(kb, i);
                    u32x4 v = {0u, 0u, 0u, 0u};
                    if (row < row_end) {
                        if (!EDGE || k + 8 <= p.K) {
                            __builtin_memcpy(&v, x + k, 16);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (k + e < p.K) v[e / 2] |= static_cast<uint32_t>(x[k + e]) << (16 * (e % 2));
                        }
                    }
                    xv[c][m][i] = v;
                }
            }
        }
        const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int h = 0; h < LOADS; ++h) {
                f32x4 dot[MT] = {}, sum[MT] = {};
#pragma unroll
                for (int i = h * PER; i < (h + 1) * PER; ++i) {
                    const bf16x8 wv = weights_of(w[c][i]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const bf16x8 a = ordered(xv[c][m][i]);
                        dot[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, wv, dot[m], 0, 0, 0);
                        sum[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ones, sum[m], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int v = 0; v < 4; ++v) total[m][v] = __builtin_fmaf(s[c][h], __builtin_fmaf(-z[c][h], sum[m][v], dot[m][v]), total[m][v]);
            }
    };
    const int whole = p.K / kW4Block, steps = (p.K + kW4Block - 1) / kW4Block;
    int b = wave;
    int kbs[U];
    for (; b + (U - 1) * kW4Waves < whole; b += U * kW4Waves) {
#pragma unroll
        for (int c = 0; c < U; ++c) kbs[c] = (b + c * kW4Waves) * kW4Block;
        step(std::false_type{}, std::integral_constant<int, U>{}, kbs);
    }
    for (; b < whole; b += kW4Waves) {
        kbs[0] = b * kW4Block;
        step(std::false_type{}, std::integral_constant<int, 1>{}, kbs);
    }
    if (b < steps) {  // the partial last step
        kbs[0] = b * kW4Block;
        step(std::true_type{}, std::integral_constant<int, 1>{}, kbs);
    }
    // The wavefronts' parts, added in their order.
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][m][lane] = total[m];
    __syncthreads();
    if (wave >= MT) return;
    f32x4 r = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kW4Waves; ++w) r += part[w][wave][lane];
    OutT* y = static_cast<OutT*>(p.y);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int row = row0 + wave * 16 + 4 * lq + v;
        if (row < row_end && n0 + l16 < p.N) store_y(y + row * p.ldy + n0 + l16, r[v]);
    }
}

template <int RUN, int MT>
void go(const W4Problem& p, int out_type, dim3 grid, hipStream_t s) {
    const dim3 block(kW4Waves * kWave);
    if (p.zeros != nullptr) {
        if (out_type == kTypeF32) gemv_w4_kernel<RUN, MT, true, float><<<grid, block, 0, s>>>(p);
        else gemv_w4_kernel<RUN, MT, true, uint16_t><<<grid, block, 0, s>>>(p);
    } else {
        if (out_type == kTypeF32) gemv_w4_kernel<RUN, MT, false, float><<<grid, block, 0, s>>>(p);
        else gemv_w4_kernel<RUN, MT, false, uint16_t><<<grid, block, 0, s>>>(p);
    }
}

template <int RUN>
void go_tiles(const W4Problem& p, int mt, int out_type, dim3 grid, hipStream_t s) {
    if (mt == 1) go<RUN, 1>(p, out_type, grid, s);
    else if (mt == 2) go<RUN, 2>(p, out_type, grid, s);
    else go<RUN, 4>(p, out_type, grid, s);
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
    p.tiles_n = ceil_div(N, 16);
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
    if (tiles * p.tiles_n > 0x7fffffffll) return fail(1, "%s: too many tiles", who);
    const dim3 grid(static_cast<unsigned>(tiles * p.tiles_n));
    if (group_size % 128 == 0) go_tiles<32>(p, mt, out_type, grid, s);
    else if (group_size % 64 == 0) go_tiles<16>(p, mt, out_type, grid, s);
    else go_tiles<8>(p, mt, out_type, grid, s);
    return check_launch("gemv_w4_kernel");
}

}  // namespace prism
