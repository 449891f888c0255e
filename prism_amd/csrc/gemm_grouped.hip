// Products grouped by expert, bf16 in and fp32 accumulation on MFMA, and their gradients:
//   forward   D[r][n]    = sum_k A[r][k]  B[g(r)][n][k]          (A: rows x K, B: groups x N x K, D: rows x N)
//   grad_a    dA[r][k]   = sum_n dD[r][n] B[g(r)][n][k]
//   grad_b    dB[g][n][k] = sum over the rows r of group g of dD[r][n] A[r][k]   (an empty group: zeros)
// g(r) is the group with offsets[g] <= r < offsets[g + 1] (expert_groups.h). All three are
//   OUT[i][j] = sum_c P[i][c] Q[j][c]
// with operands that lie in memory with c running along the rows ("straight": A and B in the forward product, dD in
// grad_a) or down the columns ("turned": B in grad_a, both in grad_b). A straight operand's tile lies in LDS as rows of
// 64 c, and a matrix fragment (8 consecutive c of one row) is one 16 B read. A turned operand's tile lies in LDS as 64
// rows of c, as in memory, and is turned by the transposing LDS read (ds_read_b64_tr_b16: the 16 lanes of a quarter
// wave read a 4 x 16 block of 16-bit values and each receives one column of it), two reads to a fragment.
//
// What a tile reads beyond its rows, columns or c arrives as zero: rows of other groups never enter a sum, whatever
// they hold.
#include <type_traits>

#include "common.h"
#include "direct_load.h"
#include "expert_groups.h"

namespace prism {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// fp32 -> bf16, round to nearest even (v_cvt_pk_bf16_f32). The results' only rounding below 32 bits.
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(uint16_t* p, float v) { *p = to_bf16(v); }

// One problem, as OUT = P Q^T. Element strides; `groups` weight matrices (or, with RAGGED_C, results) `group_stride`
// elements apart.
struct GroupedProblem {
    const uint16_t *P, *Q;
    const int32_t* offsets;
    void* OUT;
    long long ldp, ldq, ldo, group_stride;
    int groups, rows;     // rows: of the row operand, all groups
    int cols;             // of OUT
    int depth;            // extent of c (forms with whole groups along c: unused)
    int out_rows;         // rows of one group's OUT (those forms only)
    int tiles_n;          // column tiles
};

constexpr int kBK = 64;

// The tile of one operand in LDS: `LINES` rows (or columns) of the product by 64 c.
//   straight: [LINES][64], 128 B a line; the 16 B chunk of c = 8 q .. 8 q + 7 of line r in slot q ^ ((r >> 1) & 7):
//             the sixteen lines a fragment read touches spread over all banks.
//   turned:   [64][LINES]; the 32 B block b (16 lines) of row c in slot b ^ f(c), f(c) = (c & 3) | (c & 8) >> 1: the
//             eight rows that half a wave reads at a time lie in eight different blocks.
// A wave-wide direct load fills 1 KiB of consecutive LDS, so the permutation is applied to the addresses it reads.
template <int LINES, bool TURNED, int WAVES>
struct OperandTile {
    static constexpr int ROW_ELEMS = TURNED ? LINES : kBK;            // elements of a row in LDS
    static constexpr int ROWS = TURNED ? kBK : LINES;
    static constexpr int CHUNKS = ROW_ELEMS / 8;
    static constexpr int ROWS_PER_LOAD = kWave / CHUNKS;
    static constexpr int ROWS_PER_PASS = ROWS_PER_LOAD * WAVES;
    static constexpr int PASSES = ROWS / ROWS_PER_PASS;
    static_assert(kWave % CHUNKS == 0 && ROWS % ROWS_PER_PASS == 0, "whole loads and passes");
    static constexpr int ELEMS = LINES * kBK;

    static __device__ __forceinline__ int slot_of(int row, int chunk) {
        if constexpr (TURNED) return chunk ^ (2 * ((row & 3) | ((row & 8) >> 1)));
        else return chunk ^ ((row >> 1) & 7);
    }
    // Row and chunk that lane `lane` of wave `wave` fetches in pass `pass` (it lands at LDS byte 16 lane of that load).
    static __device__ __forceinline__ int row_of(int pass, int wave, int lane) { return pass * ROWS_PER_PASS + wave * ROWS_PER_LOAD + lane / CHUNKS; }
    static __device__ __forceinline__ int chunk_of(int pass, int wave, int lane) { return slot_of(row_of(pass, wave, lane), lane % CHUNKS); }
    static __device__ __forceinline__ int lds_elem(int pass, int wave) { return (pass * ROWS_PER_PASS + wave * ROWS_PER_LOAD) * ROW_ELEMS; }

    // The fragment of 16 lines from `line0` (a multiple of 16) and 32 c from `c0`: lane l gets c0 + 8 (l / 16) .. + 7 of
    // line line0 + l % 16.
    static __device__ __forceinline__ bf16x8 fragment(const uint16_t* tile, int line0, int c0, int lane) {
        const int l16 = lane & 15, lq = lane >> 4;
        if constexpr (!TURNED) {
            const int row = line0 + l16;
            return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(&tile[row * kBK + slot_of(row, c0 / 8 + lq) * 8]));
        } else {
            const int row = c0 + 8 * lq + (l16 >> 2);
            const uint16_t* at = &tile[row * LINES + slot_of(row, (line0 + 4 * (l16 & 3)) / 8) * 8 + 4 * (l16 & 1)];
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * LINES));  // c + 4: the same slot
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            return __builtin_bit_cast(bf16x8, both);
        }
    }
};

// What one operand's tile covers in memory: `lines` lines from `base` on and c in [0, depth); everything else is zero.
struct OperandSource {
    const uint16_t* base;  // the tile's first line, c = 0
    long long ld;
    int lines;             // lines that exist from the tile's first on (may exceed the tile)
    int depth;
};

// A 16 B packet from memory by ordinary loads, for rows and bases of any alignment: whole packets in one access,
// packets that end outside element by element.
__device__ __forceinline__ u32x4 load_packet(const uint16_t* at, int there) {
    u32x4 r = {0u, 0u, 0u, 0u};
    if (there >= 8) {
        __builtin_memcpy(&r, at, 16);
    } else {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < there ? at[i] : uint16_t{0};
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = static_cast<uint32_t>(e[2 * i]) | (static_cast<uint32_t>(e[2 * i + 1]) << 16);
    }
    return r;
}

template <int LINES, bool TURNED, int WAVES, bool ALIGNED>
__device__ __forceinline__ void load_operand(uint16_t* tile, const OperandSource& src, int c0, int wave, int lane) {
    using T = OperandTile<LINES, TURNED, WAVES>;
    // Rows and row elements in memory that exist from the tile's corner on.
    const uint16_t* corner = src.base + (TURNED ? static_cast<long long>(c0) * src.ld : static_cast<long long>(c0));
    const int rows = TURNED ? src.depth - c0 : src.lines;
    const int elems = TURNED ? src.lines : src.depth - c0;
    if constexpr (ALIGNED) {
        // Lines, depth and rows are multiples of 8 elements along memory, so a chunk is whole or absent; rows beyond
        // the last are beyond the descriptor's extent (at most LINES or 64 rows of it: below 2 GiB by the launcher).
        const int in_tile = rows < T::ROWS ? (rows > 0 ? rows : 0) : T::ROWS;
        const i32x4 rsrc = buffer_descriptor(corner, static_cast<uint32_t>(in_tile * src.ld * 2));
#pragma unroll
        for (int p = 0; p < T::PASSES; ++p) {
            const int chunk = T::chunk_of(p, wave, lane);
            const uint32_t off = chunk * 8 < elems ? static_cast<uint32_t>((T::row_of(p, wave, lane) * src.ld + chunk * 8) * 2) : kBeyondExtent;
            direct_load16_buffer(rsrc, off, 0u, &tile[T::lds_elem(p, wave)]);
        }
    } else {
#pragma unroll
        for (int p = 0; p < T::PASSES; ++p) {
            const int row = T::row_of(p, wave, lane), chunk = T::chunk_of(p, wave, lane);
            const int there = row < rows ? elems - chunk * 8 : 0;
            const u32x4 v = load_packet(corner + (there > 0 ? row * src.ld + chunk * 8 : 0), there);
            *reinterpret_cast<u32x4*>(&tile[T::lds_elem(p, wave) + lane * 8]) = v;
        }
    }
}

// BM x BN tiles, four waves of BM/2 x BN/2, two LDS stages of 64 c. RAGGED_C: the groups lie along c (grad_b).
template <int BM, int BN, bool P_TURNED, bool Q_TURNED, bool RAGGED_C, bool ALIGNED, typename OutT>
__global__ __launch_bounds__(256) void gemm_grouped_kernel(GroupedProblem g) {
    constexpr int WAVES = 4, WM = BM / 2, WN = BN / 2, MI = WM / 16, NI = WN / 16;
    using PT = OperandTile<BM, P_TURNED, WAVES>;
    using QT = OperandTile<BN, Q_TURNED, WAVES>;
    __shared__ __attribute__((aligned(1024))) uint16_t Ps[2][PT::ELEMS];
    __shared__ __attribute__((aligned(1024))) uint16_t Qs[2][QT::ELEMS];

    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int tm = blockIdx.x / g.tiles_n, col0 = (blockIdx.x % g.tiles_n) * BN;
    OperandSource ps, qs;
    OutT* out;
    int rows_left;  // rows of OUT from the tile's first on
    if constexpr (RAGGED_C) {
        const int tiles_m = (g.out_rows + BM - 1) / BM;
        const int group = tm / tiles_m, row0 = (tm % tiles_m) * BM;
        const int lo = clamp_offset(g.offsets[group], g.rows), hi = clamp_offset(g.offsets[group + 1], g.rows);
        const int depth = hi > lo ? hi - lo : 0;
        ps = {g.P + lo * g.ldp + row0, g.ldp, g.out_rows - row0, depth};
        qs = {g.Q + lo * g.ldq + col0, g.ldq, g.cols - col0, depth};
        rows_left = g.out_rows - row0;
        out = static_cast<OutT*>(g.OUT) + group * g.group_stride + row0 * g.ldo + col0;
    } else {
        const GroupTile t = find_group_tile(g.offsets, g.groups, g.rows, tm, BM);
        if (t.group < 0) return;
        rows_left = t.row_end - t.row0;
        ps = {g.P + t.row0 * g.ldp, g.ldp, rows_left, g.depth};
        qs = {g.Q + t.group * g.group_stride + (Q_TURNED ? col0 : col0 * g.ldq), g.ldq, g.cols - col0, g.depth};
        out = static_cast<OutT*>(g.OUT) + t.row0 * g.ldo + col0;
    }
    const int wave_m = wave / 2, wave_n = wave % 2;
    f32x4 acc[MI][NI] = {};
    const int tiles = (ps.depth + kBK - 1) / kBK;
    auto load = [&](int t) {
        load_operand<BM, P_TURNED, WAVES, ALIGNED>(Ps[t & 1], ps, t * kBK, wave, lane);
        load_operand<BN, Q_TURNED, WAVES, ALIGNED>(Qs[t & 1], qs, t * kBK, wave, lane);
    };
    auto landed = [&] {
        asm volatile("" ::: "memory");  // the compiler knows neither the loads' writes to LDS nor what the barrier orders
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (tiles > 0) load(0);
    landed();
    for (int t = 0; t < tiles; ++t) {
        if (t + 1 < tiles) load(t + 1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fp[MI], fq[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) fp[i] = PT::fragment(Ps[t & 1], wave_m * WM + i * 16, kk * 32, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) fq[j] = QT::fragment(Qs[t & 1], wave_n * WN + j * 16, kk * 32, lane);
            // Q first: a lane then holds four consecutive columns of one row of OUT.
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fq[j], fp[i], acc[i][j], 0, 0, 0);
        }
        landed();
    }
    const int cols_left = g.cols - col0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = wave_m * WM + i * 16 + (lane & 15);
        if (row >= rows_left) continue;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int col = wave_n * WN + j * 16 + 4 * (lane >> 4);
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (col + v < cols_left) store_out(out + row * g.ldo + col + v, acc[i][j][v]);
        }
    }
}

template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C, typename OutT>
int run(GroupedProblem g, const char* who, hipStream_t s) {
    constexpr int BM = 128, BN = 128;
    g.tiles_n = ceil_div(g.cols, BN);
    const long long tiles_m = RAGGED_C ? static_cast<long long>(g.groups) * ceil_div(g.out_rows, BM) : most_row_tiles(g.rows, g.groups, BM);
    if (tiles_m == 0) return 0;
    if (tiles_m * g.tiles_n > 0x7fffffffll) return fail(1, "%s: too many tiles", who);
    const dim3 grid(static_cast<unsigned>(tiles_m * g.tiles_n));
    // Direct-to-LDS loads need 16 B chunks that are whole or absent (bases, strides and the extents along memory in
    // multiples of 8 elements) and 32-bit offsets inside a tile.
    const int p_along = P_TURNED ? g.out_rows : g.depth, q_along = Q_TURNED ? g.cols : g.depth;
    const bool aligned = aligned16(g.P) && aligned16(g.Q) && g.ldp % 8 == 0 && g.ldq % 8 == 0 && (RAGGED_C || g.group_stride % 8 == 0) &&
                         p_along % 8 == 0 && q_along % 8 == 0 && g.ldp < (1 << 21) && g.ldq < (1 << 21);
    if (aligned) gemm_grouped_kernel<BM, BN, P_TURNED, Q_TURNED, RAGGED_C, true, OutT><<<grid, dim3(256), 0, s>>>(g);
    else gemm_grouped_kernel<BM, BN, P_TURNED, Q_TURNED, RAGGED_C, false, OutT><<<grid, dim3(256), 0, s>>>(g);
    return check_launch("gemm_grouped_kernel");
}

// The bytes from p that a rows x cols matrix of row stride ld occupies.
uintptr_t span_bytes(long long rows, long long cols, long long ld, int size) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<uintptr_t>((rows - 1) * ld + cols) * size;
}
bool overlap(const void* a, uintptr_t a_bytes, const void* b, uintptr_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

}  // namespace

int launch_gemm_grouped(GroupedForm form, int groups, long long rows, int N, int K, const uint16_t* first, long long ld_first,
                        const uint16_t* second, long long ld_second, long long group_stride, const int32_t* offsets, void* out,
                        long long ld_out, int out_type, hipStream_t s) {
    const char* who = form == GroupedForm::kForward ? "prism_gemm_bf16_grouped"
                      : form == GroupedForm::kGradA ? "prism_gemm_bf16_grouped_grad_a" : "prism_gemm_bf16_grouped_grad_b";
    if (groups < 0 || rows < 0 || N < 0 || K < 0) return fail(1, "%s: negative dimension (%d groups, %lld rows, N=%d, K=%d)", who, groups, rows, N, K);
    if (rows > 0x7fffffffll - 256) return fail(1, "%s: %lld rows, at most 2^31 - 257 are supported", who, rows);
    if (out_type != kTypeF32 && out_type != kTypeBf16) return fail(1, "%s: unknown output type %d", who, out_type);
    const int size = out_type == kTypeF32 ? 4 : 2;
    const bool grad_b = form == GroupedForm::kGradB;
    // Row lengths of the operands, and the group matrices' shape (always N x K).
    const long long first_cols = form == GroupedForm::kForward ? K : N;
    const long long out_cols = form == GroupedForm::kForward ? N : K;
    const long long ld_group = grad_b ? ld_out : ld_second, ld_rows2 = grad_b ? ld_second : ld_out;
    if (groups == 0 || (grad_b ? N == 0 || K == 0 : rows == 0 || out_cols == 0)) return 0;
    if (ld_first < first_cols || ld_group < K || ld_rows2 < (grad_b ? K : out_cols))
        return fail(1, "%s: a row stride is shorter than its row", who);
    if (groups > 1 && group_stride < (N > 0 ? static_cast<long long>(N - 1) * ld_group + K : 0))
        return fail(1, "%s: the stride between group matrices is shorter than a matrix", who);
    const long long depth = form == GroupedForm::kForward ? K : (grad_b ? rows : N);
    if (offsets == nullptr || out == nullptr || (depth > 0 && (first == nullptr || second == nullptr))) return fail(1, "%s: null pointer", who);
    if (!aligned2(first) || !aligned2(second) || !aligned4(offsets) || !(size == 4 ? aligned4(out) : aligned2(out)))
        return fail(1, "%s: misaligned pointer", who);
    const uintptr_t group_bytes = (static_cast<uintptr_t>(groups - 1) * group_stride) * (grad_b ? size : 2) + span_bytes(N, K, ld_group, grad_b ? size : 2);
    const uintptr_t out_bytes = grad_b ? group_bytes : span_bytes(rows, out_cols, ld_out, size);
    if (overlap(out, out_bytes, first, span_bytes(rows, first_cols, ld_first, 2)) ||
        overlap(out, out_bytes, second, grad_b ? span_bytes(rows, K, ld_second, 2) : group_bytes) ||
        overlap(out, out_bytes, offsets, (static_cast<uintptr_t>(groups) + 1) * 4))
        return fail(1, "%s: the output overlaps an input", who);

    GroupedProblem g{};
    g.P = first; g.Q = second; g.offsets = offsets; g.OUT = out;
    g.ldp = ld_first; g.ldq = ld_second; g.ldo = ld_out; g.group_stride = group_stride;
    g.groups = groups; g.rows = static_cast<int>(rows); g.cols = static_cast<int>(out_cols);
    g.depth = grad_b ? 0 : static_cast<int>(depth); g.out_rows = N;
    auto with = [&](auto p_turned, auto q_turned, auto ragged) {
        constexpr bool PT = decltype(p_turned)::value, QT = decltype(q_turned)::value, RC = decltype(ragged)::value;
        return out_type == kTypeF32 ? run<PT, QT, RC, float>(g, who, s) : run<PT, QT, RC, uint16_t>(g, who, s);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (form == GroupedForm::kForward) return with(no{}, no{}, no{});
    if (form == GroupedForm::kGradA) return with(no{}, yes{}, no{});
    return with(yes{}, yes{}, yes{});
}

}  // namespace prism
