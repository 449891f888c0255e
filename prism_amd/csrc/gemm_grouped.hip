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
//
// 2 R N K flop. With many rows a group the matrix pipe bounds them, with few reading B (at 1.4 PFLOP/s and 6 TB/s both take as
// long at some 230 rows). Three kernels (choose_kernel): 16, 128 or 256 rows a tile. Calls among others, three sets of inputs in
// turn, from box to box, 2048 x 4096 matrices: forward 65536 rows of 64 groups 870 to 910 us (1.21 to 1.26 PFLOP/s; the dense
// product of this library reaches 1.5), grad_a 32768 rows of 32 groups 470 to 496 us (1.11 to 1.17), grad_b of the same 613 to
// 631 us (0.87 to 0.90, and 1.07 GB of fp32 results). 32 rows of 64 groups, 1536 x 2048, 160 MB of B: 30 to 36 us (4.5 to 5.3 TB/s).
#include <type_traits>

#include "common.h"
#include "direct_load.h"
#include "expert_groups.h"
#include "few_rows.h"
#include "tile_map.h"

namespace prism {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// fp32 -> bf16, round to nearest even (v_cvt_pk_bf16_f32). The results' only rounding below 32 bits.
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(uint16_t* p, float v) { *p = to_bf16(v); }

// v_mfma_f32_16x16x32_bf16 on an accumulator in place, from inline assembly: through the builtin the compiler moves
// accumulators between registers around the instruction (a hundred moves per 32 of them in the general kernel, spills in the
// big one). It then does not know the result's latency: an accumulator is read by nothing but the same instruction within 64
// clocks of its last one (grouped_settle), and a register that the vector ALU has just written is not an operand.
__device__ __forceinline__ void mfma_in_place(f32x4& c, bf16x8 a, bf16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void grouped_settle() { asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory"); }

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
    bool near;            // rows of a tile within 32-bit offsets of each other
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

// A stage of an operand by direct-to-LDS loads. Bases and rows may lie anywhere (16 B loads take 2-byte aligned addresses),
// but a chunk must be whole or absent, and the range check works on dwords: the depth is a multiple of 8 or the stage lies
// inside it, and (turned) the lines are a multiple of 8 or the stage is not the last. A stage beyond the depth: zeros.
template <int LINES, bool TURNED, int WAVES>
__device__ __forceinline__ void load_direct(uint16_t* tile, const OperandSource& src, int c0, int wave, int lane) {
    using T = OperandTile<LINES, TURNED, WAVES>;
    // Rows in memory that exist from the tile's corner on; those beyond the last are beyond the descriptor's extent (at most
    // LINES or 65 rows of it: below 2 GiB by the launcher). Beyond the lines of a row of a turned operand lies the next row's
    // head, which only enters lines that are not written; the extent ends with the lines of the stage's last row, or of the
    // row behind it where there is one.
    const uint16_t* corner = src.base + (TURNED ? static_cast<long long>(c0) * src.ld : static_cast<long long>(c0));
    const int c_left = src.depth - c0, lines = src.lines < LINES ? src.lines : LINES;
    const int elems = TURNED ? lines : c_left;
    const int rows = TURNED ? (c_left < kBK + 1 ? c_left : kBK + 1) : lines;
    uint32_t extent = TURNED ? static_cast<uint32_t>((rows - 1) * src.ld + lines) * 2u : static_cast<uint32_t>(rows * src.ld * 2);
    if (c_left <= 0) extent = 0;
    const i32x4 rsrc = buffer_descriptor(corner, extent);
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
        const int chunk = T::chunk_of(p, wave, lane);
        const uint32_t at = static_cast<uint32_t>((T::row_of(p, wave, lane) * src.ld + chunk * 8) * 2);
        direct_load16_buffer(rsrc, TURNED || chunk * 8 < elems ? at : kBeyondExtent, 0u, &tile[T::lds_elem(p, wave)]);
    }
}

// The same by ordinary loads, for any stage of any operand.
template <int LINES, bool TURNED, int WAVES>
__device__ __forceinline__ void load_packets(uint16_t* tile, const OperandSource& src, int c0, int wave, int lane) {
    using T = OperandTile<LINES, TURNED, WAVES>;
    const uint16_t* corner = src.base + (TURNED ? static_cast<long long>(c0) * src.ld : static_cast<long long>(c0));
    const int rows = TURNED ? src.depth - c0 : src.lines, elems = TURNED ? src.lines : src.depth - c0;
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
        const int row = T::row_of(p, wave, lane), chunk = T::chunk_of(p, wave, lane);
        const int there = row < rows ? elems - chunk * 8 : 0;
        const u32x4 v = load_packet(corner + (there > 0 ? row * src.ld + chunk * 8 : 0), there);
        *reinterpret_cast<u32x4*>(&tile[T::lds_elem(p, wave) + lane * 8]) = v;
    }
}

// ------------------------------------------------------------------------------------------- the general kernel --
// 128 x 128 tiles, four waves of 64 x 64, one tile a workgroup: operands of any alignment, and problems with too few big
// tiles for the chip. RAGGED_C: the groups lie along c (grad_b), whose rows one workgroup walks by itself: with few results that
// leaves compute units idle (16384 rows of 4 groups by 256 x 256: 16 workgroups, 48 us; 65 with a long group among them). Bound by
// the latency of its loads: a stage of two workgroups on a unit takes 1.1 us for 0.42 us of matrix instructions. 5003 rows of 24
// groups by 1000 x 1048, fp32 results: 30 us a call (0.35 PFLOP/s; matrix pipe 19 % busy, 143 MB read for 61 of operands).
// Direct-to-LDS loads into a ring of STAGES stages of 64 c. Four, three ahead, where there is a tile to a CU and nothing else
// hides the memory's latency (with two stages, one ahead, a stage took 0.65 us, memory latency, instead of 0.45); two where
// there are more tiles and two workgroups share a CU (choose_kernel). Not ALIGNED: the last stage, or every one of rows too
// far apart for 32-bit offsets, comes by ordinary loads.
template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C, bool ALIGNED, int STAGES, typename OutT>
__global__ __launch_bounds__(256) void gemm_grouped_kernel(GroupedProblem g) {
    constexpr int BM = 128, BN = 128, WAVES = 4, WM = BM / 2, WN = BN / 2, MI = WM / 16, NI = WN / 16;
    using PT = OperandTile<BM, P_TURNED, WAVES>;
    using QT = OperandTile<BN, Q_TURNED, WAVES>;
    constexpr int LOADS = PT::PASSES + QT::PASSES;  // of a wave and stage
    __shared__ __attribute__((aligned(1024))) uint16_t Ps[STAGES][PT::ELEMS];
    __shared__ __attribute__((aligned(1024))) uint16_t Qs[STAGES][QT::ELEMS];

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
    const int tiles = __builtin_amdgcn_readfirstlane(ps.depth > 0 ? (ps.depth + kBK - 1) / kBK : 1);  // without depth: a stage of zeros
    auto load = [&](int t) {  // beyond the last: zeros, so that every stage has its loads in flight
        uint16_t *to_p = Ps[t % STAGES], *to_q = Qs[t % STAGES];
        // The counting in front of the barriers takes every stage's direct loads to be under way. Where this one comes by ordinary
        // loads, of which a wavefront may have none, the direct loads of the stages before are waited for here.
        if (!ALIGNED && t < tiles && (t == tiles - 1 || !g.near)) {
            load_packets<BM, P_TURNED, WAVES>(to_p, ps, t * kBK, wave, lane);
            load_packets<BN, Q_TURNED, WAVES>(to_q, qs, t * kBK, wave, lane);
            __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kLgkmMax));
        } else {
            load_direct<BM, P_TURNED, WAVES>(to_p, ps, t * kBK, wave, lane);
            load_direct<BN, Q_TURNED, WAVES>(to_q, qs, t * kBK, wave, lane);
        }
    };
    auto barrier = [&](auto in_flight) {  // of this wave's loads at most so many are still on their way
        asm volatile("" ::: "memory");    // the compiler knows neither the loads' writes to LDS nor what the barrier orders
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(decltype(in_flight)::value, 0));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto multiply = [&](int t) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fp[MI], fq[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) fp[i] = PT::fragment(Ps[t % STAGES], wave_m * WM + i * 16, kk * 32, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) fq[j] = QT::fragment(Qs[t % STAGES], wave_n * WN + j * 16, kk * 32, lane);
            // Q first: a lane then holds four consecutive columns of one row of OUT.
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) mfma_in_place(acc[i][j], fq[j], fp[i]);
        }
    };
    // The barrier in front of stage t: it has landed, and everybody is done with stage t - 1, whose place t + 3 takes.
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) load(t);
    int t = 0;
    do {
        barrier(std::integral_constant<int, (STAGES - 2) * LOADS>{});
        load(t + STAGES - 1);
        multiply(t);
    } while (++t < tiles);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kLgkmMax));  // the loads beyond the last stage write LDS
    grouped_settle();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) asm volatile("" : "+a"(acc[i][j]));  // every later use comes behind the wait
    const int cols_left = g.cols - col0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = wave_m * WM + i * 16 + (lane & 15);
        if (row >= rows_left) continue;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int col = wave_n * WN + j * 16 + 4 * (lane >> 4);
            OutT* at = out + row * g.ldo + col;
            if (col + 4 <= cols_left) {
                typedef OutT Out4 __attribute__((ext_vector_type(4), aligned(sizeof(OutT))));
                if constexpr (sizeof(OutT) == 4) *reinterpret_cast<Out4*>(at) = acc[i][j];
                else *reinterpret_cast<Out4*>(at) = Out4{to_bf16(acc[i][j][0]), to_bf16(acc[i][j][1]), to_bf16(acc[i][j][2]), to_bf16(acc[i][j][3])};
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (col + v < cols_left) store_out(at + v, acc[i][j][v]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------- many rows: 256 x 256 tiles --
// The pipeline of gemm_bf16_early_kernel (gemm_bf16.hip) for ragged groups and turned operands: four waves of 128 x 128
// with all 256 accumulation registers, one workgroup per CU that walks its tiles, direct-to-LDS loads into two stages of
// 64 c, all fragments of a stage read behind the first 32 matrix instructions of its phase, a barrier in mid-phase that
// frees the stage, the loads of the tile after next spread over the rest, and the last two phases of a tile fetching the
// first two stages of the workgroup's next tile. What that kernel's comments say about the matrix instruction from inline
// assembly and about scalar operands of direct loads holds here too:
//   * an accumulator is read by nothing but that instruction within 64 clocks of its last one (grouped_settle);
//   * a fragment register written by the vector ALU is not used by the next few instructions (s_nop at the loop's head);
//   * descriptors and scalar offsets are in scalar registers well before the load that reads them.
// Bound by the matrix pipe: a stage takes 1.35 us (straight operands; 1.45 turned), a tile 9 to 12 us besides: its first
// fragments, half-empty last row tiles of the groups, and the write-back, which a CU's next tile waits for where all CUs write
// at once (in-order waits). Tried: non-temporal stores (+1 % on grad_b), other paces of the turned reads, staggered starts
// (slower).
// New here: every load goes through its descriptor's extent, which ends with the group (straight: the lines that exist;
// turned: the c that exist), so that ragged tiles need no code of their own, and the walk over the tiles of all groups
// reads a table that the workgroup makes of the offsets in LDS at its start.
// On the scalar ALU by name: a minimum inside a maximum becomes v_med3_i32 otherwise, and a descriptor with a word from
// the vector ALU cannot be an operand of the load.
__device__ __forceinline__ int scalar_min(int a, int b) {
    int r;
    asm("s_min_i32 %0, %1, %2" : "=s"(r) : "s"(a), "s"(b) : "scc");
    return r;
}
__device__ __forceinline__ int scalar_max(int a, int b) {
    int r;
    asm("s_max_i32 %0, %1, %2" : "=s"(r) : "s"(a), "s"(b) : "scc");
    return r;
}

constexpr int kBigGroups = 1024;  // groups that the table in LDS holds
constexpr int kBigBlockM = 8;     // row tiles of a group that are walked together (see list_tiles)
constexpr int kList = 32;         // tiles of a workgroup that are worked out together

// Behind how many of a phase's 128 matrix instructions the barrier that frees the stage sits, and the instructions
// between two loads.
template <int TURNED>
struct BigPace {
    static constexpr int kReads = 1 + (TURNED > 0), kBarrierAt = 36, kGap = 6;
};

// Register address of a fragment in LDS and how the fragment is read from it; ROW0: the wave's first line of the tile.
template <bool TURNED>
struct BigFragments {
    uint32_t at[TURNED ? 8 : 2];  // byte addresses in LDS
    __device__ __forceinline__ void init(const uint16_t* tile, int row0, int lane) {
        const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)tile));
        const int l16 = lane & 15, lq = lane >> 4;
        if constexpr (!TURNED) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) at[kk] = base + ((row0 + l16) * kBK + ((4 * kk + lq) ^ ((l16 >> 1) & 7)) * 8) * 2;
        } else {
            const int row = 8 * lq + (l16 >> 2), f = (row & 3) | ((row & 8) >> 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) at[i] = base + (row * 256 + ((row0 / 16 + i) ^ f) * 16 + 4 * (l16 & 3)) * 2;
        }
        // As they are from here on: taken apart into a constant and the rest, the constant parts of the reads no longer
        // fit their instructions' offsets, which costs a vector addition between two matrix instructions for every read.
#pragma unroll
        for (uint32_t& a : at) asm volatile("" : "+v"(a));
    }
    // Fragment i (16 lines) of c 32 kk .. 32 kk + 31 of stage S. HALF (turned): which four of the lane's eight c.
    template <int S, int KK>
    __device__ __forceinline__ u32x4 straight(int i) const {
        return *(const __attribute__((address_space(3))) u32x4*)(at[KK] + S * 32768 + i * (16 * kBK * 2));
    }
    template <int S, int KK, int HALF>
    __device__ __forceinline__ s16x4 turned(int i) const {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at[i] + S * 32768 + KK * 16384 + HALF * 2048));
    }
};

template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C, typename OutT>
__global__ __launch_bounds__(256) void gemm_grouped_big_kernel(GroupedProblem g) {
    constexpr int BM = 256, BN = 256, WM = 128, WN = 128, MI = 8, NI = 8, LOADS = 16;
    constexpr int OUT_LD = WN + 8;
    using Pace = BigPace<P_TURNED + Q_TURNED>;
    __shared__ __attribute__((aligned(1024))) uint16_t Ps[2][BM * kBK];
    __shared__ __attribute__((aligned(1024))) uint16_t Qs[2][BN * kBK];
    __shared__ __attribute__((aligned(16))) uint16_t Out_s[4][16 * OUT_LD];
    // The groups: their first tile (and the number of all tiles behind them), first row and end.
    __shared__ int first_tile[kBigGroups + 1], group_lo[kBigGroups], group_hi[kBigGroups];
    __shared__ long long list_at[kList][3];
    __shared__ int list_left[kList][3];

    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wave_m = wave / 2, wave_n = wave % 2;
    const int l16 = lane & 15, lq = lane >> 4;
    const int out_tiles_m = RAGGED_C ? (g.out_rows + BM - 1) / BM : 0;

    if (wave == 0) {
        int before = 0;
        for (int base = 0; base < g.groups; base += kWave) {
            const int e = base + lane;
            int lo = 0, hi = 0;
            if (e < g.groups) {
                lo = clamp_offset(g.offsets[e], g.rows);
                hi = clamp_offset(g.offsets[e + 1], g.rows);
                if (hi < lo) hi = lo;
            }
            const int tiles = e < g.groups ? (RAGGED_C ? out_tiles_m : (hi - lo + BM - 1) / BM) * g.tiles_n : 0;
            const int upto = before + wave_inclusive_sum(tiles, lane);
            if (e < g.groups) {
                first_tile[e] = upto - tiles;
                group_lo[e] = lo;
                group_hi[e] = hi;
            }
            before = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        if (lane == 0) first_tile[g.groups] = before;
    }
    __syncthreads();
    const int all_tiles = __builtin_amdgcn_readfirstlane(first_tile[g.groups]);
    const int grid = gridDim.x;  // a multiple of 8
    if (static_cast<int>(blockIdx.x) >= all_tiles) return;

    // One tile of the walk: what the loads and the write-back need of it, all scalar.
    struct Tile {
        const uint16_t *p, *q;   // first line (straight: c = 0 of it; turned: its element of row c = 0)
        int p_lines, q_lines;    // lines that exist, at most 256 of them
        int depth;
        long long out;           // first element of OUT
        int rows_left, cols_left;
    };
    // The workgroup's next tiles, kList at a time: a lane of the first wavefront works one out (some 200 instructions and a
    // dozen dependent LDS reads, 2 us if every tile did it for itself at its head).
    // 256 consecutive numbers of the walk run at a time, the workgroups of XCD x being those with number % 8 == x: they take
    // consecutive tiles, which share operand panels in that XCD's L2. Within a group eight row tiles are walked together,
    // column tile by column tile: 32 consecutive tiles are an 8 x 4 patch.
    auto list_tiles = [&](int first_id) {
        const int id = first_id + lane * grid;
        if (lane >= kList || id >= all_tiles) return;
        const int round0 = id / grid * grid, w = id - round0;
        const int count = all_tiles - round0 < grid ? all_tiles - round0 : grid;
        const int x = w % 8, per = count / 8, rem = count % 8;
        const int tile = round0 + x * per + (x < rem ? x : rem) + w / 8;
        int group = 0;  // the last one whose first tile is not behind this one
        for (int step = kBigGroups / 2; step > 0; step /= 2)
            if (group + step < g.groups && first_tile[group + step] <= tile) group += step;
        const int in_group = tile - first_tile[group], lo = group_lo[group], hi = group_hi[group];
        const int tiles_m = RAGGED_C ? out_tiles_m : (hi - lo + BM - 1) / BM;
        const int block = in_group / (kBigBlockM * g.tiles_n), in_block = in_group - block * kBigBlockM * g.tiles_n;
        const int height = tiles_m - block * kBigBlockM < kBigBlockM ? tiles_m - block * kBigBlockM : kBigBlockM;
        const int row0 = (block * kBigBlockM + in_block % height) * BM, col0 = in_block / height * BN;
        long long p, q, out;
        if constexpr (RAGGED_C) {
            p = lo * g.ldp + row0;
            q = lo * g.ldq + col0;
            out = group * g.group_stride + row0 * g.ldo + col0;
        } else {
            p = (lo + row0) * g.ldp;
            q = group * g.group_stride + (Q_TURNED ? static_cast<long long>(col0) : col0 * g.ldq);
            out = (lo + row0) * g.ldo + col0;
        }
        list_at[lane][0] = p;
        list_at[lane][1] = q;
        list_at[lane][2] = out;
        list_left[lane][0] = (RAGGED_C ? g.out_rows : hi - lo) - row0;
        list_left[lane][1] = g.cols - col0;
        list_left[lane][2] = RAGGED_C ? hi - lo : g.depth;
    };
    auto listed_tile = [&](int i) {
        auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        auto scalar64 = [&](long long v) {
            return static_cast<long long>((static_cast<unsigned long long>(static_cast<uint32_t>(scalar(static_cast<int>(v >> 32)))) << 32) |
                                          static_cast<uint32_t>(scalar(static_cast<int>(v & 0xffffffffll))));
        };
        Tile t;
        t.p = g.P + scalar64(list_at[i][0]);
        t.q = g.Q + scalar64(list_at[i][1]);
        t.out = scalar64(list_at[i][2]);
        t.rows_left = scalar(list_left[i][0]);
        t.cols_left = scalar(list_left[i][1]);
        t.depth = scalar(list_left[i][2]);
        t.p_lines = t.rows_left < BM ? t.rows_left : BM;
        t.q_lines = t.cols_left < BN ? t.cols_left : BN;
        return t;
    };

    // Load side. Straight: a wave-wide load covers 8 lines of 128 B, a pass of the four waves 32 lines; turned: 2 rows c of
    // 512 B, a pass 8 rows. Lane offsets are the same for every tile; `odd` for the odd passes of a turned operand, whose
    // rows have bit 3 set (see OperandTile).
    using PT = OperandTile<BM, P_TURNED, 4>;
    using QT = OperandTile<BN, Q_TURNED, 4>;
    static_assert(PT::PASSES == 8 && QT::PASSES == 8, "sixteen direct loads per wave and stage");
    const uint32_t p_ld = static_cast<uint32_t>(g.ldp) * 2u, q_ld = static_cast<uint32_t>(g.ldq) * 2u;  // bytes; below 2^22
    const uint32_t p_off = PT::row_of(0, wave, lane) * p_ld + PT::chunk_of(0, wave, lane) * 16u;
    const uint32_t q_off = QT::row_of(0, wave, lane) * q_ld + QT::chunk_of(0, wave, lane) * 16u;
    const uint32_t p_odd = PT::row_of(0, wave, lane) * p_ld + PT::chunk_of(1, wave, lane) * 16u;
    const uint32_t q_odd = QT::row_of(0, wave, lane) * q_ld + QT::chunk_of(1, wave, lane) * 16u;
    const uint32_t p_pass = __builtin_amdgcn_readfirstlane(PT::ROWS_PER_PASS * p_ld), q_pass = __builtin_amdgcn_readfirstlane(QT::ROWS_PER_PASS * q_ld);
    // Descriptor of stage t of a tile: straight: the lines that exist, columns from 64 t on; turned: rows 64 t on, of
    // which the last reaches to its last line only (a chunk beyond the lines of another row is the next row's head:
    // finite or not, it only enters lines that are not written).
    auto descriptor_of = [&](auto turned, const uint16_t* base, int lines, int depth, uint32_t ld_bytes, int stage) {
        constexpr bool T = decltype(turned)::value;
        uint64_t a = reinterpret_cast<uint64_t>(base);
        int extent;
        if constexpr (!T) {
            a += static_cast<uint64_t>(static_cast<uint32_t>(stage)) * (kBK * 2);
            extent = lines * static_cast<int>(ld_bytes);
        } else {
            a += static_cast<uint64_t>(static_cast<uint32_t>(stage)) * (kBK * ld_bytes);
            const int rows = scalar_max(scalar_min(depth - stage * kBK, kBK), 0);
            extent = scalar_max((rows - 1) * static_cast<int>(ld_bytes) + lines * 2, 0);  // no rows: not above 0, as lines * 2 <= ld_bytes
        }
        i32x4 d;
        d[0] = static_cast<int>(a & 0xffffffffu);
        d[1] = static_cast<int>((a >> 32) & 0xffffu);
        d[2] = extent;
        d[3] = 0x00020000;
        return d;
    };
    // Lane offset of a straight operand at stage t: the partial last stage ends inside a line, the padding stages beyond.
    auto straight_offset = [&](uint32_t off, int chunk, int depth, int stage) -> uint32_t {
        const int left = depth - stage * kBK;
        return chunk * 8 < left ? off : kBeyondExtent;
    };
    const int p_chunk = PT::chunk_of(0, wave, lane), q_chunk = QT::chunk_of(0, wave, lane);
    auto lds_of = [&](int stage, int m) -> const uint16_t* {
        return m < 8 ? &Ps[stage][PT::lds_elem(m, wave)] : &Qs[stage][QT::lds_elem(m - 8, wave)];
    };
    auto aim_load = [&](int stage, int m) { set_direct_load_destination(lds_of(stage, m)); };
    auto fire_load = [&](const i32x4& pd, const i32x4& qd, uint32_t po, uint32_t qo, uint32_t po_odd, uint32_t qo_odd, int m) {
        if (m < 8) direct_load16_buffer_to_destination(pd, m % 2 ? po_odd : po, m * p_pass);
        else direct_load16_buffer_to_destination(qd, m % 2 ? qo_odd : qo, (m - 8) * q_pass);
    };

    // Operand side. Fragment sets: [0] c 0..31 of the current stage; [1], [2] c 32..63 of stage 0 / stage 1.
    BigFragments<P_TURNED> p_at;
    BigFragments<Q_TURNED> q_at;
    p_at.init(Ps[0], wave_m * WM, lane);
    q_at.init(Qs[0], wave_n * WN, lane);
    union Fragment {
        u32x4 whole;
        s16x4 half[2];
    };
    Fragment fp[3][MI], fq[3][NI];
    f32x4 acc[MI][NI];
    // A phase's reads in order: per fragment one (straight) or two (turned).
    constexpr int P_READS = 8 * (1 + P_TURNED), Q_READS = 8 * (1 + Q_TURNED), SET_READS = P_READS + Q_READS;
    auto read_one = [&](auto stage_c, auto kk_c, int set, int r) {
        constexpr int S = decltype(stage_c)::value, KK = decltype(kk_c)::value;
        if (r < P_READS) {
            if constexpr (!P_TURNED) fp[set][r].whole = p_at.template straight<S, KK>(r);
            else if (r % 2 == 0) fp[set][r / 2].half[0] = p_at.template turned<S, KK, 0>(r / 2);
            else fp[set][r / 2].half[1] = p_at.template turned<S, KK, 1>(r / 2);
        } else {
            r -= P_READS;
            if constexpr (!Q_TURNED) fq[set][r].whole = q_at.template straight<S, KK>(r);
            else if (r % 2 == 0) fq[set][r / 2].half[0] = q_at.template turned<S, KK, 0>(r / 2);
            else fq[set][r / 2].half[1] = q_at.template turned<S, KK, 1>(r / 2);
        }
    };
    auto mfma_block = [&](int set, auto after) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int jj = 0; jj < NI; ++jj) {
                const int j = (i & 1) ? NI - 1 - jj : jj;
                mfma_in_place(acc[i][j], __builtin_bit_cast(bf16x8, fq[set][j].whole), __builtin_bit_cast(bf16x8, fp[set][i].whole));
                __builtin_amdgcn_sched_barrier(0);
                after(i * NI + jj);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    // One phase, for the stage S that holds K tile t; it fetches what `from` says at stage number `next` into S.
    auto phase = [&](auto stage_c, const Tile& from, int next, bool wait_at_end) {
        constexpr int S = decltype(stage_c)::value;
        constexpr int MINE = 1 + S, OTHER = 2 - S;
        constexpr int BARRIER_AT = Pace::kBarrierAt, GAP = Pace::kGap, READS = Pace::kReads;
        static_assert(2 * SET_READS <= READS * BARRIER_AT && BARRIER_AT <= 64 && BARRIER_AT + (LOADS - 1) * GAP < 128, "reads and loads fit the phase");
        const i32x4 pd = descriptor_of(std::integral_constant<bool, P_TURNED>{}, from.p, from.p_lines, from.depth, p_ld, next);
        const i32x4 qd = descriptor_of(std::integral_constant<bool, Q_TURNED>{}, from.q, from.q_lines, from.depth, q_ld, next);
        const uint32_t po = P_TURNED ? p_off : straight_offset(p_off, p_chunk, from.depth, next);
        const uint32_t qo = Q_TURNED ? q_off : straight_offset(q_off, q_chunk, from.depth, next);
        const uint32_t po_odd = P_TURNED ? p_odd : po, qo_odd = Q_TURNED ? q_odd : qo;
        auto maybe_load = [&](int at) {
            if (at + 1 >= BARRIER_AT && (at + 1 - BARRIER_AT) % GAP == 0 && (at + 1 - BARRIER_AT) / GAP < LOADS) aim_load(S, (at + 1 - BARRIER_AT) / GAP);
            if (at >= BARRIER_AT && (at - BARRIER_AT) % GAP == 0 && (at - BARRIER_AT) / GAP < LOADS)
                fire_load(pd, qd, po, qo, po_odd, qo_odd, (at - BARRIER_AT) / GAP);
        };
        using k0 = std::integral_constant<int, 0>;
        using k1 = std::integral_constant<int, 1>;
        mfma_block(OTHER, [&](int m) {
#pragma unroll
            for (int u = 0; u < READS; ++u) {
                const int r = m * READS + u;
                if (r < SET_READS) read_one(stage_c, k0{}, 0, r);
                else if (r < 2 * SET_READS) read_one(stage_c, k1{}, MINE, r - SET_READS);
            }
            if (m == BARRIER_AT - 1) {
                __builtin_amdgcn_s_waitcnt(waitcnt_imm(kVmMax, 0));
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
            maybe_load(m);
        });
        mfma_block(0, [&](int m) { maybe_load(64 + m); });
        if (wait_at_end) __builtin_amdgcn_s_waitcnt(waitcnt_imm(LOADS, kLgkmMax));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    using s0 = std::integral_constant<int, 0>;
    using s1 = std::integral_constant<int, 1>;

    int id = blockIdx.x, at = 0;  // the current tile and its place in the list
    if (wave == 0) list_tiles(id);
    __syncthreads();
    Tile tile = listed_tile(0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const i32x4 pd = descriptor_of(std::integral_constant<bool, P_TURNED>{}, tile.p, tile.p_lines, tile.depth, p_ld, t);
        const i32x4 qd = descriptor_of(std::integral_constant<bool, Q_TURNED>{}, tile.q, tile.q_lines, tile.depth, q_ld, t);
        const uint32_t po = P_TURNED ? p_off : straight_offset(p_off, p_chunk, tile.depth, t);
        const uint32_t qo = Q_TURNED ? q_off : straight_offset(q_off, q_chunk, tile.depth, t);
        const i32x4 pd_s = scalar_descriptor(pd), qd_s = scalar_descriptor(qd);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 4" ::: "memory");  // between a scalar register's write by the vector ALU and a load that reads it
#pragma unroll
        for (int m = 0; m < LOADS; ++m) {
            aim_load(t, m);
            asm volatile("s_nop 0" ::: "memory");  // between the write of M0 and the load
            fire_load(pd_s, qd_s, po, qo, P_TURNED ? p_odd : po, Q_TURNED ? q_odd : qo, m);
        }
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kLgkmMax));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  while (true) {  // one tile per trip, its first stages complete in LDS
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < MI; ++i) fp[2][i].whole = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < NI; ++j) fq[2][j].whole = u32x4{0u, 0u, 0u, 0u};
    const int next_id = id + grid;
    const bool has_next = next_id < all_tiles;
    Tile next = tile;
    if (has_next) {
        if (++at == kList) {
            at = 0;
            lds_barrier();  // every wavefront has its copy of the last tile of the list
            if (wave == 0) list_tiles(next_id);
            lds_barrier();
        }
        next = listed_tile(at);
    }
    // Stages of 64 c, an even number of at least two (those beyond the depth are zeros).
    const int have = (tile.depth + kBK - 1) / kBK, stages = have < 2 ? 2 : have + (have & 1);
    int t = 0;
    do {
        asm volatile("s_nop 4");
        const bool last = t + 2 >= stages;
        const int fetch = last ? (has_next ? 0 : stages - 2) : t + 2;
        Tile from = tile;  // selected field by field, not branched on: the trips stay the same straight-line code
        from.p = last ? next.p : tile.p;
        from.q = last ? next.q : tile.q;
        from.p_lines = last ? next.p_lines : tile.p_lines;
        from.q_lines = last ? next.q_lines : tile.q_lines;
        from.depth = last ? next.depth : tile.depth;
        phase(s0{}, from, fetch, t != 0);  // a tile's first phase: its second stage has landed, and the last tile's stores may drain
        phase(s1{}, from, fetch + 1, true);
        t += 2;
    } while (t < stages);
    grouped_settle();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fq[2][j].whole), __builtin_bit_cast(bf16x8, fp[2][i].whole), acc[i][j], 0, 0, 0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kLgkmMax));  // the next tile's first stages, before the stores queue up behind them
    OutT* out = static_cast<OutT*>(g.OUT) + tile.out;
    const int rows_left = tile.rows_left - wave_m * WM, cols_left = tile.cols_left - wave_n * WN;
    out += wave_m * WM * g.ldo + wave_n * WN;
    // 16 rows at a time through the wave's own patch of LDS, so that they leave as runs of 256 B.
    char* mine = reinterpret_cast<char*>(Out_s[wave]);
    constexpr int RUN = 16 / sizeof(OutT);               // values of a lane's packet
    constexpr int SPLIT = sizeof(OutT) == 4 ? 2 : 1;     // parts of 256 B in a wave's 128 columns
    typedef OutT OutRun __attribute__((ext_vector_type(RUN)));
    typedef OutT OutRunAny __attribute__((ext_vector_type(RUN), aligned(sizeof(OutT))));
    OutT* to = out + lq * g.ldo + RUN * l16;  // row 16 i + 4 p + lq
    int row = lq;
    const long long row4 = 4 * g.ldo;
    auto write_rows = [&](auto inside) {  // inside: the wave's 128 x 128 lie inside OUT
        constexpr bool INSIDE = decltype(inside)::value;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
#pragma unroll
            for (int part = 0; part < SPLIT; ++part) {
#pragma unroll
                for (int jj = 0; jj < NI / SPLIT; ++jj) {
                    asm volatile("" : "+a"(acc[i][part * (NI / SPLIT) + jj]));  // conversions stay here: moved in front of the branch they spill
                    const f32x4& r = acc[i][part * (NI / SPLIT) + jj];
                    if constexpr (sizeof(OutT) == 4) *reinterpret_cast<f32x4*>(mine + l16 * (OUT_LD * 2) + jj * 64 + lq * 16) = r;
                    else *reinterpret_cast<u16x4*>(mine + l16 * (OUT_LD * 2) + jj * 32 + lq * 8) = u16x4{to_bf16(r[0]), to_bf16(r[1]), to_bf16(r[2]), to_bf16(r[3])};
                }
                OutRun v[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) v[p] = *reinterpret_cast<const OutRun*>(mine + (4 * p + lq) * (OUT_LD * 2) + 16 * l16);
                OutT* at = to + part * (WN / SPLIT);
                if constexpr (INSIDE) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) *reinterpret_cast<OutRunAny*>(at + p * row4) = v[p];
                } else {
                    const int left = cols_left - part * (WN / SPLIT) - RUN * l16;
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        if (row + 4 * p >= rows_left) continue;
                        if (left >= RUN) *reinterpret_cast<OutRunAny*>(at + p * row4) = v[p];
                        else
#pragma unroll
                            for (int e = 0; e < RUN; ++e)
                                if (e < left) at[p * row4 + e] = v[p][e];
                    }
                }
            }
            to += 4 * row4;
            row += 16;
            asm volatile("" : "+v"(to), "+v"(row));  // one address and one row number carried along, not eight of each kept
        }
    };
    if (rows_left >= WM && cols_left >= WN) write_rows(std::true_type{});
    else if (rows_left > 0 && cols_left > 0) write_rows(std::false_type{});
    if (!has_next) break;
    id = next_id;
    tile = next;
  }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kLgkmMax));  // the last, redundant loads write LDS
}

// ------------------------------------------------------------------------------------------- few rows: 16 a tile --
// The forward product where a group has few rows: reading B bounds it. A wavefront takes 16 columns and a slice of K, 128 k
// to a step; its lane reads 16 B of the column's row of B for every instruction (the four lanes of a row 64 B, the next
// instruction's the rest of the line), so the rows need no alignment. The parts of a column tile meet in LDS. 64 matrices of
// 1536 x 2048, 32 rows: 30 to 36 us a call, box to box, 4.5 to 5.3 TB/s.
constexpr int kFewWaves = 8, kFewLeast = 2, kFewStep = 128;

struct FewProblem {
    const uint16_t *A, *B;
    const int32_t* offsets;
    void* D;
    long long lda, ldb, ldd, group_stride;
    int groups, rows, N, K;
    int tiles_n, row_tiles, k_parts, n_parts;
};

// What a wavefront works on (as W4Slice of the 4-bit weights): its lane's row of B, its complete steps first .. end - 1,
// and whether it also has the partial last one.
struct FewSlice {
    const uint16_t *b, *x;
    long long ldx;
    int rows, first, end, K;
    bool partial;
};

template <int ROWS>
__device__ __forceinline__ f32x4 multiply_few(const FewSlice& p) {
    constexpr int U = ROWS == 16 ? 1 : 2;  // steps of a round
    constexpr int BRINGS = 16 / ROWS, I = U * 4, X_LOADS = (I + BRINGS - 1) / BRINGS;
    const int lane = threadIdx.x % kWave, l16 = lane % 16, lq = lane / 16;
    const uint16_t* x_row = p.x + (l16 % ROWS < p.rows ? l16 % ROWS : p.rows - 1) * p.ldx + 8 * lq;
    const uint16_t* b_row = p.b + 8 * lq;
    // A round: U steps of B and the x they meet, fetched two rounds ahead. Loads are waited for in order: x is not asked
    // for later than its weights, and nothing is fetched under a condition (where two paths with different loads meet, the
    // wait has to assume the shorter one and waits for the rounds ahead as well).
    struct Round {
        u32x4 b[I], x[X_LOADS];
    };
    auto fetch = [&](Round& r, int step) {
#pragma unroll
        for (int i = 0; i < I; ++i) __builtin_memcpy(&r.b[i], b_row + static_cast<long long>(step) * kFewStep + 32 * i, 16);
#pragma unroll
        for (int j = 0; j < X_LOADS; ++j) {
            const int c = j * BRINGS + l16 / ROWS;  // the lane's instruction; beyond the round's, the last one's
            __builtin_memcpy(&r.x[j], x_row + static_cast<long long>(step) * kFewStep + 32 * (c < I ? c : I - 1), 16);
        }
    };
    f32x4 even = {0.0f, 0.0f, 0.0f, 0.0f}, odd = even;
    auto compute = [&](const Round& r) {
        bf16x8 x[X_LOADS];
#pragma unroll
        for (int j = 0; j < X_LOADS; ++j) x[j] = __builtin_bit_cast(bf16x8, r.x[j]);
        auto pair = [&](auto c) {
            constexpr int C = decltype(c)::value;
            bf16x8 a, b;
            instruction_x<ROWS, C>(x, a);
            instruction_x<ROWS, C + 1>(x, b);
            even = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, r.b[C]), even, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, __builtin_bit_cast(bf16x8, r.b[C + 1]), odd, 0, 0, 0);
        };
        pair(std::integral_constant<int, 0>{});
        pair(std::integral_constant<int, 2>{});
        if constexpr (U == 2) {
            pair(std::integral_constant<int, 4>{});
            pair(std::integral_constant<int, 6>{});
        }
    };
    const int rounds = p.end > p.first ? (p.end - p.first) / U : 0;
    if (rounds > 0) {
        auto round_at = [&](int r) { return p.first + (r < rounds ? r : rounds - 1) * U; };
        Round a, b;
        fetch(a, p.first);
        fetch(b, round_at(1));
        for (int r = 0;; r += 2) {
            compute(a);
            if (r + 2 >= rounds) {
                if (r + 1 < rounds) compute(b);
                break;
            }
            fetch(a, round_at(r + 2));
            compute(b);
            fetch(b, round_at(r + 3));
        }
    }
    // What is left: complete steps that fill no round, and the partial last one, whose packets are cut at K.
    const uint16_t* x_own = p.x + (l16 < p.rows ? l16 : p.rows - 1) * p.ldx + 8 * lq;
    for (int step = p.first + rounds * U; step < p.end + p.partial; ++step) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = step * kFewStep + 32 * i, there = p.K - k - 8 * lq;
            const u32x4 x = load_packet(x_own + k, there), b = load_packet(b_row + k, there);
            even = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, b), even, 0, 0, 0);
        }
    }
    return even + odd;
}

template <typename OutT>
__global__ __launch_bounds__(kFewWaves * kWave) void gemm_grouped_few_kernel(FewProblem p) {
    __shared__ f32x4 parts[kFewWaves * kWave];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane % 16, lq = lane / 16;
    const int k_part = wave % p.k_parts, n_part = wave / p.k_parts;
    // The row tiles of a column tile follow each other on one XCD (workgroups 8 apart), whose L2 then has its part of B.
    const int xcd = blockIdx.x % kXcds, local = blockIdx.x / kXcds;
    const int column = (local / p.row_tiles) * kXcds + xcd;
    if (column >= p.tiles_n) return;
    const GroupTile t = find_group_tile(p.offsets, p.groups, p.rows, local % p.row_tiles, 16);
    if (t.group < 0) return;
    const int n0 = (column * p.n_parts + n_part) * 16;
    const int whole = p.K / kFewStep, steps = (p.K + kFewStep - 1) / kFewStep, slice = (steps + p.k_parts - 1) / p.k_parts;
    FewSlice s;
    s.b = p.B + t.group * p.group_stride + (n0 + l16 < p.N ? n0 + l16 : p.N - 1) * p.ldb;  // columns beyond the last repeat it
    s.x = p.A + t.row0 * p.lda;
    s.ldx = p.lda;
    s.rows = t.row_end - t.row0 < 16 ? t.row_end - t.row0 : 16;
    s.first = k_part * slice;
    s.end = s.first + slice < whole ? s.first + slice : whole;
    s.partial = whole < steps && s.first <= whole && whole < s.first + slice;
    if (s.end < s.first) s.end = s.first;  // a slice beyond the last step
    s.K = p.K;
    f32x4 total;
    if (s.rows == 1) total = multiply_few<1>(s);
    else if (s.rows <= 4) total = multiply_few<4>(s);
    else total = multiply_few<16>(s);
    if (p.k_parts > 1) {  // the parts of a column tile, added in their order
        parts[wave * kWave + lane] = total;
        __syncthreads();
        if (k_part != 0) return;
        for (int o = 1; o < p.k_parts; ++o) total += parts[(wave + o) * kWave + lane];
    }
    if (n0 + l16 >= p.N) return;
    OutT* out = static_cast<OutT*>(p.D);
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (4 * lq + v < s.rows) store_out(out + (t.row0 + 4 * lq + v) * p.ldd + n0 + l16, total[v]);
}

template <typename OutT>
int run_few(const GroupedProblem& g, const char* who, hipStream_t s) {
    FewProblem p{};
    p.A = g.P; p.B = g.Q; p.offsets = g.offsets; p.D = g.OUT;
    p.lda = g.ldp; p.ldb = g.ldq; p.ldd = g.ldo; p.group_stride = g.group_stride;
    p.groups = g.groups; p.rows = g.rows; p.N = g.cols; p.K = g.depth;
    const long long row_tiles = most_row_tiles(g.rows, g.groups, 16);
    p.row_tiles = static_cast<int>(row_tiles);
    p.k_parts = few_rows_k_parts(busy_row_tiles(g.rows, g.groups, row_tiles), p.N, p.K, kFewStep, kFewWaves, 16);
    p.n_parts = p.k_parts < kFewLeast ? kFewLeast / p.k_parts : 1;
    p.tiles_n = ceil_div(p.N, 16 * p.n_parts);
    const long long blocks = row_tiles * ceil_div(p.tiles_n, kXcds) * kXcds;
    if (!launchable(blocks, kFewWaves * kWave)) return fail(1, "%s: too many tiles", who);
    gemm_grouped_few_kernel<OutT><<<dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(p.k_parts * p.n_parts * kWave)), 0, s>>>(p);
    return check_launch("gemm_grouped_few_kernel");
}

// Which kernel: the one with the smallest estimate, in us, of these simple costs (all figures measured on one MI355X with
// 8 to 64 groups; `used` groups have rows, which the host takes to be as many as there can be, and a group wastes half a
// row tile):
//   few      5 + B read once per 16-row tile at 5.3 TB/s with up to 4 rows a group, 3.9 with more (see instruction_x)
//   general  rounds of 256 tiles of 128 x 128 at 4 + 0.48 a stage with a ring of four stages, of 512 at 4 + 1.1 with one of
//            two, or B once at 4.3 TB/s
//   big      rounds of 256 tiles of 256 x 256 at 8 + 1.2 a stage (stages in pairs), or B once at 4.3 TB/s
// (gradient of B: instead of B, results beyond the memory-side cache at 5.3 TB/s from big tiles and 4.2 from general ones).
// Measured, few / general / big: 64 rows of 32 groups, 2048 x 2048: 56 / 57 / 65 us; 512 rows: 101 / 63 / 70; 2048 rows:
// 252 / 67 / 73; 8192 rows: - / 106 / 82; 100 rows of 8 groups, 256 x 4096: 10 / 34 / 69; 2000 rows of 16, 768 x 768: 38 /
// 12 / 21. Gradient of B, general / big: 512 rows of 32 groups, 2048 x 2048: 137 / 66; 1000 rows of 32, 304 x 512: 10 / 12.
// General, four stages / two: 5003 rows of 24 groups, 1000 x 1048: 32.9 / 28.7; 4000 of 8, 2048 x 1024: 30.4 / 25.3; 2000 of 16,
// 768 x 768: 12.2 / 13.4; 6000 of 16, 1536 x 2048: 79 / 83; gradient of B, 1000 rows of 32, 304 x 512: 10.0 / 7.8. Gradient
// of B, two / big: 1000 rows of 64, 2048 x 1024, 537 MB: 127 / 102; 717 of 64, 704 x 1216: 46 / 51.
enum class Kernel { kFew, kGeneral, kGeneralPairs, kBig };
template <bool RAGGED_C>
Kernel choose_kernel(const GroupedProblem& g, int out_size, bool can_few, bool can_big) {
    const double rows = g.rows, groups = g.groups, used = rows < groups ? rows : groups;
    auto row_tiles = [&](double tile) { const double t = rows / tile + used / 2; return t > used ? t : used; };
    auto rounds = [](double tiles) { return static_cast<double>(static_cast<long long>((tiles + 255.0) / 256.0)); };
    const double depth = RAGGED_C ? rows / groups : static_cast<double>(g.depth), stages = static_cast<double>(static_cast<long long>((depth + 63) / 64));
    const double results = RAGGED_C ? groups * g.out_rows * g.cols * out_size : 0.0;
    auto tiled = [&](int edge, int per_cu, double fixed, double stage_us, double n_stages) {
        const double b_us = !RAGGED_C ? used * g.cols * depth * 2 / 4.3e6 : (results > (256 << 20) ? results / (edge == 256 ? 5.3e6 : 4.2e6) : 0.0);
        const double tiles = (RAGGED_C ? groups * ceil_div(g.out_rows, edge) : row_tiles(edge)) * ceil_div(g.cols, edge);
        const double us = rounds(tiles / per_cu) * (fixed + stage_us * n_stages);
        return 2 + (us > b_us ? us : b_us);
    };
    const double single = tiled(128, 1, 4, 0.48, stages > 1 ? stages : 1), pairs = tiled(128, 2, 4, 1.1, stages > 1 ? stages : 1);
    const double general = single <= pairs ? single : pairs;
    const double big = can_big ? tiled(256, 1, 8, 1.2, stages > 2 ? stages + static_cast<long long>(stages) % 2 : 2) : 1e30;
    const double few = can_few ? 5 + row_tiles(16) * g.cols * depth * 2 / (rows <= 4 * groups ? 5.3e6 : 3.9e6) : 1e30;
    if (few <= general && few <= big) return Kernel::kFew;
    if (big < general) return Kernel::kBig;
    return single <= pairs ? Kernel::kGeneral : Kernel::kGeneralPairs;
}

// Rows of a tile of 32-bit offsets from each other.
bool near_rows(const GroupedProblem& g) { return g.ldp < (1 << 21) && g.ldq < (1 << 21); }
// 16 B chunks are whole or absent throughout (bases, strides and the extents along memory in multiples of 8 elements), with
// 32-bit offsets inside a tile. What is not runs on the general kernel, or on the one for few rows.
template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C>
bool whole_chunks(const GroupedProblem& g) {
    const int p_along = P_TURNED ? g.out_rows : g.depth, q_along = Q_TURNED ? g.cols : g.depth;
    return aligned16(g.P) && aligned16(g.Q) && g.ldp % 8 == 0 && g.ldq % 8 == 0 && (RAGGED_C || g.group_stride % 8 == 0) && p_along % 8 == 0 &&
           q_along % 8 == 0 && near_rows(g);
}
template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C>
Kernel choose_kernel(const GroupedProblem& g, int out_size) {
    return choose_kernel<RAGGED_C>(g, out_size, !P_TURNED && !Q_TURNED,
                                   whole_chunks<P_TURNED, Q_TURNED, RAGGED_C>(g) && g.groups <= kBigGroups && cu_count() >= 8);
}

template <bool P_TURNED, bool Q_TURNED, bool RAGGED_C, typename OutT>
int run(GroupedProblem g, const char* who, hipStream_t s) {
    constexpr bool FORWARD = !P_TURNED && !Q_TURNED;
    g.near = near_rows(g);
    const bool aligned = whole_chunks<P_TURNED, Q_TURNED, RAGGED_C>(g);
    const Kernel kernel = choose_kernel<P_TURNED, Q_TURNED, RAGGED_C>(g, static_cast<int>(sizeof(OutT)));
    if constexpr (FORWARD)
        if (kernel == Kernel::kFew) return run_few<OutT>(g, who, s);
    const int edge = kernel == Kernel::kBig ? 256 : 128;
    g.tiles_n = ceil_div(g.cols, edge);
    const long long tiles_m = RAGGED_C ? static_cast<long long>(g.groups) * ceil_div(g.out_rows, edge) : most_row_tiles(g.rows, g.groups, edge);
    if (!launchable(tiles_m * g.tiles_n, 256)) return fail(1, "%s: too many tiles", who);
    if (kernel == Kernel::kBig) {
        gemm_grouped_big_kernel<P_TURNED, Q_TURNED, RAGGED_C, OutT><<<dim3(static_cast<unsigned>(cu_count() / 8 * 8)), dim3(256), 0, s>>>(g);
        return check_launch("gemm_grouped_big_kernel");
    }
    const dim3 grid(static_cast<unsigned>(tiles_m * g.tiles_n));
    auto start = [&](auto stages) {
        constexpr int STAGES = decltype(stages)::value;
        if (aligned) gemm_grouped_kernel<P_TURNED, Q_TURNED, RAGGED_C, true, STAGES, OutT><<<grid, dim3(256), 0, s>>>(g);
        else gemm_grouped_kernel<P_TURNED, Q_TURNED, RAGGED_C, false, STAGES, OutT><<<grid, dim3(256), 0, s>>>(g);
    };
    if (kernel == Kernel::kGeneralPairs) start(std::integral_constant<int, 2>{});
    else start(std::integral_constant<int, 4>{});
    return check_launch("gemm_grouped_kernel");
}

}  // namespace

static int check_grouped_sizes(const char* who, int groups, long long rows, int N, int K, int out_type) {
    if (groups < 0 || rows < 0 || N < 0 || K < 0) return fail(1, "%s: negative dimension (%d groups, %lld rows, N=%d, K=%d)", who, groups, rows, N, K);
    if (rows > 0x7fffffffll - 256) return fail(1, "%s: %lld rows, at most 2^31 - 257 are supported", who, rows);
    if (groups > 0x7fffffff - 4096 || N > 0x7fffffff - 4096 || K > 0x7fffffff - 4096)
        return fail(1, "%s: %d groups, N=%d, K=%d: at most 2^31 - 4097 are supported", who, groups, N, K);
    if (out_type != kTypeF32 && out_type != kTypeBf16) return fail(1, "%s: unknown output type %d", who, out_type);
    return 0;
}

int gemm_grouped_plan(int form, int groups, long long rows, int N, int K, int out_type, int* tile_rows, int* stages) {
    const char* who = "prism_gemm_bf16_grouped_plan";
    if (form < 0 || form > static_cast<int>(GroupedForm::kGradB)) return fail(1, "%s: unknown form %d", who, form);
    if (int rc = check_grouped_sizes(who, groups, rows, N, K, out_type)) return rc;
    const GroupedForm f = static_cast<GroupedForm>(form);
    const bool empty = groups == 0 || (f == GroupedForm::kGradB ? N == 0 || K == 0 : rows == 0 || (f == GroupedForm::kForward ? N : K) == 0);
    GroupedProblem g{};  // contiguous, bases at address 0
    g.ldp = f == GroupedForm::kForward ? K : N;
    g.ldq = K;
    g.group_stride = static_cast<long long>(N) * K;
    g.groups = groups; g.rows = static_cast<int>(rows); g.cols = f == GroupedForm::kForward ? N : K;
    g.depth = f == GroupedForm::kForward ? K : (f == GroupedForm::kGradA ? N : 0); g.out_rows = N;
    const int size = out_type == kTypeF32 ? 4 : 2;
    Kernel kernel = Kernel::kFew;
    if (!empty)
        kernel = f == GroupedForm::kForward ? choose_kernel<false, false, false>(g, size)
                 : f == GroupedForm::kGradA ? choose_kernel<false, true, false>(g, size) : choose_kernel<true, true, true>(g, size);
    if (tile_rows) *tile_rows = empty ? 0 : (kernel == Kernel::kFew ? 16 : (kernel == Kernel::kBig ? 256 : 128));
    if (stages) *stages = empty || kernel == Kernel::kFew ? 0 : (kernel == Kernel::kGeneral ? 4 : 2);
    return 0;
}

int launch_gemm_grouped(GroupedForm form, int groups, long long rows, int N, int K, const uint16_t* first, long long ld_first,
                        const uint16_t* second, long long ld_second, long long group_stride, const int32_t* offsets, void* out,
                        long long ld_out, int out_type, hipStream_t s) {
    const char* who = form == GroupedForm::kForward ? "prism_gemm_bf16_grouped"
                      : form == GroupedForm::kGradA ? "prism_gemm_bf16_grouped_grad_a" : "prism_gemm_bf16_grouped_grad_b";
    if (int rc = check_grouped_sizes(who, groups, rows, N, K, out_type)) return rc;
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
    const int group_size = grad_b ? size : 2;
    Span matrices = matrix_span(grad_b ? out : second, N, K, ld_group, group_size);
    if (matrices.bytes != 0) matrices.bytes += static_cast<uintptr_t>(groups - 1) * group_stride * group_size;
    if (outputs_overlap({grad_b ? matrices : matrix_span(out, rows, out_cols, ld_out, size)},
                        {matrix_span(first, rows, first_cols, ld_first, 2), grad_b ? matrix_span(second, rows, K, ld_second, 2) : matrices,
                         entries_span(offsets, groups + 1ll)}))
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
