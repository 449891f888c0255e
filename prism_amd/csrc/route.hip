// The router of an expert layer: the k largest of a token's E logits with their softmax weights, the gradient of that
// choice, and the plan that turns the choice into groups of rows (counts into offsets: a stable counting sort).
//
//   choice    the j-th chosen expert has the j-th largest logit; equal logits (also -0 and 0) go to the lower index; a
//             logit of -inf is never chosen (expert -1, weight 0); NaN counts as the largest.
//   weights   exp(z_j - z_0) / sum, summed over the chosen (renormalise) or over all E logits
//   gradient  with g the weights' gradient and c = sum_j w_j g_j:  chosen experts w_j (g_j - c), the others 0
//             (renormalise) or -c p_e, p_e = w_0 exp(z_e - z_0)
//   plan      entries (t, j) = t k + j in the order of their experts, equal experts in the order of the entries:
//             offsets[e] entries go to experts below e, rows[s] is the entry in slot s, slots[t][j] its inverse.
// Ranks come from counts and from positions inside a wavefront, never from the order in which atomics arrive.
//
// Launches and dependent steps bound it, not bytes. Router and plan, calls from C back to back: 1 token, 64 experts, k = 4:
// 4.8 us, one kernel; 16384 tokens, 256 experts bf16, k = 8: 14.7 us (bf16 keys struck out one by one and counts summed one by
// one: 17.2). Its kernels, each by itself in a trace: choice and counts 7.3 us (8.4 MB; eight rounds of a 16-lane maximum), sums
// 3.4, places 5.8. Above 256 experts a lane holds 64 keys whatever their number, which costs where it is not near 1024: choice
// and counts of 16384 bf16 tokens 12.6 us with 384 experts, 13.5 with 512, 16.3 with 1024; fp32 12.1 with 256, 27.9 with 384, 32.2 with
// 1024 (128 registers, and 12 B of scratch in the form for rows of any alignment). Gradient of 32768 x 128 fp32: 8.2 us,
// 4.5 TB/s.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace prism {
namespace {

constexpr int kMaxExperts = 1024, kMaxChosen = 32;
constexpr int kLanes = 16;  // lanes of a token: a DPP row, so that its sums and maxima need no LDS

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int N>
__device__ __forceinline__ uint32_t rotated(uint32_t v) { return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, true); }  // row_ror
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, rotated<8>(v));
    v = max(v, rotated<4>(v));
    v = max(v, rotated<2>(v));
    return max(v, rotated<1>(v));
}
__device__ __forceinline__ float row_sum(float v) {
    auto turn = [](uint32_t u) { return __builtin_bit_cast(float, u); };
    auto bits = [](float f) { return __builtin_bit_cast(uint32_t, f); };
    v += turn(rotated<8>(bits(v)));
    v += turn(rotated<4>(bits(v)));
    v += turn(rotated<2>(bits(v)));
    return v + turn(rotated<1>(bits(v)));
}
// Lane 0's value of every row.
__device__ __forceinline__ uint32_t row_first(uint32_t v) { return __builtin_amdgcn_update_dpp(0, v, 0x150, 0xf, 0xf, true); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ void from_float(float& to, float v) { to = v; }
__device__ __forceinline__ void from_float(uint16_t& to, float v) { to = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }  // nearest even

// PACK consecutive values in one access (16 B, or one value).
template <typename T, int PACK>
struct Logits {
    T v[PACK];
    static __device__ __forceinline__ Logits load(const T* p) {
        Logits r;
        __builtin_memcpy(r.v, __builtin_assume_aligned(p, PACK * sizeof(T)), PACK * sizeof(T));
        return r;
    }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(__builtin_assume_aligned(p, PACK * sizeof(T)), v, PACK * sizeof(T)); }
};

// Logits as unsigned integers of the same order: -0 as 0, any NaN above +inf. bf16 logits leave the lower 16 bits free.
__device__ __forceinline__ uint32_t order_of(float z) {
    z += 0.0f;
    const uint32_t u = z != z ? 0x7fff0000u : __builtin_bit_cast(uint32_t, z);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t o) { return __builtin_bit_cast(float, (o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
constexpr uint32_t kOrderNone = 0x007fffffu;  // order_of(-inf): this and below is not there

// One token by the 16 lanes of a row, VALUES logits each: value v of a lane is expert (v / PACK) 16 PACK + lane PACK + v % PACK.
// Picking is k rounds of: the row's largest key that is left, its expert. bf16: the key holds the order in its upper
// half and the complement of the expert in its lower one, so that one maximum finds both; fp32: the order is the key, the
// lowest expert that has it is found by a second maximum (of complements).
template <typename T, int VALUES, int PACK>
__device__ __forceinline__ void choose_experts(const T* z, int experts, int k, bool renormalise, float* weights, int32_t* chosen) {
    constexpr bool PACKED = sizeof(T) == 2;
    const int lane = threadIdx.x & (kLanes - 1);
    auto expert_of = [&](int v) { return (v / PACK) * (kLanes * PACK) + lane * PACK + v % PACK; };
    uint32_t key[VALUES];
#pragma unroll
    for (int v = 0; v < VALUES; v += PACK) {
        const int e = expert_of(v);
        if (e < experts) {
            const Logits<T, PACK> at = Logits<T, PACK>::load(z + e);
#pragma unroll
            for (int i = 0; i < PACK; ++i) {
                const uint32_t o = order_of(as_float(at.v[i]));
                key[v + i] = o <= kOrderNone ? 0u : (PACKED ? (o & 0xffff0000u) | static_cast<uint16_t>(~(e + i)) : o);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PACK; ++i) key[v + i] = 0u;
        }
    }
    // Lane j keeps the j-th and the (j + 16)-th.
    uint32_t my_key[2] = {0u, 0u};
    int my_expert[2] = {-1, -1};
    uint32_t top = 0, last = 0;
    for (int j = 0; j < k; ++j) {
        // PACKED: the largest key below the last one. Relative to that one and modulo 2^32, the keys from it on are small and
        // those below it large, in their order: a subtraction each, and nothing is struck out.
        uint32_t best = key[0] - last;
#pragma unroll
        for (int v = 1; v < VALUES; ++v) best = max(best, key[v] - last);
        const uint32_t won = row_max(best) + last;
        if (won == 0) break;  // the same for the 16 lanes
        int expert;
        if constexpr (PACKED) {
            expert = static_cast<uint16_t>(~won);
            last = won;
        } else {
            uint32_t other = 0;  // complement of the lowest expert with this order, among this lane's
#pragma unroll
            for (int v = VALUES - 1; v >= 0; --v) other = key[v] == won ? ~static_cast<uint32_t>(expert_of(v)) : other;
            expert = static_cast<int>(~row_max(other));
#pragma unroll
            for (int v = 0; v < VALUES; ++v) key[v] = expert_of(v) == expert ? 0u : key[v];
        }
        if (j == 0) top = won;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (j == lane + i * kLanes) { my_key[i] = won; my_expert[i] = expert; }
    }
    // (the order of a negative bf16 logit has ones in its lower half)
    auto logit = [](uint32_t o) { return logit_of(!PACKED ? o : ((o & 0x80000000u) ? o & 0xffff0000u : o | 0xffffu)); };
    const float z0 = logit(top);
    float total = 0.0f, up[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        up[i] = my_key[i] ? expf(logit(my_key[i]) - z0) : 0.0f;
        total += up[i];
    }
    if (!renormalise)  // and those that were not chosen
#pragma unroll
        for (int v = 0; v < VALUES; ++v) total += key[v] != 0u && (!PACKED || key[v] < last) ? expf(logit(key[v]) - z0) : 0.0f;
    total = row_sum(total);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane + i * kLanes;
        if (j < k) {
            weights[j] = my_key[i] ? up[i] / total : 0.0f;
            chosen[j] = my_expert[i];
        }
    }
}

constexpr int kRouteBlock = 256;

template <typename T, int VALUES, int PACK>
__global__ __launch_bounds__(kRouteBlock) void route_topk_kernel(const T* __restrict__ logits, long long ld, int tokens, int experts, int k,
                                                                 int renormalise, float* __restrict__ weights, int32_t* __restrict__ chosen) {
    const int token = blockIdx.x * (kRouteBlock / kLanes) + threadIdx.x / kLanes;
    if (token >= tokens) return;  // whole rows of lanes
    const long long at = static_cast<long long>(token) * k;
    choose_experts<T, VALUES, PACK>(logits + token * ld, experts, k, renormalise != 0, weights + at, chosen + at);
}

// 16 lanes a token: the gradient as if nothing had been chosen (0, or -c p_e), then the chosen experts' over it: every
// w_j (g_j - c), since p_e = w_j for a chosen expert of weights that are not renormalised.
template <typename T, int PACK>
__global__ __launch_bounds__(kRouteBlock) void route_backward_kernel(const float* __restrict__ grad, const T* __restrict__ logits, long long ld,
                                                                     const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                                                                     int tokens, int experts, int k, int renormalise, T* out, long long ldo) {
    const int token = blockIdx.x * (kRouteBlock / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x & (kLanes - 1);
    if (token >= tokens) return;
    const long long at = static_cast<long long>(token) * k;
    const T* z = logits + token * ld;
    T* to = out + token * ldo;
    float w[2], g[2], c = 0.0f;
    int e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane + i * kLanes;
        e[i] = j < k ? chosen[at + j] : -1;
        const bool there = e[i] >= 0 && e[i] < experts;
        w[i] = there ? weights[at + j] : 0.0f;
        g[i] = there ? grad[at + j] : 0.0f;
        if (!there) e[i] = -1;
        c = __builtin_fmaf(w[i], g[i], c);
    }
    c = row_sum(c);
    const int first = static_cast<int>(row_first(static_cast<uint32_t>(e[0])));
    const bool dense = !renormalise && first >= 0;  // else zeros
    const float w0 = __builtin_bit_cast(float, row_first(__builtin_bit_cast(uint32_t, w[0])));
    const float z0 = dense ? as_float(z[first]) : 0.0f, scale = -c * w0;
    for (int i = lane * PACK; i < experts; i += kLanes * PACK) {
        Logits<T, PACK> d;
        if (dense) {
            const Logits<T, PACK> v = Logits<T, PACK>::load(z + i);
#pragma unroll
            for (int j = 0; j < PACK; ++j) from_float(d.v[j], scale * expf(as_float(v.v[j]) - z0));
        } else {
#pragma unroll
            for (int j = 0; j < PACK; ++j) from_float(d.v[j], 0.0f);
        }
        d.store(to + i);
    }
    // The same wavefront writes these again: behind its first stores.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (e[i] >= 0) from_float(to[e[i]], w[i] * (g[i] - c));
}

// ------------------------------------------------------------------------------------------------------------ plan --
// A wavefront takes a chunk of consecutive entries, 64 at a time. `mine` is the expert of this lane's entry, -1 for
// none; peers(): the lanes with the same expert.
__device__ __forceinline__ unsigned long long peers(int mine, int bits) {
    unsigned long long mask = __ballot(mine >= 0);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((mine >> b) & 1);
        mask &= ((mine >> b) & 1) ? set : ~set;
    }
    return mask;
}
__device__ __forceinline__ unsigned long long lanes_below() { return (1ull << (threadIdx.x & (kWave - 1))) - 1; }

__device__ __forceinline__ int entry_expert(const int32_t* chosen, int entry, int end, int experts) {
    const int e = entry < end ? chosen[entry] : -1;
    return e >= 0 && e < experts ? e : -1;
}

// Places a chunk: `next` (this wavefront's own, in LDS) holds the next slot of every expert.
__device__ __forceinline__ void place_chunk(const int32_t* chosen, int first, int end, int experts, int bits, int* next, int32_t* rows, int32_t* slots) {
    const int lane = threadIdx.x & (kWave - 1);
    for (int base = first; base < end; base += kWave) {
        const int entry = base + lane;
        const int mine = entry_expert(chosen, entry, end, experts);
        const unsigned long long same = peers(mine, bits);
        int slot = -1;
        if (mine >= 0) slot = next[mine] + __popcll(same & lanes_below());
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // LDS runs a wavefront's accesses in order; the compiler must keep it too
        if (mine >= 0) {
            if ((same & lanes_below()) == 0) next[mine] += __popcll(same);  // the first of its peers
            rows[slot] = entry;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (entry < end) slots[entry] = slot;
    }
}

// Exclusive sums over the experts of `value` (LDS, experts <= kMaxExperts entries) by the first wavefront; the total
// goes to value[experts]. Called by all; ends with a barrier.
__device__ __forceinline__ void scan_experts(int* value, int experts) {
    if (threadIdx.x < kWave) {
        const int lane = threadIdx.x, per = (experts + kWave - 1) / kWave, first = lane * per;
        int mine = 0;
        for (int i = 0; i < per; ++i)
            if (first + i < experts) mine += value[first + i];
        int upto = mine;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        int before = upto - mine;
        for (int i = 0; i < per; ++i)
            if (first + i < experts) {
                const int v = value[first + i];
                value[first + i] = before;
                before += v;
            }
        if (lane == kWave - 1) value[experts] = upto;
    }
    __syncthreads();
}

// One workgroup of 16 wavefronts does a run of up to kRun entries: counts them per wavefront in LDS, sums the counts over
// the wavefronts, places them. A plan of one run takes the experts' offsets from its own counts; in longer ones they come
// from the counts of all runs (plan_count_kernel), which every run adds up for itself, or, with many runs, plan_sum_kernel.
constexpr int kRunWaves = 16, kRun = 4096, kShortRun = 512;
// Runs up to which each adds up all counts. Router and plan, 64 experts, k = 4, this way / with plan_sum_kernel: 32 runs 8.6 /
// 10.2 us, 40 runs 8.9 / 10.2, 63 runs 11.0 / 10.2.
constexpr int kSelfSum = 48;

__device__ __forceinline__ void count_run(const int32_t* chosen, int first, int end, int per, int experts, int* count) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int i = threadIdx.x; i < kRunWaves * experts; i += blockDim.x) count[i] = 0;
    __syncthreads();
    for (int base = first + wave * per; base < min(first + (wave + 1) * per, end); base += kWave) {
        const int mine = entry_expert(chosen, base + lane, min(first + (wave + 1) * per, end), experts);
        if (mine >= 0) atomicAdd(&count[wave * experts + mine], 1);  // sums of ones: no order
    }
    __syncthreads();
}

// count[wave][expert] becomes the next slot of every wavefront and expert, given start[expert], the run's own first slots.
__device__ __forceinline__ void place_run(const int32_t* chosen, int first, int end, int per, int experts, int bits, int* count, const int* start,
                                          int total, int32_t* rows, int32_t* slots) {
    const int wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int next = start[e], c[kRunWaves];  // all read before the first is written: one LDS latency, not sixteen
#pragma unroll
        for (int w = 0; w < kRunWaves; ++w) c[w] = count[w * experts + e];
#pragma unroll
        for (int w = 0; w < kRunWaves; ++w) {
            count[w * experts + e] = next;
            next += c[w];
        }
    }
    __syncthreads();
    for (int i = max(first, total) + threadIdx.x; i < end; i += blockDim.x) rows[i] = -1;  // slots that are not used
    place_chunk(chosen, min(first + wave * per, end), min(first + (wave + 1) * per, end), experts, bits, count + wave * experts, rows, slots);
}

__device__ __forceinline__ int per_wave(int run) { return (run + kRunWaves * kWave - 1) / (kRunWaves * kWave) * kWave; }

// A whole plan by one workgroup. lds: (16 + 1) * experts + 1 ints.
__device__ __forceinline__ void plan_in_workgroup(const int32_t* chosen, int entries, int experts, int bits, int32_t* offsets, int32_t* rows,
                                                  int32_t* slots, int* lds) {
    int *count = lds, *start = lds + kRunWaves * experts;
    const int per = per_wave(entries);
    count_run(chosen, 0, entries, per, experts, count);
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < kRunWaves; ++w) sum += count[w * experts + e];
        start[e] = sum;
    }
    __syncthreads();
    scan_experts(start, experts);
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
    place_run(chosen, 0, entries, per, experts, bits, count, start, start[experts], rows, slots);
}

__global__ __launch_bounds__(kRunWaves * kWave) void plan_small_kernel(const int32_t* chosen, int entries, int experts, int bits, int32_t* offsets,
                                                                       int32_t* rows, int32_t* slots) {
    extern __shared__ int plan_lds[];
    plan_in_workgroup(chosen, entries, experts, bits, offsets, rows, slots, plan_lds);
}

// Router and plan of up to 64 tokens (16 lanes each) in one launch (1 token: 4.8 us a call from C, 7.0 as two).
template <typename T, int VALUES, int PACK>
__global__ __launch_bounds__(kRunWaves * kWave) void route_small_kernel(const T* logits, long long ld, int tokens, int experts, int k, int renormalise,
                                                                        float* weights, int32_t* chosen, int bits, int32_t* offsets, int32_t* rows,
                                                                        int32_t* slots) {
    extern __shared__ int plan_lds[];
    const int token = threadIdx.x / kLanes;
    if (token < tokens) choose_experts<T, VALUES, PACK>(logits + token * ld, experts, k, renormalise != 0, weights + token * k, chosen + token * k);
    __syncthreads();  // what this workgroup wrote to memory it may read behind this
    plan_in_workgroup(chosen, tokens * k, experts, bits, offsets, rows, slots, plan_lds);
}

// counts[run][expert]
__global__ __launch_bounds__(kRunWaves * kWave) void plan_count_kernel(const int32_t* __restrict__ chosen, int entries, int experts, int run,
                                                                       int* __restrict__ counts) {
    extern __shared__ int plan_lds[];
    for (int e = threadIdx.x; e < experts; e += blockDim.x) plan_lds[e] = 0;
    __syncthreads();
    const int first = blockIdx.x * run, end = min(first + run, entries);
    for (int i = first + threadIdx.x; i < end; i += blockDim.x) {
        const int mine = entry_expert(chosen, i, end, experts);
        if (mine >= 0) atomicAdd(&plan_lds[mine], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[static_cast<long long>(blockIdx.x) * experts + e] = plan_lds[e];
}

// Router of 64 tokens a workgroup, and their counts: the plan's first step rides along (16384 tokens, 256 experts,
// k = 8: 14.7 us with its plan, 16.5 as calls of their own).
template <typename T, int VALUES, int PACK>
__global__ __launch_bounds__(kRunWaves * kWave) void route_count_kernel(const T* __restrict__ logits, long long ld, int tokens, int experts, int k, int renormalise,
                                                                        float* weights, int32_t* chosen, int* __restrict__ counts) {
    extern __shared__ int plan_lds[];
    for (int e = threadIdx.x; e < experts; e += blockDim.x) plan_lds[e] = 0;
    const int token0 = blockIdx.x * (kRunWaves * kWave / kLanes), token = token0 + threadIdx.x / kLanes;
    const long long at = static_cast<long long>(token) * k;
    if (token < tokens) choose_experts<T, VALUES, PACK>(logits + token * ld, experts, k, renormalise != 0, weights + at, chosen + at);
    __syncthreads();
    const int first = token0 * k, end = min(first + kRunWaves * kWave / kLanes * k, tokens * k);
    for (int i = first + threadIdx.x; i < end; i += blockDim.x) {
        const int mine = entry_expert(chosen, i, end, experts);
        if (mine >= 0) atomicAdd(&plan_lds[mine], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[static_cast<long long>(blockIdx.x) * experts + e] = plan_lds[e];
}

// counts[run][expert] becomes its sum over the runs before; totals[expert] the sum over all. 16 experts a workgroup, the
// runs in 64 parts, four to a wavefront. A part's first counts stay in registers, loaded all at a time.
__global__ __launch_bounds__(1024) void plan_sum_kernel(int* __restrict__ counts, int runs, int experts, int* __restrict__ totals) {
    constexpr int WAVES = 16, HELD = 8;
    __shared__ int wave_sum[WAVES][16];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, l16 = lane % 16;
    const int e = blockIdx.x * 16 + l16, part = threadIdx.x / 16;
    const int per = (runs + 63) / 64, first = min(part * per, runs), end = e < experts ? min(first + per, runs) : first;
    int* at = counts + static_cast<long long>(first) * experts + e;  // of run `first`
    int held[HELD], sum = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        held[i] = first + i < end ? at[static_cast<long long>(i) * experts] : 0;
        sum += held[i];
    }
#pragma unroll 8
    for (int i = HELD; i < end - first; ++i) sum += at[static_cast<long long>(i) * experts];
    int upto = sum;
#pragma unroll
    for (int d = 16; d < kWave; d *= 2) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane >= kWave - 16) wave_sum[wave][l16] = upto;
    __syncthreads();
    int before = upto - sum;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) before += w < wave ? wave_sum[w][l16] : 0;
    if (e < experts && part == 63) totals[e] = before + sum;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (first + i < end) at[static_cast<long long>(i) * experts] = before;
        before += held[i];
    }
    for (int i = HELD; i < end - first; ++i) {
        const int v = at[static_cast<long long>(i) * experts];
        at[static_cast<long long>(i) * experts] = before;
        before += v;
    }
}

// totals == nullptr: counts are the runs' own, and this run adds them up.
__global__ __launch_bounds__(kRunWaves * kWave) void plan_place_kernel(const int32_t* __restrict__ chosen, int entries, int experts, int bits, int run,
                                                                       const int* __restrict__ counts, const int* __restrict__ totals, int runs,
                                                                       int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    extern __shared__ int plan_lds[];
    int *count = plan_lds, *start = plan_lds + kRunWaves * experts;  // [wave][expert], [expert + 1]
    const int first = blockIdx.x * run, end = min(first + run, entries), per = per_wave(run);
    // Entries of an expert in the runs before, kept in a register across the scan (an expert is one thread's).
    int before = 0;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {  // one trip: at most 1024 experts
        int total = 0;
        if (totals != nullptr) {
            before = counts[static_cast<long long>(blockIdx.x) * experts + e];
            total = totals[e];
        } else {
#pragma unroll 8  // loads under way at a time: 2000 tokens, 64 experts, k = 4, 32 runs: 15.9 -> 9.0 us
            for (int r = 0; r < runs; ++r) {
                const int c = counts[static_cast<long long>(r) * experts + e];
                before += r < static_cast<int>(blockIdx.x) ? c : 0;
                total += c;
            }
        }
        start[e] = total;
    }
    count_run(chosen, first, end, per, experts, count);
    scan_experts(start, experts);
    const int total = start[experts];
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) start[e] += before;
    __syncthreads();
    place_run(chosen, first, end, per, experts, bits, count, start, total, rows, slots);
}

int bits_of(int experts) {
    int b = 0;
    while ((1 << b) < experts) ++b;
    return b;
}

int check_route(const char* who, long long tokens, int experts, int k) {
    if (tokens < 0) return fail(1, "%s: negative number of tokens", who);
    if (experts < 1 || experts > kMaxExperts) return fail(1, "%s: %d experts, 1 to %d are supported", who, experts, kMaxExperts);
    if (k < 1 || k > kMaxChosen || k > experts) return fail(1, "%s: k=%d, 1 to %d and at most the number of experts (%d) are supported", who, k, kMaxChosen, experts);
    if (tokens > 0x7fffffffll || tokens * k > 0x7fffffffll - 4096) return fail(1, "%s: %lld tokens x %d: beyond 31 bits", who, tokens, k);
    if (!launchable(ceil_div(tokens, 64ll), 64 * kLanes)) return fail(1, "%s: %lld tokens are too much work for one launch", who, tokens);
    return 0;
}

// Runs of a plan: shorter ones where the longest would leave CUs without one.
int run_entries(long long entries) { return entries >= 256ll * kRun ? kRun : kShortRun; }
long long plan_runs(long long entries, int run) { return entries > 0 ? ceil_div(entries, static_cast<long long>(run)) : 1; }
// One workgroup does it all: its counters fit 64 KiB of LDS.
bool one_run(long long entries, int experts) { return entries <= kRun && experts <= 512; }
size_t run_lds(int experts) { return (static_cast<size_t>(kRunWaves + 1) * experts + 1) * sizeof(int); }

// The plan behind the counts of its runs.
int place_runs(const int32_t* chosen, int entries, int experts, int run, long long runs, int* counts, int32_t* offsets, int32_t* rows, int32_t* slots,
               hipStream_t s) {
    int* totals = nullptr;
    if (runs > kSelfSum) {
        totals = counts + runs * experts;
        plan_sum_kernel<<<dim3(static_cast<unsigned>(ceil_div(experts, 16))), dim3(1024), 0, s>>>(counts, static_cast<int>(runs), experts, totals);
        if (int rc = check_launch("plan_sum_kernel")) return rc;
    }
    const size_t lds = run_lds(experts);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(plan_place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (e != hipSuccess) return hip_fail(e, "hipFuncSetAttribute(plan_place_kernel)");
    }
    plan_place_kernel<<<dim3(static_cast<unsigned>(runs)), dim3(kRunWaves * kWave), lds, s>>>(chosen, entries, experts, bits_of(experts), run, counts, totals,
                                                                                             static_cast<int>(runs), offsets, rows, slots);
    return check_launch("plan_place_kernel");
}

int check_plan(const char* who, const int32_t* chosen, long long tokens, int k, int experts, int32_t* offsets, int32_t* rows, int32_t* slots, void* ws,
               size_t ws_bytes) {
    if (tokens < 0) return fail(1, "%s: negative number of tokens", who);
    if (experts < 1 || experts > kMaxExperts) return fail(1, "%s: %d experts, 1 to %d are supported", who, experts, kMaxExperts);
    if (k < 1) return fail(1, "%s: k=%d, at least 1 expert per token is needed", who, k);
    if (tokens > 0x7fffffffll || tokens * k > 0x7fffffffll - 4096) return fail(1, "%s: %lld tokens x %d: beyond 31 bits", who, tokens, k);
    if (offsets == nullptr || !aligned4(offsets)) return fail(1, "%s: offsets must be a 4-byte aligned device pointer", who);
    if (tokens > 0 && (chosen == nullptr || rows == nullptr || slots == nullptr || !aligned4(chosen) || !aligned4(rows) || !aligned4(slots)))
        return fail(1, "%s: experts, rows and slots must be 4-byte aligned device pointers", who);
    const size_t need = expert_plan_workspace_bytes(tokens, k, experts);
    if (!one_run(tokens * k, experts) && (ws == nullptr || !aligned4(ws) || ws_bytes < need))
        return fail(1, "%s: workspace of %zu bytes, %zu needed", who, ws == nullptr ? size_t{0} : ws_bytes, need);
    return 0;
}

Span logits_span(const void* at, int type, long long tokens, int experts, long long ld) { return matrix_span(at, tokens, experts, ld, type == kTypeF32 ? 4 : 2); }
// Of a workspace only what the plan needs.
Span plan_workspace_span(const void* ws, long long tokens, int k, int experts) {
    return {ws, one_run(tokens * k, experts) ? 0 : expert_plan_workspace_bytes(tokens, k, experts)};
}

// The router's kernels for a logit type, a number of experts and an alignment: f(T, values of a lane, values of an access).
template <typename F>
int with_logits(int type, const void* logits, long long ld, int experts, F&& f) {
    auto sized = [&](auto t, auto wide) {
        using T = decltype(t);
        using std::integral_constant;
        constexpr int WIDE = decltype(wide)::value;
        const bool packed = aligned16(logits) && ld % WIDE == 0 && experts % WIDE == 0;
        auto go = [&](auto values) {
            if (packed) return f(T{}, values, integral_constant<int, WIDE>{});
            return f(T{}, values, integral_constant<int, 1>{});
        };
        if (experts <= 128) return go(integral_constant<int, 8>{});
        if (experts <= 256) return go(integral_constant<int, 16>{});
        return go(integral_constant<int, 64>{});
    };
    return type == kTypeF32 ? sized(float{}, std::integral_constant<int, 4>{}) : sized(uint16_t{}, std::integral_constant<int, 8>{});
}

}  // namespace

// Room for the shortest runs: those of the router's 64 tokens, or of kShortRun entries.
size_t expert_plan_workspace_bytes(long long tokens, int k, int experts) {
    if (tokens < 0 || k < 1 || experts < 1 || experts > kMaxExperts || tokens > 0x7fffffffll || one_run(tokens * k, experts)) return 16;
    const long long by_entries = plan_runs(tokens * k, run_entries(tokens * k)), by_tokens = ceil_div(tokens, 64ll);
    return static_cast<size_t>((by_entries > by_tokens ? by_entries : by_tokens) + 1) * experts * sizeof(int);
}

int launch_expert_plan(const int32_t* chosen, long long tokens, int k, int experts, int32_t* offsets, int32_t* rows, int32_t* slots, void* ws,
                       size_t ws_bytes, hipStream_t s) {
    const char* who = "prism_expert_plan";
    if (int rc = check_plan(who, chosen, tokens, k, experts, offsets, rows, slots, ws, ws_bytes)) return rc;
    const int entries = static_cast<int>(tokens * k);
    if (outputs_overlap({entries_span(offsets, experts + 1ll), entries_span(rows, entries), entries_span(slots, entries), plan_workspace_span(ws, tokens, k, experts)},
                        {entries_span(chosen, entries)}))
        return fail(1, "%s: a result or the workspace overlaps the experts or another one", who);
    if (one_run(entries, experts)) {
        plan_small_kernel<<<dim3(1), dim3(kRunWaves * kWave), run_lds(experts), s>>>(chosen, entries, experts, bits_of(experts), offsets, rows, slots);
        return check_launch("plan_small_kernel");
    }
    const int run = run_entries(entries);
    const long long runs = plan_runs(entries, run);
    int* counts = static_cast<int*>(ws);
    plan_count_kernel<<<dim3(static_cast<unsigned>(runs)), dim3(kRunWaves * kWave), static_cast<size_t>(experts) * sizeof(int), s>>>(chosen, entries, experts, run, counts);
    if (int rc = check_launch("plan_count_kernel")) return rc;
    return place_runs(chosen, entries, experts, run, runs, counts, offsets, rows, slots, s);
}

int check_route_call(const char* who, int type, const void* logits, long long ld, long long tokens, int experts, int k, const float* weights,
                     const int32_t* chosen) {
    if (type != kTypeF32 && type != kTypeBf16) return fail(1, "%s: unknown logit type %d", who, type);
    if (int rc = check_route(who, tokens, experts, k)) return rc;
    if (tokens == 0) return 0;
    if (logits == nullptr || weights == nullptr || chosen == nullptr) return fail(1, "%s: null pointer", who);
    if (reinterpret_cast<uintptr_t>(logits) % (type == kTypeF32 ? 4 : 2) != 0 || !aligned4(weights) || !aligned4(chosen)) return fail(1, "%s: misaligned pointer", who);
    if (tokens > 1 && ld < experts) return fail(1, "%s: a row stride (%lld) is shorter than its row (%d)", who, ld, experts);
    return 0;
}

int launch_route_topk(int type, const void* logits, long long ld, long long tokens, int experts, int k, int renormalise, float* weights, int32_t* chosen,
                      hipStream_t s) {
    const char* who = "prism_route_topk";
    if (int rc = check_route_call(who, type, logits, ld, tokens, experts, k, weights, chosen)) return rc;
    if (tokens == 0) return 0;
    if (outputs_overlap({entries_span(weights, tokens * k), entries_span(chosen, tokens * k)}, {logits_span(logits, type, tokens, experts, ld)}))
        return fail(1, "%s: a result overlaps the logits or the other result", who);
    return with_logits(type, logits, ld, experts, [&](auto t, auto values, auto pack) {
        using T = decltype(t);
        constexpr int V = decltype(values)::value, P = decltype(pack)::value;
        const unsigned blocks = static_cast<unsigned>(ceil_div(tokens, static_cast<long long>(kRouteBlock / kLanes)));
        route_topk_kernel<T, V, P><<<dim3(blocks), dim3(kRouteBlock), 0, s>>>(static_cast<const T*>(logits), ld, static_cast<int>(tokens), experts, k, renormalise,
                                                                             weights, chosen);
        return check_launch("route_topk_kernel");
    });
}

int launch_route_plan(int type, const void* logits, long long ld, long long tokens, int experts, int k, int renormalise, float* weights, int32_t* chosen,
                      int32_t* offsets, int32_t* rows, int32_t* slots, void* ws, size_t ws_bytes, hipStream_t s) {
    const char* who = "prism_route_plan";
    if (int rc = check_route_call(who, type, logits, ld, tokens, experts, k, weights, chosen)) return rc;
    if (int rc = check_plan(who, chosen, tokens, k, experts, offsets, rows, slots, ws, ws_bytes)) return rc;
    if (tokens == 0) return launch_expert_plan(chosen, tokens, k, experts, offsets, rows, slots, ws, ws_bytes, s);
    if (outputs_overlap({entries_span(weights, tokens * k), entries_span(chosen, tokens * k), entries_span(offsets, experts + 1ll), entries_span(rows, tokens * k),
                         entries_span(slots, tokens * k), plan_workspace_span(ws, tokens, k, experts)},
                        {logits_span(logits, type, tokens, experts, ld)}))
        return fail(1, "%s: a result or the workspace overlaps the logits or another one", who);
    constexpr int TOKENS = kRunWaves * kWave / kLanes;  // of a workgroup
    if (tokens > TOKENS && one_run(tokens * k, experts)) {  // too many for one workgroup's router, and no workspace to count in
        if (int rc = launch_route_topk(type, logits, ld, tokens, experts, k, renormalise, weights, chosen, s)) return rc;
        return launch_expert_plan(chosen, tokens, k, experts, offsets, rows, slots, ws, ws_bytes, s);
    }
    const long long runs = ceil_div(tokens, static_cast<long long>(TOKENS));
    const bool small = one_run(tokens * k, experts);  // else check_plan has seen to the workspace
    const int rc = with_logits(type, logits, ld, experts, [&](auto t, auto values, auto pack) {
        using T = decltype(t);
        constexpr int V = decltype(values)::value, P = decltype(pack)::value;
        const T* z = static_cast<const T*>(logits);
        if (small)
            route_small_kernel<T, V, P><<<dim3(1), dim3(kRunWaves * kWave), run_lds(experts), s>>>(z, ld, static_cast<int>(tokens), experts, k, renormalise, weights,
                                                                                                  chosen, bits_of(experts), offsets, rows, slots);
        else
            route_count_kernel<T, V, P><<<dim3(static_cast<unsigned>(runs)), dim3(kRunWaves * kWave), static_cast<size_t>(experts) * sizeof(int), s>>>(
                z, ld, static_cast<int>(tokens), experts, k, renormalise, weights, chosen, static_cast<int*>(ws));
        return check_launch("route_small_kernel or route_count_kernel");
    });
    if (rc != 0 || small) return rc;
    return place_runs(chosen, static_cast<int>(tokens * k), experts, TOKENS * k, runs, static_cast<int*>(ws), offsets, rows, slots, s);
}

int launch_route_backward(int type, const float* grad, const void* logits, long long ld, const float* weights, const int32_t* chosen, long long tokens,
                          int experts, int k, int renormalise, void* out, long long ldo, hipStream_t s) {
    const char* who = "prism_route_topk_backward";
    if (int rc = check_route_call(who, type, logits, ld, tokens, experts, k, weights, chosen)) return rc;
    if (tokens == 0) return 0;
    if (grad == nullptr || out == nullptr) return fail(1, "%s: null pointer", who);
    const unsigned size = type == kTypeF32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % size != 0 || !aligned4(grad)) return fail(1, "%s: misaligned pointer", who);
    if (tokens > 1 && ldo < experts) return fail(1, "%s: a row stride is shorter than its row (%d)", who, experts);
    if (outputs_overlap({logits_span(out, type, tokens, experts, ldo)},
                        {logits_span(logits, type, tokens, experts, ld), entries_span(grad, tokens * k), entries_span(weights, tokens * k), entries_span(chosen, tokens * k)}))
        return fail(1, "%s: the result overlaps an input", who);
    const dim3 grid(static_cast<unsigned>(ceil_div(tokens, static_cast<long long>(kRouteBlock / kLanes))));
    auto go = [&](auto t, auto pack) {
        using T = decltype(t);
        route_backward_kernel<T, decltype(pack)::value><<<grid, dim3(kRouteBlock), 0, s>>>(grad, static_cast<const T*>(logits), ld, weights, chosen,
                                                                                          static_cast<int>(tokens), experts, k, renormalise, static_cast<T*>(out), ldo);
        return check_launch("route_backward_kernel");
    };
    const int wide = 16 / static_cast<int>(size);
    const bool packed = aligned16(logits) && aligned16(out) && ld % wide == 0 && ldo % wide == 0 && experts % wide == 0;
    if (type == kTypeF32) return packed ? go(float{}, std::integral_constant<int, 4>{}) : go(float{}, std::integral_constant<int, 1>{});
    return packed ? go(uint16_t{}, std::integral_constant<int, 8>{}) : go(uint16_t{}, std::integral_constant<int, 1>{});
}

}  // namespace prism
