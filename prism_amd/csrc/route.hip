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
#include <cmath>
#include <type_traits>

#include "common.h"

namespace prism {
namespace {

constexpr int kRouteBlock = 256;
constexpr int kMaxExperts = 1024, kMaxChosen = 32;

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return __builtin_bit_cast(float, static_cast<uint32_t>(*p) << 16); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }

// Logits as unsigned integers of the same order: -0 as 0, any NaN above +inf.
__device__ __forceinline__ uint32_t order_of(float z) {
    z += 0.0f;
    const uint32_t u = z != z ? 0x7fffffffu : __builtin_bit_cast(uint32_t, z);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t o) { return __builtin_bit_cast(float, (o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
constexpr uint32_t kOrderNone = 0x007fffffu;  // order_of(-inf): this and below is not there

// One token by LANES consecutive lanes, VALUES logits each (lane i has experts i, i + LANES, ...).
template <typename T, int LANES, int VALUES>
__device__ __forceinline__ void choose_experts(const T* z, int experts, int k, bool renormalise, float* weights, int32_t* chosen) {
    const int lane = threadIdx.x & (LANES - 1);
    uint32_t order[VALUES];
    float logit[VALUES];
#pragma unroll
    for (int v = 0; v < VALUES; ++v) {
        const int e = lane + v * LANES;
        logit[v] = e < experts ? load_logit(z + e) : -INFINITY;
        order[v] = order_of(logit[v]);
    }
    // The chosen ones, one after the other: lane j (and j - LANES) keeps the j-th.
    constexpr int KEEP = kMaxChosen / LANES > 0 ? kMaxChosen / LANES : 1;
    uint32_t my_order[KEEP];
    int my_expert[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) { my_order[i] = kOrderNone; my_expert[i] = -1; }
    uint32_t top = kOrderNone;
    for (int j = 0; j < k; ++j) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int v = 0; v < VALUES; ++v)
            if (order[v] > best) { best = order[v]; at = v; }  // strictly: the lower index stays
        unsigned long long key = (static_cast<unsigned long long>(best) << 32) | static_cast<uint32_t>(~(lane + at * LANES));
#pragma unroll
        for (int d = LANES / 2; d > 0; d /= 2) {
            const unsigned long long other = __shfl_xor(key, d);
            key = other > key ? other : key;
        }
        const uint32_t won = static_cast<uint32_t>(key >> 32);
        if (won <= kOrderNone) break;  // the same for all LANES lanes
        const int expert = static_cast<int>(~static_cast<uint32_t>(key));
        if (j == 0) top = won;
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (j == lane + i * LANES) { my_order[i] = won; my_expert[i] = expert; }
#pragma unroll
        for (int v = 0; v < VALUES; ++v)
            if (lane + v * LANES == expert) order[v] = 0;
    }
    const float z0 = logit_of(top);
    float total = 0.0f, up[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        up[i] = my_order[i] > kOrderNone ? expf(logit_of(my_order[i]) - z0) : 0.0f;
        if (renormalise) total += up[i];
    }
    if (!renormalise && top > kOrderNone)
#pragma unroll
        for (int v = 0; v < VALUES; ++v) total += logit[v] == -INFINITY ? 0.0f : expf(logit[v] - z0);
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) total += __shfl_xor(total, d);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int j = lane + i * LANES;
        if (j < k) {
            weights[j] = my_order[i] > kOrderNone ? up[i] / total : 0.0f;
            chosen[j] = my_expert[i];
        }
    }
}

template <typename T, int LANES, int VALUES>
__global__ __launch_bounds__(kRouteBlock) void route_topk_kernel(const T* __restrict__ logits, long long ld, int tokens, int experts, int k,
                                                                 int renormalise, float* __restrict__ weights, int32_t* __restrict__ chosen) {
    const int token = blockIdx.x * (kRouteBlock / LANES) + threadIdx.x / LANES;
    if (token >= tokens) return;  // whole groups of LANES lanes
    const long long at = static_cast<long long>(token) * k;
    choose_experts<T, LANES, VALUES>(logits + token * ld, experts, k, renormalise != 0, weights + at, chosen + at);
}

// One thread group of 16 lanes per token.
template <typename T>
__global__ __launch_bounds__(kRouteBlock) void route_backward_kernel(const float* __restrict__ grad, const T* __restrict__ logits, long long ld,
                                                                     const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                                                                     int tokens, int experts, int k, int renormalise, T* __restrict__ out, long long ldo) {
    const int token = blockIdx.x * (kRouteBlock / 16) + threadIdx.x / 16;
    if (token >= tokens) return;
    const long long at = static_cast<long long>(token) * k;
    float c = 0.0f;
    for (int j = 0; j < k; ++j)
        if (chosen[at + j] >= 0) c = __builtin_fmaf(weights[at + j], grad[at + j], c);
    const int first = chosen[at];
    const bool any = first >= 0 && first < experts;
    const float w0 = any ? weights[at] : 0.0f, z0 = any && !renormalise ? load_logit(logits + token * ld + first) : 0.0f;
    for (int e = threadIdx.x & 15; e < experts; e += 16) {
        float d = 0.0f;
        if (!renormalise && any) d = -c * w0 * expf(load_logit(logits + token * ld + e) - z0);
        for (int j = 0; j < k; ++j)
            if (chosen[at + j] == e) d = renormalise ? weights[at + j] * (grad[at + j] - c) : __builtin_fmaf(weights[at + j], grad[at + j], d);
        store_logit(out + token * ldo + e, d);
    }
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

// One workgroup does the whole plan up to here: its counters fit 64 KiB of LDS.
constexpr int kSmallWaves = 16, kSmallEntries = 4096, kSmallExperts = 512;
inline bool one_workgroup(long long entries, int experts) { return entries <= kSmallEntries && experts <= kSmallExperts; }

// The plan by one workgroup of 16 wavefronts: counts per wavefront, sums over wavefronts and experts, places.
__device__ __forceinline__ void plan_in_workgroup(const int32_t* chosen, int entries, int experts, int bits, int32_t* offsets, int32_t* rows,
                                                  int32_t* slots, int* lds /* (16 + 1) * experts + 1 */) {
    int* count = lds;                              // [wave][expert]
    int* total = lds + kSmallWaves * experts;      // [expert + 1]
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int i = threadIdx.x; i < kSmallWaves * experts; i += blockDim.x) count[i] = 0;
    __syncthreads();
    const int per = (entries + kSmallWaves * kWave - 1) / (kSmallWaves * kWave) * kWave;
    const int first = min(wave * per, entries), end = min(first + per, entries);
    for (int base = first; base < end; base += kWave) {
        const int mine = entry_expert(chosen, base + lane, end, experts);
        if (mine >= 0) atomicAdd(&count[wave * experts + mine], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < kSmallWaves; ++w) {
            const int c = count[w * experts + e];
            count[w * experts + e] = sum;
            sum += c;
        }
        total[e] = sum;
    }
    __syncthreads();
    scan_experts(total, experts);
    for (int e = threadIdx.x; e < experts; e += blockDim.x)
        for (int w = 0; w < kSmallWaves; ++w) count[w * experts + e] += total[e];
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = total[e];
    __syncthreads();
    for (int i = total[experts] + threadIdx.x; i < entries; i += blockDim.x) rows[i] = -1;
    place_chunk(chosen, first, end, experts, bits, count + wave * experts, rows, slots);
}

__global__ __launch_bounds__(kSmallWaves * kWave) void plan_small_kernel(const int32_t* chosen, int entries, int experts, int bits, int32_t* offsets,
                                                                          int32_t* rows, int32_t* slots) {
    extern __shared__ int plan_lds[];
    plan_in_workgroup(chosen, entries, experts, bits, offsets, rows, slots, plan_lds);
}

// Larger plans: chunks of kChunk entries, one per wavefront. counts[chunk][expert], then its exclusive sums over the
// chunks and the experts' totals, then the places.
constexpr int kChunk = 512, kChunkWaves = 4;

__global__ __launch_bounds__(kChunkWaves * kWave) void plan_count_kernel(const int32_t* __restrict__ chosen, int entries, int experts, int* __restrict__ counts) {
    extern __shared__ int plan_lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int i = threadIdx.x; i < kChunkWaves * experts; i += blockDim.x) plan_lds[i] = 0;
    __syncthreads();
    const int chunk = blockIdx.x * kChunkWaves + wave;
    const long long first = static_cast<long long>(chunk) * kChunk;
    if (first < entries) {
        const int end = static_cast<int>(first + kChunk < entries ? first + kChunk : entries);
        for (int base = static_cast<int>(first); base < end; base += kWave) {
            const int mine = entry_expert(chosen, base + lane, end, experts);
            if (mine >= 0) atomicAdd(&plan_lds[wave * experts + mine], 1);
        }
    }
    __syncthreads();
    if (first < entries)
        for (int e = lane; e < experts; e += kWave) counts[static_cast<long long>(chunk) * experts + e] = plan_lds[wave * experts + e];
}

// 16 experts a workgroup, the chunks in 64 runs.
__global__ __launch_bounds__(1024) void plan_sum_kernel(int* __restrict__ counts, int chunks, int experts, int* __restrict__ totals) {
    __shared__ int run_sum[64][17];
    const int e = blockIdx.x * 16 + threadIdx.x % 16, run = threadIdx.x / 16;
    const int per = (chunks + 63) / 64, first = min(run * per, chunks), end = min(first + per, chunks);
    int sum = 0;
    if (e < experts)
        for (int c = first; c < end; ++c) sum += counts[static_cast<long long>(c) * experts + e];
    run_sum[run][threadIdx.x % 16] = sum;
    __syncthreads();
    if (e >= experts) return;
    int before = 0;
    for (int r = 0; r < run; ++r) before += run_sum[r][threadIdx.x % 16];
    for (int c = first; c < end; ++c) {
        const long long at = static_cast<long long>(c) * experts + e;
        const int v = counts[at];
        counts[at] = before;
        before += v;
    }
    if (run == 63) totals[e] = before;
}

__global__ __launch_bounds__(kChunkWaves * kWave) void plan_place_kernel(const int32_t* __restrict__ chosen, int entries, int experts, int bits,
                                                                         const int* __restrict__ counts, const int* __restrict__ totals,
                                                                         int32_t* __restrict__ offsets, int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    extern __shared__ int plan_lds[];
    int* start = plan_lds + kChunkWaves * experts;  // [expert + 1]
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) start[e] = totals[e];
    __syncthreads();
    scan_experts(start, experts);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
    const int chunk = blockIdx.x * kChunkWaves + wave;
    const long long first = static_cast<long long>(chunk) * kChunk;
    if (first >= entries) return;
    const int end = static_cast<int>(first + kChunk < entries ? first + kChunk : entries);
    int* next = plan_lds + wave * experts;  // this wavefront's own: no barrier needed
    for (int e = lane; e < experts; e += kWave) next[e] = start[e] + counts[static_cast<long long>(chunk) * experts + e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = static_cast<int>(first) + lane; i < end; i += kWave)
        if (i >= start[experts]) rows[i] = -1;
    place_chunk(chosen, static_cast<int>(first), end, experts, bits, next, rows, slots);
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
    if (tokens * k > 0x7fffffffll - 4096) return fail(1, "%s: %lld tokens x %d: beyond 31 bits", who, tokens, k);
    return 0;
}

}  // namespace

size_t expert_plan_workspace_bytes(long long tokens, int k, int experts) {
    const long long entries = tokens * k;
    if (tokens < 0 || k < 1 || experts < 1 || one_workgroup(entries, experts)) return 16;
    return static_cast<size_t>((entries > 0 ? ceil_div(entries, static_cast<long long>(kChunk)) : 1) + 1) * experts * sizeof(int);
}

int launch_expert_plan(const int32_t* chosen, long long tokens, int k, int experts, int32_t* offsets, int32_t* rows, int32_t* slots, void* ws,
                       size_t ws_bytes, hipStream_t s) {
    const char* who = "prism_expert_plan";
    if (tokens < 0) return fail(1, "%s: negative number of tokens", who);
    if (experts < 1 || experts > kMaxExperts) return fail(1, "%s: %d experts, 1 to %d are supported", who, experts, kMaxExperts);
    if (k < 1) return fail(1, "%s: k=%d, at least 1 expert per token is needed", who, k);
    if (tokens > 0x7fffffffll || tokens * k > 0x7fffffffll - 4096) return fail(1, "%s: %lld tokens x %d: beyond 31 bits", who, tokens, k);
    const int entries = static_cast<int>(tokens * k);
    if (offsets == nullptr || !aligned4(offsets)) return fail(1, "%s: offsets must be a 4-byte aligned device pointer", who);
    if (entries > 0 && (chosen == nullptr || rows == nullptr || slots == nullptr || !aligned4(chosen) || !aligned4(rows) || !aligned4(slots)))
        return fail(1, "%s: experts, rows and slots must be 4-byte aligned device pointers", who);
    const int bits = bits_of(experts);
    if (one_workgroup(entries, experts)) {
        const size_t lds = (static_cast<size_t>(kSmallWaves + 1) * experts + 1) * sizeof(int);
        plan_small_kernel<<<dim3(1), dim3(kSmallWaves * kWave), lds, s>>>(chosen, entries, experts, bits, offsets, rows, slots);
        return check_launch("plan_small_kernel");
    }
    if (ws == nullptr || !aligned4(ws) || ws_bytes < expert_plan_workspace_bytes(tokens, k, experts))
        return fail(1, "%s: workspace of %zu bytes, %zu needed", who, ws == nullptr ? size_t{0} : ws_bytes, expert_plan_workspace_bytes(tokens, k, experts));
    const int chunks = entries > 0 ? ceil_div(entries, kChunk) : 1;
    int* counts = static_cast<int*>(ws);
    int* totals = counts + static_cast<size_t>(chunks) * experts;
    const dim3 grid(static_cast<unsigned>(ceil_div(chunks, kChunkWaves)));
    const size_t lds = static_cast<size_t>(kChunkWaves) * experts * sizeof(int);
    plan_count_kernel<<<grid, dim3(kChunkWaves * kWave), lds, s>>>(chosen, entries, experts, counts);
    if (int rc = check_launch("plan_count_kernel")) return rc;
    plan_sum_kernel<<<dim3(static_cast<unsigned>(ceil_div(experts, 16))), dim3(1024), 0, s>>>(counts, chunks, experts, totals);
    if (int rc = check_launch("plan_sum_kernel")) return rc;
    plan_place_kernel<<<grid, dim3(kChunkWaves * kWave), lds + (static_cast<size_t>(experts) + 1) * sizeof(int), s>>>(chosen, entries, experts, bits, counts, totals,
                                                                                                                     offsets, rows, slots);
    return check_launch("plan_place_kernel");
}

int launch_route_topk(int type, const void* logits, long long ld, long long tokens, int experts, int k, int renormalise, float* weights, int32_t* chosen,
                      hipStream_t s) {
    const char* who = "prism_route_topk";
    if (type != kTypeF32 && type != kTypeBf16) return fail(1, "%s: unknown logit type %d", who, type);
    if (int rc = check_route(who, tokens, experts, k)) return rc;
    if (tokens == 0) return 0;
    if (logits == nullptr || weights == nullptr || chosen == nullptr) return fail(1, "%s: null pointer", who);
    if (reinterpret_cast<uintptr_t>(logits) % (type == kTypeF32 ? 4 : 2) != 0 || !aligned4(weights) || !aligned4(chosen)) return fail(1, "%s: misaligned pointer", who);
    if (tokens > 1 && ld < experts) return fail(1, "%s: a row stride (%lld) is shorter than its row (%d)", who, ld, experts);
    auto go = [&](auto t, auto lanes, auto values) {
        using T = decltype(t);
        constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
        const unsigned blocks = static_cast<unsigned>(ceil_div(tokens, static_cast<long long>(kRouteBlock / L)));
        route_topk_kernel<T, L, V><<<dim3(blocks), dim3(kRouteBlock), 0, s>>>(static_cast<const T*>(logits), ld, static_cast<int>(tokens), experts, k, renormalise,
                                                                             weights, chosen);
        return check_launch("route_topk_kernel");
    };
    auto sized = [&](auto t) {
        using std::integral_constant;
        if (experts <= 64) return go(t, integral_constant<int, 16>{}, integral_constant<int, 4>{});
        if (experts <= 128) return go(t, integral_constant<int, 16>{}, integral_constant<int, 8>{});
        if (experts <= 256) return go(t, integral_constant<int, 16>{}, integral_constant<int, 16>{});
        if (experts <= 512) return go(t, integral_constant<int, 64>{}, integral_constant<int, 8>{});
        return go(t, integral_constant<int, 64>{}, integral_constant<int, 16>{});
    };
    return type == kTypeF32 ? sized(float{}) : sized(uint16_t{});
}

int launch_route_backward(int type, const float* grad, const void* logits, long long ld, const float* weights, const int32_t* chosen, long long tokens,
                          int experts, int k, int renormalise, void* out, long long ldo, hipStream_t s) {
    const char* who = "prism_route_topk_backward";
    if (type != kTypeF32 && type != kTypeBf16) return fail(1, "%s: unknown logit type %d", who, type);
    if (int rc = check_route(who, tokens, experts, k)) return rc;
    if (tokens == 0) return 0;
    if (grad == nullptr || logits == nullptr || weights == nullptr || chosen == nullptr || out == nullptr) return fail(1, "%s: null pointer", who);
    const unsigned size = type == kTypeF32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size != 0 || reinterpret_cast<uintptr_t>(out) % size != 0 || !aligned4(weights) || !aligned4(chosen) || !aligned4(grad))
        return fail(1, "%s: misaligned pointer", who);
    if (tokens > 1 && (ld < experts || ldo < experts)) return fail(1, "%s: a row stride is shorter than its row (%d)", who, experts);
    const uintptr_t a = reinterpret_cast<uintptr_t>(logits), b = reinterpret_cast<uintptr_t>(out);
    if (a < b + ((tokens - 1) * ldo + experts) * size && b < a + ((tokens - 1) * ld + experts) * size) return fail(1, "%s: the result overlaps the logits", who);
    const dim3 grid(static_cast<unsigned>(ceil_div(tokens, static_cast<long long>(kRouteBlock / 16))));
    if (type == kTypeF32)
        route_backward_kernel<float><<<grid, dim3(kRouteBlock), 0, s>>>(grad, static_cast<const float*>(logits), ld, weights, chosen, static_cast<int>(tokens), experts, k,
                                                                        renormalise, static_cast<float*>(out), ldo);
    else
        route_backward_kernel<uint16_t><<<grid, dim3(kRouteBlock), 0, s>>>(grad, static_cast<const uint16_t*>(logits), ld, weights, chosen, static_cast<int>(tokens), experts,
                                                                           k, renormalise, static_cast<uint16_t*>(out), ldo);
    return check_launch("route_backward_kernel");
}

}  // namespace prism
