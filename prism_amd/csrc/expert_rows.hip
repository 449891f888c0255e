// The row moves on both sides of the experts' products. A token's j-th chosen expert holds the token's row in slot
// slots[t][j] (-1: nowhere); rows[s] = t k + j is the inverse (-1: the slot is not used).
//   gather            xs[s] = x[rows[s] / k]
//   weighted sum      out[t] = sum_j w[t][j] y[slots[t][j]]       (w absent: 1, the gather's backward)
//   its backward      dy[slots[t][j]] = w[t][j] dout[t],   dw[t][j] = <dout[t], y[slots[t][j]]>
// Unused slots are left as they are, a token without experts gets zeros. Sums run over j (and, in the dot products,
// over the row) in 32 bits and in a fixed order: the same bits on every run.
//
// HBM-bound: every row is read once and written once. 8192 tokens x 8 x 4096 bf16, a random choice of 64 experts: sum 117 us
// (604 MB, 5.2 TB/s), its backward 218 us (1.14 GB, 5.2 TB/s), gather 142 us (604 MB, 4.3 TB/s). What the L2s move for the last two is
// more: a token's row is wanted by wavefronts of up to eight XCDs and fetched by each of their L2s, 496 MB of reads for 67 MB
// of rows in the gather (7.2 TB/s with its writes), 810 MB in the backward (6.1 TB/s).
#include <initializer_list>
#include <type_traits>

#include "common.h"

namespace prism {
namespace {

constexpr int kRowsBlock = 256, kRowsWaves = kRowsBlock / kWave;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ void from_float(float& to, float v) { to = v; }
__device__ __forceinline__ void from_float(uint16_t& to, float v) { to = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }  // nearest even

// A lane's packet: 16 B of consecutive elements of a row, at any element (16 B accesses need no more alignment than that;
// as packets of 4 B, rows of 4100 B ran at half the bandwidth), the last of a row cut to what is there. ONCE: non-temporal,
// for rows that no other wavefront touches: stores always (8192 tokens x 8 x 4096 bf16, gather: 172 -> 139 us), loads where
// there is more of them than the memory-side cache holds (backward of the sum: 231 -> 219 us; 32 MB of them: 8.1 -> 12.5).
template <typename T>
struct Packet {
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    typedef T Vector __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    T v[N];
    template <bool ONCE>
    static __device__ __forceinline__ Packet load(const T* p, int there) {
        Packet r;
        if (there >= N) {
            const Vector* at = reinterpret_cast<const Vector*>(p);
            const Vector raw = ONCE ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
            for (int i = 0; i < N; ++i) r.v[i] = raw[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) r.v[i] = i < there ? p[i] : T{};
        }
        return r;
    }
    template <bool ONCE>
    __device__ __forceinline__ void store(T* p, int there) const {
        if (there >= N) {
            Vector raw;
#pragma unroll
            for (int i = 0; i < N; ++i) raw[i] = v[i];
            if constexpr (ONCE) __builtin_nontemporal_store(raw, reinterpret_cast<Vector*>(p));
            else *reinterpret_cast<Vector*>(p) = raw;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < there) p[i] = v[i];
        }
    }
};

// One wavefront per 64 packets of a slot's row.
template <typename T>
__global__ __launch_bounds__(kRowsBlock) void expert_gather_kernel(const T* __restrict__ x, long long ldx, int tokens, int k,
                                                                   const int32_t* __restrict__ rows, T* __restrict__ out, long long ldo,
                                                                   int n_slots, int width, int parts) {
    using P = Packet<T>;
    const long long unit = static_cast<long long>(blockIdx.x) * kRowsWaves + threadIdx.x / kWave;
    const int slot = static_cast<int>(unit / parts);
    const int at = (static_cast<int>(unit % parts) * kWave + threadIdx.x % kWave) * P::N;
    if (slot >= n_slots || at >= width) return;
    const int row = rows[slot], token = row / k;
    if (row < 0 || token >= tokens) return;
    P::template load<false>(x + token * ldx + at, width - at).template store<true>(out + slot * ldo + at, width - at);
}

// One wavefront per 64 packets of a token's row; U rows in flight.
template <typename T, bool WEIGHTED, bool STREAM>
__global__ __launch_bounds__(kRowsBlock) void expert_sum_kernel(const T* __restrict__ y, long long ldy, int n_slots,
                                                                const float* __restrict__ weights, const int32_t* __restrict__ slots, int k,
                                                                T* __restrict__ out, long long ldo, int tokens, int width, int parts) {
    using P = Packet<T>;
    constexpr int U = 4;
    const long long unit = static_cast<long long>(blockIdx.x) * kRowsWaves + threadIdx.x / kWave;
    const int token = static_cast<int>(unit / parts);
    const int at = (static_cast<int>(unit % parts) * kWave + threadIdx.x % kWave) * P::N;
    if (token >= tokens || at >= width) return;
    float sum[P::N] = {};
    for (int j0 = 0; j0 < k; j0 += U) {
        P v[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u;
            const int slot = j < k ? slots[static_cast<long long>(token) * k + j] : -1;
            const bool there = slot >= 0 && slot < n_slots;
            w[u] = there ? (WEIGHTED ? weights[static_cast<long long>(token) * k + j] : 1.0f) : 0.0f;
            v[u] = P::template load<STREAM>(y + (there ? slot * ldy + at : 0), there ? width - at : 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < P::N; ++i) sum[i] = __builtin_fmaf(w[u], as_float(v[u].v[i]), sum[i]);
    }
    P r;
#pragma unroll
    for (int i = 0; i < P::N; ++i) from_float(r.v[i], sum[i]);
    r.template store<false>(out + token * ldo + at, width - at);
}

// One wavefront per (token, j), or two (STREAM): its slot's row of dy, and the dot product of its row of y. The wavefronts of
// a token follow each other: dout's row is in the caches for all but the first. Where the rows come from and go to memory in
// an order of no locality, two wavefronts a row keep half as many rows under way: 8192 tokens x 8 x 4096 bf16 235 -> 219 us
// (5.2 TB/s; slots in the tokens' order: 188), x 2048 119 -> 112, 16384 x 2 x 7168 230 -> 233; where the caches hold a good part,
// one is better (2048 x 4 x 4096: 24.6 against 26.3 us, 600 x 8 x 4096 fp32: 30 against 36).
template <typename T, bool STREAM>
__global__ __launch_bounds__(kRowsBlock) void expert_sum_backward_kernel(const T* __restrict__ dout, long long ldd, const T* __restrict__ y,
                                                                         long long ldy, const float* __restrict__ weights,
                                                                         const int32_t* __restrict__ slots, int n_slots, T* __restrict__ dy,
                                                                         long long lddy, float* __restrict__ dw, long long entries, int k, int width) {
    using P = Packet<T>;
    constexpr int SHARE = STREAM ? 2 : 1;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, part = wave % SHARE;
    const long long entry = static_cast<long long>(blockIdx.x) * (kRowsWaves / SHARE) + wave / SHARE;
    const int slot = entry < entries ? slots[entry] : -1;
    float dot = 0.0f;
    if (slot >= 0 && slot < n_slots) {
        const float w = weights[entry];
        const T* up = dout + entry / k * ldd;
#pragma unroll 2
        for (int at = (part * kWave + lane) * P::N; at < width; at += SHARE * kWave * P::N) {
            const P a = P::template load<false>(up + at, width - at), b = P::template load<STREAM>(y + slot * ldy + at, width - at);
            P r;
#pragma unroll
            for (int i = 0; i < P::N; ++i) {
                dot = __builtin_fmaf(as_float(a.v[i]), as_float(b.v[i]), dot);
                from_float(r.v[i], w * as_float(a.v[i]));
            }
            r.template store<true>(dy + slot * lddy + at, width - at);
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d /= 2) dot += __shfl_xor(dot, d);
    if constexpr (SHARE == 2) {
        __shared__ float behind[kRowsWaves];
        if (lane == 0) behind[wave] = dot;
        __syncthreads();
        dot += behind[wave | 1];  // of the first wavefront; the second one's is not used
    }
    if (lane == 0 && part == 0 && entry < entries) dw[entry] = dot;
}

// More than the 256 MiB memory-side cache would keep of the rows.
bool streams(long long rows, long long width, int size) { return rows * width * size > (192ll << 20); }

template <typename F>
int with_type(int type, F&& f) { return type == kTypeF32 ? f(float{}) : f(uint16_t{}); }

int check_rows(const char* who, int type, long long tokens, int k, long long n_slots, long long width, std::initializer_list<const void*> bases,
               std::initializer_list<long long> strides) {
    if (type != kTypeF32 && type != kTypeBf16) return fail(1, "%s: unknown element type %d", who, type);
    if (tokens < 0 || n_slots < 0 || width < 0) return fail(1, "%s: negative dimension (%lld tokens, %lld slots, width %lld)", who, tokens, n_slots, width);
    if (k < 1) return fail(1, "%s: k=%d, at least 1 expert per token is needed", who, k);
    if (tokens > 0x7fffffffll || n_slots > 0x7fffffffll || width > 0x3fffffffll || tokens * k > 0x7fffffffll)
        return fail(1, "%s: %lld tokens x %d, %lld slots, width %lld: beyond 31 bits", who, tokens, k, n_slots, width);
    if (tokens == 0 || n_slots == 0 || width == 0) return 0;
    for (long long s : strides)
        if (s < width) return fail(1, "%s: a row stride (%lld) is shorter than its row (%lld)", who, s, width);
    for (const void* b : bases) {
        if (b == nullptr) return fail(1, "%s: null pointer", who);
        if (reinterpret_cast<uintptr_t>(b) % (type == kTypeF32 ? 4 : 2) != 0) return fail(1, "%s: misaligned pointer", who);
    }
    return 0;
}

}  // namespace

int launch_expert_gather(int type, const void* x, long long ldx, long long tokens, int k, const int32_t* rows, void* out, long long ldo,
                         long long n_slots, long long width, hipStream_t s) {
    const char* who = "prism_expert_gather";
    if (int rc = check_rows(who, type, tokens, k, n_slots, width, {x, out}, {ldx, ldo})) return rc;
    if (tokens == 0 || n_slots == 0 || width == 0) return 0;
    if (rows == nullptr || !aligned4(rows)) return fail(1, "%s: rows must be a 4-byte aligned device pointer", who);
    const int size = type == kTypeF32 ? 4 : 2;
    if (outputs_overlap({matrix_span(out, n_slots, width, ldo, size)}, {matrix_span(x, tokens, width, ldx, size), entries_span(rows, n_slots)}))
        return fail(1, "%s: the result overlaps an input", who);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int parts = static_cast<int>(ceil_div(width, static_cast<long long>(kWave * Packet<T>::N)));
        const long long blocks = ceil_div(n_slots * parts, static_cast<long long>(kRowsWaves));
        if (!launchable(blocks, kRowsBlock)) return fail(1, "%s: too much work for one launch", who);
        expert_gather_kernel<T><<<dim3(static_cast<unsigned>(blocks)), dim3(kRowsBlock), 0, s>>>(
            static_cast<const T*>(x), ldx, static_cast<int>(tokens), k, rows, static_cast<T*>(out), ldo, static_cast<int>(n_slots), static_cast<int>(width), parts);
        return check_launch("expert_gather_kernel");
    });
}

int launch_expert_sum(int type, const void* y, long long ldy, long long n_slots, const float* weights, const int32_t* slots, long long tokens, int k,
                      void* out, long long ldo, long long width, hipStream_t s) {
    const char* who = "prism_expert_combine";
    if (int rc = check_rows(who, type, tokens, k, n_slots, width, {y, out}, {ldy, ldo})) return rc;
    if (tokens == 0 || width == 0) return 0;
    if (slots == nullptr || !aligned4(slots) || !aligned4(weights)) return fail(1, "%s: slots and weights must be 4-byte aligned device pointers", who);
    const int size = type == kTypeF32 ? 4 : 2;
    // Written also where there are no slots, which check_rows takes for an empty call.
    if (out == nullptr || ldo < width) return fail(1, "%s: null result or a row stride shorter than its row", who);
    if (reinterpret_cast<uintptr_t>(out) % size != 0) return fail(1, "%s: misaligned pointer", who);
    if (outputs_overlap({matrix_span(out, tokens, width, ldo, size)},
                        {matrix_span(y, n_slots, width, ldy, size), entries_span(weights, tokens * k), entries_span(slots, tokens * k)}))
        return fail(1, "%s: the result overlaps an input", who);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int parts = static_cast<int>(ceil_div(width, static_cast<long long>(kWave * Packet<T>::N)));
        const long long blocks = ceil_div(tokens * parts, static_cast<long long>(kRowsWaves));
        if (!launchable(blocks, kRowsBlock)) return fail(1, "%s: too much work for one launch", who);
        auto go = [&](auto weighted, auto stream) {
            expert_sum_kernel<T, weighted, stream><<<dim3(static_cast<unsigned>(blocks)), dim3(kRowsBlock), 0, s>>>(
                static_cast<const T*>(y), ldy, static_cast<int>(n_slots), weights, slots, k, static_cast<T*>(out), ldo, static_cast<int>(tokens),
                static_cast<int>(width), parts);
        };
        const bool stream = streams(n_slots, width, size);
        if (weights != nullptr) stream ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
        else stream ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
        return check_launch("expert_sum_kernel");
    });
}

int launch_expert_sum_backward(int type, const void* dout, long long ldd, const void* y, long long ldy, const float* weights, const int32_t* slots,
                               long long tokens, int k, void* dy, long long lddy, float* dw, long long n_slots, long long width, hipStream_t s) {
    const char* who = "prism_expert_combine_backward";
    if (int rc = check_rows(who, type, tokens, k, n_slots, width, {dout, y, dy}, {ldd, ldy, lddy})) return rc;
    if (tokens == 0) return 0;
    if (slots == nullptr || weights == nullptr || dw == nullptr || !aligned4(slots) || !aligned4(weights) || !aligned4(dw))
        return fail(1, "%s: slots, weights and their gradient must be 4-byte aligned device pointers", who);
    const int size = type == kTypeF32 ? 4 : 2;
    const long long entries = tokens * k;
    if (outputs_overlap({matrix_span(dy, n_slots, width, lddy, size), entries_span(dw, entries)},
                        {matrix_span(dout, tokens, width, ldd, size), matrix_span(y, n_slots, width, ldy, size), entries_span(weights, entries),
                         entries_span(slots, entries)}))
        return fail(1, "%s: a result overlaps an input or the other result", who);
    const bool stream = streams(n_slots, width, size);
    const long long blocks = ceil_div(entries, static_cast<long long>(stream ? kRowsWaves / 2 : kRowsWaves));
    if (!launchable(blocks, kRowsBlock)) return fail(1, "%s: too much work for one launch", who);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto streaming) {
            expert_sum_backward_kernel<T, streaming><<<dim3(static_cast<unsigned>(blocks)), dim3(kRowsBlock), 0, s>>>(
                static_cast<const T*>(dout), ldd, static_cast<const T*>(y), ldy, weights, slots, static_cast<int>(n_slots), static_cast<T*>(dy), lddy, dw, entries, k,
                static_cast<int>(width));
        };
        stream ? go(std::true_type{}) : go(std::false_type{});
        return check_launch("expert_sum_backward_kernel");
    });
}

}  // namespace prism
