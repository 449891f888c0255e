// The row moves on both sides of the experts' products. A token's j-th chosen expert holds the token's row in slot
// slots[t][j] (-1: nowhere); rows[s] = t k + j is the inverse (-1: the slot is not used).
//   gather            xs[s] = x[rows[s] / k]
//   weighted sum      out[t] = sum_j w[t][j] y[slots[t][j]]       (w absent: 1, the gather's backward)
//   its backward      dy[slots[t][j]] = w[t][j] dout[t],   dw[t][j] = <dout[t], y[slots[t][j]]>
// Unused slots are left as they are, a token without experts gets zeros. Sums run over j (and, in the dot products,
// over the row) in 32 bits and in a fixed order: the same bits on every run.
//
// HBM-bound: every row is read once and written once.
#include <initializer_list>
#include <type_traits>

#include "common.h"

namespace prism {
namespace {

constexpr int kRowsBlock = 256, kRowsWaves = kRowsBlock / kWave;

// A lane's packet: BYTES of consecutive elements, as fp32 values and back.
template <typename T, int BYTES>
struct Packet {
    static constexpr int N = BYTES / static_cast<int>(sizeof(T));
    T raw[N];
    static __device__ __forceinline__ Packet load(const T* p) {
        Packet r;
        __builtin_memcpy(r.raw, __builtin_assume_aligned(p, BYTES), BYTES);
        return r;
    }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(__builtin_assume_aligned(p, BYTES), raw, BYTES); }
};
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ void from_float(float& to, float v) { to = v; }
__device__ __forceinline__ void from_float(uint16_t& to, float v) { to = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }  // nearest even

// One wavefront per 64 packets of a slot's row.
template <typename T, int BYTES>
__global__ __launch_bounds__(kRowsBlock) void expert_gather_kernel(const T* __restrict__ x, long long ldx, int tokens, int k,
                                                                   const int32_t* __restrict__ rows, T* __restrict__ out, long long ldo,
                                                                   int n_slots, int width, int parts) {
    using P = Packet<T, BYTES>;
    const long long unit = static_cast<long long>(blockIdx.x) * kRowsWaves + threadIdx.x / kWave;
    const int slot = static_cast<int>(unit / parts);
    const int at = (static_cast<int>(unit % parts) * kWave + threadIdx.x % kWave) * P::N;
    if (slot >= n_slots || at >= width) return;
    const int row = rows[slot], token = row / k;
    if (row < 0 || token >= tokens) return;
    P::load(x + token * ldx + at).store(out + slot * ldo + at);
}

// One wavefront per 64 packets of a token's row; U rows in flight.
template <typename T, int BYTES, bool WEIGHTED>
__global__ __launch_bounds__(kRowsBlock) void expert_sum_kernel(const T* __restrict__ y, long long ldy, int n_slots,
                                                                const float* __restrict__ weights, const int32_t* __restrict__ slots, int k,
                                                                T* __restrict__ out, long long ldo, int tokens, int width, int parts) {
    using P = Packet<T, BYTES>;
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
            if (there) v[u] = P::load(y + slot * ldy + at);
            else
#pragma unroll
                for (int i = 0; i < P::N; ++i) v[u].raw[i] = T{};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < P::N; ++i) sum[i] = __builtin_fmaf(w[u], as_float(v[u].raw[i]), sum[i]);
    }
    P r;
#pragma unroll
    for (int i = 0; i < P::N; ++i) from_float(r.raw[i], sum[i]);
    r.store(out + token * ldo + at);
}

// One wavefront per (token, j): its slot's row of dy, and the dot product of its row of y.
template <typename T, int BYTES>
__global__ __launch_bounds__(kRowsBlock) void expert_sum_backward_kernel(const T* __restrict__ dout, long long ldd, const T* __restrict__ y,
                                                                         long long ldy, const float* __restrict__ weights,
                                                                         const int32_t* __restrict__ slots, int n_slots, T* __restrict__ dy,
                                                                         long long lddy, float* __restrict__ dw, long long entries, int k, int width) {
    using P = Packet<T, BYTES>;
    const int lane = threadIdx.x % kWave;
    const long long entry = static_cast<long long>(blockIdx.x) * kRowsWaves + threadIdx.x / kWave;
    if (entry >= entries) return;
    const int slot = slots[entry];
    float dot = 0.0f;
    if (slot >= 0 && slot < n_slots) {
        const float w = weights[entry];
        const T* up = dout + entry / k * ldd;
        for (int at = lane * P::N; at < width; at += kWave * P::N) {
            const P a = P::load(up + at), b = P::load(y + slot * ldy + at);
            P r;
#pragma unroll
            for (int i = 0; i < P::N; ++i) {
                dot = __builtin_fmaf(as_float(a.raw[i]), as_float(b.raw[i]), dot);
                from_float(r.raw[i], w * as_float(a.raw[i]));
            }
            r.store(dy + slot * lddy + at);
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d /= 2) dot += __shfl_xor(dot, d);
    if (lane == 0) dw[entry] = dot;
}

// The widest packet that every row start, and the row length, is a multiple of.
int packet_bytes(int size, long long width, std::initializer_list<const void*> bases, std::initializer_list<long long> strides) {
    uintptr_t all = static_cast<uintptr_t>(width) * size;
    for (const void* b : bases) all |= reinterpret_cast<uintptr_t>(b);
    for (long long s : strides) all |= static_cast<uintptr_t>(s) * size;
    for (int bytes = 16; bytes > size; bytes /= 2)
        if (all % bytes == 0) return bytes;
    return size;
}

template <typename F>
int with_packet(int type, int bytes, F&& f) {
    if (type == kTypeF32) {
        if (bytes == 16) return f(float{}, std::integral_constant<int, 16>{});
        if (bytes == 8) return f(float{}, std::integral_constant<int, 8>{});
        return f(float{}, std::integral_constant<int, 4>{});
    }
    if (bytes == 16) return f(uint16_t{}, std::integral_constant<int, 16>{});
    if (bytes == 8) return f(uint16_t{}, std::integral_constant<int, 8>{});
    if (bytes == 4) return f(uint16_t{}, std::integral_constant<int, 4>{});
    return f(uint16_t{}, std::integral_constant<int, 2>{});
}

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
bool rows_overlap(const void* a, long long a_rows, long long lda, const void* b, long long b_rows, long long ldb, long long width, int size) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const uintptr_t xs = static_cast<uintptr_t>((a_rows - 1) * lda + width) * size, ys = static_cast<uintptr_t>((b_rows - 1) * ldb + width) * size;
    return a_rows > 0 && b_rows > 0 && width > 0 && x < y + ys && y < x + xs;
}

}  // namespace

int launch_expert_gather(int type, const void* x, long long ldx, long long tokens, int k, const int32_t* rows, void* out, long long ldo,
                         long long n_slots, long long width, hipStream_t s) {
    const char* who = "prism_expert_gather";
    if (int rc = check_rows(who, type, tokens, k, n_slots, width, {x, out}, {ldx, ldo})) return rc;
    if (tokens == 0 || n_slots == 0 || width == 0) return 0;
    if (rows == nullptr || !aligned4(rows)) return fail(1, "%s: rows must be a 4-byte aligned device pointer", who);
    const int size = type == kTypeF32 ? 4 : 2;
    if (rows_overlap(x, tokens, ldx, out, n_slots, ldo, width, size)) return fail(1, "%s: x and the result overlap", who);
    return with_packet(type, packet_bytes(size, width, {x, out}, {ldx, ldo}), [&](auto t, auto bytes) {
        using T = decltype(t);
        const int parts = static_cast<int>(ceil_div(width, static_cast<long long>(kWave * Packet<T, bytes>::N)));
        const long long blocks = ceil_div(n_slots * parts, static_cast<long long>(kRowsWaves));
        if (blocks > 0x7fffffffll) return fail(1, "%s: too much work for one launch", who);
        expert_gather_kernel<T, bytes><<<dim3(static_cast<unsigned>(blocks)), dim3(kRowsBlock), 0, s>>>(
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
    if (out == nullptr || ldo < width) return fail(1, "%s: null result or a row stride shorter than its row", who);
    const int size = type == kTypeF32 ? 4 : 2;
    if (rows_overlap(y, n_slots, ldy, out, tokens, ldo, width, size)) return fail(1, "%s: y and the result overlap", who);
    return with_packet(type, packet_bytes(size, width, {y, out}, {ldy, ldo}), [&](auto t, auto bytes) {
        using T = decltype(t);
        const int parts = static_cast<int>(ceil_div(width, static_cast<long long>(kWave * Packet<T, bytes>::N)));
        const long long blocks = ceil_div(tokens * parts, static_cast<long long>(kRowsWaves));
        if (blocks > 0x7fffffffll) return fail(1, "%s: too much work for one launch", who);
        auto go = [&](auto weighted) {
            expert_sum_kernel<T, bytes, weighted><<<dim3(static_cast<unsigned>(blocks)), dim3(kRowsBlock), 0, s>>>(
                static_cast<const T*>(y), ldy, static_cast<int>(n_slots), weights, slots, k, static_cast<T*>(out), ldo, static_cast<int>(tokens),
                static_cast<int>(width), parts);
        };
        if (weights != nullptr) go(std::true_type{});
        else go(std::false_type{});
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
    if (rows_overlap(y, n_slots, ldy, dy, n_slots, lddy, width, size) || rows_overlap(dout, tokens, ldd, dy, n_slots, lddy, width, size))
        return fail(1, "%s: the gradient of y overlaps an input", who);
    const long long entries = tokens * k;
    return with_packet(type, packet_bytes(size, width, {dout, y, dy}, {ldd, ldy, lddy}), [&](auto t, auto bytes) {
        using T = decltype(t);
        expert_sum_backward_kernel<T, bytes><<<dim3(static_cast<unsigned>(ceil_div(entries, static_cast<long long>(kRowsWaves)))), dim3(kRowsBlock), 0, s>>>(
            static_cast<const T*>(dout), ldd, static_cast<const T*>(y), ldy, weights, slots, static_cast<int>(n_slots), static_cast<T*>(dy), lddy, dw, entries, k,
            static_cast<int>(width));
        return check_launch("expert_sum_backward_kernel");
    });
}

}  // namespace prism
