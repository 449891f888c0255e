// Shared host-side helpers for libprism_amd.so (gfx950 only).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

namespace prism {

constexpr int kWave = 64;  // CDNA wavefront width; every kernel here assumes it

// Thread-local error text behind prism_last_error_string().
char* error_buffer();
constexpr size_t kErrorBufferLen = 512;

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_buffer(), kErrorBufferLen, fmt, ap);
    va_end(ap);
    return code;
}

inline int hip_fail(hipError_t e, const char* what) {
    return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
}

// Launch check: hipGetLastError() clears and returns the launch error, if any.
inline int check_launch(const char* kernel) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, kernel);
    return 0;
}

// A launch has fewer than 2^32 threads along x.
inline bool launchable(long long blocks, int threads) { return blocks <= 0xffffffffll / threads; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

template <typename T>
constexpr T ceil_div(T a, T b) { return (a + b - 1) / b; }

// Memory that a call reads or writes, and whether any of its outputs shares some with an input or another output.
struct Span {
    const void* at;
    uintptr_t bytes;
};
// A row-major matrix, from its first element to its last.
inline Span matrix_span(const void* at, long long rows, long long cols, long long ld, int size) {
    return {at, rows <= 0 || cols <= 0 ? 0 : static_cast<uintptr_t>((rows - 1) * ld + cols) * size};
}
// An array of 4-byte entries.
inline Span entries_span(const void* at, long long entries) { return {at, static_cast<uintptr_t>(entries) * 4}; }
inline bool overlap(const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.at != nullptr && b.at != nullptr && a.bytes != 0 && b.bytes != 0 && x < y + b.bytes && y < x + a.bytes;
}
inline bool outputs_overlap(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
    for (const Span* o = outputs.begin(); o != outputs.end(); ++o) {
        for (const Span& i : inputs)
            if (overlap(*o, i)) return true;
        for (const Span* p = outputs.begin(); p != o; ++p)
            if (overlap(*o, *p)) return true;
    }
    return false;
}

// Compute units of the current device (the launchers size their tile choices by it).
inline int cu_count() {
    static int cached[64] = {};  // per device; a racing first call writes the same value
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (cached[dev] == 0) {
        int cus = 0;
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
        cached[dev] = cus;
    }
    return cached[dev];
}

// Internal launchers, one per kernel family (defined in the .hip files).
int launch_add_m(const int32_t* x, int32_t* y, int32_t m, size_t n, hipStream_t s);
// Scan flags and error code: the values of PRISM_SCAN_* / PRISM_ERROR_SCAN_ORDER in include/prism_amd.h.
constexpr unsigned kFlagExclusive = 1u, kFlagTicket = 2u, kFlagNoHelp = 4u;
constexpr unsigned kFlagOpMask = 0x30u, kFlagOpSum = 0x00u, kFlagOpMax = 0x10u, kFlagOpMin = 0x20u;
constexpr int kScanOrderError = 10001, kScanWorkspaceError = 10002;
size_t scan_workspace_bytes(size_t n);
int scan_workspace_init(void* ws, size_t ws_bytes, hipStream_t s);
// spin_limit < 0: the library's bound on the polls of a look-back window; 0: a look-back never waits.
int launch_scan(const uint32_t* in, uint32_t* out, size_t n, void* ws, size_t ws_bytes, unsigned flags,
                long long spin_limit, hipStream_t s);
int scan_status(void* ws, size_t ws_bytes, hipStream_t s);
// flags: kFlagNoHelp or 0; spin_limit as for launch_scan.
int launch_segmented_scan(const uint32_t* in, const uint8_t* heads, uint32_t* out, size_t n, void* ws, size_t ws_bytes,
                          unsigned flags, long long spin_limit, hipStream_t s);
int launch_scan64(const unsigned long long* in, unsigned long long* out, size_t n, void* ws, size_t ws_bytes, unsigned flags,
                  long long spin_limit, hipStream_t s);
int launch_scan_static(const uint32_t* in, uint32_t* out, size_t n, hipStream_t s);
int launch_wave_regroup(const int32_t* in, int32_t* out, size_t n, int items_per_lane, int direction, hipStream_t s);
int launch_sgemm(int variant, int M, int N, int K, float alpha, const float* A, const float* B,
                 float beta, float* C, hipStream_t s);
// 0 if the arguments are ones launch_sgemm accepts, else the error (and the error string is set).
int check_sgemm_arguments(int variant, int M, int N, int K, const float* A, const float* B, const float* C);
size_t sgemm_workspace_bytes(int M, int N, int K);
// What launch_sgemm_ws does for this shape with 16 B-aligned operands and ws_bytes of workspace: the number of
// workgroups that share K ranges and of the tiles they share (both 0: the call is launch_sgemm).
int sgemm_ws_plan(int M, int N, int K, size_t ws_bytes, int* groups, int* sk_tiles);
int launch_sgemm_ws(int variant, int M, int N, int K, float alpha, const float* A, const float* B, float beta,
                    float* C, void* ws, size_t ws_bytes, hipStream_t s);
int launch_gemm_bf16(int M, int N, int K, const uint16_t* A, const uint16_t* B, float* D_f32,
                     uint16_t* C_bf16_colmajor, hipStream_t s);

// Element types of the expert-layer operators: the values of PRISM_TYPE_* in include/prism_amd.h.
constexpr int kTypeF32 = 0, kTypeBf16 = 1;
// The grouped products; (first, second, out) are (A, B, D), (dD, B, dA) or (dD, A, dB), group_stride the elements
// between the matrices of B or dB.
enum class GroupedForm { kForward, kGradA, kGradB };
int launch_gemm_grouped(GroupedForm form, int groups, long long rows, int N, int K, const uint16_t* first, long long ld_first,
                        const uint16_t* second, long long ld_second, long long group_stride, const int32_t* offsets, void* out,
                        long long ld_out, int out_type, hipStream_t s);
// Which kernel a product of contiguous operands takes: the rows of its tiles and the stages of its ring.
int gemm_grouped_plan(int form, int groups, long long rows, int N, int K, int out_type, int* tile_rows, int* stages);
int launch_gemv_w4(int groups, long long rows, int N, int K, const uint16_t* x, long long ldx, const uint8_t* q, long long ldq, long long q_stride,
                   const uint16_t* scales, const uint8_t* zeros, int group_size, const int32_t* offsets, void* y, long long ldy, int out_type, hipStream_t s);
int launch_route_topk(int type, const void* logits, long long ld, long long tokens, int experts, int k, int renormalise, float* weights, int32_t* chosen,
                      hipStream_t s);
// The choice and its plan in as few launches as they take together.
int launch_route_plan(int type, const void* logits, long long ld, long long tokens, int experts, int k, int renormalise, float* weights, int32_t* chosen,
                      int32_t* offsets, int32_t* rows, int32_t* slots, void* ws, size_t ws_bytes, hipStream_t s);
int launch_route_backward(int type, const float* grad, const void* logits, long long ld, const float* weights, const int32_t* chosen, long long tokens,
                          int experts, int k, int renormalise, void* out, long long ldo, hipStream_t s);
size_t expert_plan_workspace_bytes(long long tokens, int k, int experts);
int launch_expert_plan(const int32_t* chosen, long long tokens, int k, int experts, int32_t* offsets, int32_t* rows, int32_t* slots, void* ws,
                       size_t ws_bytes, hipStream_t s);
int launch_expert_gather(int type, const void* x, long long ldx, long long tokens, int k, const int32_t* rows, void* out, long long ldo,
                         long long n_slots, long long width, hipStream_t s);
int launch_expert_sum(int type, const void* y, long long ldy, long long n_slots, const float* weights, const int32_t* slots, long long tokens, int k,
                      void* out, long long ldo, long long width, hipStream_t s);
int launch_expert_sum_backward(int type, const void* dout, long long ldd, const void* y, long long ldy, const float* weights, const int32_t* slots,
                               long long tokens, int k, void* dy, long long lddy, float* dw, long long n_slots, long long width, hipStream_t s);

}  // namespace prism
