// Shared helpers of the C-ABI library: status codes, the per-thread error string, launch checks.
#pragma once
#include <cuda_runtime.h>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/e3nn_b200.h"

namespace e3b {

// Per-thread message of the last failing call (returned by e3b_last_error()).
inline char* error_buffer() {
    static thread_local char buf[512] = {0};
    return buf;
}

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

inline int check_launch(const char* what) {
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return fail(E3B_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return E3B_OK;
}

#define E3B_CUDA_TRY(expr)                                                                   \
    do {                                                                                     \
        cudaError_t _e = (expr);                                                             \
        if (_e != cudaSuccess) return ::e3b::fail(E3B_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
    } while (0)

constexpr int kNumSMs = 148;  // B200

// Lets a kernel be launched with `smem` bytes of dynamic shared memory.  Always the same large limit, so that no call lowers the
// one that another thread is about to launch with.
template <typename K>
int allow_smem(K kernel, size_t smem) {
    constexpr int kMost = 226 * 1024;      // (what is static counts against the 48 KB of a plain launch too)
    if (smem > kMost) return fail(E3B_ERR_UNSUPPORTED, "%lld bytes of shared memory are needed", static_cast<long long>(smem));
    if (smem > 32 * 1024) E3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    return E3B_OK;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace e3b
