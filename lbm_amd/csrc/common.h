// Shared host-side helpers for liblbm_hip.so (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/lbm_abi.h"

namespace lbm {

// thread-local last-error message, written by every failing entry point
char* last_error_buf();
int fail(int code, const char* fmt, ...);

inline hipStream_t as_stream(lbm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

// after a kernel launch: report (and clear) a launch error without synchronising
inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(LBM_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
    return LBM_OK;
}

// A launch of 2^32 threads and more along one dimension runs the rest beyond 2^32 only, and reports no error.
inline bool grid_fits(int64_t blocks, int64_t threads) { return blocks <= 0xffffffffLL / threads; }

constexpr int kWave = 64;

// n bytes set to v by a kernel: memset nodes of a captured graph have given wrong results on replays after the first
static __global__ __launch_bounds__(256) void fill_bytes_kernel(uint8_t* p, uint8_t v, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = v;
}
inline int fill_bytes(const char* what, uint8_t* p, uint8_t v, int64_t n, hipStream_t st) {
    const int64_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(fill_bytes_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, p, v, n);
    return check_launch(what);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_min(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fminf(v, __shfl_xor(v, o, 64));
    return v;
}

}  // namespace lbm

#define LBM_REQUIRE(cond, code, ...) \
    do {                             \
        if (!(cond)) return lbm::fail(code, __VA_ARGS__); \
    } while (0)
