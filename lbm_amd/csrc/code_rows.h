// Rows of scores [N, K] (fp32, fp16 or bf16) held in the registers of a team of wavefronts: what the usage-balance and the sampling kernels
// share.  A team is W waves; its thread t holds V scores of the row, four neighbours at a time: value 4c + i of thread t is column
// (c * 64 W + t) * 4 + i, so a wave's loads are 1 KiB (fp32) or 512 bytes in one piece and ascending columns are chunk, thread, i.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace lbm {

template <typename T>
__device__ __forceinline__ float score_to_f32(T v);
template <>
__device__ __forceinline__ float score_to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float score_to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float score_to_f32<__hip_bfloat16>(__hip_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T score_from_f32(float v);   // one rounding to nearest even
template <>
__device__ __forceinline__ float score_from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half score_from_f32<__half>(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ __hip_bfloat16 score_from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

template <typename T>
struct alignas(4 * sizeof(T)) Quad {
    T v[4];
};

// v[] = the row's scores of thread t, -inf past column K.  vec: four scores in one access (aligned base and row stride, K % 4 == 0).
template <typename T, int V, int W>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int K, int t, int vec, float* v) {
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        const int col = (c * 64 * W + t) * 4;
        if (vec) {
            Quad<T> q;
            if (col < K) {
                q = *reinterpret_cast<const Quad<T>*>(row + col);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * c + i] = score_to_f32<T>(q.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * c + i] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * c + i] = col + i < K ? score_to_f32<T>(row[col + i]) : -INFINITY;
        }
    }
}

// reductions over a team, the result in every thread.  W = 1: one wave, no barrier.  W > 1: the team is the workgroup; s holds two rounds
// of W values and `round` alternates between them, so one barrier per reduction suffices (a slot is rewritten only after the next one).
template <typename A, int W, typename Op>
__device__ __forceinline__ A team_reduce(A v, A* s, int& round, Op op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    if constexpr (W > 1) {
        A* slot = s + round * W;
        round ^= 1;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = op(v, slot[w]);
    }
    return v;
}

struct OpMax {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a > b ? a : b; }
};
struct OpMin {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a < b ? a : b; }
};
struct OpAdd {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};

// exp(x) for x <= 0 to about 1.5 ulp, NaN for NaN: the part of x log2(e) that its product rounds away is added back behind the exponential
__device__ __forceinline__ float exp_f32(float x) {
    constexpr float kLog2e = 1.44269502e+0f, kLog2eLo = 1.92596303e-8f, kLn2 = 0.693147182f;
    x = x < -150.f ? -150.f : x;     // 2^-216: zero in fp32 either way, and -inf would make the residual NaN
    const float t = x * kLog2e;
    const float r = fmaf(x, kLog2eLo, fmaf(x, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * kLn2, e);
}

}  // namespace lbm

// CALL(type) for an LBM_F32 / LBM_F16 / LBM_BF16 argument
#define LBM_CODE_TYPES(dtype, CALL)                      \
    do {                                                 \
        if ((dtype) == LBM_F32) { CALL(float); }         \
        else if ((dtype) == LBM_F16) { CALL(__half); }   \
        else { CALL(__hip_bfloat16); }                   \
    } while (0)
