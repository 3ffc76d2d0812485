// Rows of scores (fp32, fp16 or bf16) in the registers of a wave: conversions, loads and wave-wide sums, maxima and running sums, shared by the
// usage-balance and the sampling kernels.
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

// The row's scores of one wave's lanes, -inf past column K: value 4c + i of lane t is column (64 c + t) * 4 + i, so ascending columns are chunk,
// lane, i.  Four scores in one access; VEC: of aligned rows with K % 4 == 0, else of any, one by one where the row ends.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int K, int t, float* v) {
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        const int col = (c * 64 + t) * 4;
        if constexpr (VEC) {
            Quad<T> q;
#pragma unroll
            for (int i = 0; i < 4; ++i) q.v[i] = score_from_f32<T>(-INFINITY);
            if (col < K) q = *reinterpret_cast<const Quad<T>*>(row + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * c + i] = score_to_f32<T>(q.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * c + i] = -INFINITY;
            if (col + 4 <= K) {
                Quad<T> q;
                __builtin_memcpy(&q, row + col, sizeof(q));
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * c + i] = score_to_f32<T>(q.v[i]);
            } else if (col < K) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (col + i < K) v[4 * c + i] = score_to_f32<T>(row[col + i]);
            }
        }
    }
}

// Sums and maxima over a wave by DPP moves (4 shifts inside rows of 16 lanes, 2 row broadcasts), no LDS.  All 64 lanes must be active.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_move(float old, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_move(int old, int x) {
    return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_move(double old, double x) {
    return __hiloint2double(dpp_move<CTRL, ROWS>(__double2hiint(old), __double2hiint(x)),
                            dpp_move<CTRL, ROWS>(__double2loint(old), __double2loint(x)));
}
__device__ __forceinline__ float lane_value(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }
__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ double lane_value(double x, int lane) {
    return __hiloint2double(lane_value(__double2hiint(x), lane), lane_value(__double2loint(x), lane));
}
// inclusive running value over the lanes; `none` is op's neutral element
template <typename A, typename Op>
__device__ __forceinline__ A wave_scan(A x, A none, Op op) {
    x = op(x, dpp_move<0x111, 0xf>(none, x));
    x = op(x, dpp_move<0x112, 0xf>(none, x));
    x = op(x, dpp_move<0x114, 0xf>(none, x));
    x = op(x, dpp_move<0x118, 0xf>(none, x));
    x = op(x, dpp_move<0x142, 0xa>(none, x));
    x = op(x, dpp_move<0x143, 0xc>(none, x));
    return x;
}

struct OpMax {      // floats: NaN loses
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ int operator()(int a, int b) const { return a > b ? a : b; }
};
struct OpMin {
    __device__ __forceinline__ int operator()(int a, int b) const { return a < b ? a : b; }
};
struct OpAdd {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};

template <typename A>
__device__ __forceinline__ A wave_total(A x) { return lane_value(wave_scan<A>(x, A(0), OpAdd()), 63); }
__device__ __forceinline__ float wave_best(float x) { return lane_value(wave_scan<float>(x, -INFINITY, OpMax()), 63); }
__device__ __forceinline__ int wave_first(int x) { return lane_value(wave_scan<int>(x, 0x7fffffff, OpMin()), 63); }

// op over the L neighbouring lanes of a row, the result in each of them.  L < 64: exchanges inside rows of 16 lanes (pairs, quads, halves,
// the row's mirror image) and one across two rows; other rows' lanes may be off.
template <int L, typename A, typename Op>
__device__ __forceinline__ A group_all(A x, A none, Op op) {
    static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes of a row");
    if constexpr (L == 64) {
        return lane_value(wave_scan<A>(x, none, op), 63);
    } else {
        x = op(x, dpp_move<0xB1, 0xf>(x, x));
        x = op(x, dpp_move<0x4E, 0xf>(x, x));
        x = op(x, dpp_move<0x141, 0xf>(x, x));
        if constexpr (L > 8) x = op(x, dpp_move<0x140, 0xf>(x, x));
        if constexpr (L > 16) x = op(x, __shfl_xor(x, 16, 64));
        return x;
    }
}
template <int L>
__device__ __forceinline__ float group_total(float x) { return group_all<L>(x, 0.f, OpAdd()); }
template <int L>
__device__ __forceinline__ float group_best(float x) { return group_all<L>(x, -INFINITY, OpMax()); }
template <int L>
__device__ __forceinline__ int group_first(int x) { return group_all<L>(x, 0x7fffffff, OpMin()); }

}  // namespace lbm

// CALL(type) for an LBM_F32 / LBM_F16 / LBM_BF16 argument
#define LBM_CODE_TYPES(dtype, CALL)                      \
    do {                                                 \
        if ((dtype) == LBM_F32) { CALL(float); }         \
        else if ((dtype) == LBM_F16) { CALL(__half); }   \
        else { CALL(__hip_bfloat16); }                   \
    } while (0)
