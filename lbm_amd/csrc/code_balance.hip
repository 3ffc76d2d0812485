// Usage-balance loss of a codebook (or of experts behind a router) and its gradient.
//
//   p_n = softmax(s_n),  P = mean of p_n over the M rows that count,  c = number of times each code was picked in them,
//   f = c / sum(c),      loss = K sum_k f_k P_k          (1 where use is even, K where one code takes all)
//   ds_n = p_n (a - p_n.a) / M   with   a = g_loss K f + g_P   (f is a count: no gradient runs through it)
//
// A row counts if its keep flag is set and it holds a score above -inf.  Both passes are bound by HBM: the forward reads the scores once
// (4 operations per score), the gradient reads them again and writes as much.  A row lives in registers between its load, its maximum, its
// sum and its use; every thread adds p of its own columns over all rows it sees, so the column sums cost no traffic until the end, where
// each workgroup leaves one partial row.  Partial sums are joined in a fixed order in 64 bits: results do not change from run to run.
// The gradient takes a relative to its value at the row's best score: where one p is near 1 its a - p.a is a difference of near equals
// otherwise, and loses what it should return.
#include "code_rows.h"

namespace {

using lbm::OpAdd;
using lbm::OpMax;
using lbm::OpMin;

constexpr int kMaxK = 8192;   // a workgroup counts picks in LDS

// per row (float2): maximum, 1 / sum (0: the row does not count)
// workspace of the forward pass: partial sums [G][K] f32, partial counts [G][K] u32, rows counted [G] u32
struct Plan {
    int64_t G;
    size_t off_cnt, off_rows, total;
};

template <int W>
constexpr int teams() { return W == 1 ? 4 : 1; }   // rows a workgroup works on at a time

int waves_for(int K) { return K <= 2048 ? 1 : 4; }

Plan make_plan(int64_t N, int K) {
    const int T = waves_for(K) == 1 ? 4 : 1;
    Plan p;
    p.G = (N + 8 * T - 1) / (8 * T);      // eight rows per team at least, so that the partial rows stay small beside the scores
    const int64_t cap = T == 4 ? 2048 : 1024;
    if (p.G > cap) p.G = cap;
    if (p.G < 1) p.G = 1;
    auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
    size_t o = up((size_t)p.G * K * sizeof(float));
    p.off_cnt = o;
    o = up(o + (size_t)p.G * K * sizeof(unsigned));
    p.off_rows = o;
    o = up(o + (size_t)p.G * sizeof(unsigned));
    p.total = o;
    return p;
}

template <typename T, int V, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void balance_rows_kernel(const T* __restrict__ scores, int64_t lds, int vec,
                                                                            const int64_t* __restrict__ codes, int slots,
                                                                            const uint8_t* __restrict__ keep, float2* __restrict__ stat,
                                                                            float* __restrict__ part, unsigned* __restrict__ part_cnt,
                                                                            unsigned* __restrict__ part_rows, int64_t N, int K) {
    constexpr int TEAMS = teams<W>();
    extern __shared__ unsigned s_cnt[];                  // [K] picks; then, W == 1, the teams' column sums one after the other
    __shared__ float s_f[2 * W];
    __shared__ int s_i[2 * W];
    const int team = W == 1 ? threadIdx.x >> 6 : 0, t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    int rf = 0, ri = 0;
    for (int k = threadIdx.x; k < K; k += blockDim.x) s_cnt[k] = 0u;
    __syncthreads();

    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    unsigned rows = 0;
    for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < N; row += (int64_t)gridDim.x * TEAMS) {
        if (keep != nullptr && keep[row] == 0) {
            if (t == 0) stat[row] = make_float2(0.f, 0.f);
            continue;
        }
        float v[V];
        lbm::load_row<T, V, W>(scores + row * lds, K, t, vec, v);
        float m = -INFINITY;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m = fmaxf(m, v[i]);
            nan |= v[i] != v[i];
        }
        m = lbm::team_join<float, W>(lbm::wave_best(m), s_f, rf, OpMax());
        if (m == -INFINITY) {                            // nothing but -inf (does not count) or NaN (its sums are NaN, as softmax's)
            const int any = lbm::team_join<int, W>(__any(nan) ? 1 : 0, s_i, ri, OpMax());
            if (any == 0) {
                if (t == 0) stat[row] = make_float2(0.f, 0.f);
                continue;
            }
        }
        float e[V], s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            e[i] = lbm::exp_f32(v[i] - m);
            s += e[i];
        }
        s = lbm::team_join<float, W>(lbm::wave_total(s), s_f, rf, OpAdd());
        const float r = 1.f / s;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(e[i], r, acc[i]);
        ++rows;
        if (t == 0) stat[row] = make_float2(m, r);
        if (codes != nullptr) {
            for (int q = t; q < slots; q += 64 * W) {
                const int64_t k = codes[row * slots + q];
                if (k >= 0 && k < K) atomicAdd(&s_cnt[(int)k], 1u);
            }
        } else {
            int best = 0x7fffffff;                       // lowest column that holds the maximum
#pragma unroll
            for (int i = V - 1; i >= 0; --i) best = v[i] == m ? ((i >> 2) * 64 * W + t) * 4 + (i & 3) : best;
            best = lbm::team_join<int, W>(lbm::wave_first(best), s_i, ri, OpMin());
            if (t == 0 && best < K) atomicAdd(&s_cnt[best], 1u);
        }
    }
    __syncthreads();
    unsigned* pc = part_cnt + (int64_t)blockIdx.x * K;
    for (int k = threadIdx.x; k < K; k += blockDim.x) pc[k] = s_cnt[k];
    float* pp = part + (int64_t)blockIdx.x * K;
    if constexpr (W == 1) {
        __shared__ unsigned s_rows[4];
        float* s_sum = reinterpret_cast<float*>(s_cnt);
        if (t == 0) s_rows[team] = rows;
        for (int g = 0; g < TEAMS; ++g) {                // the teams in order
            __syncthreads();
            if (team == g) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int k = ((i >> 2) * 64 + t) * 4 + (i & 3);
                    if (k < K) s_sum[k] = g == 0 ? acc[i] : s_sum[k] + acc[i];
                }
            }
        }
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += blockDim.x) pp[k] = s_sum[k];
        if (threadIdx.x == 0) part_rows[blockIdx.x] = (s_rows[0] + s_rows[1]) + (s_rows[2] + s_rows[3]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int k = ((i >> 2) * 64 * W + t) * 4 + (i & 3);
            if (k < K) pp[k] = acc[i];
        }
        if (t == 0) part_rows[blockIdx.x] = rows;
    }
}

// column sums over the partial rows, 16 columns x 16 groups of rows per workgroup; totals[0] = rows counted (every workgroup adds them up
// for itself, workgroup 0 leaves them)
__global__ __launch_bounds__(256) void balance_join_kernel(const float* __restrict__ part, const unsigned* __restrict__ part_cnt,
                                                           const unsigned* __restrict__ part_rows, float* __restrict__ mean,
                                                           int64_t* __restrict__ counts, double* __restrict__ totals, int64_t G, int K) {
    __shared__ double s_p[16][17];
    __shared__ unsigned long long s_c[16][17];
    __shared__ unsigned long long s_m[4];
    unsigned long long m = 0;
    for (int64_t g = threadIdx.x; g < G; g += 256) m += part_rows[g];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
    if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m;
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int k = blockIdx.x * 16 + col;
    double p = 0.0;
    unsigned long long c = 0;
    if (k < K)
        for (int64_t g = grp; g < G; g += 16) {
            p += (double)part[g * K + k];
            c += part_cnt[g * K + k];
        }
    s_p[grp][col] = p;
    s_c[grp][col] = c;
    __syncthreads();
    m = (s_m[0] + s_m[1]) + (s_m[2] + s_m[3]);
    if (threadIdx.x < 16 && k < K) {
        for (int g = 1; g < 16; ++g) {
            p += s_p[g][col];
            c += s_c[g][col];
        }
        mean[k] = m > 0 ? (float)(p / (double)m) : 0.f;
        counts[k] = (int64_t)c;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) totals[0] = (double)m;
}

__device__ __forceinline__ double block_sum(double v, double* s) {
    v = lbm::wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// loss = K sum f P; totals[1] = picks counted
__global__ __launch_bounds__(256) void balance_loss_kernel(const float* __restrict__ mean, const int64_t* __restrict__ counts,
                                                           float* __restrict__ loss, double* __restrict__ totals, int K) {
    __shared__ double s[4];
    double c = 0.0, l = 0.0;
    for (int k = threadIdx.x; k < K; k += 256) {
        c += (double)counts[k];
        l += (double)counts[k] * (double)mean[k];
    }
    c = block_sum(c, s);
    l = block_sum(l, s);
    if (threadIdx.x == 0) {
        loss[0] = (float)((double)K * l / (c > 0.0 ? c : 1.0));   // NaN in mean shows even where nothing was picked
        totals[1] = c;
    }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void balance_grad_kernel(const T* __restrict__ scores, int64_t lds, int vec,
                                                                            const float2* __restrict__ stat, const int64_t* __restrict__ counts,
                                                                            const double* __restrict__ totals, const float* __restrict__ g_loss,
                                                                            const float* __restrict__ g_mean, T* __restrict__ ds, int vec_out,
                                                                            int64_t N, int K) {
    constexpr int TEAMS = teams<W>();
    __shared__ float s_f[2 * W];
    const int team = W == 1 ? threadIdx.x >> 6 : 0, t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    int rf = 0;
    const double M = totals[0], C = totals[1];
    const double gl = g_loss != nullptr && C > 0.0 ? (double)g_loss[0] * K / C : 0.0;
    const float inv_m = M > 0.0 ? (float)(1.0 / M) : 0.f;
    float a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = ((i >> 2) * 64 * W + t) * 4 + (i & 3);
        a[i] = k < K ? (float)(gl * (double)counts[k] + (g_mean != nullptr ? (double)g_mean[k] : 0.0)) : 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < N; row += (int64_t)gridDim.x * TEAMS) {
        const float m = stat[row].x, r = stat[row].y;
        float d[V];
        if (r == 0.f) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 0.f;
        } else {
            float v[V], ref = -INFINITY;
            lbm::load_row<T, V, W>(scores + row * lds, K, t, vec, v);
#pragma unroll
            for (int i = 0; i < V; ++i) ref = v[i] == m ? fmaxf(ref, a[i]) : ref;
            ref = lbm::team_join<float, W>(lbm::wave_best(ref), s_f, rf, OpMax());
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[i] = lbm::exp_f32(v[i] - m) * r;
                dot = fmaf(d[i], a[i] - ref, dot);
            }
            dot = lbm::team_join<float, W>(lbm::wave_total(dot), s_f, rf, OpAdd());
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = d[i] * ((a[i] - ref) - dot) * inv_m;
        }
        T* out = ds + row * (int64_t)K;
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            const int col = (c * 64 * W + t) * 4;
            if (vec_out) {
                if (col < K) {
                    lbm::Quad<T> q;
#pragma unroll
                    for (int i = 0; i < 4; ++i) q.v[i] = lbm::score_from_f32<T>(d[4 * c + i]);
                    *reinterpret_cast<lbm::Quad<T>*>(out + col) = q;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < K) out[col + i] = lbm::score_from_f32<T>(d[4 * c + i]);
            }
        }
    }
}

template <typename T>
int vec_ok(const void* p, int64_t ld, int K) {
    return ((uintptr_t)p % (4 * sizeof(T))) == 0 && (ld & 3) == 0 && (K & 3) == 0 ? 1 : 0;
}

template <typename T>
int run_rows(const void* scores, int64_t lds, const int64_t* codes, int slots, const uint8_t* keep, float2* stat, float* part, unsigned* cnt,
             unsigned* rows, int64_t G, int64_t N, int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    const int vec = vec_ok<T>(scores, lds, K);
    const size_t shm = (size_t)K * 4;
#define LBM_ROWS(V, W)                                                                                                                     \
    hipLaunchKernelGGL((balance_rows_kernel<T, V, W>), dim3((unsigned)G), dim3(W == 1 ? 256 : 64 * W), shm, st, s, lds, vec, codes, slots, \
                       keep, stat, part, cnt, rows, N, K)
    if (K <= 256) LBM_ROWS(4, 1);
    else if (K <= 512) LBM_ROWS(8, 1);
    else if (K <= 1024) LBM_ROWS(16, 1);
    else if (K <= 2048) LBM_ROWS(32, 1);
    else if (K <= 4096) LBM_ROWS(16, 4);
    else LBM_ROWS(32, 4);
#undef LBM_ROWS
    return lbm::check_launch("lbm_code_balance");
}

template <typename T>
int run_grad(const void* scores, int64_t lds, const float2* stat, const int64_t* counts, const double* totals, const float* g_loss,
             const float* g_mean, void* ds, int64_t G, int64_t N, int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    T* o = static_cast<T*>(ds);
    const int vec = vec_ok<T>(scores, lds, K), vo = vec_ok<T>(ds, K, K);
#define LBM_GRAD(V, W)                                                                                                                       \
    hipLaunchKernelGGL((balance_grad_kernel<T, V, W>), dim3((unsigned)G), dim3(W == 1 ? 256 : 64 * W), 0, st, s, lds, vec, stat, counts, totals, \
                       g_loss, g_mean, o, vo, N, K)
    if (K <= 256) LBM_GRAD(4, 1);
    else if (K <= 512) LBM_GRAD(8, 1);
    else if (K <= 1024) LBM_GRAD(16, 1);
    else if (K <= 2048) LBM_GRAD(32, 1);
    else if (K <= 4096) LBM_GRAD(16, 4);
    else LBM_GRAD(32, 4);
#undef LBM_GRAD
    return lbm::check_launch("lbm_code_balance_grad");
}

}  // namespace

extern "C" size_t lbm_code_balance_workspace_bytes(int64_t N, int32_t K) {
    if (N < 0 || K < 1 || K > kMaxK) return 0;
    return make_plan(N, K).total;
}

extern "C" int lbm_code_balance(const void* scores, int32_t dtype, int64_t lds, const int64_t* codes_or_null, int32_t slots,
                                const uint8_t* keep_or_null, float* loss, int64_t* counts, float* mean, float* row_stat, double* totals,
                                void* workspace, int64_t N, int32_t K, lbm_stream_t stream) {
    const char* what = "lbm_code_balance";
    LBM_REQUIRE(N >= 0 && K >= 1, LBM_EINVAL, "%s: bad sizes (N=%lld K=%d)", what, (long long)N, K);
    LBM_REQUIRE(K <= kMaxK, LBM_EUNSUPPORTED, "%s: K=%d > %d", what, K, kMaxK);
    LBM_REQUIRE(dtype == LBM_F32 || dtype == LBM_F16 || dtype == LBM_BF16, LBM_EINVAL, "%s: unknown score type %d", what, dtype);
    LBM_REQUIRE(loss && counts && mean && totals && workspace, LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(N == 0 || (scores && row_stat), LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(((uintptr_t)row_stat & 7) == 0, LBM_EINVAL, "%s: row_stat must be 8-byte aligned", what);
    LBM_REQUIRE(N <= 1 || lds >= 0, LBM_EINVAL, "%s: negative row stride", what);
    LBM_REQUIRE(codes_or_null == nullptr || slots >= 1, LBM_EINVAL, "%s: slots must be >= 1 with codes", what);
    LBM_REQUIRE(((uintptr_t)workspace & 15) == 0, LBM_EINVAL, "%s: workspace must be 16-byte aligned", what);
    const Plan p = make_plan(N, K);
    char* ws = static_cast<char*>(workspace);
    float* part = reinterpret_cast<float*>(ws);
    unsigned* cnt = reinterpret_cast<unsigned*>(ws + p.off_cnt);
    unsigned* rows = reinterpret_cast<unsigned*>(ws + p.off_rows);
    hipStream_t st = lbm::as_stream(stream);
    int rc = LBM_OK;
#define LBM_CALL(T) rc = run_rows<T>(scores, lds, codes_or_null, slots, keep_or_null, reinterpret_cast<float2*>(row_stat), part, cnt, rows, p.G, N, K, st)
    LBM_CODE_TYPES(dtype, LBM_CALL);
#undef LBM_CALL
    if (rc != LBM_OK) return rc;
    hipLaunchKernelGGL(balance_join_kernel, dim3((unsigned)((K + 15) / 16)), dim3(256), 0, st, part, cnt, rows, mean, counts, totals, p.G, K);
    hipLaunchKernelGGL(balance_loss_kernel, dim3(1), dim3(256), 0, st, mean, counts, loss, totals, K);
    return lbm::check_launch(what);
}

extern "C" int lbm_code_balance_grad(const void* scores, int32_t dtype, int64_t lds, const float* row_stat, const int64_t* counts,
                                     const double* totals, const float* g_loss_or_null, const float* g_mean_or_null, void* dscores,
                                     int64_t N, int32_t K, lbm_stream_t stream) {
    const char* what = "lbm_code_balance_grad";
    LBM_REQUIRE(N >= 0 && K >= 1, LBM_EINVAL, "%s: bad sizes (N=%lld K=%d)", what, (long long)N, K);
    LBM_REQUIRE(K <= kMaxK, LBM_EUNSUPPORTED, "%s: K=%d > %d", what, K, kMaxK);
    LBM_REQUIRE(dtype == LBM_F32 || dtype == LBM_F16 || dtype == LBM_BF16, LBM_EINVAL, "%s: unknown score type %d", what, dtype);
    if (N == 0) return LBM_OK;
    LBM_REQUIRE(scores && row_stat && counts && totals && dscores, LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(N <= 1 || lds >= 0, LBM_EINVAL, "%s: negative row stride", what);
    const int64_t T = waves_for(K) == 1 ? 4 : 1, cap = T == 4 ? 2048 : 1024;
    int64_t G = (N + T - 1) / T;
    if (G > cap) G = cap;
    int rc = LBM_OK;
#define LBM_CALL(T) rc = run_grad<T>(scores, lds, reinterpret_cast<const float2*>(row_stat), counts, totals, g_loss_or_null, g_mean_or_null, dscores, G, N, K, lbm::as_stream(stream))
    LBM_CODE_TYPES(dtype, LBM_CALL);
#undef LBM_CALL
    return rc;
}
