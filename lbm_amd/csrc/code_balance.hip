// Usage-balance loss of a codebook (or of experts behind a router) and its gradient.
//
//   p_n = softmax(s_n),  P = mean of p_n over the M rows that count,  c = number of times each code was picked in them,
//   f = c / sum(c),      loss = K sum_k f_k P_k          (1 where use is even, K where one code takes all)
//   ds_n = p_n (a - p_n.a) / M   with   a = g_loss K f + g_P   (f is a count: no gradient runs through it)
//
// A row counts if its keep flag is set and it holds a score above -inf.  Both passes are bound by HBM: the forward reads the scores once
// (4 operations per score), the gradient reads them again and writes as much.  A row lives in registers between its load, its maximum, its
// sum and its use, the next row's load runs under that, and every thread adds p of its own columns over all rows it sees, so the column
// sums cost no traffic until the end, where each workgroup leaves one partial row.  Partial sums are joined in a fixed order in 64 bits:
// results do not change from run to run.  Up to 2048 codes a wave holds a row, or eight, four or two short ones (no barrier); above
// that four waves share one and exchange their maxima and sums once per row (100000 rows with the gradient in four waves: 2048 codes 408 us
// for 270 in bf16 and 551 for 514 in fp32, 1100 codes 375 for 301 in fp32; 2047 codes 413 for 367 in bf16, but 545 for 775 in fp32, where a
// wave's registers spill; 8192 codes in eight waves with half the registers each: 217 us for 172 at 40000 rows; 5 codes, a row to a wave: 653
// us for 108 at 1043158 rows of bf16 with the gradient).
// The gradient takes a relative to its value at the row's best score: where one p is near 1 its a - p.a is a difference of near equals
// otherwise, and loses what it should return.
#include "code_rows.h"

namespace {

using lbm::OpMax;
using lbm::OpMin;

constexpr int kMaxK = 8192;   // a workgroup counts picks in LDS
constexpr int kJoinCols = 64;

// workspace of the forward pass: partial sums [G][K] f32, partial counts [G][K] u32, rows counted [G] u32; second stage: sums [S][K] f64,
// counts [S][K] u64
struct Plan {
    int64_t G;
    int S;            // pieces of the G partial rows in the second stage
    size_t off_cnt, off_rows, off_sum2, off_cnt2, total;
};

// lanes that share a row (256: the workgroup)
int lanes_for(int K) { return K <= 8 ? 8 : (K <= 64 ? 16 : (K <= 128 ? 32 : (K <= 2048 ? 64 : 256))); }

Plan make_plan(int64_t N, int K) {
    const int T = 256 / lanes_for(K);     // rows a workgroup works on at a time
    Plan p;
    // eight rows per team at least, so that the partial rows stay small beside the scores -- two where that leaves CUs without work
    p.G = (N + 8 * T - 1) / (8 * T);
    if (p.G < 512) {
        p.G = (N + 2 * T - 1) / (2 * T);
        if (p.G > 512) p.G = 512;
    }
    // as many as the registers let run at a time: 8, 7, 4, 3, 4 and 3 per CU (7 at 1536000 x 512 fp32: 603 us, 8 in two rounds 660)
    const int64_t cap = 256 * (K <= 128 ? 8 : (K <= 512 ? 7 : (K <= 1024 ? 4 : (K <= 2048 ? 3 : (K <= 4096 ? 4 : 3)))));
    if (p.G > cap) p.G = cap;
    if (p.G < 1) p.G = 1;
    const int groups = (K + kJoinCols - 1) / kJoinCols;
    p.S = 256 / groups;                   // one workgroup per CU
    if (p.S > (p.G + 15) / 16) p.S = (int)((p.G + 15) / 16);
    if (p.S < 1) p.S = 1;
    auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
    size_t o = up((size_t)p.G * K * sizeof(float));
    p.off_cnt = o;  o = up(o + (size_t)p.G * K * sizeof(unsigned));
    p.off_rows = o; o = up(o + (size_t)p.G * sizeof(unsigned));
    p.off_sum2 = o; o = up(o + (size_t)p.S * K * sizeof(double));
    p.off_cnt2 = o; o = up(o + (size_t)p.S * K * sizeof(unsigned long long));
    p.total = o;
    return p;
}

// A row's scores as loaded by its L lanes, E at a time: value E c + i of lane t is column (c * L + t) * E + i.  E is 16 bytes at most, or 1
// where rows or their addresses are no multiples of that: then one load takes L neighbouring scores
template <typename T, int V, int L, bool VEC>
struct Held {
    static constexpr int E = !VEC ? 1 : (V < 16 / (int)sizeof(T) ? V : 16 / (int)sizeof(T));
    struct alignas(E * sizeof(T)) Pack { T v[E]; };
    Pack q[V / E];

    static __device__ __forceinline__ int column(int i, int t) { return ((i / E) * L + t) * E + i % E; }
    __device__ __forceinline__ void load(const T* __restrict__ row, int K, int t) {
#pragma unroll
        for (int c = 0; c < V / E; ++c) {
            const int col = (c * L + t) * E;
            if (col < K) {
                q[c] = *reinterpret_cast<const Pack*>(row + col);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) q[c].v[i] = lbm::score_from_f32<T>(-INFINITY);
            }
        }
    }
    __device__ __forceinline__ float at(int i) const { return lbm::score_to_f32<T>(q[i / E].v[i % E]); }
};

// E scores, each rounded once to the nearest, in one access
template <typename T, int E>
__device__ __forceinline__ void store_pack(T* out, const float* f) {
    if constexpr (E * sizeof(T) < 4) {
        out[0] = lbm::score_from_f32<T>(f[0]);
    } else {
        constexpr int W = E * sizeof(T) / 4;
        unsigned w[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(f[i]);
            } else {
                const T a = lbm::score_from_f32<T>(f[2 * i]), b = lbm::score_from_f32<T>(f[2 * i + 1]);
                w[i] = (unsigned)__builtin_bit_cast(unsigned short, a) | (unsigned)__builtin_bit_cast(unsigned short, b) << 16;
            }
        }
        if constexpr (W == 4) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (W == 2) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<unsigned*>(out) = w[0];
    }
}

constexpr float kLog2e = 1.44269502f;

// exp(x), x <= 0: (2 |x| + 2) 2^-24 relative
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// exp(v - m) times a factor that all scores of a row share: 2^(v log2(e) - ml) with ml = m log2(e) rounded, one fused operation and so one
// rounding of the exponent, where the difference and its product are two (errors of a row's gradients: 3e-7 for 1e-6).  The factor is
// 2^(m log2(e) - ml); it drops out of e / sum(e).  Scores of 10^6 and more, where ml is no longer near the exponents, take the difference.
struct RowExp {
    float m, ml;
    bool near;
    __device__ __forceinline__ explicit RowExp(float best) : m(best), ml(best * kLog2e), near(fabsf(best) < 1e6f) {}
    template <int V>
    __device__ __forceinline__ void apply(float* v) const {
        if (near) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __builtin_amdgcn_exp2f(fmaf(v[i], kLog2e, -ml));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = exp_neg(v[i] - m);
        }
    }
    // log2 of the factor
    __device__ __forceinline__ float excess() const { return near ? fmaf(m, kLog2e, -ml) : 0.f; }
};

// the team; one wave to a row: the same in all its lanes, and the row's addresses are scalar.  (Where four waves share a row that costs
// registers that the longest rows do not have: 40000 x 8192 fp32 370 us for 267.)
template <int L>
__device__ __forceinline__ int team_of() {
    return L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / L;
}

template <typename T, int V, int L, bool VEC>
__global__ __launch_bounds__(256, V == 32 ? 3 : 4) void balance_rows_kernel(const T* __restrict__ scores, int64_t lds,
                                                                           const int64_t* __restrict__ codes, int slots,
                                                                           const uint8_t* __restrict__ keep, float2* __restrict__ stat,
                                                                           float* __restrict__ part, unsigned* __restrict__ part_cnt,
                                                                           unsigned* __restrict__ part_rows, int64_t N, int K) {
    constexpr int TEAMS = 256 / L, W = L > 64 ? L / 64 : 1, LW = L > 64 ? 64 : L;
    using H = Held<T, V, L, VEC>;
    extern __shared__ unsigned s_cnt[];                  // [K] picks; then the teams' column sums [TEAMS][K]
    __shared__ float2 s_ms[2][W];                        // W > 1: (maximum, sum) of each wave
    __shared__ int s_best[2][W];
    __shared__ unsigned s_rows[TEAMS];
    const int team = team_of<L>(), t = threadIdx.x % L, wave = threadIdx.x >> 6;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    for (int k = threadIdx.x; k < K; k += 256) s_cnt[k] = 0u;
    __syncthreads();

    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    unsigned rows = 0;
    int round = 0;
    // What the next row needs is loaded while this one is worked on: its scores, its picks, and the keep byte of the row behind it.  Loads
    // return in order, so nothing that this row waits for is loaded behind them -- but for the picks of the longest rows, whose registers
    // are all taken.
    constexpr bool AHEAD = V < 32;
    auto kept = [&](int64_t r) -> unsigned {
        unsigned v = 0u;
        if (r < N) v = keep != nullptr ? keep[r] : 1u;
        return v;
    };
    auto picked = [&](int64_t r) -> int64_t {
        int64_t v = -1;
        if (codes != nullptr && t < slots && r < N) v = codes[r * slots + t];
        return v;
    };
    int64_t row = (int64_t)blockIdx.x * TEAMS + team;
    unsigned on = kept(row), on_next = kept(row + step);
    int64_t pick_next = AHEAD ? picked(row) : -1;
    H held;
    if (on) held.load(scores + row * lds, K, t);
    for (; row < N; row += step) {
        const bool now = on != 0u;
        int64_t pick = pick_next;
        float e[V];
        if (now) {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = held.at(i);
        }
        on = on_next;
        if (on) held.load(scores + (row + step) * lds, K, t);
        if constexpr (AHEAD) pick_next = picked(row + step);
        else pick = picked(row);
        on_next = kept(row + 2 * step);
        if (!now) {
            if (t == 0) stat[row] = make_float2(0.f, 0.f);
            continue;
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, e[i]);
        m = lbm::group_best<LW>(m);
        int best = 0x7fffffff;
        if (codes == nullptr && m > -INFINITY) {         // lowest column that holds the (wave's) maximum
#pragma unroll
            for (int i = V - 1; i >= 0; --i) best = e[i] == m ? H::column(i, t) : best;
            best = lbm::group_first<LW>(best);
        }
        const RowExp x(m);
        float s = 0.f, scale = 1.f;
        if (m == -INFINITY) {                            // nothing but -inf, or NaN, which shows
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s = e[i] != e[i] ? e[i] : s;
                e[i] = e[i] != e[i] ? e[i] : 0.f;
            }
        } else {
            x.template apply<V>(e);
#pragma unroll
            for (int i = 0; i < V; ++i) s += e[i];
        }
        s = lbm::group_total<LW>(s);
        if constexpr (W > 1) {                           // the waves' pairs joined: one barrier per row, since the other half of s_ms is
            scale = __builtin_amdgcn_exp2f(-x.excess()); // written only behind the next row's
            if ((threadIdx.x & 63) == 0) {
                s_ms[round][wave] = make_float2(m, m == -INFINITY ? s : s * scale);
                s_best[round][wave] = best;
            }
            __syncthreads();
            const float m_wave = m;
            float2 ms[W];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                ms[w] = s_ms[round][w];
                m = fmaxf(m, ms[w].x);
            }
            s = 0.f;
            best = 0x7fffffff;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s += ms[w].x == m ? ms[w].y : ms[w].y * exp_neg(ms[w].x - m);
                const int bw = s_best[round][w];
                best = ms[w].x == m && bw < best ? bw : best;
            }
            round ^= 1;
            scale *= m_wave == m ? 1.f : exp_neg(m_wave - m);
        }
        if (m == -INFINITY && s == 0.f) {
            if (t == 0) stat[row] = make_float2(0.f, 0.f);
            continue;
        }
        float r = __builtin_amdgcn_rcpf(s);              // within a unit in the last place
        scale *= r;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(e[i], scale, acc[i]);
        ++rows;
        if constexpr (W > 1) r *= __builtin_amdgcn_exp2f(-RowExp(m).excess());
        if (t == 0) stat[row] = make_float2(m, r);       // p = r exp(), with the row's factor
        if (codes != nullptr) {
            if (pick >= 0 && pick < K) atomicAdd(&s_cnt[(int)pick], 1u);
            for (int q = t + L; q < slots; q += L) {
                const int64_t k = codes[row * slots + q];
                if (k >= 0 && k < K) atomicAdd(&s_cnt[(int)k], 1u);
            }
        } else if (t == 0 && best < K) {
            atomicAdd(&s_cnt[best], 1u);
        }
    }
    __syncthreads();
    unsigned* pc = part_cnt + (int64_t)blockIdx.x * K;
    for (int k = threadIdx.x; k < K; k += 256) pc[k] = s_cnt[k];
    float* pp = part + (int64_t)blockIdx.x * K;
    if (t == 0) s_rows[team] = rows;
    if constexpr (TEAMS > 1) {
        float* s_sum = reinterpret_cast<float*>(s_cnt);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int k = H::column(i, t);
            if (k < K) s_sum[team * K + k] = acc[i];
        }
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += 256) {     // the teams in order
            float v = 0.f;
#pragma unroll
            for (int g = 0; g < TEAMS; ++g) v += s_sum[g * K + k];
            pp[k] = v;
        }
        if (threadIdx.x == 0) {
            rows = 0;
            for (int g = 0; g < TEAMS; ++g) rows += s_rows[g];
            part_rows[blockIdx.x] = rows;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int k = H::column(i, t);
            if (k < K) pp[k] = acc[i];
        }
        if (t == 0) part_rows[blockIdx.x] = rows;
    }
}

// column sums over the G partial rows: workgroup (64 columns, piece of the rows)
__global__ __launch_bounds__(256) void balance_join_kernel(const float* __restrict__ part, const unsigned* __restrict__ part_cnt,
                                                           double* __restrict__ sum2, unsigned long long* __restrict__ cnt2, int64_t G, int K) {
    __shared__ double s_p[4][kJoinCols];
    __shared__ unsigned long long s_c[4][kJoinCols];
    const int S = gridDim.y, piece = blockIdx.y, col = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const int k = blockIdx.x * kJoinCols + col;
    const int64_t g0 = G * piece / S, g1 = G * (piece + 1) / S;
    double p = 0.0;
    unsigned long long c = 0;
    if (k < K) {
        int64_t g = g0 + grp;
        for (; g + 12 < g1; g += 16) {                   // four loads of each kind on their way at a time
            float f[4];
            unsigned n[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f[u] = part[(g + 4 * u) * K + k];
                n[u] = part_cnt[(g + 4 * u) * K + k];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                p += (double)f[u];
                c += n[u];
            }
        }
        for (; g < g1; g += 4) {
            p += (double)part[g * K + k];
            c += part_cnt[g * K + k];
        }
    }
    s_p[grp][col] = p;
    s_c[grp][col] = c;
    __syncthreads();
    if (threadIdx.x < kJoinCols && k < K) {
        sum2[(int64_t)piece * K + k] = (s_p[0][col] + s_p[1][col]) + (s_p[2][col] + s_p[3][col]);
        cnt2[(int64_t)piece * K + k] = (s_c[0][col] + s_c[1][col]) + (s_c[2][col] + s_c[3][col]);
    }
}

constexpr int kFinish = 1024;

__device__ __forceinline__ double block_sum(double v, double* s) {
    v = lbm::wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kFinish / 64; ++w) v += s[w];
    return v;
}

// one workgroup: the pieces joined in order, the means, the loss; totals: rows that count, picks that count.  (A last-workgroup-to-arrive
// join inside the kernel above cost more than this launch: 33 us for both against 9 at 24000 x 512, its fences write an XCD's L2 back.)
__global__ __launch_bounds__(kFinish) void balance_finish_kernel(const double* __restrict__ sum2, const unsigned long long* __restrict__ cnt2,
                                                                 const unsigned* __restrict__ part_rows, float* __restrict__ mean,
                                                                 int64_t* __restrict__ counts, float* __restrict__ loss,
                                                                 double* __restrict__ totals, int S, int64_t G, int K) {
    __shared__ double s_sum[kFinish / 64];
    double m = 0.0;
    for (int64_t g = threadIdx.x; g < G; g += kFinish) m += (double)part_rows[g];
    m = block_sum(m, s_sum);
    double picks = 0.0, l = 0.0;
    for (int k = threadIdx.x; k < K; k += kFinish) {
        double p = 0.0;
        unsigned long long c = 0;
        for (int z0 = 0; z0 < S; z0 += 8) {              // eight of each kind on their way at a time
            double f[8];
            unsigned long long n[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int z = z0 + u < S ? z0 + u : S - 1;
                f[u] = sum2[(int64_t)z * K + k];
                n[u] = cnt2[(int64_t)z * K + k];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                p += z0 + u < S ? f[u] : 0.0;
                c += z0 + u < S ? n[u] : 0ull;
            }
        }
        const float f = m > 0.0 ? (float)(p / m) : 0.f;
        mean[k] = f;
        counts[k] = (int64_t)c;
        picks += (double)c;
        l += (double)c * (double)f;
    }
    picks = block_sum(picks, s_sum);
    l = block_sum(l, s_sum);
    if (threadIdx.x == 0) {
        loss[0] = (float)((double)K * l / (picks > 0.0 ? picks : 1.0));   // NaN in mean shows even where nothing was picked
        totals[0] = m;
        totals[1] = picks;
    }
}

template <typename T, int V, int L, bool VEC>
__global__ __launch_bounds__(256, V == 32 ? 3 : 4) void balance_grad_kernel(const T* __restrict__ scores, int64_t lds,
                                                                           const float2* __restrict__ stat, const int64_t* __restrict__ counts,
                                                                           const double* __restrict__ totals, const float* __restrict__ g_loss,
                                                                           const float* __restrict__ g_mean, T* __restrict__ ds, int64_t N,
                                                                           int K) {
    constexpr int TEAMS = 256 / L, W = L > 64 ? L / 64 : 1, LW = L > 64 ? 64 : L;
    using H = Held<T, V, L, VEC>;
    __shared__ float4 s_x[2][W];                         // W > 1: each wave's p.(a - ref), its sum of p, its ref, whether it holds the best
    const int team = team_of<L>(), t = threadIdx.x % L, wave = threadIdx.x >> 6;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    const double M = totals[0], C = totals[1];
    const double gl = g_loss != nullptr && C > 0.0 ? (double)g_loss[0] * K / C : 0.0;
    const float inv_m = M > 0.0 ? (float)(1.0 / M) : 0.f;
    float a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = H::column(i, t);
        a[i] = k < K ? (float)(gl * (double)counts[k] + (g_mean != nullptr ? (double)g_mean[k] : 0.0)) : 0.f;
    }
    int round = 0;
    int64_t row = (int64_t)blockIdx.x * TEAMS + team;
    auto row_stat = [&](int64_t q) {
        float2 v = make_float2(0.f, 0.f);
        if (q < N) v = stat[q];
        return v;
    };
    float2 st = row_stat(row), st_next = row_stat(row + step);
    H held;
    if (st.y != 0.f) held.load(scores + row * lds, K, t);
    for (; row < N; row += step) {
        const float m = st.x, r = st.y;
        float d[V];
        if (r != 0.f) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = held.at(i);
        }
        st = st_next;
        if (st.y != 0.f) held.load(scores + (row + step) * lds, K, t);
        st_next = row_stat(row + 2 * step);
        if (r == 0.f) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 0.f;
        } else {
            float ref = -INFINITY, dot = 0.f, mass = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) ref = d[i] == m ? fmaxf(ref, a[i]) : ref;
            ref = lbm::group_best<LW>(ref);
            const bool best = ref > -INFINITY;
            if (W > 1 && !best) ref = 0.f;
            RowExp(m).template apply<V>(d);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dot = fmaf(d[i], a[i] - ref, dot);
                if constexpr (W > 1) mass += d[i];
            }
            dot = lbm::group_total<LW>(dot) * r;
            if constexpr (W > 1) {                       // p.(a - ref of the best score), from each wave's own reference
                mass = lbm::group_total<LW>(mass) * r;
                if ((threadIdx.x & 63) == 0) s_x[round][wave] = make_float4(dot, mass, ref, best ? 1.f : 0.f);
                __syncthreads();
                float4 xs[W];
                ref = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    xs[w] = s_x[round][w];
                    ref = xs[w].w != 0.f ? fmaxf(ref, xs[w].z) : ref;
                }
                dot = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) dot += fmaf(xs[w].z - ref, xs[w].y, xs[w].x);
                round ^= 1;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] *= ((a[i] - ref) - dot) * (r * inv_m);
        }
        T* out = ds + row * (int64_t)K;
#pragma unroll
        for (int c = 0; c < V / H::E; ++c) {
            const int col = (c * L + t) * H::E;
            if (col < K) store_pack<T, H::E>(out + col, d + H::E * c);
        }
    }
}

// E scores at a time: aligned base and rows, and the last access of a row ends with it
template <typename T, int V>
bool vec_ok(const void* p, int64_t ld, int K) {
    constexpr int E = Held<T, V, 64, true>::E;
    return (uintptr_t)p % (E * sizeof(T)) == 0 && ld % E == 0 && K % E == 0;
}

// CALL(V, L): V scores in each of the L = lanes_for(K) lanes of a row
#define LBM_BALANCE_SIZES(CALL)       \
    if (K <= 8) CALL(1, 8);           \
    else if (K <= 64) CALL(4, 16);    \
    else if (K <= 128) CALL(4, 32);   \
    else if (K <= 512) CALL(8, 64);   \
    else if (K <= 1024) CALL(16, 64); \
    else if (K <= 2048) CALL(32, 64); \
    else if (K <= 4096) CALL(16, 256); \
    else CALL(32, 256);

template <typename T>
int run_rows(const void* scores, int64_t lds, const int64_t* codes, int slots, const uint8_t* keep, float2* stat, float* part, unsigned* cnt,
             unsigned* rows, int64_t G, int64_t N, int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    const size_t shm = (size_t)K * 4 * (256 / lanes_for(K));
#define LBM_ROWS(V, L)                                                                                                             \
    hipLaunchKernelGGL((vec_ok<T, V>(scores, lds, K) ? balance_rows_kernel<T, V, L, true> : balance_rows_kernel<T, V, L, false>), \
                       dim3((unsigned)G), dim3(256), shm, st, s, lds, codes, slots, keep, stat, part, cnt, rows, N, K)
    LBM_BALANCE_SIZES(LBM_ROWS)
#undef LBM_ROWS
    return lbm::check_launch("lbm_code_balance");
}

template <typename T>
int run_grad(const void* scores, int64_t lds, const float2* stat, const int64_t* counts, const double* totals, const float* g_loss,
             const float* g_mean, void* ds, int64_t G, int64_t N, int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    T* o = static_cast<T*>(ds);
#define LBM_GRAD(V, L)                                                                                                      \
    hipLaunchKernelGGL((vec_ok<T, V>(scores, lds, K) && vec_ok<T, V>(ds, K, K) ? balance_grad_kernel<T, V, L, true>        \
                                                                              : balance_grad_kernel<T, V, L, false>),      \
                       dim3((unsigned)G), dim3(256), 0, st, s, lds, stat, counts, totals, g_loss, g_mean, o, N, K)
    LBM_BALANCE_SIZES(LBM_GRAD)
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
    double* sum2 = reinterpret_cast<double*>(ws + p.off_sum2);
    unsigned long long* cnt2 = reinterpret_cast<unsigned long long*>(ws + p.off_cnt2);
    const int groups = (K + kJoinCols - 1) / kJoinCols;
    hipStream_t st = lbm::as_stream(stream);
    int rc = LBM_OK;
#define LBM_CALL(T) rc = run_rows<T>(scores, lds, codes_or_null, slots, keep_or_null, reinterpret_cast<float2*>(row_stat), part, cnt, rows, p.G, N, K, st)
    LBM_CODE_TYPES(dtype, LBM_CALL);
#undef LBM_CALL
    if (rc != LBM_OK) return rc;
    hipLaunchKernelGGL(balance_join_kernel, dim3((unsigned)groups, (unsigned)p.S), dim3(256), 0, st, part, cnt, sum2, cnt2, p.G, K);
    hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(kFinish), 0, st, sum2, cnt2, rows, mean, counts, loss, totals, p.S, p.G, K);
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
    LBM_REQUIRE(((uintptr_t)row_stat & 7) == 0, LBM_EINVAL, "%s: row_stat must be 8-byte aligned", what);
    LBM_REQUIRE(N <= 1 || lds >= 0, LBM_EINVAL, "%s: negative row stride", what);
    const int64_t T = 256 / lanes_for(K), cap = T >= 4 ? 2048 : (K <= 4096 ? 1024 : 512);
    int64_t G = (N + T - 1) / T;
    if (G > cap) G = cap;
    int rc = LBM_OK;
#define LBM_CALL(T) rc = run_grad<T>(scores, lds, reinterpret_cast<const float2*>(row_stat), counts, totals, g_loss_or_null, g_mean_or_null, dscores, G, N, K, lbm::as_stream(stream))
    LBM_CODE_TYPES(dtype, LBM_CALL);
#undef LBM_CALL
    return rc;
}
