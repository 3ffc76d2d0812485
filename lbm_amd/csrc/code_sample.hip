// One code per row, drawn with a given uniform number: temperature, top-k, top-p and min-p over a row of scores.
//
//   w_k = exp((s_k - max s) / T) in 64 bits (so the best code's weight is 1);   T = 0: the best code, lowest index
//   top-k: the k best scores stay (equal scores: lowest index first)
//   top-p: in descending order (equal scores: lowest index first) a code stays while the weights before it sum to less than p times the sum
//          of what top-k left
//   min-p: a code stays if w_k >= min_p
//   answer: the first index at which the running sum of what stayed exceeds u times its total
// Scores of +inf share all the weight, whatever T; NaN counts as -inf; a row without a score above -inf answers -1.
//
// The definition is one of real numbers: which side of a border a row falls on must not depend on how the sums were formed.  Weights and the
// sums that decide are therefore 64-bit (an fp64 operation issues as fast as an unpacked fp32 one here), and the answers equal any other
// 64-bit evaluation's but where a border is met to 1e-15.
//
// Borders are found without sorting: a border is a score, and how many scores (what weight) lie at or above a trial score is one pass over the
// row's registers.  Trial scores halve the interval by value, then, for scores that lie too close together or are equal, by ordered bit
// patterns.  The search for top-p sums fp32 copies of the weights (a third of the instructions); the score it ends at is then checked with
// the 64-bit sums and moved where they disagree.
#include "code_rows.h"

namespace {

struct Params {           // per-row arrays where not NULL, else the value
    const float *T_row, *p_row, *min_row;
    const int* k_row;
    double T, top_p, min_p;
    int top_k;
};

// order-preserving bit pattern of a score (no NaN, no -0)
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_score(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// 2^t for t <= 0 (NaN: 0): t = n + f with |f| <= 1/2, 2^f by the polynomial of degree 11 that interpolates it at the Chebyshev nodes of
// [-1/2, 1/2] (2e-17 relative in exact arithmetic): 18 instructions
__device__ __forceinline__ double exp2_f64(double t) {
    t = fmax(t, -1100.0);
    const double n = rint(t), f = t - n;
    double p = 4.4558179083360645e-10;
    p = fma(p, f, 7.074194297288521e-09);
    p = fma(p, f, 1.0178057087733941e-07);
    p = fma(p, f, 1.3215432535912375e-06);
    p = fma(p, f, 1.5252733841556773e-05);
    p = fma(p, f, 0.00015403530463724353);
    p = fma(p, f, 0.001333355814640647);
    p = fma(p, f, 0.009618129107587256);
    p = fma(p, f, 0.055504108664821625);
    p = fma(p, f, 0.24022650695910158);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

// A row in the registers of a team of W waves, V scores a thread; slots ascend by chunk of 256 W, thread, i.
template <int V, int W>
struct Row {
    float v[V];           // -inf once a code is out
    double w[V];
    int t;                // thread of the team
    double* s_d;          // LDS, W > 1: [2][W], [2][W], [V / 4][W]
    int* s_i;
    double* s_tot;
    int rd = 0, ri = 0;

    __device__ __forceinline__ int slot(int i) const { return ((i >> 2) * 64 * W + t) * 4 + (i & 3); }
    __device__ __forceinline__ int lane() const { return threadIdx.x & 63; }
    __device__ __forceinline__ int wave() const { return W == 1 ? 0 : (int)(threadIdx.x >> 6); }

    __device__ __forceinline__ int join(int c) { return lbm::team_join<int, W>(c, s_i, ri, lbm::OpAdd()); }
    __device__ __forceinline__ double sum(double x) { return lbm::team_join<double, W>(lbm::wave_total(x), s_d, rd, lbm::OpAdd()); }
    __device__ __forceinline__ float best(float x) {
        x = lbm::wave_best(x);
        if constexpr (W > 1) x = __int_as_float(lbm::team_join<int, W>(__float_as_int(x), s_i, ri, [](int a, int b) {
            return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
        }));
        return x;
    }
    __device__ __forceinline__ int count_from(float x) {          // scores >= x
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(v[i] >= x));
        return join(c);
    }
    __device__ __forceinline__ int count_equal(float x) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(v[i] == x));
        return join(c);
    }
    __device__ __forceinline__ double weight_above(float x) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i] > x ? w[i] : 0.0;
        return sum(s);
    }
    // fp32 weight (from the copies wf) and number of the scores >= x
    __device__ __forceinline__ float probe(const float* wf, float x, int* n) {
        float s = 0.f;
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool in = v[i] >= x;
            s += in ? wf[i] : 0.f;
            c += __popcll(__ballot(in));
        }
        s = lbm::wave_total(s);
        if constexpr (W > 1) {                                    // both in one exchange
            const double both = lbm::team_join<double, W>(__hiloint2double(c, __float_as_int(s)), s_d, rd, [](double a, double b) {
                return __hiloint2double(__double2hiint(a) + __double2hiint(b),
                                        __float_as_int(__int_as_float(__double2loint(a)) + __int_as_float(__double2loint(b))));
            });
            c = __double2hiint(both);
            s = __int_as_float(__double2loint(both));
        }
        *n = c;
        return s;
    }
    __device__ __forceinline__ float next_below(float x) {
        float b = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) b = fmaxf(b, v[i] < x ? v[i] : -INFINITY);
        return best(b);
    }
    __device__ __forceinline__ float next_above(float x) {
        float b = -INFINITY;                                      // of the negatives
#pragma unroll
        for (int i = 0; i < V; ++i) b = fmaxf(b, v[i] > x ? -v[i] : -INFINITY);
        return -best(b);
    }
    __device__ __forceinline__ void drop_below(float x) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = v[i] < x ? 0.0 : w[i];
            v[i] = v[i] < x ? -INFINITY : v[i];
        }
    }
    // of the scores equal to x only the first n in index order stay: where a border cuts through equal scores
    __device__ void keep_first_equal(float x, int n) {
        int base = 0;
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine += v[4 * c + i] == x ? 1 : 0;
            const int scan = lbm::wave_scan<int>(mine, 0, lbm::OpAdd());
            int before = base + scan - mine, total = lbm::lane_value(scan, 63);
            if constexpr (W > 1) {
                int* s = s_i + ri * W;
                ri ^= 1;
                if (lane() == 0) s[wave()] = total;
                __syncthreads();
                total = 0;
#pragma unroll
                for (int q = 0; q < W; ++q) {
                    if (q < wave()) before += s[q];
                    total += s[q];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v[4 * c + i] == x) {
                    if (before >= n) {
                        w[4 * c + i] = 0.0;
                        v[4 * c + i] = -INFINITY;
                    }
                    ++before;
                }
            base += total;
        }
    }
    // m: the best score; c = log2(e) / T
    __device__ __forceinline__ void weigh(float m, double c) {
        if (m == INFINITY) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = v[i] == m ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = exp2_f64(((double)v[i] - (double)m) * c);
        }
    }
    __device__ __forceinline__ double weight() {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += w[i];
        return sum(s);
    }
};

constexpr int kByValue = 12;             // steps that halve by value; 32 by bit pattern end the search whatever the scores
constexpr int kSteps = kByValue + 32;

// trial score of step `it` strictly inside (lo, hi); false when no number lies between
__device__ __forceinline__ bool trial(int it, float lo, float hi, float* mid) {
    if (it < kByValue) {
        *mid = 0.5f * lo + 0.5f * hi;
        if (*mid > lo && *mid < hi) return true;
    }
    const unsigned kl = order_key(lo), kh = order_key(hi);
    if (kh - kl <= 1u) return false;
    *mid = key_score(kl + (kh - kl) / 2);
    return true;
}

// the k best scores stay; lo: the lowest score, m: the best one
template <int V, int W>
__device__ __forceinline__ void keep_top_k(Row<V, W>& R, float lo, float m, int k) {
    int c = R.count_from(m);
    float b = m;
    if (c < k) {
        float hi = m;                    // fewer than k from hi on
        c = 0;
        for (int it = 0; it < kSteps; ++it) {
            float mid;
            if (!trial(it, lo, hi, &mid)) break;
            c = R.count_from(mid);
            if (c >= k) lo = mid;
            else hi = mid;
            if (c == k) break;
        }
        b = lo;
        if (c != k) c = R.count_from(b);
    }
    if (c > k) R.keep_first_equal(b, k - (c - R.count_equal(b)));
    R.drop_below(b);
}

// scores below this one weigh together less than (1 - p) of a total that is 1 at least: K exp((s - m) / T) < 1 - p, with room for the rounding
__device__ __forceinline__ float top_p_floor(float m, float lo, double temp, double top_p, int K) {
    const double f = (double)m + temp * (double)(logf((float)((1.0 - top_p) / K)) - 1e-3f);
    return f > (double)lo && f < (double)m ? (float)f : lo;
}

// the codes of the smallest descending prefix that reaches `target` stay; the scores >= lo reach it, lo <= m
template <int V, int W>
__device__ __forceinline__ void keep_top_p(Row<V, W>& R, float lo, float m, double target, double c) {
    float wf[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wf[i] = (float)R.w[i];
    float l = lo, hi = m, b = m;
    int n_hi;
    if (R.probe(wf, m, &n_hi) < (float)target) {
        for (int it = 0; it < kSteps; ++it) {
            float mid;
            int n;
            if (!trial(it, l, hi, &mid)) break;
            if (R.probe(wf, mid, &n) >= (float)target) {
                l = mid;
                if (n - n_hi == 1) break;
            } else {
                hi = mid;
                n_hi = n;
            }
        }
        b = R.next_below(hi);
    }
    // the 64-bit sums decide: above b lies less than the target, with b's scores at least it
    double above = 0.0, wb = 1.0;
    int eq = 0;
    bool settled = false;
    for (int tries = 0; tries < 4 && !settled; ++tries) {
        above = R.weight_above(b);
        eq = R.count_equal(b);
        wb = b == m ? 1.0 : exp2_f64(((double)b - (double)m) * c);
        settled = true;
        if (above >= target && b < m) {
            b = R.next_above(b);
            settled = false;
        } else if (above + eq * wb < target) {
            const float below = R.next_below(b);
            if (below != -INFINITY) {
                b = below;
                settled = false;
            }
        }
    }
    if (!settled) {                      // fp32 sums led too far astray (a border among weights below 1e-7 of the total): search on the 64-bit sums
        l = lo;
        hi = m;
        for (int it = 0; it < kSteps; ++it) {
            float mid;
            if (!trial(it, l, hi, &mid)) break;
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) s += R.v[i] >= mid ? R.w[i] : 0.0;
            if (R.sum(s) >= target) l = mid;
            else hi = mid;
        }
        b = R.next_below(hi);
        above = R.weight_above(b);
        eq = R.count_equal(b);
        wb = exp2_f64(((double)b - (double)m) * c);
    }
    double keep = ceil((target - above) / wb);
    keep = keep >= 1.0 ? fmin(keep, 1e9) : 1.0;
    if (eq > (int)keep) R.keep_first_equal(b, (int)keep);
    R.drop_below(b);
}

// the slot the draw falls on
template <int V, int W>
__device__ __forceinline__ int draw(Row<V, W>& R, double u) {
    double inc[V / 4], s4[V / 4], base[V / 4], total = 0.0;
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        s4[c] = (R.w[4 * c] + R.w[4 * c + 1]) + (R.w[4 * c + 2] + R.w[4 * c + 3]);
        inc[c] = lbm::wave_scan<double>(s4[c], 0.0, lbm::OpAdd());
    }
    if constexpr (W == 1) {
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            base[c] = total;
            total += lbm::lane_value(inc[c], 63);
        }
    } else {
        if (R.lane() == 63)
#pragma unroll
            for (int c = 0; c < V / 4; ++c) R.s_tot[c * W + R.wave()] = inc[c];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < V / 4; ++c)
#pragma unroll
            for (int q = 0; q < W; ++q) {
                if (q == R.wave()) base[c] = total;
                total += R.s_tot[c * W + q];
            }
    }
    const double goal = u * total;
    int hit = 0x7fffffff;
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        const unsigned long long over = __ballot(base[c] + inc[c] > goal && s4[c] > 0.0);
        if (hit == 0x7fffffff && over != 0) {
            const int first = __ffsll((long long)over) - 1;
            // in that lane: the first weight that carries the sum past the goal, or its last one where rounding keeps all from it
            double run = base[c] + (first == 0 ? 0.0 : lbm::lane_value(inc[c], first == 0 ? 0 : first - 1));
            int at = 0;
            bool done = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double w = lbm::lane_value(R.w[4 * c + i], first);
                run += w;
                if (!done && w > 0.0) {
                    at = i;
                    done = run > goal;
                }
            }
            hit = (c * 64 * W + R.wave() * 64 + first) * 4 + at;
        }
    }
    hit = lbm::team_join<int, W>(hit, R.s_i, R.ri, lbm::OpMin());
    if (hit == 0x7fffffff) {             // u of 1 or more, or NaN: the last code that stayed
        int last = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) last = R.w[i] > 0.0 ? R.slot(i) : last;
        last = -lbm::wave_first(-last);
        hit = lbm::team_join<int, W>(last, R.s_i, R.ri, lbm::OpMax());
    }
    return hit;
}

struct Setting {
    double temp, c, top_p, min_p, u;
    int top_k;
};

// everything behind the best score m; lo: the lowest score above -inf; total: the weight top-p refers to where it is not that of this row's
// own scores (negative: it is)
template <int V, int W>
__device__ __forceinline__ int settle(Row<V, W>& R, const Setting& s, float lo, float m, int K, bool weighed, double total) {
    if (s.top_k > 0 && s.top_k < K) keep_top_k<V, W>(R, lo, m, s.top_k);
    if (!weighed) R.weigh(m, s.c);
    if (s.top_p < 1.0) {
        if (total < 0.0) total = R.weight();
        if (m == INFINITY) {             // equal weights of 1
            const double keep = ceil(s.top_p * total);
            R.keep_first_equal(m, keep < 1.0 ? 1 : (int)keep);
        } else {
            keep_top_p<V, W>(R, top_p_floor(m, lo, s.temp, s.top_p, K), m, s.top_p * total, s.c);
        }
    }
    if (s.min_p > 0.0) {
        const double lim = fmin(s.min_p, 1.0);
#pragma unroll
        for (int i = 0; i < V; ++i) R.w[i] = R.w[i] >= lim ? R.w[i] : 0.0;
    }
    return draw<V, W>(R, s.u);
}

constexpr int kCand = 512;               // scores one wave finishes alone (8 a lane)

template <typename T, int V, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void code_sample_kernel(const T* __restrict__ scores, int64_t lds, int vec,
                                                                           const float* __restrict__ u, Params par,
                                                                           const uint8_t* __restrict__ allowed, int64_t allowed_ld,
                                                                           int64_t* __restrict__ out, int64_t N, int K) {
    __shared__ double s_d[2 * W];
    __shared__ int s_i[2 * W];
    __shared__ double s_tot[V / 4 * W];
    const int team = W == 1 ? threadIdx.x >> 6 : 0;
    const int64_t row = (int64_t)blockIdx.x * (W == 1 ? 4 : 1) + team;
    if (row >= N) return;                // W = 1: a whole wave, and no barriers follow
    Row<V, W> R;
    R.t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    R.s_d = s_d;
    R.s_i = s_i;
    R.s_tot = s_tot;
    lbm::load_row<T, V, W>(scores + row * lds, K, R.t, vec, R.v);
    if (allowed != nullptr) {
        const uint8_t* a = allowed + row * allowed_ld;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (R.slot(i) < K && a[R.slot(i)] == 0) R.v[i] = -INFINITY;
    }
    Setting s;
    s.temp = par.T_row != nullptr ? (double)par.T_row[row] : par.T;
    s.top_p = par.p_row != nullptr ? (double)par.p_row[row] : par.top_p;
    s.min_p = par.min_row != nullptr ? (double)par.min_row[row] : par.min_p;
    s.top_k = par.k_row != nullptr ? par.k_row[row] : par.top_k;
    s.u = (double)u[row];

    float m = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        R.v[i] = R.v[i] != R.v[i] ? -INFINITY : R.v[i] + 0.f;     // + 0: -0 and 0 are one score
        m = fmaxf(m, R.v[i]);
        lo = fminf(lo, R.v[i] == -INFINITY ? INFINITY : R.v[i]);
    }
    m = R.best(m);
    if (m == -INFINITY) {
        if (R.t == 0) out[row] = -1;
        return;
    }
    if (!(s.temp > 0.0)) {
        int first = 0x7fffffff;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) first = R.v[i] == m ? R.slot(i) : first;
        first = lbm::team_join<int, W>(lbm::wave_first(first), R.s_i, R.ri, lbm::OpMin());
        if (R.t == 0) out[row] = first;
        return;
    }
    s.c = fmin(1.4426950408889634 / s.temp, 1e300);
    const bool by_k = s.top_k > 0 && s.top_k < K;
    if (by_k || s.top_p < 1.0) lo = -R.best(-lo);
    const int hit = settle<V, W>(R, s, lo, m, K, false, -1.0);
    if (R.t == 0) out[row] = hit;
}

template <typename T>
int run_sample(const void* scores, int64_t lds, const float* u, const Params& par, const uint8_t* allowed, int64_t allowed_ld, int64_t* out,
               int64_t N, int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    const int vec = ((uintptr_t)scores % (4 * sizeof(T))) == 0 && (lds & 3) == 0 && (K & 3) == 0 ? 1 : 0;
#define LBM_SAMPLE(V, W)                                                                                                                  \
    hipLaunchKernelGGL((code_sample_kernel<T, V, W>), dim3((unsigned)(W == 1 ? (N + 3) / 4 : N)), dim3(W == 1 ? 256 : 64 * W), 0, st, s, lds, \
                       vec, u, par, allowed, allowed_ld, out, N, K)
    if (K <= 256) LBM_SAMPLE(4, 1);
    else if (K <= 512) LBM_SAMPLE(8, 1);
    else if (K <= 1024) LBM_SAMPLE(16, 1);
    else if (K <= 2048) LBM_SAMPLE(8, 4);
    else if (K <= 4096) LBM_SAMPLE(16, 4);
    else LBM_SAMPLE(8, 16);
#undef LBM_SAMPLE
    return lbm::check_launch("lbm_code_sample");
}

constexpr int kMaxK = 8192;   // 16 waves x 64 lanes x 8 scores

}  // namespace

// shared with vq.hip: usage counts of int64 codes, added to hist
int lbm_vq_hist_launch(const int64_t* idx, unsigned long long* hist, int64_t N, int K, hipStream_t st);

extern "C" int lbm_code_sample(const void* scores, int32_t dtype, int64_t lds, const float* u, const float* temperature_row_or_null,
                               double temperature, const int32_t* top_k_row_or_null, int32_t top_k, const float* top_p_row_or_null,
                               double top_p, const float* min_p_row_or_null, double min_p, const uint8_t* allowed_or_null,
                               int64_t allowed_ld, int64_t* codes, unsigned long long* hist_or_null, int64_t N, int32_t K,
                               lbm_stream_t stream) {
    const char* what = "lbm_code_sample";
    LBM_REQUIRE(N >= 0 && K >= 1, LBM_EINVAL, "%s: bad sizes (N=%lld K=%d)", what, (long long)N, K);
    LBM_REQUIRE(K <= kMaxK, LBM_EUNSUPPORTED, "%s: K=%d > %d", what, K, kMaxK);
    LBM_REQUIRE(dtype == LBM_F32 || dtype == LBM_F16 || dtype == LBM_BF16, LBM_EINVAL, "%s: unknown score type %d", what, dtype);
    LBM_REQUIRE(temperature_row_or_null || temperature >= 0.0, LBM_EINVAL, "%s: temperature must be >= 0", what);
    LBM_REQUIRE(top_k_row_or_null || top_k >= 0, LBM_EINVAL, "%s: top_k must be >= 0 (0: all codes)", what);
    LBM_REQUIRE(top_p_row_or_null || (top_p >= 0.0 && top_p <= 1.0), LBM_EINVAL, "%s: top_p must lie in [0, 1]", what);
    LBM_REQUIRE(min_p_row_or_null || (min_p >= 0.0 && min_p <= 1.0), LBM_EINVAL, "%s: min_p must lie in [0, 1]", what);
    if (N == 0) return LBM_OK;
    LBM_REQUIRE(scores && u && codes, LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(N <= 0x7fffffffLL, LBM_EUNSUPPORTED, "%s: N must be < 2^31", what);
    LBM_REQUIRE(N <= 1 || (lds >= 0 && allowed_ld >= 0), LBM_EINVAL, "%s: negative row stride", what);
    const Params par{temperature_row_or_null, top_p_row_or_null, min_p_row_or_null, top_k_row_or_null, temperature, top_p, min_p, top_k};
    hipStream_t st = lbm::as_stream(stream);
    int rc = LBM_OK;
#define LBM_CALL(T) rc = run_sample<T>(scores, lds, u, par, allowed_or_null, allowed_ld, codes, N, K, st)
    LBM_CODE_TYPES(dtype, LBM_CALL);
#undef LBM_CALL
    if (rc == LBM_OK && hist_or_null != nullptr) rc = lbm_vq_hist_launch(codes, hist_or_null, N, K, st);
    return rc;
}
