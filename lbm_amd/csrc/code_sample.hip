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
// The definition is one of real numbers: which side of a border a row falls on must not depend on how the sums were formed.  Sums and weights
// are therefore 64-bit (an fp64 operation issues as fast as an unpacked fp32 one here), and the answers equal any other 64-bit evaluation's
// but where a border is met to 1e-15.
//
// Borders are found without sorting: a border is a score, and how many scores (what weight) lie at or above a trial score is one pass over the
// row's registers.  The trial interval is halved by value first, which separates neighbouring scores in about log2(K) + 4 steps, and by
// the scores' ordered bit patterns after 16 steps, which ends in 32 more whatever the values.
#include "code_rows.h"

namespace {

using lbm::OpAdd;
using lbm::OpMax;
using lbm::OpMin;

struct Params {           // per-row arrays where not NULL, else the value
    const float *T_row, *p_row, *min_row;
    const int* k_row;
    double T, top_p, min_p;
    int top_k;
};

// order-preserving bit pattern of a score (no NaN)
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_score(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <int V, int W>
struct Row {
    float v[V];
    double w[V];          // 0 once a code is out
    int t;
    double* s_d;          // [2][W]
    int* s_i;             // [2][W]
    double* s_tot;        // [V/4 * W]
    int rd = 0, ri = 0;

    __device__ __forceinline__ int col(int i) const { return ((i >> 2) * 64 * W + t) * 4 + (i & 3); }

    // number of scores >= x / their weight
    __device__ __forceinline__ int count_from(float x) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(v[i] >= x));
        if constexpr (W > 1) {
            int* slot = s_i + ri * W;
            ri ^= 1;
            if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = c;
            __syncthreads();
            c = slot[0];
#pragma unroll
            for (int q = 1; q < W; ++q) c += slot[q];
        }
        return c;
    }
    __device__ __forceinline__ double weight_from(float x) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i] >= x ? w[i] : 0.0;
        return lbm::team_reduce<double, W>(s, s_d, rd, OpAdd());
    }
    // how many codes with score == x come before mine in index order, i = my value: only where a border cuts through equal scores
    __device__ void keep_first_equal(float x, int n) {
        int base = 0;
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine += v[4 * c + i] == x ? 1 : 0;
            int scan = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int up = __shfl_up(scan, o, 64);
                if ((threadIdx.x & 63) >= o) scan += up;
            }
            int before = base + scan - mine, total = __shfl(scan, 63, 64);
            if constexpr (W > 1) {
                int* slot = s_i + ri * W;
                ri ^= 1;
                if ((threadIdx.x & 63) == 63) slot[threadIdx.x >> 6] = scan;
                __syncthreads();
                total = 0;
#pragma unroll
                for (int q = 0; q < W; ++q) {
                    if (q < (int)(threadIdx.x >> 6)) before += slot[q];
                    total += slot[q];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v[4 * c + i] == x) {
                    if (before >= n) w[4 * c + i] = 0.0;
                    ++before;
                }
            base += total;
        }
    }
};

// The border score b of `enough(count or weight from x)`: enough holds at b and not above it.  lo: a score where it holds; hi: past the best.
// stop(x): an exact hit at x, nothing left to separate.
template <typename F>
__device__ __forceinline__ float find_border(float lo, float hi, F enough) {
    // enough(x) returns 0: not enough at x, 1: enough, 2: enough and x separates exactly (every score >= x stays)
    for (int it = 0; it < 48; ++it) {
        float mid;
        if (it < 16) {
            mid = 0.5f * lo + 0.5f * hi;
            if (!(mid > lo && mid < hi)) continue;
        } else {
            const unsigned kl = order_key(lo), kh = order_key(hi);
            if (kh - kl <= 1u) break;
            mid = key_score(kl + (kh - kl) / 2);
        }
        const int e = enough(mid);
        if (e == 2) return mid;
        if (e == 1) lo = mid;
        else hi = mid;
    }
    return lo;
}

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
    if (row >= N) return;
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
            if (R.col(i) < K && a[R.col(i)] == 0) R.v[i] = -INFINITY;
    }
    const double temp = par.T_row != nullptr ? (double)par.T_row[row] : par.T;
    const double top_p = par.p_row != nullptr ? (double)par.p_row[row] : par.top_p;
    const double min_p = par.min_row != nullptr ? (double)par.min_row[row] : par.min_p;
    const int top_k = par.k_row != nullptr ? par.k_row[row] : par.top_k;
    const double uu = (double)u[row];

    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        R.v[i] = R.v[i] != R.v[i] ? -INFINITY : R.v[i] + 0.f;   // + 0: -0 and 0 are one score
        m = fmaxf(m, R.v[i]);
    }
    float mn = INFINITY;                                        // lowest score above -inf
#pragma unroll
    for (int i = 0; i < V; ++i) mn = R.v[i] == -INFINITY ? mn : fminf(mn, R.v[i]);
    {
        const double mm = lbm::team_reduce<double, W>((double)m, R.s_d, R.rd, OpMax());
        m = (float)mm;
    }
    if (m == -INFINITY) {
        if (R.t == 0) out[row] = -1;
        return;
    }
    if (!(temp > 0.0)) {
        int best = 0x7fffffff;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) best = R.v[i] == m ? R.col(i) : best;
        best = lbm::team_reduce<int, W>(best, R.s_i, R.ri, OpMin());
        if (R.t == 0) out[row] = best;
        return;
    }
    mn = (float)lbm::team_reduce<double, W>((double)mn, R.s_d, R.rd, OpMin());
#pragma unroll
    for (int i = 0; i < V; ++i)
        R.w[i] = R.v[i] == m ? 1.0 : (R.v[i] == -INFINITY || m == INFINITY ? 0.0 : exp(((double)R.v[i] - (double)m) / temp));

    // past the best score: the next float above it, +inf for the largest (a trial score there holds nothing unless m is +inf itself)
    const float above = m == INFINITY ? INFINITY : key_score(order_key(m) + 1u);
    if (top_k > 0 && top_k < K && m != INFINITY) {
        float b = mn;
        if (R.count_from(mn) > top_k) {
            b = find_border(mn, above, [&](float x) {
                const int c = R.count_from(x);
                return c == top_k ? 2 : (c > top_k ? 1 : 0);
            });
            const int over = R.count_from(b);
            if (over > top_k) {
                const int strictly = R.count_from(key_score(order_key(b) + 1u));
                R.keep_first_equal(b, top_k - strictly);
            }
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (R.v[i] < b) R.w[i] = 0.0;
        }
    } else if (top_k > 0 && top_k < K) {                        // scores of +inf: only they have weight
        R.keep_first_equal(INFINITY, top_k);
    }
    if (top_p < 1.0 && m != INFINITY) {
        const double target = top_p * R.weight_from(mn);
        const float b = find_border(mn, above, [&](float x) { return R.weight_from(x) >= target ? 1 : 0; });
        // scores above b weigh less than the target; of those equal to b the first n that it takes
        const float next = key_score(order_key(b) + 1u);
        const double strictly = b == m ? 0.0 : R.weight_from(next);
        const double at = b == m ? 1.0 : exp(((double)b - (double)m) / temp);
        double n = ceil((target - strictly) / at);
        n = n < 1.0 ? 1.0 : (n > 2e9 ? 2e9 : n);
        // equal scores that top-k took out stand behind those it left: the order is the same
        R.keep_first_equal(b, (int)n);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (R.v[i] < b) R.w[i] = 0.0;
    } else if (top_p < 1.0) {                                   // n equal weights of 1
        const double target = top_p * R.weight_from(INFINITY);
        double n = ceil(target);
        R.keep_first_equal(INFINITY, n < 1.0 ? 1 : (int)n);
    }
    if (min_p > 0.0) {
        const double lim = min_p < 1.0 ? min_p : 1.0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (R.w[i] < lim) R.w[i] = 0.0;
    }

    // running sums in index order: chunk, wave, lane
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6;
    double inc[V / 4];
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        double s = (R.w[4 * c] + R.w[4 * c + 1]) + (R.w[4 * c + 2] + R.w[4 * c + 3]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(s, o, 64);
            if (lane >= o) s += up;
        }
        inc[c] = s;
    }
    double base[V / 4], total = 0.0;
    if constexpr (W == 1) {
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            base[c] = total;
            total += __shfl(inc[c], 63, 64);
        }
    } else {
        if (lane == 63)
#pragma unroll
            for (int c = 0; c < V / 4; ++c) s_tot[c * W + wave] = inc[c];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < V / 4; ++c)
            for (int q = 0; q < W; ++q) {
                if (q == wave) base[c] = total;
                total += s_tot[c * W + q];
            }
    }
    const double goal = uu * total;
    int hit = 0x7fffffff, last = -1;
#pragma unroll
    for (int c = V / 4 - 1; c >= 0; --c) {
        double before = __shfl_up(inc[c], 1, 64);
        if (lane == 0) before = 0.0;
        double run = base[c] + before;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double w = R.w[4 * c + i];
            run += w;
            if (w > 0.0) {
                if (run > goal) hit = R.col(4 * c + i) < hit ? R.col(4 * c + i) : hit;
                if (R.col(4 * c + i) > last) last = R.col(4 * c + i);
            }
        }
    }
    hit = lbm::team_reduce<int, W>(hit, R.s_i, R.ri, OpMin());
    last = lbm::team_reduce<int, W>(last, R.s_i, R.ri, OpMax());
    if (R.t == 0) out[row] = hit <= last ? hit : last;
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
