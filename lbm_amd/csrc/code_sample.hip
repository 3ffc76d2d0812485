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
// row.  Rows in registers cut the range of scores into 64 parts at a time and sum each in LDS (384000 x 512, top-k 100: 586 -> 463 us
// against halving); longer rows halve it by trial scores.  Scores that lie too close together or are equal are left to ordered bit
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

// Scores in the registers of one wave, V a lane; slots ascend by chunk of 256, lane, i.
template <int V>
struct Row {
    float v[V];           // -inf once a code is out
    double w[V];

    static __device__ __forceinline__ int lane() { return threadIdx.x & 63; }
    static __device__ __forceinline__ int slot(int i) { return ((i >> 2) * 64 + lane()) * 4 + (i & 3); }

    __device__ __forceinline__ int count_from(float x) const {    // scores >= x
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(v[i] >= x));
        return c;
    }
    __device__ __forceinline__ int count_equal(float x) const {
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(v[i] == x));
        return c;
    }
    __device__ __forceinline__ double weight_above(float x) const {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[i] > x ? w[i] : 0.0;
        return lbm::wave_total(s);
    }
    // fp32 weight (from the copies wf) and number of the scores >= x
    __device__ __forceinline__ float probe(const float* wf, float x, int* n) const {
        float s = 0.f;
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool in = v[i] >= x;
            s += in ? wf[i] : 0.f;
            c += __popcll(__ballot(in));
        }
        *n = c;
        return lbm::wave_total(s);
    }
    __device__ __forceinline__ float next_below(float x) const {
        float b = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) b = fmaxf(b, v[i] < x ? v[i] : -INFINITY);
        return lbm::wave_best(b);
    }
    // lowest score >= x
    __device__ __forceinline__ float next_from(float x) const {
        float b = -INFINITY;                                      // of the negatives
#pragma unroll
        for (int i = 0; i < V; ++i) b = fmaxf(b, v[i] >= x ? -v[i] : -INFINITY);
        return -lbm::wave_best(b);
    }
    __device__ __forceinline__ float next_above(float x) const {
        float b = -INFINITY;                                      // of the negatives
#pragma unroll
        for (int i = 0; i < V; ++i) b = fmaxf(b, v[i] > x ? -v[i] : -INFINITY);
        return -lbm::wave_best(b);
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
            int before = base + scan - mine;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v[4 * c + i] == x) {
                    if (before >= n) {
                        w[4 * c + i] = 0.0;
                        v[4 * c + i] = -INFINITY;
                    }
                    ++before;
                }
            base += lbm::lane_value(scan, 63);
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
    __device__ __forceinline__ double weight() const {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += w[i];
        return lbm::wave_total(s);
    }
    __device__ __forceinline__ int first_of(float x) const {      // lowest slot of a score that is there
        int first = 0x7fffffff;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) first = v[i] == x ? slot(i) : first;
        return lbm::wave_first(first);
    }
};

constexpr int kByValue = 10;             // trial scores that halve by value; then by ordered bit pattern, which 32 end whatever the scores
constexpr int kSteps = 64;

// trial score of (lo, hi]: lo < hi
__device__ __forceinline__ float trial(int it, float lo, float hi) {
    if (it < kByValue) {
        const float mid = 0.5f * lo + 0.5f * hi;
        if (mid > lo && mid <= hi) return mid;
    }
    const unsigned kl = order_key(lo), kh = order_key(hi);
    return key_score(kl + (kh - kl + 1u) / 2);
}

// Where the sum over descending scores of [lo, m], lo < m, reaches `goal`: the range is cut into 64 equal parts, the parts' sums are taken in
// LDS (h[64], the wave's own) and added up over the lanes, and the part in which the goal is reached is cut again, three times at most or
// until it holds one score.  A level costs about three trial scores and does the work of six.  *lowest, *highest: the last part's scores;
// *upto: the sum with all of them.  Parts are monotone in the score whatever rounds, so only sums that round (A = float) can mislead.
template <typename A, int V, typename Weight>
__device__ __forceinline__ int narrow(const Row<V>& R, float lo, float m, A goal, A* h, Weight weight, float* lowest, float* highest, A* upto) {
    const int lane = R.lane();
    const float scale = 64.f / (0.5f * m - 0.5f * lo);
    float part[V];                       // < 0: not in it
#pragma unroll
    for (int i = 0; i < V; ++i) part[i] = R.v[i] >= lo ? fminf(fmaxf((0.5f * m - 0.5f * R.v[i]) * scale, 0.f), 63.9999f) : -1.f;
    A base = A(0);
    int n = 0;
    for (int level = 0; level < 3; ++level) {
        h[lane] = A(0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (part[i] >= 0.f) atomicAdd(&h[(int)part[i]], weight(i));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const A mine = h[lane];
        const A sum = lbm::wave_scan<A>(mine, A(0), lbm::OpAdd());
        const unsigned long long full = __ballot(mine > A(0)), over = __ballot(base + sum >= goal) & full;
        const int at = over != 0 ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)full);
        *upto = base + lbm::lane_value(sum, at);
        base = at == 0 ? base : base + lbm::lane_value(sum, at - 1);
        n = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool in = part[i] >= 0.f && (int)part[i] == at;
            part[i] = in ? fminf((part[i] - (float)at) * 64.f, 63.9999f) : -1.f;
            n += __popcll(__ballot(in));
        }
        if (n == 1) break;
    }
    float hi = -INFINITY, low = INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        hi = fmaxf(hi, part[i] >= 0.f ? R.v[i] : -INFINITY);
        low = fminf(low, part[i] >= 0.f ? R.v[i] : INFINITY);
    }
    *highest = lbm::wave_best(hi);
    *lowest = n == 1 ? *highest : -lbm::wave_best(-low);
    return n;
}

// the k best scores stay; lo: a score at or below all of them, m: the best one
template <int V>
__device__ __forceinline__ void keep_top_k(Row<V>& R, float lo, float m, int k, int* h) {
    int c = 0;
    if (lo < m) {
        float low, hi;                   // the border is one of the scores in [low, hi]
        narrow<int>(R, lo, m, k, h, [](int) { return 1; }, &low, &hi, &c);
        lo = low;
        if (c != k) {
            for (int it = kByValue; it < kSteps && lo < hi; ++it) {       // between scores that are there: equal ones end the search
                const float mid = trial(it, lo, hi);
                if (R.count_from(mid) >= k) lo = R.next_from(mid);
                else hi = R.next_below(mid);
            }
            c = R.count_from(lo);
        }
    } else {
        c = R.count_from(lo);
    }
    if (c > k) R.keep_first_equal(lo, k - (c - R.count_equal(lo)));
    R.drop_below(lo);
}

// scores below this one weigh together less than (1 - p) of a total that is 1 at least: K exp((s - m) / T) < 1 - p, with room for the rounding
__device__ __forceinline__ float top_p_floor(float m, float lo, double temp, double top_p, int K) {
    const double f = (double)m + temp * (double)(logf((float)((1.0 - top_p) / K)) - 1e-3f);
    return f > (double)lo && f < (double)m ? (float)f : lo;
}

// the codes of the smallest descending prefix that reaches `target` > 1 stay; the scores >= lo reach it, lo <= m
template <int V>
__device__ __forceinline__ void keep_top_p(Row<V>& R, float lo, float m, double target, double c, float* h) {
    float wf[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wf[i] = (float)R.w[i];
    float b = m;
    if (lo < m) {
        float l, up;
        narrow<float>(R, lo, m, (float)target, h, [&](int i) { return wf[i]; }, &l, &b, &up);
        for (int it = kByValue; it < kSteps && l < b; ++it) {     // between scores that are there: equal ones end the search
            const float mid = trial(it, l, b);
            int n;
            if (R.probe(wf, mid, &n) >= (float)target) l = R.next_from(mid);
            else b = R.next_below(mid);
        }
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
        float l = R.next_from(lo);
        b = m;
        for (int it = 0; it < kSteps && l < b; ++it) {
            const float mid = trial(it, l, b);
            if (R.weight_above(R.next_below(mid)) >= target) l = R.next_from(mid);
            else b = R.next_below(mid);
        }
        above = R.weight_above(b);
        eq = R.count_equal(b);
        wb = exp2_f64(((double)b - (double)m) * c);
    }
    double keep = ceil((target - above) / wb);
    keep = keep >= 1.0 ? fmin(keep, 1e9) : 1.0;
    if (eq > (int)keep) R.keep_first_equal(b, (int)keep);
    R.drop_below(b);
}

// four weights at lane `first` that carry a running sum past the goal: which of them does (its last one where rounding keeps all from it)
__device__ __forceinline__ int crossing(double run, double goal, const double* w4, int first) {
    int at = 0;
    bool done = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double w = lbm::lane_value(w4[i], first);
        run += w;
        if (!done && w > 0.0) {
            at = i;
            done = run > goal;
        }
    }
    return at;
}

// the slot the draw falls on
template <int V>
__device__ __forceinline__ int draw(Row<V>& R, double u) {
    double inc[V / 4], s4[V / 4], total = 0.0;
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        s4[c] = (R.w[4 * c] + R.w[4 * c + 1]) + (R.w[4 * c + 2] + R.w[4 * c + 3]);
        inc[c] = lbm::wave_scan<double>(s4[c], 0.0, lbm::OpAdd());
        total += lbm::lane_value(inc[c], 63);
    }
    const double goal = u * total;
    double base = 0.0;
    int hit = -1;
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
        const unsigned long long over = __ballot(base + inc[c] > goal && s4[c] > 0.0);
        if (hit < 0 && over != 0) {
            const int first = __ffsll((long long)over) - 1;
            const double run = base + (first == 0 ? 0.0 : lbm::lane_value(inc[c], first == 0 ? 0 : first - 1));
            hit = (c * 64 + first) * 4 + crossing(run, goal, R.w + 4 * c, first);
        }
        base += lbm::lane_value(inc[c], 63);
    }
    if (hit < 0) {                       // u of 1 or more, or NaN: the last code that stayed
        int last = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) last = R.w[i] > 0.0 ? R.slot(i) : last;
        hit = -lbm::wave_first(-last);
    }
    return hit;
}

struct Setting {
    double temp, c, top_p, min_p, u;
    int top_k;
    bool by_k, by_p;
};

__device__ __forceinline__ Setting row_setting(const Params& par, const float* u, int64_t row, int K) {
    Setting s;
    s.temp = par.T_row != nullptr ? (double)par.T_row[row] : par.T;
    s.c = fmin(1.4426950408889634 / s.temp, 1e300);
    s.top_p = par.p_row != nullptr ? (double)par.p_row[row] : par.top_p;
    s.min_p = par.min_row != nullptr ? (double)par.min_row[row] : par.min_p;
    s.top_k = par.k_row != nullptr ? par.k_row[row] : par.top_k;
    if (s.top_k == 1) s.temp = 0.0;      // the best code
    s.u = (double)u[row];
    s.by_k = s.top_k > 0 && s.top_k < K;
    s.by_p = s.top_p < 1.0;
    return s;
}

// everything behind the best score m; lo: a score at or below all others; total: the weight that top-p refers to where the scores here are
// not all of them (negative: they are); h: 64 words of LDS, the wave's own.  -1: they do not reach top-p's share of that total.
template <int V>
__device__ __forceinline__ int settle(Row<V>& R, const Setting& s, float lo, float m, int K, double total, float* h) {
    if (s.by_p && m < INFINITY) {
        // Where top-p's share of all weight is less than the best code's 1, that code is all that stays (top-k only takes weight away).  On
        // fp32 weights: w errs by 1.3e-7 |log2 w| w, where |log2 w| w <= 0.54, and their sum by 2^-20 of itself, together less than 10^-4 at
        // 1024 codes.  Peaked rows end here: 384000 x 512, top-p 0.9 374 -> 153 us, with top-k and min-p 580 -> 152; flat ones pay 3 %.
        float all = 0.f;
        if (total < 0.0) {
            const float c = (float)s.c;
#pragma unroll
            for (int i = 0; i < V; ++i) all += __builtin_amdgcn_exp2f((R.v[i] - m) * c);
            all = lbm::wave_total(all);
        } else {
            all = (float)total;
        }
        if (s.top_p * all < 0.999) return R.first_of(m);
    }
    if (s.by_k) keep_top_k<V>(R, lo, m, s.top_k, reinterpret_cast<int*>(h));
    R.weigh(m, s.c);
    if (s.by_p) {
        const double here = R.weight();
        if (total < 0.0) total = here;
        const double target = s.top_p * total;
        if (here < target) return -1;
        if (target <= 1.0) return R.first_of(m);
        if (m == INFINITY) {             // equal weights of 1
            const double keep = ceil(target);
            R.keep_first_equal(m, (int)keep);
        } else {
            keep_top_p<V>(R, top_p_floor(m, lo, s.temp, s.top_p, K), m, target, s.c, h);
        }
    }
    if (s.min_p > 0.0) {
        const double lim = fmin(s.min_p, 1.0);
#pragma unroll
        for (int i = 0; i < V; ++i) R.w[i] = R.w[i] >= lim ? R.w[i] : 0.0;
    }
    return draw<V>(R, s.u);
}

// K <= 64 V: the whole row in registers, a wave to a row.  384000 x 512 fp32: greedy 122 - 134 us and top-p of peaked rows 150 - 180 (HBM), then
// vector instructions and LDS atomics bound it: no filter 260 - 310 (64-bit exponentials), top-k 100 435 - 465, top-p 0.9 with a nucleus of 35 codes
// 610, of hundreds 1040.
template <typename T, int V, bool VEC>
__global__ __launch_bounds__(256) void code_sample_kernel(const T* __restrict__ scores, int64_t lds, const float* __restrict__ u,
                                                          Params par, const uint8_t* __restrict__ allowed, int64_t allowed_ld,
                                                          int64_t* __restrict__ out, int64_t N, int K) {
    // one value per wave, and the compiler is told so: branches on a row's settings are the scalar unit's (3 % at 384000 x 512, top-k 100)
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ float s_part[4][64];
    if (row >= N) return;                // a whole wave
    Row<V> R;
    lbm::load_row<T, V, VEC>(scores + row * lds, K, R.lane(), R.v);
    if (allowed != nullptr) {
        const uint8_t* a = allowed + row * allowed_ld;
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            const int col = R.slot(4 * c);
            uint8_t q[4] = {0, 0, 0, 0};
            if (col + 4 <= K) {
                __builtin_memcpy(q, a + col, 4);
            } else if (col < K) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (col + i < K) q[i] = a[col + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) R.v[4 * c + i] = q[i] == 0 ? -INFINITY : R.v[4 * c + i];
        }
    }
    const Setting s = row_setting(par, u, row, K);
    float m = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        R.v[i] = R.v[i] != R.v[i] ? -INFINITY : R.v[i] + 0.f;     // + 0: -0 and 0 are one score
        m = fmaxf(m, R.v[i]);
        lo = fminf(lo, R.v[i] == -INFINITY ? INFINITY : R.v[i]);
    }
    m = lbm::wave_best(m);
    int hit;
    if (m == -INFINITY) {
        hit = -1;
    } else if (!(s.temp > 0.0)) {
        hit = R.first_of(m);
    } else {
        if (s.by_k || s.by_p) lo = -lbm::wave_best(-lo);
        hit = settle<V>(R, s, lo, m, K, -1.0, s_part[threadIdx.x >> 6]);
    }
    if (R.lane() == 0) out[row] = hit;
}

// ---- longer rows: one wave still, which reads the row in chunks of 256 and keeps only what can be drawn.
//
// 512 samples of the row give a score t that a few hundred scores reach; one pass takes the best score, the total fp32 weight where top-p
// asks for it, and the scores >= t with their columns into LDS, where they are a short row again: up to 512 in registers (8 a lane), up to kCand by
// passes over LDS.  The pass is repeated with a corrected t where too many or too few came, and a row whose nucleus does not fit (or that has
// no filter at all) is answered by the same passes over memory.  No barrier anywhere: rows do not wait for each other.  40000 x 8192 fp16: greedy
// 117 - 133 us (HBM), top-k 100 250, top-p 0.9 of peaked rows 247 - 277, no filter 384 - 432, a nucleus of 400 codes 935, of thousands 3.3 ms; top-k
// under a mask 520.  One row alone: 4 to 15 us, 42 where the nucleus has 480 codes, 107 - 119 thousands.
constexpr int kReg = 512, kCand = 1536;

// passes over scores of a row, in memory or taken into LDS
template <typename S>
struct Passes {       // S::request loads four scores that are in range, S::convert makes floats of them, S::four is both with the row's end
    static __device__ __forceinline__ int lane() { return threadIdx.x & 63; }
    __device__ __forceinline__ const S& self() const { return *static_cast<const S*>(this); }

    // f(four scores, slot of the first) in index order across calls; U chunks' loads are on their way at a time
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each_<false, 4>(f);
    }
    template <typename F>
    __device__ __forceinline__ void each_raw(F f) const {
        each_<true, 8>(f);
    }
    template <bool RAW, int U, typename F>
    __device__ __forceinline__ void each_(F f) const {
        int c = 0;
        for (; c + U * 256 <= self().n; c += U * 256) {
            typename S::Four q[U];
#pragma unroll
            for (int i = 0; i < U; ++i) q[i] = self().request(c + i * 256 + lane() * 4);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float v[4];
                if constexpr (RAW) self().convert_raw(q[i], c + i * 256 + lane() * 4, v);
                else self().convert(q[i], c + i * 256 + lane() * 4, v);
                f(v, c + i * 256 + lane() * 4);
            }
        }
        for (; c < self().n; c += 256) {
            float q[4];
            self().four(c + lane() * 4, q);
            f(q, c + lane() * 4);
        }
    }
    // scores above x and equal to it
    __device__ void counts(float x, int* above, int* equal) const {
        int a = 0, e = 0;
        each([&](const float* q, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) a += q[i] > x ? 1 : 0, e += q[i] == x ? 1 : 0;
        });
        *above = lbm::wave_total(a);
        *equal = lbm::wave_total(e);
    }
    __device__ __forceinline__ double weight_of_all(float m, double c) const {
        double s = 0.0;
        each_raw([&](const float* q, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s += exp2_f64(((double)q[i] - (double)m) * c);
        });
        return lbm::wave_total(s);
    }
    __device__ double weight_above(float x, float m, double c) const {
        double s = 0.0;
        each([&](const float* q, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s += q[i] > x ? exp2_f64(((double)q[i] - (double)m) * c) : 0.0;
        });
        return lbm::wave_total(s);
    }
    // the highest score x with reached(scores >= x): one of those in [lo, hi], reached(lo).  add(q) is summed over the scores >= the trial.
    // The first trial is hi itself where `top` (a distribution may have one code).
    template <typename A, typename Add, typename Reached>
    __device__ __forceinline__ float border(float lo, float hi, bool top, Add add, Reached reached) const {
        for (int it = 0; it < kSteps && lo < hi; ++it) {
            const float mid = it == 0 && top ? hi : trial(it, lo, hi);
            A sum = A(0);
            float from = -INFINITY, below = -INFINITY;            // from: of the negatives
            each([&](const float* q, int) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = q[i] >= mid;
                    sum += in ? add(q[i]) : A(0);
                    from = fmaxf(from, in ? -q[i] : -INFINITY);
                    below = fmaxf(below, in ? -INFINITY : q[i]);
                }
            });
            if (reached(lbm::wave_total(sum))) lo = -lbm::wave_best(from);
            else hi = lbm::wave_best(below);
        }
        return lo;
    }
    // weight above x, number of scores equal to x, the nearest scores above and below
    __device__ void around(float x, float m, double c, double* above, int* equal, float* up, float* down) const {
        double s = 0.0;
        int e = 0;
        float u = -INFINITY, d = -INFINITY;                       // u: of the negatives
        each([&](const float* q, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s += q[i] > x ? exp2_f64(((double)q[i] - (double)m) * c) : 0.0;
                e += q[i] == x ? 1 : 0;
                u = fmaxf(u, q[i] > x ? -q[i] : -INFINITY);
                d = fmaxf(d, q[i] < x ? q[i] : -INFINITY);
            }
        });
        *above = lbm::wave_total(s);
        *equal = lbm::wave_total(e);
        *up = -lbm::wave_best(u);
        *down = lbm::wave_best(d);
    }
    // slot of the j-th (from 0) score equal to x; -1: there are fewer
    __device__ int nth_equal(float x, int j) const {
        for (int c = 0; c < self().n; c += 256) {
            float q[4];
            self().four(c + lane() * 4, q);
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine += q[i] == x ? 1 : 0;
            const int scan = lbm::wave_scan<int>(mine, 0, lbm::OpAdd()), here = lbm::lane_value(scan, 63);
            if (j < here) {
                int before = scan - mine, at = 0x7fffffff;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (q[i] == x && before++ == j) at = c + lane() * 4 + i;
                return lbm::wave_first(at);
            }
            j -= here;
        }
        return -1;
    }
};

// VEC: accesses of four scores are aligned and the row ends with one (n % 4 == 0); MASK: codes that may not be drawn.  (Both at compile time: a
// branch round a load makes the compiler wait for it there, and one access was on its way at a time.)
template <typename T, bool VEC, bool MASK>
struct Memory : Passes<Memory<T, VEC, MASK>> {
    const T* row;
    const uint8_t* allowed;
    int n;

    __device__ __forceinline__ float one(int col) const {
        const float f = lbm::score_to_f32<T>(row[col]) + 0.f;
        return f != f || (MASK && allowed[col] == 0) ? -INFINITY : f;
    }
    using Four = lbm::Quad<T>;
    __device__ __forceinline__ Four request(int col) const {
        Four q;
        if constexpr (VEC) q = *reinterpret_cast<const Four*>(row + col);
        else __builtin_memcpy(&q, row + col, sizeof(q));
        return q;
    }
    __device__ __forceinline__ void convert(const Four& q, int col, float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = lbm::score_to_f32<T>(q.v[i]) + 0.f;
            f[i] = f[i] != f[i] ? -INFINITY : f[i];
        }
        mask(col, f);
    }
    // where NaN and the sign of 0 do not matter: maxima, comparisons with a score, weights
    __device__ __forceinline__ void convert_raw(const Four& q, int col, float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = lbm::score_to_f32<T>(q.v[i]);
        mask(col, f);
    }
    __device__ __forceinline__ void mask(int col, float* f) const {
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = allowed[col + i] == 0 ? -INFINITY : f[i];
        }
    }
    // -inf past the row's end, where the last four scores are read and moved up (there are four: rows here have more than 1024)
    __device__ __forceinline__ void four(int col, float* f) const {
        const int at = col + 4 <= n ? col : n - 4, by = col - at;
        float q[4];
        convert(request(at), at, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = by == 0 ? q[i] : -INFINITY;
            if constexpr (!VEC) {
#pragma unroll
                for (int k = 1; i + k < 4; ++k) f[i] = by == k ? q[i + k] : f[i];
            }
        }
    }
};

struct Taken : Passes<Taken> {
    const float* val;     // LDS
    int n;
    struct Four { float v[4]; };
    __device__ __forceinline__ Four request(int at) const {
        const float4 q = *reinterpret_cast<const float4*>(val + at);
        return {q.x, q.y, q.z, q.w};
    }
    __device__ __forceinline__ void convert(const Four& q, int, float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = q.v[i];
    }
    __device__ __forceinline__ void convert_raw(const Four& q, int at, float* f) const { convert(q, at, f); }
    __device__ __forceinline__ void four(int at, float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = at + i < n ? val[at + i] : -INFINITY;
    }
};

// the draw by passes; lo, m: lowest and best score; total as for settle (-1 likewise); below: top-p's border is known to lie below this score
template <typename S>
__device__ __forceinline__ int draw_by_passes(const S& R, const Setting& s, float lo, float m, int K, double total, float below) {
    int above, equal;
    if (m == INFINITY) {                 // equal weights of 1
        R.counts(m, &above, &equal);
        double n = s.by_k && s.top_k < equal ? s.top_k : equal;
        if (s.by_p) n = fmax(1.0, ceil(s.top_p * n));
        const double j = floor(s.u * n);
        return R.nth_equal(m, j >= 0.0 && j < n ? (int)j : (s.u < 0.0 ? 0 : (int)n - 1));
    }
    auto weight = [&](float q) { return exp2_f64(((double)q - (double)m) * s.c); };
    // what stays: scores above b and the first `keep` of those equal to it
    float b = -INFINITY;
    int keep = 0;
    equal = 0;
    if (s.by_k) {
        b = R.template border<int>(lo, m, false, [](float) { return 1; }, [&](int c) { return c >= s.top_k; });
        R.counts(b, &above, &equal);
        keep = s.top_k - above < equal ? s.top_k - above : equal;
    }
    double here = 0.0;
    if (s.by_p) {
        here = b == -INFINITY ? R.weight_of_all(m, s.c) : R.weight_above(b, m, s.c) + keep * weight(b);
        const double target = s.top_p * (total < 0.0 ? here : total);
        if (here < target) return -1;
        const float l = fmaxf(b == -INFINITY ? lo : b, top_p_floor(m, lo, s.temp, s.top_p, K));
        const bool top = !(below < m);
        const float h = top ? m : below;
        // searched on fp32 sums, settled by 64-bit ones as in keep_top_p
        const float cf = (float)s.c, goal = (float)target;
        float x = l < h ? R.template border<float>(l, h, top, [&](float q) { return __builtin_amdgcn_exp2f((q - m) * cf); },
                                                   [&](float w) { return w >= goal; })
                        : l;
        double over = 0.0;
        bool settled = false;
        for (int tries = 0; tries < 4 && !settled; ++tries) {
            float up, down;
            R.around(x, m, s.c, &over, &equal, &up, &down);
            settled = true;
            if (over >= target && x < m) {
                x = up;
                settled = false;
            } else if (equal == 0 || over + equal * weight(x) < target) {
                if (down > -INFINITY) {
                    x = down;
                    settled = false;
                }
            }
        }
        if (!settled) {
            x = R.template border<double>(l, m, true, weight, [&](double w) { return w >= target; });
            float up, down;
            R.around(x, m, s.c, &over, &equal, &up, &down);
        }
        if (x > b) {
            b = x;
            keep = equal;
        } else {                         // top-k's border, where `keep` of the equals stay
            int above_b;
            R.counts(b, &above_b, &equal);
            over = R.weight_above(b, m, s.c);
        }
        const double n = ceil((target - over) / weight(b));
        keep = n >= 1.0 ? (n < keep ? (int)n : keep) : 1;
    }
    const double lim = s.min_p > 0.0 ? fmin(s.min_p, 1.0) : 0.0;
    // weights that stay, four at a time; `seen` counts the equals of b so far
    auto weights = [&](const float* q, double* w, int& seen) {
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += q[i] == b ? 1 : 0;
        const int scan = lbm::wave_scan<int>(mine, 0, lbm::OpAdd());
        int before = seen + scan - mine;
        seen += lbm::lane_value(scan, 63);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = q[i] > b || (q[i] == b && before < keep);
            before += q[i] == b ? 1 : 0;
            w[i] = weight(q[i]);
            w[i] = in && w[i] >= lim ? w[i] : 0.0;
        }
    };
    // Sums of 2048 scores at a time, which lead to the group the draw falls into; where the border cuts through equal scores their order
    // counts and the row is walked from its start.
    double base = 0.0;
    int start = 0;
    if (keep >= equal) {
        const double least = lim;
        auto group = [&](int g) {        // the lanes' sums of group g
            double w = 0.0;
            if (b == -INFINITY && least == 0.0 && g * 2048 + 2048 <= R.n) {       // everything: loads at once, no comparisons
                typename S::Four at_once[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) at_once[i] = R.request(g * 2048 + i * 256 + R.lane() * 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float q[4];
                    R.convert_raw(at_once[i], g * 2048 + i * 256 + R.lane() * 4, q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) w += weight(q[j]);
                }
                return lbm::wave_total(w);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = g * 2048 + i * 256 + R.lane() * 4;
                float q[4];
                R.four(c, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double x = weight(q[j]);
                    w += q[j] >= b && x >= least ? x : 0.0;
                }
            }
            return lbm::wave_total(w);
        };
        const int groups = (R.n + 2047) / 2048;
        here = 0.0;
        double mine = 0.0;               // lane g % 64 keeps group g's sum of the last 64
        for (int g = 0; g < groups; ++g) {
            const double w = group(g);
            here += w;
            if ((g & 63) == R.lane()) mine = w;
        }
        const double goal = s.u * here;
        if (groups <= 64) {
            double run = 0.0;
            for (int g = 0; g < groups; ++g) {
                const double w = lbm::lane_value(mine, g);
                if (w > 0.0) {           // where none passes the goal (u of 1 or more, NaN) the last group that holds a weight
                    start = g * 2048;
                    base = run;
                }
                run += w;
                if (run > goal) break;
            }
        }
    } else {
        double sum = 0.0;
        int seen = 0;
        R.each([&](const float* q, int) {
            double w[4];
            weights(q, w, seen);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        });
        here = lbm::wave_total(sum);
    }
    const double goal = s.u * here;
    int seen = 0, last = -1;
    for (int c = start; c < R.n; c += 256) {
        float q[4];
        double w[4];
        R.four(c + R.lane() * 4, q);
        weights(q, w, seen);
        const double s4 = (w[0] + w[1]) + (w[2] + w[3]);
        const double inc = lbm::wave_scan<double>(s4, 0.0, lbm::OpAdd());
        const unsigned long long over = __ballot(base + inc > goal && s4 > 0.0);
        if (over != 0) {
            const int first = __ffsll((long long)over) - 1;
            const double run = base + (first == 0 ? 0.0 : lbm::lane_value(inc, first == 0 ? 0 : first - 1));
            return c + first * 4 + crossing(run, goal, w, first);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) last = w[i] > 0.0 ? c + R.lane() * 4 + i : last;
        base += lbm::lane_value(inc, 63);
    }
    return -lbm::wave_first(-last);      // u of 1 or more, NaN, or a goal that rounding keeps out of reach: the last code that stayed
}

constexpr float kLowest = -3.402823466e+38f;

template <typename T, bool VEC, bool MASK>
__global__ __launch_bounds__(256, 3) void code_sample_long_kernel(const T* __restrict__ scores, int64_t lds, const float* __restrict__ u,
                                                               Params par, const uint8_t* __restrict__ allowed, int64_t allowed_ld,
                                                               int64_t* __restrict__ out, int64_t N, int K) {
    __shared__ __align__(16) float s_val[4][kCand];
    __shared__ unsigned short s_col[4][kCand], s_four[4][kCand];
    __shared__ float s_part[4][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= N) return;                // a whole wave
    Memory<T, VEC, MASK> S;
    S.row = scores + row * lds;
    S.allowed = MASK ? allowed + row * allowed_ld : nullptr;
    S.n = K;
    const Setting s = row_setting(par, u, row, K);
    float* val = s_val[wave];
    unsigned short *col = s_col[wave], *four = s_four[wave];
    constexpr int V = kReg / 64;
    int hit = -2;                        // not answered yet
    float below = INFINITY;              // top-p's border is known to lie below this score
    float m = -INFINITY, lo = INFINITY;
    const bool greedy = !(s.temp > 0.0), p_alone = s.by_p && !s.by_k;
    if (!greedy && K <= 65536 && (s.by_k ? s.top_k <= 1280 : s.by_p || s.min_p > 0.0)) {
        Row<V> R;                        // samples: every (K / 512)-th score
        float t_lo = INFINITY, t_hi = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            R.v[i] = S.one((int)((int64_t)(lane + 64 * i) * K / kReg));
            t_hi = fmaxf(t_hi, R.v[i]);
            t_lo = fminf(t_lo, R.v[i] == -INFINITY ? INFINITY : R.v[i]);
        }
        t_hi = lbm::wave_best(t_hi);
        t_lo = -lbm::wave_best(-t_lo);
        const float ref = t_hi, cf = (float)s.c;       // weights of the pass are relative to the best sample
        double total = -1.0;
        // how many scores to take: what top-k needs and as much again, at most what fits; the square root of the samples that reach t is
        // their spread, a sixth at 320 of 8192
        int aim = !s.by_k ? 320 : (s.top_k <= 128 ? 256 : (s.top_k <= 384 ? (s.top_k + kReg) / 2 : (s.top_k + kCand) / 2));
        int want = (int)fmax(1.f, (float)aim * kReg / (float)K);
        for (int tries = 0; tries < 3 && hit == -2; ++tries) {
            float t = kLowest, l = t_lo, h = t_hi;
            if (R.count_from(t_lo) > want) {
                for (int it = 0; it < kByValue && l < h; ++it) {
                    t = trial(it, l, h);
                    const int c = R.count_from(t);
                    if (c > want + want / 8) l = t;
                    else if (c < want - want / 8) h = t;
                    else break;
                }
            }
            // first the groups of four that hold a score >= t, by their number; then, of those alone, the scores themselves
            int fours = 0;
            float sum = 0.f;
            m = -INFINITY;
            S.each_raw([&](const float* q, int c) {
                const float best = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
                m = fmaxf(m, best);
                if (p_alone) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f((q[i] - ref) * cf);
                }
                const unsigned long long b = __ballot(best >= t);
                const int at = fours + __builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)b, 0));
                if (best >= t && at < kCand) four[at] = (unsigned short)(c >> 2);
                fours += __popcll(b);
            });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            int n = fours > kCand ? kCand + 1 : 0;
            for (int f0 = 0; f0 < fours && n <= kCand; f0 += 64) {
                float q[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                int c = 0;
                if (f0 + lane < fours) {
                    c = four[f0 + lane] * 4;
                    S.four(c, q);
                }
                int pre = n, tot = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned long long b = __ballot(q[i] >= t);
                    pre = __builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)b, pre));
                    tot += __popcll(b);
                }
                if (n + tot <= kCand) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (q[i] >= t) {
                            val[pre] = q[i];
                            col[pre] = (unsigned short)(c + i);
                            ++pre;
                        }
                }
                n += tot;
            }
            m = lbm::wave_best(m);
            if (m == -INFINITY) {
                hit = -1;
                break;
            }
            if (m == INFINITY) break;
            int next = want;
            // (a list that outgrew the registers is worth another pass where a shorter one does)
            const int room = tries == 0 && (!s.by_k || s.top_k <= 384) ? kReg : kCand;
            if (n > room || (s.by_k && n < s.top_k && t > kLowest)) {
                next = (int)fmin(fmax(1.f, (float)want * (float)aim / (float)(n > 0 ? n : 1)), (float)kReg);
            } else {
                if (p_alone && total < 0.0) {
                    // all weight: on fp32 weights where that shows that the best code fills top-p's share (as in settle, whose bound grows
                    // with the codes), else by a pass of 64-bit ones.  40000 x 8192 fp16, top-p 0.9: peaked rows 380 -> 257 us against 64
                    // bits at once; rows spread over tens of codes 524 -> 509 at 48828 x 4096, 687 -> 775 at 133333 x 1500.
                    // The fp32 sum is relative to the best sample.  A best code 2^120 above that (NaN: no finite sample, or a temperature
                    // whose reciprocal is no float) is left to the 64-bit pass: the factor that brings the sum back to it falls below the
                    // smallest normal float, where the exponential gives 0, before the sum overflows.
                    const float up = (m - ref) * cf;
                    const float all = lbm::wave_total(sum) * __builtin_amdgcn_exp2f(-up);
                    total = up < 120.f && s.top_p * all < 0.999 - 1e-7 * K ? (double)all : S.weight_of_all(m, s.c);
                }
                // min-p alone: everything it leaves must have been taken
                const bool all = s.by_k || s.by_p || t == kLowest || exp2_f64(((double)t - (double)m) * s.c) < fmin(s.min_p, 1.0);
                int at = -1;
                if (all) {
                    // LDS serves a wave's accesses in order: the compiler only has to keep the order too
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    lo = INFINITY;
                    if (n <= kReg) {
                        Row<V> Q;
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const bool in = Row<V>::slot(i) < n;
                            Q.v[i] = in ? val[Row<V>::slot(i)] : -INFINITY;
                            lo = fminf(lo, in ? Q.v[i] : INFINITY);
                        }
                        at = settle<V>(Q, s, -lbm::wave_best(-lo), m, K, total, s_part[wave]);
                    } else {
                        Taken Q;
                        Q.val = val;
                        Q.n = n;
                        for (int i = lane; i < n; i += 64) lo = fminf(lo, val[i]);
                        at = draw_by_passes(Q, s, -lbm::wave_best(-lo), m, K, total, INFINITY);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
                if (at >= 0) {
                    hit = col[at];
                    break;
                }
                if (p_alone && all) below = t;
                aim = kCand * 3 / 4;     // the nucleus is larger
                next = (int)fmax(1.f, (float)aim * kReg / (float)K);
            }
            if (next == want) break;
            want = next;
        }
    }
    if (hit == -2 && greedy) {
        int at = 0x7fffffff;             // each lane's first best score
        m = -INFINITY;
        S.each([&](const float* q, int c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                at = q[i] > m ? c + i : at;
                m = fmaxf(m, q[i]);
            }
        });
        const float best = lbm::wave_best(m);
        hit = best == -INFINITY ? -1 : lbm::wave_first(m == best ? at : 0x7fffffff);
    }
    if (hit == -2) {
        m = -INFINITY;
        lo = INFINITY;
        S.each([&](const float* q, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m = fmaxf(m, q[i]);
                lo = fminf(lo, q[i] == -INFINITY ? INFINITY : q[i]);
            }
        });
        m = lbm::wave_best(m);
        lo = -lbm::wave_best(-lo);
        hit = m == -INFINITY ? -1 : draw_by_passes(S, s, lo, m, K, -1.0, below);
    }
    if (lane == 0) out[row] = hit;
}

constexpr int64_t kLaunchRows = 1 << 25;       // a launch holds fewer than 2^32 threads; a wave works on a row

template <typename T>
int run_sample(const void* scores, int64_t lds, const float* u, Params par, const uint8_t* allowed, int64_t allowed_ld, int64_t* out, int64_t N,
               int K, hipStream_t st) {
    const T* s = static_cast<const T*>(scores);
    const bool vec = ((uintptr_t)scores % (4 * sizeof(T))) == 0 && (lds & 3) == 0 && (K & 3) == 0;
    for (;;) {
        const int64_t n = N < kLaunchRows ? N : kLaunchRows;
        const dim3 grid((unsigned)((n + 3) / 4)), block(256);
#define LBM_SAMPLE(kernel) hipLaunchKernelGGL((kernel), grid, block, 0, st, s, lds, u, par, allowed, allowed_ld, out, n, K)
        if (K <= 256) LBM_SAMPLE((vec ? code_sample_kernel<T, 4, true> : code_sample_kernel<T, 4, false>));
        else if (K <= 512) LBM_SAMPLE((vec ? code_sample_kernel<T, 8, true> : code_sample_kernel<T, 8, false>));
        else if (K <= 1024) LBM_SAMPLE((vec ? code_sample_kernel<T, 16, true> : code_sample_kernel<T, 16, false>));
        else if (allowed == nullptr) LBM_SAMPLE((vec ? code_sample_long_kernel<T, true, false> : code_sample_long_kernel<T, false, false>));
        else LBM_SAMPLE((vec ? code_sample_long_kernel<T, true, true> : code_sample_long_kernel<T, false, true>));
#undef LBM_SAMPLE
        const int rc = lbm::check_launch("lbm_code_sample");
        if (rc != LBM_OK || n == N) return rc;
        s += n * lds;
        u += n;
        out += n;
        if (allowed != nullptr) allowed += n * allowed_ld;
        if (par.T_row != nullptr) par.T_row += n;
        if (par.k_row != nullptr) par.k_row += n;
        if (par.p_row != nullptr) par.p_row += n;
        if (par.min_row != nullptr) par.min_row += n;
        N -= n;
    }
}

constexpr int kMaxK = 1 << 24;

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
    LBM_REQUIRE(hist_or_null == nullptr || K <= 32768, LBM_EUNSUPPORTED, "%s: histogram supports K <= 32768", what);
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
