// Scores of every code for every row, and their gradients: three fp32 matrix products on one tile kernel.
//
//   s[n, k]  = (2 x_n . e_k - |e_k|^2) / T                 forward   [N, D] x [K, D]^T
//   dx[n, d] = (2 / T) sum_k g[n, k] e_k[d]                 rows      [N, K] x [K, D]
//   de[k, d] = (2 / T) (sum_n g[n, k] x_n[d] - c_k e_k[d])  codebook  [N, K]^T x [N, D],  c_k = sum_n g[n, k]
//
// s is minus the squared distance over the temperature without its row constant |x_n|^2 / T, which softmax, argmax and every ordering
// of a row ignore and whose size would only cost the differences their low bits.
//
// Products: every fp32 operand is cut into three bf16 pieces, each the nearest bf16 of what is left (the remainders are exact, the three
// hold 24 bits and more), and a product keeps six terms of the nine, accumulated in fp32 on v_mfma_f32_32x32x16_bf16; the three left out lie
// below 2^-26 of it.  That is as exact as a chain of fp32 products (7.5e-8 of the scores' size against 64 bits either way) at 16/6 of the fp32
// matrix rate.  An operand whose nearest bf16 is an infinity (0x1.ffp127 = 3.396e38 and more) makes NaN of what it enters: inf - inf among
// its pieces.  (Clamping the first piece would let finite ones through; two instructions per pair of values: 40000 x 8192 x 256 1067 -> 1094 us.)
//
// Bound: the matrix pipe and the power it draws; an output element costs 12 D FLOP of bf16 products for 4 bytes of store.  That is also why
// the scores are stored at all: forming them a second time for the gradient costs more than writing and reading them.
//
// Tile: 4 waves, each (TM/2) x (TN/2) outputs in 32 x 32 accumulators.  The contraction runs 32 steps at a time: operands are requested into
// registers while the products of the previous 32 steps run, cut into pieces and written to LDS as three planes [row][32 + 8] of bf16, which the
// waves read eight steps at a time (ds_read_b128; the pitch of 80 bytes spreads rows over the banks).
#include <type_traits>

#include "common.h"

namespace {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using b16x2 = __attribute__((ext_vector_type(2))) __bf16;
using b16x8 = __attribute__((ext_vector_type(8))) __bf16;

constexpr int kThreads = 256;
constexpr int kBK = 32;
constexpr int kPitch = 80;        // bytes of a row of one plane

// operand contiguous along the contraction (KC) or along its rows (MC), read 4 bytes or (V) 16 bytes at a time
enum { KC = 0, MC = 1, KCV = 2, MCV = 3 };
constexpr bool along_k(int mode) { return (mode & 1) == 0; }
constexpr bool wide(int mode) { return (mode & 2) != 0; }

// Operand `rows x steps`: element (r, k) is p[r * ld + k] (KC) or p[off(r) + k * ld] (MC; off(r) = r, or b * pitch + s for channel-major rows
// r = b * S + s).
struct Operand {
    const float* p;
    int64_t ld;       // KC: row stride; MC: stride of one contraction step
    int64_t S, pitch; // MC: S = 0: rows are contiguous
    int64_t rows;
};

// N consecutive steps of one row -> their three pieces
template <int N>
__device__ __forceinline__ void cut(const float* v, unsigned (*p)[N / 2]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        f32x2 f = {v[2 * i], v[2 * i + 1]};
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const unsigned w = __builtin_bit_cast(unsigned, __builtin_convertvector(f, b16x2));
            p[q][i] = w;
            f.x -= __uint_as_float(w << 16);
            f.y -= __uint_as_float(w & 0xffff0000u);
        }
    }
}

// One operand's share of a tile: 32 contraction steps of T rows, in registers on the way from memory to LDS.  Rows past the operand's last
// repeat it (what they give is not stored); steps past the end are zeros and come from load_tail only, so that load has no branch in it.
//   K:    thread has steps 4 (t % 8) .. + 3 of rows t / 8 + 32 i
//   MCV:  rows 4 (t / G) .. + 3 of steps U (t % G) .. + U - 1, U = T / 32: the eight (sixteen) threads of four rows write whole LDS rows
//   MC:   row t % T of steps 4 (t / T) + 4 (256 / T) i .. + 3: the threads of a wave read neighbouring rows
template <int T, int MODE>
struct Stage {
    static constexpr bool K = along_k(MODE), WIDE = wide(MODE);
    static constexpr int kPlane = T * kPitch, kBytes = 3 * kPlane;
    static constexpr int Q = T / 32, U = T / 32, G = kBK / U;
    float v[Q][4];                    // K, MC: [quad][step]; MCV: [step][row]
    const float* base[K ? Q : 1];
    int64_t ld;

    __device__ __forceinline__ static int step(int i, int u) {       // contraction step of v[i][u]
        if constexpr (K) return (threadIdx.x & 7) * 4 + u;
        else if constexpr (WIDE) return U * (threadIdx.x % G) + i;
        else return 4 * (threadIdx.x / T) + 4 * (kThreads / T) * i + u;
    }
    __device__ __forceinline__ static int row(int i, int u) {        // tile row of v[i][u]
        if constexpr (K) return (threadIdx.x >> 3) + 32 * i;
        else if constexpr (WIDE) return 4 * (threadIdx.x / G) + u;
        else return threadIdx.x % T;
    }
    __device__ __forceinline__ void init(const Operand& o, int64_t r0, int64_t k0) {
        ld = o.ld;
        if constexpr (K) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const int64_t r = r0 + row(i, 0);
                base[i] = o.p + (r < o.rows ? r : o.rows - 1) * o.ld + step(0, 0) + k0;
            }
        } else {
            int64_t r = r0 + row(0, 0);
            if (WIDE) r = r < o.rows ? r : 0;                      // rows % 4 == 0: four at a time are all in or all out
            else r = r < o.rows ? r : o.rows - 1;
            base[0] = o.p + (o.S > 0 ? (r / o.S) * o.pitch + r % o.S : r) + (k0 + step(0, 0)) * o.ld;
        }
    }
    // 32 whole steps
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            if constexpr (WIDE) {
                const float4 f = *reinterpret_cast<const float4*>(K ? base[K ? i : 0] : base[0] + (int64_t)i * ld);
                v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) v[i][u] = K ? base[K ? i : 0][u] : base[0][(int64_t)(4 * (kThreads / T) * i + u) * ld];
            }
            if (K) base[K ? i : 0] += kBK;
        }
        if (!K) base[0] += (int64_t)kBK * ld;
    }
    // the last `left` < 32 steps
    __device__ __forceinline__ void load_tail(int left) {
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float f = 0.f;
                if (step(i, u) < left) {
                    if constexpr (K) f = base[K ? i : 0][u];
                    else if constexpr (WIDE) f = base[0][(int64_t)i * ld + u];
                    else f = base[0][(int64_t)(4 * (kThreads / T) * i + u) * ld];
                }
                v[i][u] = f;
            }
    }
    // pieces to the three planes at s
    __device__ __forceinline__ void store(char* s) const {
        if constexpr (K || !WIDE) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                unsigned p[3][2];
                cut<4>(v[i], p);
                char* at = s + row(i, 0) * kPitch + step(i, 0) * 2;
#pragma unroll
                for (int q = 0; q < 3; ++q) *reinterpret_cast<uint2*>(at + q * kPlane) = make_uint2(p[q][0], p[q][1]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float f[U];
#pragma unroll
                for (int i = 0; i < U; ++i) f[i] = v[i][r];
                unsigned p[3][U / 2];
                cut<U>(f, p);
                char* at = s + row(0, r) * kPitch + step(0, 0) * 2;
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    if constexpr (U == 4) *reinterpret_cast<uint2*>(at + q * kPlane) = make_uint2(p[q][0], p[q][1]);
                    else *reinterpret_cast<unsigned*>(at + q * kPlane) = p[q][0];
                }
            }
        }
    }
    // piece q of steps 16 g + 8 h .. + 7 of row r
    static __device__ __forceinline__ b16x8 frag(const char* s, int r, int g, int h, int q) {
        return *reinterpret_cast<const b16x8*>(s + q * kPlane + r * kPitch + g * 32 + h * 16);
    }
    // sums over the steps in registers, added to sum[4]: K: of row(i); MCV: of row(u); MC: of the one row, in sum[0]
    __device__ __forceinline__ void add_steps(float* sum) const {
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[K ? i : (WIDE ? u : 0)] += v[i][u];
    }
};

enum { EPI_SCORES = 0, EPI_SCALE = 1, EPI_PARTIAL = 2 };

struct Tiles {
    int mt, nt;     // tiles along the rows of A and of B
    int splits;     // pieces of the contraction (EPI_PARTIAL)
    int64_t piece;  // steps of one piece
};

// out[m, n] over the contraction; EPI_SCORES: out = (2 acc - e_n) * scale, e_n = sqnorm[n] or, where that is NULL, the square sum of B's
// row n taken from its staged values; EPI_SCALE: out = acc * scale; EPI_PARTIAL: piece z's sums to out[z][m][n] and A's row sums over
// the piece to rowsum[z][m] (NULL: not wanted).
template <int TM, int TN, int AM, int BM, int EPI>
__global__ __launch_bounds__(kThreads, 2) void code_mm_kernel(Operand a, Operand b, float* __restrict__ out, int64_t ldo, int64_t depth,
                                                              Tiles t, float scale, const float* __restrict__ sqnorm,
                                                              float* __restrict__ rowsum) {
    using SA = Stage<TM, AM>;
    using SB = Stage<TN, BM>;
    constexpr int MI = TM / 64, NI = TN / 64;
    __shared__ __align__(16) char s_ab[SA::kBytes + SB::kBytes];
    __shared__ float s_n[EPI == EPI_PARTIAL ? kThreads : TN];      // |e|^2 of the tile's codes; or the threads' row sums
    char* s_a = s_ab;
    char* s_b = s_ab + SA::kBytes;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = lane & 31, h = lane >> 5;
    const int wm = (wave >> 1) * (TM / 2), wn = (wave & 1) * (TN / 2);

    // Workgroups go round the 8 XCDs: each XCD works through a contiguous run of tiles, B tiles fastest, so that the tiles that share A's
    // rows meet in one L2.  A workgroup takes every n-th tile of its XCD's run and requests the next tile's first steps before it stores
    // the present one's results.
    const int64_t total = (int64_t)t.mt * t.nt * t.splits;
    const int xcd = blockIdx.x & 7, each = gridDim.x >> 3, more = gridDim.x & 7;
    const int per_xcd = each + (xcd < more ? 1 : 0), before = xcd * each + (xcd < more ? xcd : more);
    const int64_t run0 = total * before / gridDim.x, run1 = total * (before + per_xcd) / gridDim.x;
    int64_t item = run0 + (blockIdx.x >> 3);
    if (item >= run1) return;

    SA sa;
    SB sb;
    int64_t m0, n0;
    int z, whole, left;
    auto begin = [&](int64_t i) {
        const int64_t tiles = (int64_t)t.mt * t.nt, tile = i % tiles;
        z = (int)(i / tiles);
        m0 = tile / t.nt * TM;
        n0 = tile % t.nt * TN;
        const int64_t kbeg = z * t.piece, kend = kbeg + t.piece < depth ? kbeg + t.piece : depth;
        whole = (int)((kend - kbeg) / kBK);
        left = (int)((kend - kbeg) % kBK);
        sa.init(a, m0, kbeg);
        sb.init(b, n0, kbeg);
        if (whole > 0) {
            sa.load();
            sb.load();
        }
    };
    begin(item);
    for (;;) {
        f32x16 acc[MI][NI];
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int y = 0; y < NI; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
        float sq[SB::Q] = {};
        float asum[4] = {};

        auto put = [&] {
            // the waves that stage go before those that multiply: two workgroups share a SIMD, and the other one's products fill the
            // gap (40000 x 8192 x 256: 1089 -> 1054 us)
            __builtin_amdgcn_s_setprio(1);
            __syncthreads();   // the previous steps' fragments are read
            sa.store(s_a);
            sb.store(s_b);
            if constexpr (EPI == EPI_SCORES) {
#pragma unroll
                for (int i = 0; i < SB::Q; ++i)
#pragma unroll
                    for (int u = 0; u < 4; ++u) sq[i] = fmaf(sb.v[i][u], sb.v[i][u], sq[i]);
            }
            if constexpr (EPI == EPI_PARTIAL) sa.add_steps(asum);
            __syncthreads();
        };
        auto products = [&] {
            // the pieces of the second 16 steps are read while the products of the first run
            b16x8 fa[2][MI][3], fb[2][NI][3];
            auto read = [&](int g) {
#pragma unroll
                for (int q = 0; q < 3; ++q) {
#pragma unroll
                    for (int x = 0; x < MI; ++x) fa[g][x][q] = SA::frag(s_a, wm + 32 * x + j, g, h, q);
#pragma unroll
                    for (int y = 0; y < NI; ++y) fb[g][y][q] = SB::frag(s_b, wn + 32 * y + j, g, h, q);
                }
            };
            read(0);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (g == 0) read(1);
                __builtin_amdgcn_sched_barrier(0);
                // the six products, small ones first
                constexpr int qa[6] = {2, 1, 0, 1, 0, 0}, qb[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                for (int t6 = 0; t6 < 6; ++t6)
#pragma unroll
                    for (int x = 0; x < MI; ++x)
#pragma unroll
                        for (int y = 0; y < NI; ++y)
                            acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[g][x][qa[t6]], fb[g][y][qb[t6]], acc[x][y], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (int it = 1; it < whole; ++it) {
            put();
            sa.load();     // on their way while the products run
            sb.load();
            __builtin_amdgcn_sched_barrier(0);
            products();
        }
        if (whole > 0) {
            put();
            products();
        }
        if (left > 0) {
            sa.load_tail(left);
            sb.load_tail(left);
            put();
            products();
        }
        const int64_t m0_now = m0, n0_now = n0;
        const int z_now = z;
        item += per_xcd;
        if (item < run1) begin(item);
        __builtin_amdgcn_sched_barrier(0);

        if constexpr (EPI == EPI_SCORES) {
            if (sqnorm != nullptr) {
                if (threadIdx.x < TN) s_n[threadIdx.x] = n0_now + threadIdx.x < b.rows ? sqnorm[n0_now + threadIdx.x] : 0.f;
            } else {
#pragma unroll
                for (int i = 0; i < SB::Q; ++i) {
                    float s = sq[i];   // the eight lanes that staged one row of B
                    s += __shfl_xor(s, 1, 64);
                    s += __shfl_xor(s, 2, 64);
                    s += __shfl_xor(s, 4, 64);
                    if ((threadIdx.x & 7) == 0) s_n[(threadIdx.x >> 3) + 32 * i] = s;
                }
            }
            __syncthreads();           // (the next tile's first barrier keeps its s_n behind this one's reads)
        }
        float* o = out;
        if constexpr (EPI == EPI_PARTIAL) {
            o += (int64_t)z_now * a.rows * ldo;
            if (rowsum != nullptr && n0_now == 0) {
                if constexpr (AM == MCV) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        float v = asum[u];             // the threads of four rows are neighbours
#pragma unroll
                        for (int o = 1; o < SA::G; o <<= 1) v += __shfl_xor(v, o, 64);
                        const int64_t m = m0_now + SA::row(0, u);
                        if (threadIdx.x % SA::G == 0 && m < a.rows) rowsum[(int64_t)z_now * a.rows + m] = v;
                    }
                } else if constexpr (AM == MC) {
                    s_n[threadIdx.x] = asum[0];
                    __syncthreads();
                    if (threadIdx.x < TM && m0_now + threadIdx.x < a.rows) {
                        float v = 0.f;
#pragma unroll
                        for (int o = 0; o < kThreads / TM; ++o) v += s_n[threadIdx.x + o * TM];
                        rowsum[(int64_t)z_now * a.rows + m0_now + threadIdx.x] = v;
                    }
                }
            }
        }
        const bool inside = m0_now + TM <= a.rows && n0_now + TN <= b.rows;
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int y = 0; y < NI; ++y) {
                const int nl = wn + 32 * y + j;
                const int64_t n = n0_now + nl, m = m0_now + wm + 32 * x + 4 * h;
                const float e = EPI == EPI_SCORES ? s_n[nl] : 0.f;
                float* q = o + m * ldo + n;
                const bool col = n < b.rows;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int dm = (r & 3) + 8 * (r >> 2);
                    float v = acc[x][y][r];
                    if constexpr (EPI == EPI_SCORES) v = (2.f * v - e) * scale;
                    if constexpr (EPI == EPI_SCALE) v = v * scale;
                    if (inside || (col && m + dm < a.rows)) q[dm * ldo] = v;
                }
            }
        if (item >= run1) return;
    }
}

// out[m, d] = scale * (sum_z part[z][m][d] - (sum_z rowsum[z][m]) * e[m][d]); NORM = false: without the second term.  Pieces in order, eight
// loads on their way at a time.
template <bool NORM>
__global__ __launch_bounds__(256) void code_grad_join_kernel(const float* __restrict__ part, const float* __restrict__ rowsum,
                                                             const float* __restrict__ codebook, float* __restrict__ out, int splits,
                                                             int64_t M, int64_t D, float scale, int64_t first) {
    const int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x, n = M * D;
    if (i >= n) return;
    const int64_t m = NORM ? i / D : 0;
    double s = 0.0, c = 0.0;
    for (int z0 = 0; z0 < splits; z0 += 8) {
        float p[8], r[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int z = z0 + u < splits ? z0 + u : splits - 1;
            p[u] = part[z * n + i];
            r[u] = NORM ? rowsum[z * M + m] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            s += z0 + u < splits ? (double)p[u] : 0.0;
            c += z0 + u < splits ? (double)r[u] : 0.0;
        }
    }
    if (NORM) s -= c * (double)codebook[i];
    out[i] = (float)(s * (double)scale);
}

template <bool NORM>
int launch_join(const char* what, const float* part, const float* rowsum, const float* codebook, float* out, int splits, int64_t M, int64_t D,
                float scale, hipStream_t st) {
    constexpr int64_t kEntries = 1LL << 31;               // a launch holds fewer than 2^32 threads
    for (int64_t first = 0; first < M * D; first += kEntries) {
        const int64_t n = M * D - first < kEntries ? M * D - first : kEntries;
        hipLaunchKernelGGL((code_grad_join_kernel<NORM>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, rowsum, codebook, out,
                           splits, M, D, scale, first);
        const int rc = lbm::check_launch(what);
        if (rc != LBM_OK) return rc;
    }
    return LBM_OK;
}

// 2 / T is a finite float, and 1 / T
bool usable(double temperature) { return temperature > 0.0 && temperature < INFINITY && 2.0 / temperature <= 0x1.fffffep127; }

bool aligned16(const float* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }

template <int TM, int TN, int AM, int BM, int EPI>
int launch_tiles(const char* what, const Operand& a, const Operand& b, float* out, int64_t ldo, int64_t depth, int splits, int64_t piece,
                 float scale, const float* sqnorm, float* rowsum, hipStream_t st) {
    const int64_t mt = (a.rows + TM - 1) / TM, nt = (b.rows + TN - 1) / TN;
    if (mt > 0x7fffffffLL || nt > 0x7fffffffLL) return lbm::fail(LBM_EUNSUPPORTED, "%s: too many tiles", what);
    const Tiles t{(int)mt, (int)nt, splits, piece};
    const int64_t total = mt * nt * splits, fit = TM * TN >= 128 * 128 ? 512 : 1024;      // workgroups that run at a time
    hipLaunchKernelGGL((code_mm_kernel<TM, TN, AM, BM, EPI>), dim3((unsigned)(total < fit ? total : fit)), dim3(kThreads), 0, st, a, b, out, ldo,
                       depth, t, scale, sqnorm, rowsum);
    return lbm::check_launch(what);
}

template <int AM, int BM, int EPI>
int launch_mm(const char* what, const Operand& a, const Operand& b, float* out, int64_t ldo, int64_t depth, int splits, int64_t piece,
              float scale, const float* sqnorm, float* rowsum, hipStream_t st) {
    // Cost of a tile size: tiles that the busiest CU gets, their area, and what a product costs in it -- the smaller tiles read and cut more
    // per product (24000 x 512 x 256, the rows' gradient: 128 x 128 53 us, 64 x 128 60 us, 64 x 64 60 us with a third less work on the
    // busiest CU; 375 x 512 x 256: 64 x 64 9 us, 128 x 128 19 us).
    auto cost = [&](int tm, int tn, int each) {
        const int64_t n = ((a.rows + tm - 1) / tm) * ((b.rows + tn - 1) / tn) * splits;
        return (n + 255) / 256 * (tm * tn) * (n <= 256 ? each + 3 : each);     // alone on its CU a tile's gaps stay open
    };
    const int64_t c128 = cost(128, 128, 10), c64 = cost(64, 128, 14), c32 = cost(64, 64, 15);
    if (c128 <= c64 && c128 <= c32)
        return launch_tiles<128, 128, AM, BM, EPI>(what, a, b, out, ldo, depth, splits, piece, scale, sqnorm, rowsum, st);
    if (c64 <= c32)
        return launch_tiles<64, 128, AM, BM, EPI>(what, a, b, out, ldo, depth, splits, piece, scale, sqnorm, rowsum, st);
    return launch_tiles<64, 64, AM, BM, EPI>(what, a, b, out, ldo, depth, splits, piece, scale, sqnorm, rowsum, st);
}

// A contraction in pieces whose sums are joined in 64 bits: how many, and the steps of each (a multiple of 32).
// tiles: of the output; a contraction is cut where they leave CUs idle, into pieces of `least` steps at least, and where it is longer than
// `most`, the longest fp32 chain.
struct Split {
    int n;
    int64_t piece;
};
Split split_steps(int64_t tiles, int64_t depth, int64_t least, int64_t most) {
    int64_t n = 512 / (tiles > 0 ? tiles : 1);
    if (n > depth / least) n = depth / least;
    if (n < (depth + most - 1) / most) n = (depth + most - 1) / most;
    if (n < 1) n = 1;
    const int64_t piece = ((depth + n - 1) / n + kBK - 1) / kBK * kBK;
    return {(int)((depth + piece - 1) / piece), piece};
}
// the codebook's gradient sums over the N rows, the rows' over the K codes.  (The latter is cut where few rows make few tiles; the pieces cost
// a write and a read of the gradient each.)
Split split_rows(int64_t N, int32_t D, int32_t K) {
    return split_steps((((int64_t)K + 127) / 128) * (((int64_t)D + 127) / 128), N, 128, 32768);
}
Split split_codes(int64_t N, int32_t D, int32_t K) {
    return split_steps(((N + 63) / 64) * (((int64_t)D + 127) / 128), K, 256, 4096);
}

}  // namespace

extern "C" int lbm_code_logits_f32(const float* x, int64_t ldx, int32_t layout, int64_t S, const float* codebook,
                                   const float* e_sqnorm_or_null, float* logits, int64_t ldl, int64_t N, int32_t D, int32_t K,
                                   double temperature, lbm_stream_t stream) {
    const char* what = "lbm_code_logits_f32";
    LBM_REQUIRE(N >= 0 && D >= 1 && K >= 1, LBM_EINVAL, "%s: bad sizes (N=%lld D=%d K=%d)", what, (long long)N, D, K);
    LBM_REQUIRE(usable(temperature), LBM_EINVAL, "%s: temperature must be positive and finite, and 2 / temperature too", what);
    LBM_REQUIRE(layout == LBM_VQ_ROWS || layout == LBM_VQ_CHANNEL_MAJOR, LBM_EINVAL, "%s: unknown layout %d", what, layout);
    if (N == 0) return LBM_OK;
    LBM_REQUIRE(x && codebook && logits, LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(ldl >= K, LBM_EINVAL, "%s: ldl (%lld) < K (%d)", what, (long long)ldl, K);
    if (layout == LBM_VQ_ROWS)
        LBM_REQUIRE(ldx >= D, LBM_EINVAL, "%s: ldx (%lld) < D (%d)", what, (long long)ldx, D);
    else
        LBM_REQUIRE(S >= 1 && ldx >= S && N % S == 0, LBM_EINVAL,
                    "%s: channel-major needs 1 <= S <= ldx and N %% S == 0 (N=%lld, S=%lld, ldx=%lld)", what, (long long)N, (long long)S,
                    (long long)ldx);
    const Operand b{codebook, D, 0, 0, K};
    const bool wide_b = aligned16(codebook, D);
    const float scale = (float)(1.0 / temperature);
    hipStream_t st = lbm::as_stream(stream);
    if (layout == LBM_VQ_ROWS) {
        const Operand a{x, ldx, 0, 0, N};
        return wide_b && aligned16(x, ldx)
                   ? launch_mm<KCV, KCV, EPI_SCORES>(what, a, b, logits, ldl, D, 1, D, scale, e_sqnorm_or_null, nullptr, st)
                   : launch_mm<KC, KC, EPI_SCORES>(what, a, b, logits, ldl, D, 1, D, scale, e_sqnorm_or_null, nullptr, st);
    }
    const Operand a{x, ldx, S, (int64_t)D * ldx, N};
    return wide_b ? launch_mm<MC, KCV, EPI_SCORES>(what, a, b, logits, ldl, D, 1, D, scale, e_sqnorm_or_null, nullptr, st)
                  : launch_mm<MC, KC, EPI_SCORES>(what, a, b, logits, ldl, D, 1, D, scale, e_sqnorm_or_null, nullptr, st);
}

extern "C" size_t lbm_code_logits_grad_workspace_bytes(int64_t N, int32_t D, int32_t K) {
    if (N < 0 || D < 1 || K < 1) return 0;
    if (N == 0) return 16;
    const Split rows = split_rows(N, D, K), codes = split_codes(N, D, K);
    const size_t for_e = (size_t)rows.n * (size_t)K * (size_t)(D + 1) * sizeof(float);
    const size_t for_x = codes.n > 1 ? (size_t)codes.n * (size_t)N * (size_t)D * sizeof(float) : 0;
    return for_e > for_x ? for_e : for_x;
}

extern "C" int lbm_code_logits_grad_f32(const float* g, int64_t ldg, const float* x, int64_t ldx, const float* codebook, float* dx_or_null,
                                        float* de_or_null, int32_t norm_grad, void* workspace, int64_t N, int32_t D, int32_t K,
                                        double temperature, lbm_stream_t stream) {
    const char* what = "lbm_code_logits_grad_f32";
    LBM_REQUIRE(N >= 0 && D >= 1 && K >= 1, LBM_EINVAL, "%s: bad sizes (N=%lld D=%d K=%d)", what, (long long)N, D, K);
    LBM_REQUIRE(usable(temperature), LBM_EINVAL, "%s: temperature must be positive and finite, and 2 / temperature too", what);
    LBM_REQUIRE(codebook && (N == 0 || g), LBM_EINVAL, "%s: NULL pointer", what);
    LBM_REQUIRE(N == 0 || ldg >= K, LBM_EINVAL, "%s: ldg (%lld) < K (%d)", what, (long long)ldg, K);
    if (dx_or_null == nullptr && de_or_null == nullptr) return LBM_OK;
    LBM_REQUIRE(workspace != nullptr && ((uintptr_t)workspace & 15) == 0, LBM_EINVAL, "%s: needs a 16-byte aligned workspace", what);
    LBM_REQUIRE(de_or_null == nullptr || N == 0 || (x && ldx >= D), LBM_EINVAL, "%s: the codebook's gradient needs x with ldx >= D (%d)", what, D);
    hipStream_t st = lbm::as_stream(stream);
    const float scale = (float)(2.0 / temperature);
    float* part = static_cast<float*>(workspace);
    int rc = LBM_OK;
    if (dx_or_null != nullptr && N > 0) {
        const Operand a{g, ldg, 0, 0, N}, b{codebook, D, 0, 0, D};
        const bool wide_ab = aligned16(g, ldg) && aligned16(codebook, D);
        const Split sp = split_codes(N, D, K);
        if (sp.n == 1) {
            rc = wide_ab ? launch_mm<KCV, MCV, EPI_SCALE>(what, a, b, dx_or_null, D, K, 1, K, scale, nullptr, nullptr, st)
                         : launch_mm<KC, MC, EPI_SCALE>(what, a, b, dx_or_null, D, K, 1, K, scale, nullptr, nullptr, st);
        } else {
            rc = wide_ab ? launch_mm<KCV, MCV, EPI_PARTIAL>(what, a, b, part, D, K, sp.n, sp.piece, 1.f, nullptr, nullptr, st)
                         : launch_mm<KC, MC, EPI_PARTIAL>(what, a, b, part, D, K, sp.n, sp.piece, 1.f, nullptr, nullptr, st);
            if (rc == LBM_OK) rc = launch_join<false>(what, part, nullptr, codebook, dx_or_null, sp.n, N, D, scale, st);
        }
    }
    if (rc != LBM_OK || de_or_null == nullptr) return rc;
    Split sp{0, kBK};
    float* rowsum = nullptr;
    if (N > 0) {
        sp = split_rows(N, D, K);
        rowsum = part + (int64_t)sp.n * K * D;
        const Operand a{g, ldg, 0, 0, K}, b{x, ldx, 0, 0, D};
        // four rows of an operand at a time: their number has to be a multiple of four too
        rc = aligned16(g, ldg) && aligned16(x, ldx) && ((K | D) & 3) == 0
                 ? launch_mm<MCV, MCV, EPI_PARTIAL>(what, a, b, part, D, N, sp.n, sp.piece, 1.f, nullptr, rowsum, st)
                 : launch_mm<MC, MC, EPI_PARTIAL>(what, a, b, part, D, N, sp.n, sp.piece, 1.f, nullptr, rowsum, st);
        if (rc != LBM_OK) return rc;
    }
    return norm_grad ? launch_join<true>(what, part, rowsum, codebook, de_or_null, sp.n, K, D, scale, st)
                     : launch_join<false>(what, part, rowsum, codebook, de_or_null, sp.n, K, D, scale, st);
}
