// inbatch_loss.hip — the fine-tuning loss over the in-batch score matrix and its gradient on gfx950 (reference
// retrieval/criterions.py:10-27: cross entropy of [q c^T | q . neg] against the diagonal).
//
//   S = [q c^T | q . neg]  (B x B | B x 1),  lse_i = log sum_j exp S_ij,  loss = mean_i (lse_i - S_ii)
//   G = (exp(S - lse) - 1[j = i]) dloss / B,  dq = G c + G_neg neg,  dc = G^T q,  dneg = G_neg q
//
// Where the target has nearly all of a row's weight, lse - S_ii and exp(S_ii - lse) - 1 are differences of nearly equal numbers
// and a float32 gradient would be mostly rounding.  So the rows' pass keeps the OTHER columns' sum apart: with
// u = sum_(j != i) exp(S_ij - S_ii), the row's loss is log1p(u) and G_ii = -u / (1 + u) dloss / B, good to float32's last bits.
// Little work: the three products run on v_mfma_f32_32x32x2_f32 (an fma chain: no operand is rounded), G is made from S and
// lse where a product's tile is loaded.  Much work: every operand is split into two float16 planes, x = (hi + lo) 2^-e with
// one e for the elements that a sum runs over, and hi hi' + hi lo' + lo hi' run on v_mfma_f32_32x32x16_f16, sixteen times
// float32's rate for three times its products.  hi + lo is good to 22 bits of an element, or to 2^-39 of the largest one of its e
// where that is more (elements below 2^-17 of it): what a term loses is at most 3 2^-22 of it or 2^-38 of the largest one a sum
// could have, less than the float32 sums' own rounding over a row of 64 and more.  (An infinity in q or c has no second plane: its
// scores come out as NaN.)  So that rows of very different weight in
// a batch (a confident row's gradient is e^-margin of a hard one's) and of very different size keep that, S has an e for every row
// of q and of c, dq one for every row of G weighted by the sizes of c's rows, dc one for every COLUMN of G weighted by q's: two
// pairs of planes of G.  S is kept (4 B^2 bytes) instead of multiplied out again in the backward pass (2 B^2 d flops).
#include "otter_common.h"
#include "otter_device.h"

namespace {
using namespace otter;

constexpr int LOSS_MAX_B = 65536;
constexpr int MEAN_B = 48;         // up to here the rows' launch takes the mean as well
constexpr int KB = 32;             // contraction depth of a staged tile
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // 16-byte load at any 4-byte address

struct LossArgs {
    const float *q, *c, *neg;      // [B][d]; neg may be null
    float* scores;                 // [B][ld]
    float* part;                   // [splits][B][B] when splits > 1
    float *lse, *rest;             // [B]: of the row; 1 - the target's probability
    float *rowloss, *loss;         // [B], [1]
    unsigned* done;                // rows whose loss is there: cleared by the scores' launch, counted by the rows'
    const float* dloss;            // [1]
    float *dq, *dc, *dneg;
    int B, d, ld, splits, kchunk;
    float* gpart;                  // [gsplits][2][B][d] of dq and dc when gsplits > 1
    int gsplits, gchunk;           // gchunk: the contraction depth of a piece
};

// n values of a row of a matrix with `rows` rows, zeros outside: v[e] = m[row][col + e]
__device__ __forceinline__ f4u load4(const float* m, long long ld, int rows, int cols, int row, int col) {
    f4u v = {0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
        const float* p = m + (long long)row * ld + col;
        if (col + 3 < cols) return *reinterpret_cast<const f4u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < cols) v[e] = p[e];
    }
    return v;
}

struct Plain {                     // a stored matrix
    const float* m;
    int rows, cols;
    long long ld;
    __device__ __forceinline__ f4u operator()(int row, int col) const { return load4(m, ld, rows, cols, row, col); }
};

struct Grad {                      // G[i][j .. j + 3] from the scores
    const float *scores, *lse, *rest;
    long long ld;
    int B;
    float g;                       // dloss / B
    __device__ __forceinline__ f4u operator()(int i, int j) const {
        f4u v = load4(scores, ld, B, B, i, j);
        const float l = i < B ? lse[i] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i < B && j + e < B ? (j + e == i ? -rest[i] : __expf(v[e] - l)) * g : 0.0f;
        return v;
    }
};

// acc[BM x BM tile at (m0, n0)] += sum over k in [ka, kb) A(m, k) B(n, k).  An operand whose k is contiguous in memory
// (KC) lies in LDS as rows of 32 k, in 16-byte chunks swizzled by row; one whose m / n is contiguous as 32 rows of BM
// values.  Either way a lane's four values of a chunk have k = 4 (2 j + lane half) + e: both sides contract alike.
template <int BM, bool KC>
struct Stage {
    static constexpr int N4 = BM * KB / 4 / 256;       // float4 a thread
    f4u r[N4];
    template <typename F>
    __device__ __forceinline__ void load(const F& f, int m0, int k0, int kend) {
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            const int t = threadIdx.x + 256 * i;
            if constexpr (KC) {
                const int k = k0 + (t % (KB / 4)) * 4;
                r[i] = f(m0 + t / (KB / 4), k);
                if (k + 3 >= kend) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k + e >= kend) r[i][e] = 0.0f;
                }
            } else {
                const int k = k0 + t / (BM / 4);
                r[i] = f(k, m0 + (t % (BM / 4)) * 4);
                if (k >= kend) r[i] = f4u{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            const int t = threadIdx.x + 256 * i;
            int at;
            if constexpr (KC) {
                const int m = t / (KB / 4), c = t % (KB / 4);
                at = m * KB + ((c ^ ((m >> 1) & 7)) << 2);
            } else {
                at = t * 4;
            }
            *reinterpret_cast<float4*>(lds + at) = make_float4(r[i][0], r[i][1], r[i][2], r[i][3]);
        }
    }
    static __device__ __forceinline__ float4 frag(const float* lds, int m, int c) {
        if constexpr (KC) {
            return *reinterpret_cast<const float4*>(lds + m * KB + ((c ^ ((m >> 1) & 7)) << 2));
        } else {
            return make_float4(lds[(4 * c) * BM + m], lds[(4 * c + 1) * BM + m], lds[(4 * c + 2) * BM + m], lds[(4 * c + 3) * BM + m]);
        }
    }
};

template <int BM, bool AKC, bool BKC, typename FA, typename FB>
__device__ __forceinline__ void product(f32x16 (&acc)[BM / 64][BM / 64], const FA& fa, const FB& fb, int m0, int n0, int ka,
                                        int kb, float* lds) {
    constexpr int MB = BM / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BM / 2);
    float* sA = lds;
    float* sB = lds + BM * KB;
    Stage<BM, AKC> ra;
    Stage<BM, BKC> rb;
    ra.load(fa, m0, ka, kb);
    rb.load(fb, n0, ka, kb);
    for (int k0 = ka; k0 < kb; k0 += KB) {
        __syncthreads();
        ra.store(sA);
        rb.store(sB);
        __syncthreads();
        if (k0 + KB < kb) {                       // the next tile is in flight while this one is multiplied
            ra.load(fa, m0, k0 + KB, kb);
            rb.load(fb, n0, k0 + KB, kb);
        }
#pragma unroll
        for (int j = 0; j < KB / 8; ++j) {
            float4 x[MB], y[MB];
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                x[i] = Stage<BM, AKC>::frag(sA, wm + 32 * i + l31, 2 * j + h);
                y[i] = Stage<BM, BKC>::frag(sB, wn + 32 * i + l31, 2 * j + h);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int n = 0; n < MB; ++n)
                        acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(reinterpret_cast<const float*>(&x[i])[e],
                                                                        reinterpret_cast<const float*>(&y[n])[e], acc[i][n], 0, 0, 0);
        }
    }
}

template <int BM>
__device__ __forceinline__ void clear(f32x16 (&acc)[BM / 64][BM / 64]) {
#pragma unroll
    for (int i = 0; i < BM / 64; ++i)
#pragma unroll
        for (int n = 0; n < BM / 64; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][n][r] = 0.0f;
}

// row of the tile that register r of an accumulator holds (of lane half 0; half 1 has the fourth after it)
__device__ __forceinline__ constexpr int acc_row(int r) { return (r & 3) + 8 * (r >> 2); }

// out(row, col, accumulator): register r is element (row + acc_row(r), col)
template <int BM, typename F>
__device__ __forceinline__ void each(const f32x16 (&acc)[BM / 64][BM / 64], int m0, int n0, const F& out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BM / 2);
#pragma unroll
    for (int i = 0; i < BM / 64; ++i)
#pragma unroll
        for (int n = 0; n < BM / 64; ++n) out(m0 + wm + 32 * i + 4 * h, n0 + wn + 32 * n + l31, acc[i][n]);
}

// S = q c^T; grid (tiles, splits of d).  float32 products, tiles of 64: the chip is filled by pieces of d (B = 64 d = 2304:
// 36 workgroups, 5.6 us; 4096 x 63, 4096 workgroups: 37 us, 57 TFLOP/s).
template <int BM>
__global__ __launch_bounds__(256) void loss_scores_kernel(LossArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[2 * BM * KB];
    const int nt = (a.B + BM - 1) / BM;
    const int t = xcd_remap(blockIdx.x, gridDim.x);
    const int m0 = (t / nt) * BM, n0 = (t % nt) * BM;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.done = 0;
    const int ka = blockIdx.y * a.kchunk, kb = min(a.d, ka + a.kchunk);
    f32x16 acc[BM / 64][BM / 64];
    clear<BM>(acc);
    product<BM, true, true>(acc, Plain{a.q, a.B, a.d, a.d}, Plain{a.c, a.B, a.d, a.d}, m0, n0, ka, kb, lds);
    float* out = a.splits > 1 ? a.part + (size_t)blockIdx.y * a.B * a.B : a.scores;
    const long long ld = a.splits > 1 ? a.B : a.ld;
    each<BM>(acc, m0, n0, [&](int i0, int j, const f32x16& v) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (i0 + acc_row(r) < a.B && j < a.B) out[(long long)(i0 + acc_row(r)) * ld + j] = v[r];
    });
}

// the larger one, a NaN if there is one (fmaxf would drop it, and a row whose scores are not numbers would have a finite loss)
__device__ __forceinline__ float max_(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// maximum and sum of two parts of a row; parts without weight (no scores, or -inf throughout) have the sum 0
__device__ __forceinline__ void online(float& m, float& l, float m2, float l2) {
    const float n = max_(m, m2);
    if (n == -INFINITY) return;
    l = l * __expf(m - n) + l2 * __expf(m2 - n);
    m = n;
}

// one workgroup a row: the pieces of S summed in order (PIECES), the hard negative's score, lse and the row's loss; of a
// small batch the last workgroup takes the mean as well (MEAN).  That saves the host a launch and costs the GPU a fence for
// every row: forward and backward calls back to back, us, own launch and here, d = 768: B = 4 22.5 and 17.9, 32 22.8 and 19.0, 48 22.5 and
// 21.7, 64 22.2 and 23.1, 128 25.3 and 28.1; d = 2304: 48 23.0 and 22.6, 64 23.1 and 23.2, 96 24.6 and 26.7 (the kernels alone, d =
// 768: B = 4 11.2 and 11.2, 32 11.3 and 12.2, 64 11.9 and 13.6, 200 12.7 and 16.9).
template <bool PIECES, bool MEAN>
__global__ __launch_bounds__(256) void loss_rows_kernel(LossArgs a) {
    __shared__ float sm[4], sl[4], sd[4];
    __shared__ double sum[4];
    __shared__ bool last;
    const int i = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* row = a.scores + (long long)i * a.ld;
    float m = -INFINITY, l = 0.0f;
    if constexpr (PIECES) {
        for (int j = threadIdx.x; j < a.B; j += 256) {
            float s = 0.0f;
#pragma unroll 12
            for (int p = 0; p < a.splits; ++p) s += a.part[((size_t)p * a.B + i) * a.B + j];
            row[j] = s;
            if (j != i) online(m, l, s, 1.0f);
        }
    } else {
        // four scores a load: one exponential each and one for the four's maximum
#pragma unroll 2
        for (int j = threadIdx.x * 4; j < a.B; j += 1024) {
            f4u v = load4(row, 0, 1, a.B, 0, j);
#pragma unroll
            for (int e = 1; e < 4; ++e)
                if (j + e >= a.B) v[e] = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e == i) v[e] = -INFINITY;
            const float top = max_(max_(v[0], v[1]), max_(v[2], v[3])), n = max_(m, top), base = n == -INFINITY ? 0.0f : n;
            l = l * __expf(m - base) + ((__expf(v[0] - base) + __expf(v[1] - base)) + (__expf(v[2] - base) + __expf(v[3] - base)));
            m = n;
        }
    }
    float dot = 0.0f;
    if (a.neg)
#pragma unroll 4
        for (int e = threadIdx.x; e < a.d; e += 256) dot = fmaf(a.q[(long long)i * a.d + e], a.neg[(long long)i * a.d + e], dot);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o);
        online(m, l, m2, l2);
        dot += __shfl_xor(dot, o);
    }
    if (lane == 0) {
        sm[wave] = m;
        sl[wave] = l;
        sd[wave] = dot;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) online(m, l, sm[w], sl[w]);
        if (a.neg) {
            dot = sd[0] + sd[1] + sd[2] + sd[3];
            row[a.B] = dot;
            online(m, l, dot, 1.0f);
        }
        // m, l: the other columns (l = 0 if there are none)
        const float t = row[i];
        float lse, rest, loss;
        if (m <= t) {
            const float u = l * __expf(m - t) + (t - t);   // the last: 0, and NaN for a target's score of +inf (inf - inf)
            loss = log1pf(u);
            lse = t + loss;
            rest = u / (1.0f + u);
        } else {
            lse = m + logf(l + __expf(t - m));
            loss = lse - t;
            rest = 1.0f - __expf(t - lse);
        }
        a.lse[i] = lse;
        a.rest[i] = rest;
        a.rowloss[i] = loss;
        if (MEAN) {
            __threadfence();                               // the row's loss before the count of it
            last = atomicAdd(a.done, 1u) == (unsigned)a.B - 1u;
        }
    }
    if (!MEAN) return;
    __syncthreads();
    if (!last) return;
    // the workgroup that finished last takes the mean, in one fixed order whichever it is
    __threadfence();
    double s = 0.0;
    for (int k = threadIdx.x; k < a.B; k += 256) s += (double)__builtin_nontemporal_load(a.rowloss + k);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) sum[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) *a.loss = (float)((sum[0] + sum[1] + sum[2] + sum[3]) / a.B);
}

// 4 us, a launch and the latency of a few loads
__global__ __launch_bounds__(1024) void loss_mean_kernel(LossArgs a) {
    __shared__ double red[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < a.B; i += 1024) s += (double)a.rowloss[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += red[w];
        *a.loss = (float)(s / a.B);
    }
}

// Elements (row0 + acc_row(r), n) of dq (second: of dc): a piece of their sums to its place, or, where there is one piece, the
// gradients themselves with the hard negative's share.
__device__ __forceinline__ void put_grad(const LossArgs& a, bool second, int piece, float g, int row0, int n, const f32x16& v) {
    if (a.gsplits > 1 || second || !a.neg) {
        float* out = a.gsplits > 1 ? a.gpart + ((long long)piece * 2 + second) * a.B * a.d : second ? a.dc : a.dq;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (row0 + acc_row(r) < a.B && n < a.d) out[(long long)(row0 + acc_row(r)) * a.d + n] = v[r];
        return;
    }
    const int nc = min(n, a.d - 1);
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += 8) {
        float sn[8], lse[8], x[8], y[8];             // eight elements' loads before the first use
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = min(row0 + acc_row(r0 + r), a.B - 1);
            sn[r] = a.scores[(long long)row * a.ld + a.B];
            lse[r] = a.lse[row];
            x[r] = a.neg[(long long)row * a.d + nc];
            y[r] = a.q[(long long)row * a.d + nc];
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = row0 + acc_row(r0 + r);
            if (row >= a.B || n >= a.d) continue;
            const float gn = __expf(sn[r] - lse[r]) * g;
            a.dq[(long long)row * a.d + n] = fmaf(gn, x[r], v[r0 + r]);
            a.dneg[(long long)row * a.d + n] = gn * y[r];
        }
    }
}

// dq (blockIdx.y = 0) and dc from their pieces, summed in order; bound by reading them
__global__ __launch_bounds__(256) void loss_join_kernel(LossArgs a) {
    const bool second = blockIdx.y;
    const long long n = (long long)a.B * a.d, at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    const float* p = a.gpart + (second ? n : 0) + at;
    const int m = (int)min(4ll, n - at);
    f4u v = {0.f, 0.f, 0.f, 0.f};
    if (m == 4) {
#pragma unroll 4
        for (int k = 0; k < a.gsplits; ++k) v += *reinterpret_cast<const f4u*>(p + 2 * n * k);
    } else {
        for (int k = 0; k < a.gsplits; ++k)
            for (int e = 0; e < m; ++e) v[e] += p[2 * n * k + e];
    }
    const float g = *a.dloss / (float)a.B;
    float* out = second ? a.dc : a.dq;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= m) break;
        float x = v[e];
        if (!second && a.neg) {
            const long long row = (at + e) / a.d;
            const float gn = __expf(a.scores[row * a.ld + a.B] - a.lse[row]) * g;
            x = fmaf(gn, a.neg[at + e], x);
            a.dneg[at + e] = gn * a.q[at + e];
        }
        out[at + e] = x;
    }
}

// dq and dc, half the grid each; blockIdx.y: a piece of the contraction.  G is made from S where a tile of it is loaded (once for
// every 64 columns of d).  B = 64 d = 2304: 8 us; 400 x 256 in 12 pieces: 33 -> 11 us with the join.
template <int BM>
__global__ __launch_bounds__(256) void loss_grad_kernel(LossArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[2 * BM * KB];
    const int nt = (a.d + BM - 1) / BM, half = gridDim.x / 2;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const bool second = id >= half;
    const int t = second ? id - half : id;
    const int m0 = (t / nt) * BM, n0 = (t % nt) * BM;
    const int ka = blockIdx.y * a.gchunk, kb = min(a.B, ka + a.gchunk);
    const float g = *a.dloss / (float)a.B;
    const Grad G{a.scores, a.lse, a.rest, a.ld, a.B, g};
    f32x16 acc[BM / 64][BM / 64];
    clear<BM>(acc);
    if (second)
        product<BM, false, false>(acc, G, Plain{a.q, a.B, a.d, a.d}, m0, n0, ka, kb, lds);
    else
        product<BM, true, false>(acc, G, Plain{a.c, a.B, a.d, a.d}, m0, n0, ka, kb, lds);
    each<BM>(acc, m0, n0, [&](int i0, int n, const f32x16& v) { put_grad(a, second, blockIdx.y, g, i0, n, v); });
}

// ------------------------------------------------------------------ two float16 planes
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));

constexpr int SB = 32;             // contraction depth of a staged tile

struct SplitArgs {
    const float *q, *c;            // [B][d]
    unsigned short* plane[4];      // q hi, q lo, c hi, c lo: [Bp][dp], zeros outside [B][d]
    float *qs, *cs;                // [Bp]: what a row of the planes is to be multiplied by, 2^-14 of its largest element's power of two
    unsigned short* gplane[4];     // backward, of G: hi and lo for dq, hi and lo for dc; [Bp][Bp], zeros outside [B][B]
    float *gq, *gc;                // [Bp]: the scale of a row of the first pair, of a column of the second
    float *rowtop, *coltop;        // [4 colblocks][Bp], [strips][Bp]: parts of the largest weighted elements of rows and columns
    int B, d, Bp, dp;
    int strip;                     // rows of a part of coltop; Bp is a multiple of it
};

// 2^(14 - exponent of top): the largest element then lies in [2^14, 2^15), the smallest half step of a float16 (2^-25) is
// 2^-39 of it.  Exact in both directions.
__device__ __forceinline__ float plane_scale(float top) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    return top > 0.0f && e < 128 ? __uint_as_float((u32)(min(max(14 - e, -126), 126) + 127) << 23) : 1.0f;
}

__device__ __forceinline__ void split1(float x, unsigned short& hi, unsigned short& lo) {
    const _Float16 h = (_Float16)x;
    const _Float16 l = (_Float16)(x - (float)h);
    hi = __builtin_bit_cast(unsigned short, h);
    lo = __builtin_bit_cast(unsigned short, l);
}

// One wave a row of one matrix, which has its own scale.  4096 x 768: 12 us.
__global__ __launch_bounds__(256) void loss_split_kernel(SplitArgs a) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, m = blockIdx.y;
    if (row >= a.Bp) return;
    const float* x = (m ? a.c : a.q) + (long long)row * a.d;
    float t = 0.0f;
    if (row < a.B) {
        for (int i = lane; i < a.d; i += 64) t = fmaxf(t, fabsf(x[i]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o));
    }
    const float f = plane_scale(t);
    unsigned short *hi = a.plane[2 * m] + (long long)row * a.dp, *lo = a.plane[2 * m + 1] + (long long)row * a.dp;
    for (int i = lane; i < a.dp / 4; i += 64) {
        const f4u v = load4(m ? a.c : a.q, a.d, a.B, a.d, row, 4 * i);
        unsigned short h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split1(v[e] * f, h[e], l[e]);
        __builtin_memcpy(hi + 4 * i, h, 8);
        __builtin_memcpy(lo + 4 * i, l, 8);
    }
    if (lane == 0) (m ? a.cs : a.qs)[row] = 1.0f / f;
}

// a row's size as a power of two, from what its planes are multiplied by
__device__ __forceinline__ float row_size(float s) { return s * 16384.0f; }

// Parts of max_j |G_ij| size(c_j) for every row and max_i |G_ij| size(q_i) for every column: a workgroup takes `strip` rows x 1024
// columns, a thread four columns, four rows at a time and the next four on their way.  One read of S: B = 4096 25 us (2.7 TB/s).
__global__ __launch_bounds__(256) void loss_gtop_kernel(LossArgs a, SplitArgs s) {
    const int j = blockIdx.y * 1024 + threadIdx.x * 4, i0 = blockIdx.x * s.strip, last = i0 + s.strip - 1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float* rowtop = s.rowtop + (long long)(blockIdx.y * 4 + wave) * s.Bp;
    float size[4], col[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) size[e] = row_size(s.cs[min(j, s.Bp - 4) + e]);
    f4u next[4];
    auto fetch = [&](int i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) next[r] = load4(a.scores, a.ld, a.B, a.B, min(i + r, last), j);   // past the strip's end its last row again
    };
    fetch(i0);
    for (int i = i0; i <= last; i += 4) {
        float t[4];
        f4u v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = next[r];
        if (i + 4 <= last) fetch(i + 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = min(i + r, last);
            const float size_q = row_size(s.qs[row]), l = row < a.B ? a.lse[row] : 0.0f, rest = row < a.B ? a.rest[row] : 0.0f;
            t[r] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float g = row < a.B && j + e < a.B ? (j + e == row ? rest : __expf(v[r][e] - l)) : 0.0f;
                t[r] = fmaxf(t[r], g * size[e]);
                col[e] = fmaxf(col[e], g * size_q);
            }
        }
        // four maxima over 64 lanes: two steps halve the values and the lanes that hold each, lane l keeps row 2 (l & 1) + (l >> 1 & 1)
#pragma unroll
        for (int r = 0; r < 2; ++r) t[r] = fmaxf(lane & 1 ? t[2 + r] : t[r], __shfl_xor(lane & 1 ? t[r] : t[2 + r], 1));
        float top = fmaxf(lane & 2 ? t[1] : t[0], __shfl_xor(lane & 2 ? t[0] : t[1], 2));
#pragma unroll
        for (int o = 4; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const int row = i + 2 * (lane & 1) + (lane >> 1);
        if (lane < 4 && row <= last) rowtop[row] = top;
    }
    if (j < s.Bp) *reinterpret_cast<float4*>(s.coltop + (long long)blockIdx.x * s.Bp + j) = make_float4(col[0], col[1], col[2], col[3]);
}

// blockIdx.y = 0: the rows' scales, 1: the columns'; 64 of them a workgroup, a quarter of the parts a wave
__global__ __launch_bounds__(256) void loss_gscale_kernel(SplitArgs s, int nrow, int ncol) {
    __shared__ float top[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane, parts = blockIdx.y ? ncol : nrow;
    const float* p = (blockIdx.y ? s.coltop : s.rowtop) + n;
    float t = 0.0f;
#pragma unroll 8
    for (int k = wave; k < parts; k += 4) t = fmaxf(t, p[(long long)k * s.Bp]);
    top[wave][lane] = t;
    __syncthreads();
    if (wave == 0) (blockIdx.y ? s.gc : s.gq)[n] = plane_scale(fmaxf(fmaxf(top[0][lane], top[1][lane]), fmaxf(top[2][lane], top[3][lane])));
}

// G without dloss / B as the two pairs of planes: one read of B^2 float32 and a write of twice as much, B = 4096
// 33 us (6.1 TB/s).  Made where the products load it, it would be made again for every 64 of d.
__global__ __launch_bounds__(256) void loss_gplanes_kernel(LossArgs a, SplitArgs s) {
    const int nb = (s.Bp + 1023) / 1024, i = blockIdx.x / nb, j = (blockIdx.x % nb * 256 + threadIdx.x) * 4;
    if (j >= s.Bp) return;
    const Grad G{a.scores, a.lse, a.rest, a.ld, a.B, 1.0f};
    const f4u v = G(i, j);
    const float size_q = row_size(s.qs[i]), f = s.gq[i];
    const long long at = (long long)i * s.Bp + j;
    unsigned short h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split1(v[e] * row_size(s.cs[j + e]) * f, h[e], l[e]);
    __builtin_memcpy(s.gplane[0] + at, h, 8);
    __builtin_memcpy(s.gplane[1] + at, l, 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) split1(v[e] * size_q * s.gc[j + e], h[e], l[e]);
    __builtin_memcpy(s.gplane[2] + at, h, 8);
    __builtin_memcpy(s.gplane[3] + at, l, 8);
}

// A tile of one operand, both planes, on its way to LDS.  KC: SB contiguous k of W rows (80 bytes a row in LDS); otherwise W
// contiguous elements of SB k-rows (32 bytes of padding a row).  Neither the straight nor the transposed reads conflict.
template <int W, bool KC>
struct Planes {
    static constexpr int PITCH = KC ? SB * 2 + 16 : W * 2 + 32;
    static constexpr int BYTES = (KC ? W : SB) * PITCH;          // one plane
    static constexpr int N = W * SB * 2 / 16 / 256;              // 16-byte chunks a thread and plane
    static constexpr int CH = KC ? SB / 8 : W / 8;               // chunks a row
    u32x4 v[2][N];
    __device__ __forceinline__ void load(const unsigned short* hi, const unsigned short* lo, long long ld, int w0, int k0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int t = threadIdx.x + 256 * i, r = t / CH, c = t % CH;
            const long long at = (long long)(KC ? w0 + r : k0 + r) * ld + (KC ? k0 : w0) + 8 * c;
            v[0][i] = *reinterpret_cast<const u32x4*>(hi + at);
            v[1][i] = *reinterpret_cast<const u32x4*>(lo + at);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int t = threadIdx.x + 256 * i;
                *reinterpret_cast<u32x4*>(lds + p * BYTES + (t / CH) * PITCH + (t % CH) * 16) = v[p][i];
            }
    }
    // 8 values of k for row w0 + (lane & 31): k = 16 s + 8 h + (0 .. 7) where both operands are KC, otherwise the order of the
    // transposed reads, k = 16 s + 4 h + (0 .. 3) and 8 more
    template <bool BOTH>
    static __device__ __forceinline__ f16x8 frag(const char* plane, int w0, int s, int lane) {
        const int h = lane >> 5, l31 = lane & 31;
        if constexpr (KC) {
            const char* p = plane + (w0 + l31) * PITCH + s * 32;
            if constexpr (BOTH) return *reinterpret_cast<const f16x8*>(p + h * 16);
            const s16x4 x[2] = {*reinterpret_cast<const s16x4*>(p + h * 8), *reinterpret_cast<const s16x4*>(p + 16 + h * 8)};
            return __builtin_bit_cast(f16x8, x);
        } else {
            const int i16 = lane & 15;
            const char* p = plane + (16 * s + 4 * h + (i16 >> 2)) * PITCH + (w0 + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3)) * 2;
            const s16x4 x[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)p),
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)(p + 8 * PITCH))};
            return __builtin_bit_cast(f16x8, x);
        }
    }
};

// acc += A B^T over k in [ka, kb), multiples of SB: 4 waves as 2 x 2, a wave 64 x (BN / 2); lds: both operands' planes, one stage (two stages
// would halve the workgroups of a CU, which are what hides the loads)
template <int BN, bool AKC, bool BKC>
__device__ __forceinline__ void product16(f32x16 (&acc)[2][BN / 64], const unsigned short* Ahi, const unsigned short* Alo,
                                          long long lda, const unsigned short* Bhi, const unsigned short* Blo, long long ldb, int m0,
                                          int n0, int ka, int kb, char* lds) {
    constexpr int NB = BN / 64;
    constexpr bool BOTH = AKC && BKC;
    typedef Planes<128, AKC> PA;
    typedef Planes<BN, BKC> PB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * (BN / 2);
    char* sA = lds;
    char* sB = lds + 2 * PA::BYTES;
    PA ra;
    PB rb;
    ra.load(Ahi, Alo, lda, m0, ka);
    rb.load(Bhi, Blo, ldb, n0, ka);
    for (int k0 = ka; k0 < kb; k0 += SB) {
        __syncthreads();
        ra.store(sA);
        rb.store(sB);
        __syncthreads();
        if (k0 + SB < kb) {
            ra.load(Ahi, Alo, lda, m0, k0 + SB);
            rb.load(Bhi, Blo, ldb, n0, k0 + SB);
        }
#pragma unroll
        for (int s = 0; s < SB / 16; ++s) {
            f16x8 ah[2], al[2], bh[NB], bl[NB];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ah[i] = PA::template frag<BOTH>(sA, wm + 32 * i, s, lane);
                al[i] = PA::template frag<BOTH>(sA + PA::BYTES, wm + 32 * i, s, lane);
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                bh[n] = PB::template frag<BOTH>(sB, wn + 32 * n, s, lane);
                bl[n] = PB::template frag<BOTH>(sB + PB::BYTES, wn + 32 * n, s, lane);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[n], acc[i][n], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[n], acc[i][n], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[n], acc[i][n], 0, 0, 0);
        }
    }
}

template <int BN, typename F>
__device__ __forceinline__ void each16(const f32x16 (&acc)[2][BN / 64], int m0, int n0, const F& out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * (BN / 2);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < BN / 64; ++n) out(m0 + wm + 32 * i + 4 * h, n0 + wn + 32 * n + l31, acc[i][n]);
}

template <int NB>
__device__ __forceinline__ void clear16(f32x16 (&acc)[2][NB]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][n][r] = 0.0f;
}

// 128 x 128 tiles; B = 4096 d = 768: 130 us, 0.6 PFLOP/s of float16 products (a large product: 1.1), short loops of 24 steps
__global__ __launch_bounds__(256, 2) void loss_scores16_kernel(LossArgs a, SplitArgs s) {
    __shared__ __attribute__((aligned(16))) char lds[4 * Planes<128, true>::BYTES];
    const int nt = s.Bp / 128, t = xcd_remap(blockIdx.x, gridDim.x);
    const int m0 = (t / nt) * 128, n0 = (t % nt) * 128;
    const int ka = blockIdx.y * a.kchunk;
    float* out = a.splits > 1 ? a.part + (size_t)blockIdx.y * a.B * a.B : a.scores;
    const long long ld = a.splits > 1 ? a.B : a.ld;
    f32x16 acc[2][2];
    clear16<2>(acc);
    product16<128, true, true>(acc, s.plane[0], s.plane[1], s.dp, s.plane[2], s.plane[3], s.dp, m0, n0, ka, min(s.dp, ka + a.kchunk), lds);
    each16<128>(acc, m0, n0, [&](int i0, int j, const f32x16& v) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = i0 + acc_row(r);
            if (i < a.B && j < a.B) out[(long long)i * ld + j] = v[r] * s.qs[i] * s.cs[j];
        }
    });
}

// dq and dc, half the grid each; blockIdx.y: a piece of the contraction.  128 x 64 tiles, so that the 768 of B = 4096 d = 768 are
// resident at once: 240 us, 0.64 PFLOP/s.
__global__ __launch_bounds__(256, 2) void loss_grad16_kernel(LossArgs a, SplitArgs s) {
    constexpr int LDS1 = 2 * Planes<128, true>::BYTES, LDS2 = 2 * Planes<128, false>::BYTES;
    __shared__ __attribute__((aligned(16))) char lds[(LDS1 > LDS2 ? LDS1 : LDS2) + 2 * Planes<64, false>::BYTES];
    const int nt = (a.d + 63) / 64, half = gridDim.x / 2, id = xcd_remap(blockIdx.x, gridDim.x);
    const bool second = id >= half;
    const int t = second ? id - half : id, m0 = (t / nt) * 128, n0 = (t % nt) * 64;
    const float g = *a.dloss / (float)a.B;
    const float* scale = second ? s.gc : s.gq;
    const int ka = blockIdx.y * a.gchunk, kb = min(s.Bp, ka + a.gchunk);
    f32x16 acc[2][1];
    clear16<1>(acc);
    if (second)
        product16<64, false, false>(acc, s.gplane[2], s.gplane[3], s.Bp, s.plane[0], s.plane[1], s.dp, m0, n0, ka, kb, lds);
    else
        product16<64, true, false>(acc, s.gplane[0], s.gplane[1], s.Bp, s.plane[2], s.plane[3], s.dp, m0, n0, ka, kb, lds);
    each16<64>(acc, m0, n0, [&](int i0, int n, f32x16 v) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = v[r] * 0x1p-14f / scale[i0 + acc_row(r)] * g;   // a power of two, and the sizes' 2^14
        put_grad(a, second, blockIdx.y, g, i0, n, v);
    });
}

// ------------------------------------------------------------------ host side
int check_loss(const char* what, int B, int d, int ld, int ncol) {
    if (B < 1 || d < 1) return set_err(OTTER_EINVAL, "%s: bad B=%d d=%d (the mean over no rows is undefined)", what, B, d);
    if (B > LOSS_MAX_B) return set_err(OTTER_EINVAL, "%s: B=%d exceeds %d", what, B, LOSS_MAX_B);
    // the gradients' grid: two halves of 64 x 64 tiles, 256 threads each, fewer than 2^32 threads; it also keeps columns in an int
    if ((int64_t)((B + 63) / 64) * ((d - 1) / 64 + 1) > 0x7FFFFF)
        return set_err(OTTER_EINVAL, "%s: B=%d x d=%d is too large for one launch", what, B, d);
    if (ld < ncol) return set_err(OTTER_EINVAL, "%s: ld=%d is less than the %d columns of the scores", what, ld, ncol);
    return OTTER_OK;
}

// Pieces of a contraction of depth k so that `tiles` workgroups become about `want`, each at least `least` deep
int pieces(long long tiles, int k, int want, int least) {
    const int s = (int)(tiles < want ? want / tiles : 1), most = k / least;
    return max(1, min(s, most));
}

// Two float16 planes or float32, by B^2 d with d in whole tiles.  The planes cost passes over the operands, and in the
// backward pass two over S and one over G.  float32 -> planes, us: forward B = 600 d = 768 30 -> 40, 400 x 2304 44 -> 47, 500 x
// 2304 50 -> 47, 800 x 768 51 -> 43, 1500 x 256 33 -> 35, 2000 x 256 42 -> 40; backward 600 x 768 37 -> 45, 700 x 768 58 -> 49,
// 1000 x 768 90 -> 57, 1000 x 256 33 -> 40, 1200 x 256 49 -> 49, 1500 x 256 76 -> 54, 1500 x 128 41 -> 46, 2000 x 128 58 -> 57,
// 400 x 2304 45 -> 60, 500 x 2304 61 -> 61, 600 x 2304 71 -> 68, 400 x 4608 61 -> 79; of less than 128 columns the passes over
// G are as long as the products, 3000 x 64 68 -> 77, 4096 x 64 103 -> 106.  Of short sums what the planes leave out would show
// beside float32's own rounding: scores of less than 64 elements stay float32 (and take the same time: 38 and 36 us of B = 4096).
double loss_work(int B, int d) { return (double)B * B * round_up(d, 64); }
bool score_planes(int B, int d) { return B > 256 && d >= 64 && loss_work(B, d) > 4e8; }
bool grad_planes(int B, int d) { return B > 500 && loss_work(B, d) > (d < 128 ? 1e9 : 3.6e8); }

// Pieces of the scores' contraction (d) and of the gradients' (B) where there are few tiles, each piece `chunk` deep.  Fewer or
// shallower pieces and more or deeper ones measured 0 to 20 % slower; without pieces: scores of B = 600 d = 768 54 -> 40 us
// forward, gradients of 512 x 40 36 -> 11, 2000 x 63 182 -> 38, 4096 x 64 138 -> 78, 2000 x 768 106 -> 93.  Gradients of up to
// 128 rows are one piece: a launch to join pieces costs what they save.
int score_splits(int B, int d, int* chunk) {
    const bool planes = score_planes(B, d);
    const long long n = planes ? (B + 127) / 128 : (B + 63) / 64;
    const int k = round_up(d, 64), s = pieces(n * n, k, 256, planes ? 128 : 64);
    *chunk = round_up((k + s - 1) / s, KB);
    return (k + *chunk - 1) / *chunk;
}
int grad_splits(int B, int d, int* chunk) {
    const bool planes = grad_planes(B, d);
    const long long tiles = 2ll * (planes ? (B + 127) / 128 : (B + 63) / 64) * ((d + 63) / 64);
    const int k = planes ? round_up(B, 128) : B;
    const int s = planes ? pieces(tiles, k, 1024, 128) : B > 128 ? pieces(tiles, k, 512, 32) : 1;
    *chunk = round_up((k + s - 1) / s, KB);
    return (k + *chunk - 1) / *chunk;
}

int64_t align16(int64_t x) { return (x + 15) / 16 * 16; }

struct Take {                      // pieces of a workspace, 16-byte aligned
    char* p;
    int64_t used = 0;
    template <typename X>
    X* operator()(int64_t n) {
        X* r = reinterpret_cast<X*>(p + used);
        used += align16(n * (int64_t)sizeof(X));
        return r;
    }
};

void take_planes(Take& t, SplitArgs& s) {
    s.qs = t.template operator()<float>(s.Bp);
    s.cs = t.template operator()<float>(s.Bp);
    for (auto& x : s.plane) x = t.template operator()<unsigned short>((int64_t)s.Bp * s.dp);
}

SplitArgs split_args(const float* q, const float* c, int B, int d) {
    SplitArgs s = {};
    s.q = q;
    s.c = c;
    s.B = B;
    s.d = d;
    s.Bp = round_up(B, 128);
    s.dp = round_up(d, 64);
    s.strip = max(4, s.Bp / 128);
    return s;
}

// the pieces of either workspace, and its size
int64_t lay_forward(void* ws, LossArgs& a, SplitArgs& s) {
    Take t{(char*)ws};
    a.rowloss = t.template operator()<float>(a.B);
    a.done = t.template operator()<unsigned>(1);
    if (score_planes(a.B, a.d)) take_planes(t, s);
    if (a.splits > 1) a.part = t.template operator()<float>((int64_t)a.splits * a.B * a.B);
    return t.used;
}

int col_blocks(const SplitArgs& s) { return (s.Bp + 1023) / 1024; }

int64_t lay_backward(void* ws, LossArgs& a, SplitArgs& s) {
    Take t{(char*)ws};
    if (a.gsplits > 1) a.gpart = t.template operator()<float>((int64_t)a.gsplits * 2 * s.B * s.d);
    if (!grad_planes(s.B, s.d)) return t.used;
    take_planes(t, s);
    for (auto& x : s.gplane) x = t.template operator()<unsigned short>((int64_t)s.Bp * s.Bp);
    s.gq = t.template operator()<float>(s.Bp);
    s.gc = t.template operator()<float>(s.Bp);
    s.rowtop = t.template operator()<float>(4ll * col_blocks(s) * s.Bp);
    s.coltop = t.template operator()<float>((int64_t)(s.Bp / s.strip) * s.Bp);
    return t.used;
}

int check_workspace(const char* what, const void* ws, int64_t have, int64_t need) {
    if (need > 0 && (!ws || have < need || ((uintptr_t)ws & 15)))
        return set_err(OTTER_EINVAL, "%s: workspace of %lld bytes, needs %lld, 16-byte aligned", what, (long long)have, (long long)need);
    return OTTER_OK;
}

}  // namespace

extern "C" {

int64_t otter_inbatch_loss_workspace(int B, int d) {
    const int rc = check_loss("inbatch_loss_workspace", B, d, 0, 0);
    if (rc) return rc;
    LossArgs a = {};
    a.B = B;
    a.d = d;
    a.splits = score_splits(B, d, &a.kchunk);
    SplitArgs s = split_args(nullptr, nullptr, B, d);
    return lay_forward(nullptr, a, s);
}

int otter_inbatch_loss_forward(int device, const float* q, const float* c, const float* neg_c, int B, int d, float* scores,
                               int ld, float* stats, float* loss, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_loss("inbatch_loss_forward", B, d, ld, B + (neg_c ? 1 : 0));
    if (rc) return rc;
    if (!q || !c || !scores || !stats || !loss) return set_err(OTTER_EINVAL, "inbatch_loss_forward: NULL buffer");
    if ((rc = check_workspace("inbatch_loss_forward", workspace, workspace_bytes, otter_inbatch_loss_workspace(B, d)))) return rc;
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "inbatch_loss_forward: hipSetDevice(%d) failed", device);
    LossArgs a = {};
    a.q = q;
    a.c = c;
    a.neg = neg_c;
    a.scores = scores;
    a.lse = stats;
    a.rest = stats + B;
    a.loss = loss;
    a.B = B;
    a.d = d;
    a.ld = ld;
    a.splits = score_splits(B, d, &a.kchunk);
    SplitArgs s = split_args(q, c, B, d);
    lay_forward(workspace, a, s);
    hipStream_t st = (hipStream_t)stream;
    if (score_planes(B, d)) {
        loss_split_kernel<<<dim3((unsigned)(s.Bp / 4), 2), 256, 0, st>>>(s);
        loss_scores16_kernel<<<dim3((unsigned)((s.Bp / 128) * (s.Bp / 128)), (unsigned)a.splits), 256, 0, st>>>(a, s);
    } else {
        const unsigned nt = (unsigned)(B + 63) / 64;
        loss_scores_kernel<64><<<dim3(nt * nt, (unsigned)a.splits), 256, 0, st>>>(a);
    }
    if (B <= MEAN_B) {
        if (a.splits > 1)
            loss_rows_kernel<true, true><<<B, 256, 0, st>>>(a);
        else
            loss_rows_kernel<false, true><<<B, 256, 0, st>>>(a);
    } else {
        if (a.splits > 1)
            loss_rows_kernel<true, false><<<B, 256, 0, st>>>(a);
        else
            loss_rows_kernel<false, false><<<B, 256, 0, st>>>(a);
        loss_mean_kernel<<<1, 1024, 0, st>>>(a);
    }
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int64_t otter_inbatch_loss_backward_workspace(int B, int d) {
    const int rc = check_loss("inbatch_loss_backward_workspace", B, d, 0, 0);
    if (rc) return rc;
    LossArgs a = {};
    a.gsplits = grad_splits(B, d, &a.gchunk);
    SplitArgs s = split_args(nullptr, nullptr, B, d);
    return lay_backward(nullptr, a, s);
}

int otter_inbatch_loss_backward(int device, const float* dloss, const float* q, const float* c, const float* neg_c, int B, int d,
                                const float* scores, int ld, const float* stats, float* dq, float* dc, float* dneg, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    int rc = check_loss("inbatch_loss_backward", B, d, ld, B + (neg_c ? 1 : 0));
    if (rc) return rc;
    if (!dloss || !q || !c || !scores || !stats || !dq || !dc || (neg_c && !dneg))
        return set_err(OTTER_EINVAL, "inbatch_loss_backward: NULL buffer");
    if ((rc = check_workspace("inbatch_loss_backward", workspace, workspace_bytes, otter_inbatch_loss_backward_workspace(B, d)))) return rc;
    const long long tiles = (long long)((B + 63) / 64) * ((d + 63) / 64);
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "inbatch_loss_backward: hipSetDevice(%d) failed", device);
    LossArgs a = {};
    a.dloss = dloss;
    a.q = q;
    a.c = c;
    a.neg = neg_c;
    a.scores = const_cast<float*>(scores);
    a.lse = const_cast<float*>(stats);
    a.rest = a.lse + B;
    a.dq = dq;
    a.dc = dc;
    a.dneg = dneg;
    a.B = B;
    a.d = d;
    a.ld = ld;
    a.gsplits = grad_splits(B, d, &a.gchunk);
    SplitArgs s = split_args(q, c, B, d);
    lay_backward(workspace, a, s);
    hipStream_t st = (hipStream_t)stream;
    if (grad_planes(B, d)) {
        const unsigned nb = (unsigned)col_blocks(s), strips = (unsigned)(s.Bp / s.strip);
        loss_split_kernel<<<dim3((unsigned)(s.Bp / 4), 2), 256, 0, st>>>(s);
        loss_gtop_kernel<<<dim3(strips, nb), 256, 0, st>>>(a, s);
        loss_gscale_kernel<<<dim3((unsigned)(s.Bp / 64), 2), 256, 0, st>>>(s, (int)(4 * nb), (int)strips);
        loss_gplanes_kernel<<<(unsigned)s.Bp * nb, 256, 0, st>>>(a, s);
        loss_grad16_kernel<<<dim3((unsigned)(2 * (s.Bp / 128) * ((d + 63) / 64)), (unsigned)a.gsplits), 256, 0, st>>>(a, s);
    } else {
        loss_grad_kernel<64><<<dim3((unsigned)(2 * tiles), (unsigned)a.gsplits), 256, 0, st>>>(a);
    }
    if (a.gsplits > 1) loss_join_kernel<<<dim3((unsigned)(((int64_t)B * d + 1023) / 1024), 2), 256, 0, st>>>(a);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
