// inbatch_loss.hip — the fine-tuning loss over the in-batch score matrix and its gradient on gfx950 (reference
// retrieval/criterions.py:10-27: cross entropy of [q c^T | q . neg] against the diagonal).
//
//   S = [q c^T | q . neg]  (B x B | B x 1),  lse_i = log sum_j exp S_ij,  loss = mean_i (lse_i - S_ii)
//   G = (exp(S - lse) - 1[j = i]) dloss / B,  dq = G c + G_neg neg,  dc = G^T q,  dneg = G_neg q
//
// All three products are float32 products on v_mfma_f32_32x32x2_f32 (an fma chain: no operand is rounded).  S is kept
// (4 B^2 bytes, read twice) instead of multiplied out again in the backward pass (2 B^2 d flops); G is never stored, it is
// made from S and lse where a product's tile is loaded.
#include "otter_common.h"
#include "otter_device.h"

namespace {
using namespace otter;

constexpr int LOSS_MAX_B = 65536;
constexpr int KB = 32;             // contraction depth of a staged tile
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // 16-byte load at any 4-byte address

struct LossArgs {
    const float *q, *c, *neg;      // [B][d]; neg may be null
    float* scores;                 // [B][ld]
    float* part;                   // [splits][B][B] when splits > 1
    float *lse, *rowloss, *loss;   // [B], [B], [1]
    const float* dloss;            // [1]
    float *dq, *dc, *dneg;
    int B, d, ld, splits, kchunk;
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
    const float *scores, *lse;
    long long ld;
    int B;
    float g;                       // dloss / B
    __device__ __forceinline__ f4u operator()(int i, int j) const {
        f4u v = load4(scores, ld, B, B, i, j);
        const float l = i < B ? lse[i] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = i < B && j + e < B ? (__expf(v[e] - l) - (j + e == i ? 1.0f : 0.0f)) * g : 0.0f;
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

// out(row, col, value) for every element of the tile
template <int BM, typename F>
__device__ __forceinline__ void each(const f32x16 (&acc)[BM / 64][BM / 64], int m0, int n0, const F& out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BM / 2);
#pragma unroll
    for (int i = 0; i < BM / 64; ++i)
#pragma unroll
        for (int n = 0; n < BM / 64; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                out(m0 + wm + 32 * i + (r & 3) + 8 * (r >> 2) + 4 * h, n0 + wn + 32 * n + l31, acc[i][n][r]);
}

// S = q c^T; grid (tiles, splits of d)
template <int BM>
__global__ __launch_bounds__(256) void loss_scores_kernel(LossArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[2 * BM * KB];
    const int nt = (a.B + BM - 1) / BM;
    const int t = xcd_remap(blockIdx.x, gridDim.x);
    const int m0 = (t / nt) * BM, n0 = (t % nt) * BM;
    const int ka = blockIdx.y * a.kchunk, kb = min(a.d, ka + a.kchunk);
    f32x16 acc[BM / 64][BM / 64];
    clear<BM>(acc);
    product<BM, true, true>(acc, Plain{a.q, a.B, a.d, a.d}, Plain{a.c, a.B, a.d, a.d}, m0, n0, ka, kb, lds);
    float* out = a.splits > 1 ? a.part + (size_t)blockIdx.y * a.B * a.B : a.scores;
    const long long ld = a.splits > 1 ? a.B : a.ld;
    each<BM>(acc, m0, n0, [&](int i, int j, float v) {
        if (i < a.B && j < a.B) out[(long long)i * ld + j] = v;
    });
}

__device__ __forceinline__ void online(float& m, float& l, float m2, float l2) {
    const float n = fmaxf(m, m2);
    if (n == -INFINITY) return;
    l = l * __expf(m - n) + l2 * __expf(m2 - n);
    m = n;
}

// one workgroup a row: the pieces of S summed in order, the hard negative's score, lse and the row's loss
__global__ __launch_bounds__(256) void loss_rows_kernel(LossArgs a) {
    __shared__ float sm[4], sl[4], sd[4];
    const int i = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* row = a.scores + (long long)i * a.ld;
    float m = -INFINITY, l = 0.0f;
    for (int j = threadIdx.x; j < a.B; j += 256) {
        float s;
        if (a.splits > 1) {
            s = 0.0f;
            for (int p = 0; p < a.splits; ++p) s += a.part[((size_t)p * a.B + i) * a.B + j];
            row[j] = s;
        } else {
            s = row[j];
        }
        online(m, l, s, 1.0f);
    }
    float dot = 0.0f;
    if (a.neg)
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
        const float lse = m + __logf(l);
        a.lse[i] = lse;
        a.rowloss[i] = lse - row[i];
    }
}

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

// dq and dc, half the grid each
template <int BM>
__global__ __launch_bounds__(256) void loss_grad_kernel(LossArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[2 * BM * KB];
    const int nt = (a.d + BM - 1) / BM, half = gridDim.x / 2;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const bool second = id >= half;
    const int t = second ? id - half : id;
    const int m0 = (t / nt) * BM, n0 = (t % nt) * BM;
    const float g = *a.dloss / (float)a.B;
    const Grad G{a.scores, a.lse, a.ld, a.B, g};
    f32x16 acc[BM / 64][BM / 64];
    clear<BM>(acc);
    if (second) {
        product<BM, false, false>(acc, G, Plain{a.q, a.B, a.d, a.d}, m0, n0, 0, a.B, lds);
        each<BM>(acc, m0, n0, [&](int j, int n, float v) {
            if (j < a.B && n < a.d) a.dc[(long long)j * a.d + n] = v;
        });
    } else {
        product<BM, true, false>(acc, G, Plain{a.c, a.B, a.d, a.d}, m0, n0, 0, a.B, lds);
        each<BM>(acc, m0, n0, [&](int i, int n, float v) {
            if (i >= a.B || n >= a.d) return;
            const long long at = (long long)i * a.d + n;
            if (a.neg) {
                const float gn = __expf(a.scores[(long long)i * a.ld + a.B] - a.lse[i]) * g;
                v = fmaf(gn, a.neg[at], v);
                a.dneg[at] = gn * a.q[at];
            }
            a.dq[at] = v;
        });
    }
}

// ------------------------------------------------------------------ host side
int check_loss(const char* what, int B, int d, int ld, int ncol) {
    if (B < 1 || d < 1) return set_err(OTTER_EINVAL, "%s: bad B=%d d=%d (the mean over no rows is undefined)", what, B, d);
    if (B > LOSS_MAX_B) return set_err(OTTER_EINVAL, "%s: B=%d exceeds %d", what, B, LOSS_MAX_B);
    if (ld < ncol) return set_err(OTTER_EINVAL, "%s: ld=%d is less than the %d columns of the scores", what, ld, ncol);
    return OTTER_OK;
}

// pieces of d so that a small batch still has work for the chip: at least 64 of d each
int loss_splits(int B, int d, int bm) {
    const long long tiles = (long long)((B + bm - 1) / bm) * ((B + bm - 1) / bm);
    int s = (int)(tiles < 256 ? 256 / tiles : 1);
    const int most = (d + 63) / 64;
    return s < most ? (s < 1 ? 1 : s) : most;
}

int loss_tile(int B) { return B > 512 ? 128 : 64; }

}  // namespace

extern "C" {

int64_t otter_inbatch_loss_workspace(int B, int d) {
    const int rc = check_loss("inbatch_loss_workspace", B, d, 0, 0);
    if (rc) return rc;
    const int s = loss_splits(B, d, loss_tile(B));
    return (int64_t)sizeof(float) * (B + (s > 1 ? (int64_t)s * B * B : 0));
}

int otter_inbatch_loss_forward(int device, const float* q, const float* c, const float* neg_c, int B, int d, float* scores,
                               int ld, float* lse, float* loss, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_loss("inbatch_loss_forward", B, d, ld, B + (neg_c ? 1 : 0));
    if (rc) return rc;
    if (!q || !c || !scores || !lse || !loss || !workspace) return set_err(OTTER_EINVAL, "inbatch_loss_forward: NULL buffer");
    const int64_t need = otter_inbatch_loss_workspace(B, d);
    if (workspace_bytes < need)
        return set_err(OTTER_EINVAL, "inbatch_loss_forward: workspace of %lld bytes, needs %lld", (long long)workspace_bytes,
                       (long long)need);
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "inbatch_loss_forward: hipSetDevice(%d) failed", device);
    LossArgs a = {};
    a.q = q;
    a.c = c;
    a.neg = neg_c;
    a.scores = scores;
    a.lse = lse;
    a.loss = loss;
    a.rowloss = (float*)workspace;
    a.part = a.rowloss + B;
    a.B = B;
    a.d = d;
    a.ld = ld;
    const int bm = loss_tile(B), nt = (B + bm - 1) / bm;
    a.splits = loss_splits(B, d, bm);
    a.kchunk = ((d + a.splits - 1) / a.splits + KB - 1) / KB * KB;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)nt * nt, (unsigned)a.splits);
    if (bm == 128)
        loss_scores_kernel<128><<<grid, 256, 0, st>>>(a);
    else
        loss_scores_kernel<64><<<grid, 256, 0, st>>>(a);
    loss_rows_kernel<<<B, 256, 0, st>>>(a);
    loss_mean_kernel<<<1, 1024, 0, st>>>(a);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int otter_inbatch_loss_backward(int device, const float* dloss, const float* q, const float* c, const float* neg_c, int B, int d,
                                const float* scores, int ld, const float* lse, float* dq, float* dc, float* dneg, void* stream) {
    int rc = check_loss("inbatch_loss_backward", B, d, ld, B + (neg_c ? 1 : 0));
    if (rc) return rc;
    if (!dloss || !q || !c || !scores || !lse || !dq || !dc || (neg_c && !dneg))
        return set_err(OTTER_EINVAL, "inbatch_loss_backward: NULL buffer");
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "inbatch_loss_backward: hipSetDevice(%d) failed", device);
    LossArgs a = {};
    a.dloss = dloss;
    a.q = q;
    a.c = c;
    a.neg = neg_c;
    a.scores = const_cast<float*>(scores);
    a.lse = const_cast<float*>(lse);
    a.dq = dq;
    a.dc = dc;
    a.dneg = dneg;
    a.B = B;
    a.d = d;
    a.ld = ld;
    hipStream_t st = (hipStream_t)stream;
    const int bm = loss_tile(B);
    const long long tiles = (long long)((B + bm - 1) / bm) * ((d + bm - 1) / bm);
    if (tiles > 0x3FFFFFFF) return set_err(OTTER_EINVAL, "inbatch_loss_backward: B=%d x d=%d is too large for one launch", B, d);
    if (bm == 128)
        loss_grad_kernel<128><<<(unsigned)(2 * tiles), 256, 0, st>>>(a);
    else
        loss_grad_kernel<64><<<(unsigned)(2 * tiles), 256, 0, st>>>(a);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
