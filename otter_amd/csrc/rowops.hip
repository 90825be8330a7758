// rowops.hip — row operators of the training path on gfx950: dropout from counter-based draws and the layer norm of a sum
// z = dropout(x) + residual (the residual connection of every BERT layer), forward and backward.
//
//   y = (z - mean) rstd g + b                 a = dy g,  xh = (z - mean) rstd
//   dz = rstd (a - mean(a) - xh mean(a xh)),  dresidual = dz,  dx = dz keep / (1 - p)
//   dg = sum_rows dy xh,  db = sum_rows dy
//
// Nothing but mean and rstd is kept for the backward pass: z is made again from x, the residual and the same draws.  That
// moves as many bytes as storing z would (one read more, one write less), needs no buffer and keeps z unrounded.
#include "otter_common.h"
#include "otter_philox.h"

namespace {
using namespace otter;

constexpr int LN_MAX_COLS = 8192;
constexpr u32 ROW_TAG = 0xFFFFFFFFu;

// ------------------------------------------------------------------ groups of 8 elements
// VEC: the group is whole and 16-byte aligned; otherwise element by element up to `n`.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float v[8]) {
    if constexpr (VEC && sizeof(T) == 2) {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        const u32 w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else if constexpr (VEC) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f<T>(p[e]) : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float v[8]) {
    if constexpr (VEC && sizeof(T) == 2) {
        u32 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (u32)f2bf(v[2 * i]) | ((u32)f2bf(v[2 * i + 1]) << 16);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (VEC) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = from_f<T>(v[e]);
    }
}

// bit e: element e of the group is kept
__device__ __forceinline__ u32 keep8(u32 group, u32 row, const DropArgs& d, u32 k0, u32 k1) {
    const Philox4 r = philox7(group, row, ROW_TAG, d.call, k0, k1);
    u32 keep = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        keep |= (u32)((r.w[i] & 0xFFFFu) >= d.thr) << (2 * i);
        keep |= (u32)((r.w[i] >> 16) >= d.thr) << (2 * i + 1);
    }
    return keep;
}

__device__ __forceinline__ void apply_keep(float v[8], u32 keep, float scale) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (keep >> e) & 1u ? v[e] * scale : 0.0f;
}

// ------------------------------------------------------------------ dropout
// One thread per group of 8; a grid-stride loop whose (row, group) advance without a division.
struct DropoutArgs {
    const void* x;
    void* y;
    long long groups;   // rows * gpr
    int gpr, cols;      // groups a row
    DropArgs drop;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const u64 seed = (u64)*a.drop.seed;
    const u32 k0 = (u32)seed, k1 = (u32)(seed >> 32);
    const long long step = (long long)gridDim.x * 256;
    long long g = (long long)blockIdx.x * 256 + threadIdx.x;
    long long row = g / a.gpr;
    int col = (int)(g - row * a.gpr);
    const long long rstep = step / a.gpr;
    const int cstep = (int)(step - rstep * a.gpr);
    for (; g < a.groups; g += step) {
        const long long off = row * a.cols + (long long)col * 8;
        const int n = min(8, a.cols - col * 8);
        float v[8];
        load8<T, VEC>((const T*)a.x + off, n, v);
        apply_keep(v, keep8((u32)col, (u32)row, a.drop, k0, k1), a.drop.scale);
        store8<T, VEC>((T*)a.y + off, n, v);
        row += rstep;
        col += cstep;
        if (col >= a.gpr) {
            col -= a.gpr;
            ++row;
        }
    }
}

// ------------------------------------------------------------------ layer norm
struct NormArgs {
    const void* x;
    const void* residual;   // or null
    const void* weight;
    const void* bias;
    const void* dy;
    void* y;
    float* mean;
    float* rstd;
    void* dx;
    void* dresidual;        // or null
    float* part;            // [grid][2][cols]
    long long rows;
    int cols, wbf16;
    float eps;
    DropArgs drop;
};

__device__ __forceinline__ float load_w(const void* p, int i, int bf) {
    return bf ? bf2f(((const bf16_t*)p)[i]) : ((const float*)p)[i];
}

// sum over the LPR lanes of a row: half a wave, or the whole workgroup of 256
template <int LPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* lds) {
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    if constexpr (LPR > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            lds[2 * wave] = a;
            lds[2 * wave + 1] = b;
        }
        __syncthreads();
        a = lds[0] + lds[2] + lds[4] + lds[6];
        b = lds[1] + lds[3] + lds[5] + lds[7];
    }
}

// z of this lane's groups; keep[i] holds the kept bits of group i
template <typename T, bool VEC, int LPR, int NG>
__device__ __forceinline__ void load_z(const NormArgs& a, long long row, int l, u32 k0, u32 k1, float z[NG][8], u32 keep[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int c = (i * LPR + l) * 8, n = min(8, a.cols - c);
        if (n <= 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = 0.0f;
            continue;
        }
        load8<T, VEC>((const T*)a.x + row * a.cols + c, n, z[i]);
        if (a.drop.thr) {
            keep[i] = keep8((u32)(c >> 3), (u32)row, a.drop, k0, k1);
            apply_keep(z[i], keep[i], a.drop.scale);
        }
        if (a.residual) {
            float r[8];
            load8<T, VEC>((const T*)a.residual + row * a.cols + c, n, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] += r[e];
        }
    }
}

template <typename T, bool VEC, int LPR, int NG>
__global__ __launch_bounds__(256) void ln_fwd_kernel(NormArgs a) {
    __shared__ float lds[8];
    constexpr int RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    u32 k0 = 0, k1 = 0;
    if (a.drop.thr) {
        const u64 seed = (u64)*a.drop.seed;
        k0 = (u32)seed;
        k1 = (u32)(seed >> 32);
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + slot;
        const bool in = row < a.rows;             // whole half-waves: no lane of a row leaves its reductions
        float z[NG][8];
        u32 keep[NG];
        load_z<T, VEC, LPR, NG>(a, in ? row : a.rows - 1, l, k0, k1, z, keep);
        float s = 0.0f, dummy = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += z[i][e];
        row_sum2<LPR>(s, dummy, lds);
        const float mean = s / (float)a.cols;
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int c = (i * LPR + l) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = z[i][e] - mean;
                if (VEC ? c < a.cols : c + e < a.cols) v += d * d;
            }
        }
        row_sum2<LPR>(v, dummy, lds);
        const float rstd = 1.0f / sqrtf(v / (float)a.cols + a.eps);
        if (!in) continue;
        if (l == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int c = (i * LPR + l) * 8, n = min(8, a.cols - c);
            if (n <= 0) continue;
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                o[e] = e < n ? (z[i][e] - mean) * rstd * load_w(a.weight, c + e, a.wbf16) + load_w(a.bias, c + e, a.wbf16) : 0.0f;
            store8<T, VEC>((T*)a.y + row * a.cols + c, n, o);
        }
    }
}

template <typename T, bool VEC, int LPR, int NG>
__global__ __launch_bounds__(256) void ln_bwd_kernel(NormArgs a) {
    __shared__ float lds[8];
    __shared__ float red[LPR == 256 ? 1 : 256 * 8];
    constexpr int RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    u32 k0 = 0, k1 = 0;
    if (a.drop.thr) {
        const u64 seed = (u64)*a.drop.seed;
        k0 = (u32)seed;
        k1 = (u32)(seed >> 32);
    }
    float dw[NG][8], db[NG][8], w[NG][8];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int c = (i * LPR + l) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[i][e] = db[i][e] = 0.0f;
            w[i][e] = c + e < a.cols ? load_w(a.weight, c + e, a.wbf16) : 0.0f;
        }
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
        const bool in = r0 + slot < a.rows;
        const long long row = in ? r0 + slot : a.rows - 1;
        float z[NG][8], dy[NG][8];
        u32 keep[NG];
        load_z<T, VEC, LPR, NG>(a, row, l, k0, k1, z, keep);
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int c = (i * LPR + l) * 8, n = min(8, a.cols - c);
            if (n > 0) load8<T, VEC>((const T*)a.dy + row * a.cols + c, n, dy[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (n <= 0) dy[i][e] = 0.0f;
                const float xh = (z[i][e] - mean) * rstd;
                z[i][e] = xh;
                if (in) {
                    dw[i][e] += dy[i][e] * xh;
                    db[i][e] += dy[i][e];
                }
                dy[i][e] *= w[i][e];              // a = dy g (0 past the row's end)
                s1 += dy[i][e];
                s2 += dy[i][e] * xh;
            }
        }
        row_sum2<LPR>(s1, s2, lds);
        if (!in) continue;
        const float m1 = s1 / (float)a.cols, m2 = s2 / (float)a.cols;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int c = (i * LPR + l) * 8, n = min(8, a.cols - c);
            if (n <= 0) continue;
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = rstd * (dy[i][e] - m1 - z[i][e] * m2);
            if (a.dresidual) store8<T, VEC>((T*)a.dresidual + row * a.cols + c, n, o);
            if (a.drop.thr) apply_keep(o, keep[i], a.drop.scale);
            store8<T, VEC>((T*)a.dx + row * a.cols + c, n, o);
        }
    }
    // the workgroup's sums over its rows, in the order of its row slots
    float* out = a.part + (size_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = (i * LPR + l) * 8;
            if constexpr (LPR == 256) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < a.cols) out[t * a.cols + c + e] = t ? db[i][e] : dw[i][e];
            } else {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; ++e) red[(slot * 8 + e) * LPR + l] = t ? db[i][e] : dw[i][e];
                __syncthreads();
                const int e = threadIdx.x / LPR;      // 8 slots of threads: one element of the group each
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < RPB; ++k) s += red[(k * 8 + e) * LPR + l];
                if (c + e < a.cols) out[t * a.cols + c + e] = s;
            }
        }
}

// out[c] = sum over the P partial rows, in a fixed order: 32 columns x 32 row lanes a workgroup
__global__ __launch_bounds__(1024) void ln_wgrad_kernel(const float* part, int P, int cols, void* dw, void* db, int wbf16) {
    __shared__ float red[32][33];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;               // column of [dw | db]
    float s = 0.0f;
    if (c < 2 * cols)
        for (int p = rl; p < P; p += 32) s += part[(size_t)p * 2 * cols + c];
    red[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && c < 2 * cols) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += red[k][cl];
        void* dst = c < cols ? dw : db;
        const int i = c < cols ? c : c - cols;
        if (wbf16)
            ((bf16_t*)dst)[i] = f2bf(t);
        else
            ((float*)dst)[i] = t;
    }
}

// ------------------------------------------------------------------ host side
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// rows a workgroup of 256 handles at a time: half a wave a row up to 1024 columns, the workgroup a row above
int rows_per_block(int cols) { return cols <= 1024 ? 8 : 1; }

int norm_grid(long long rows, int cols) {
    const long long need = (rows + rows_per_block(cols) - 1) / rows_per_block(cols);
    return (int)(need < 1024 ? need : 1024);
}

template <bool BWD, typename T, bool VEC, int LPR>
void launch_norm(const NormArgs& a, int ng, int grid, hipStream_t st) {
#define OTTER_LN(N)                                                        \
    case N:                                                                \
        if constexpr (BWD)                                                 \
            ln_bwd_kernel<T, VEC, LPR, N><<<grid, 256, 0, st>>>(a);        \
        else                                                               \
            ln_fwd_kernel<T, VEC, LPR, N><<<grid, 256, 0, st>>>(a);        \
        break;
    switch (ng) {
        OTTER_LN(1)
        OTTER_LN(2)
        OTTER_LN(3)
        OTTER_LN(4)
    }
#undef OTTER_LN
}

template <bool BWD>
void launch_norm_any(const NormArgs& a, int dtype, bool vec, int grid, hipStream_t st) {
    const int groups = (a.cols + 7) / 8;
    const bool half = a.cols <= 1024;
    const int ng = half ? (groups + 31) / 32 : (groups + 255) / 256;
#define OTTER_LN_T(T, V) half ? launch_norm<BWD, T, V, 32>(a, ng, grid, st) : launch_norm<BWD, T, V, 256>(a, ng, grid, st)
    if (dtype == OTTER_F32) {
        if (vec) OTTER_LN_T(float, true); else OTTER_LN_T(float, false);
    } else {
        if (vec) OTTER_LN_T(bf16_t, true); else OTTER_LN_T(bf16_t, false);
    }
#undef OTTER_LN_T
}

int check_norm(const char* what, int dtype, int wdtype, int64_t rows, int cols) {
    if (dtype != OTTER_F32 && dtype != OTTER_BF16) return set_err(OTTER_EINVAL, "%s: dtype must be float32 or bfloat16", what);
    if (wdtype != OTTER_F32 && wdtype != OTTER_BF16) return set_err(OTTER_EINVAL, "%s: weight dtype must be float32 or bfloat16", what);
    if (rows < 0 || rows > 0xFFFFFFFFll || cols < 1) return set_err(OTTER_EINVAL, "%s: bad rows=%lld cols=%d", what, (long long)rows, cols);
    if (cols > LN_MAX_COLS) return set_err(OTTER_EINVAL, "%s: cols=%d exceeds %d", what, cols, LN_MAX_COLS);
    return OTTER_OK;
}

}  // namespace

namespace otter {

int make_drop(const char* what, float p, const int64_t* seed, uint32_t call, DropArgs* out) {
    if (!(p >= 0.0f && p < 1.0f)) return set_err(OTTER_EINVAL, "%s: dropout probability %g is not in [0, 1)", what, (double)p);
    const u32 thr = (u32)((double)p * 65536.0 + 0.5);
    if (thr >= 65536u) return set_err(OTTER_EINVAL, "%s: dropout probability %g rounds to 1 in steps of 2^-16", what, (double)p);
    if (thr && !seed) return set_err(OTTER_EINVAL, "%s: dropout needs a seed", what);
    out->thr = thr;
    out->call = call;
    out->scale = 65536.0f / (float)(65536u - thr);
    out->seed = (const long long*)seed;
    return OTTER_OK;
}

}  // namespace otter

extern "C" {

int otter_dropout(int device, int dtype, const void* x, void* y, int64_t rows, int64_t cols, float p, const int64_t* seed,
                  uint32_t call, void* stream) {
    if (dtype != OTTER_F32 && dtype != OTTER_BF16) return set_err(OTTER_EINVAL, "dropout: dtype must be float32 or bfloat16");
    if (rows < 0 || rows > 0xFFFFFFFFll || cols < 0 || cols > 0x7FFFFFFFll)
        return set_err(OTTER_EINVAL, "dropout: bad rows=%lld cols=%lld", (long long)rows, (long long)cols);
    DropoutArgs a;
    int rc = make_drop("dropout", p, seed, call, &a.drop);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return OTTER_OK;
    if (!x || !y) return set_err(OTTER_EINVAL, "dropout: NULL buffer");
    if (!seed) return set_err(OTTER_EINVAL, "dropout: needs a seed");
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "dropout: hipSetDevice(%d) failed", device);
    a.x = x;
    a.y = y;
    a.cols = (int)cols;
    a.gpr = (int)((cols + 7) / 8);
    a.groups = rows * a.gpr;
    const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(y);
    const long long need = (a.groups + 255) / 256;
    const int grid = (int)(need < 2048 ? need : 2048);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == OTTER_F32) {
        if (vec) dropout_kernel<float, true><<<grid, 256, 0, st>>>(a);
        else dropout_kernel<float, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (vec) dropout_kernel<bf16_t, true><<<grid, 256, 0, st>>>(a);
        else dropout_kernel<bf16_t, false><<<grid, 256, 0, st>>>(a);
    }
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int otter_layernorm_forward(int device, int dtype, int wdtype, const void* x, const void* residual, const void* weight,
                            const void* bias, int64_t rows, int cols, float eps, float p, const int64_t* seed, uint32_t call,
                            void* y, float* mean, float* rstd, void* stream) {
    NormArgs a = {};
    int rc = check_norm("layernorm_forward", dtype, wdtype, rows, cols);
    if (!rc) rc = make_drop("layernorm_forward", p, seed, call, &a.drop);
    if (rc) return rc;
    if (!(eps >= 0.0f)) return set_err(OTTER_EINVAL, "layernorm_forward: eps=%g", (double)eps);
    if (rows == 0) return OTTER_OK;
    if (!x || !weight || !bias || !y || !mean || !rstd) return set_err(OTTER_EINVAL, "layernorm_forward: NULL buffer");
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "layernorm_forward: hipSetDevice(%d) failed", device);
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.cols = cols;
    a.wbf16 = wdtype == OTTER_BF16;
    a.eps = eps;
    const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(y) && aligned16(residual);
    launch_norm_any<false>(a, dtype, vec, norm_grid(rows, cols), (hipStream_t)stream);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int64_t otter_layernorm_backward_workspace(int64_t rows, int cols) {
    if (rows < 0 || cols < 1 || cols > LN_MAX_COLS)
        return set_err(OTTER_EINVAL, "layernorm_backward_workspace: bad rows=%lld cols=%d", (long long)rows, cols);
    return (int64_t)norm_grid(rows, cols) * 2 * cols * (int64_t)sizeof(float);
}

int otter_layernorm_backward(int device, int dtype, int wdtype, const void* dy, const void* x, const void* residual,
                             const void* weight, const float* mean, const float* rstd, int64_t rows, int cols, float p,
                             const int64_t* seed, uint32_t call, void* dx, void* dresidual, void* dweight, void* dbias,
                             void* workspace, int64_t workspace_bytes, void* stream) {
    NormArgs a = {};
    int rc = check_norm("layernorm_backward", dtype, wdtype, rows, cols);
    if (!rc) rc = make_drop("layernorm_backward", p, seed, call, &a.drop);
    if (rc) return rc;
    if (!dweight || !dbias || (rows > 0 && (!dy || !x || !weight || !mean || !rstd || !dx || !workspace)))
        return set_err(OTTER_EINVAL, "layernorm_backward: NULL buffer");
    if (dresidual && !residual) return set_err(OTTER_EINVAL, "layernorm_backward: dresidual without a residual");
    const int64_t need = otter_layernorm_backward_workspace(rows, cols);
    if (rows > 0 && workspace_bytes < need)
        return set_err(OTTER_EINVAL, "layernorm_backward: workspace of %lld bytes, needs %lld", (long long)workspace_bytes,
                       (long long)need);
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "layernorm_backward: hipSetDevice(%d) failed", device);
    a.dy = dy;
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.rows = rows;
    a.cols = cols;
    a.wbf16 = wdtype == OTTER_BF16;
    a.dx = dx;
    a.dresidual = dresidual;
    a.part = (float*)workspace;
    hipStream_t st = (hipStream_t)stream;
    const int grid = norm_grid(rows, cols);
    if (rows > 0) {
        const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(residual) && aligned16(dresidual);
        launch_norm_any<true>(a, dtype, vec, grid, st);
        OTTER_HIP_TRY(hipGetLastError());
    }
    ln_wgrad_kernel<<<(2 * cols + 31) / 32, 1024, 0, st>>>(a.part, grid, cols, dweight, dbias, a.wbf16);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
