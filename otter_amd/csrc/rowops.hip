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

#include <type_traits>

namespace {
using namespace otter;

constexpr int LN_MAX_COLS = 8192;
constexpr u32 ROW_TAG = 0xFFFFFFFFu;

// ------------------------------------------------------------------ groups of 8 elements
// A group is one or two 16-byte accesses.  VEC: rows are whole groups, 16-byte aligned.  Otherwise the accesses are aligned
// to an element only (the hardware takes that; a row of 771 floats element by element cost 2.5 times as long) and a row's last
// group is cut off at `n`.
template <typename T, bool VEC> struct Chunk { typedef u32 type __attribute__((ext_vector_type(4))); };
template <> struct Chunk<float, false> { typedef u32 type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Chunk<bf16_t, false> { typedef u32 type __attribute__((ext_vector_type(4), aligned(2))); };

template <typename T> struct Raw { u32 w[2 * sizeof(T)]; };   // 8 elements as they are stored

template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(const T* p, int n, Raw<T>& r) {
    typedef typename Chunk<T, VEC>::type V;
    if (VEC || n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const V v = reinterpret_cast<const V*>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[4 * i + e] = v[e];
        }
    } else {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = e < n ? p[e] : T(0);
        __builtin_memcpy(&r, t, sizeof(t));
    }
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float v[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r.w[e]);
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float v[8]) {
    Raw<T> r;
    load_raw<T, VEC>(p, n, r);
    unpack<T>(r, v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float v[8]) {
    typedef typename Chunk<T, VEC>::type V;
    if (VEC || n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            V o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 2)
                    o[e] = (u32)f2bf(v[2 * e]) | ((u32)f2bf(v[2 * e + 1]) << 16);
                else
                    o[e] = __float_as_uint(v[4 * i + e]);
            }
            reinterpret_cast<V*>(p)[i] = o;
        }
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
// y = x keep / (1 - p): one read and one write an element, bound by memory.  One thread per group of 8, which is one generator
// call (28 instructions, hidden behind the loads); a grid-stride loop whose (row, group) advance without a division.
// 65536 x 768 float32: 78 us = 5.2 TB/s (a large copy reaches 4.8); 1120 x 768 bfloat16: 2.7 us, less than its launch.
struct DropoutArgs {
    const void* x;
    void* y;
    long long groups;   // rows * gpr
    int gpr, cols;      // groups a row
    DropArgs drop;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const u64 seed = a.drop.thr ? (u64)*a.drop.seed : 0;
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

// A lane holds the groups i LPR + l, i < NG, of a row.  Of NG groups of all lanes only the last can be cut or empty, so that one
// alone is looked at, and without a branch: a group past the row's end is the row's last 8 elements again, and the one that
// the end cuts is those, moved to their places.  (With a branch for every group and element of the cut one the kernel of odd
// rows was 19 KB of code instead of 11: 4097 x 771 float32 11.3 -> 9.2 us forward, 20.8 -> 17.8 backward; 30000 x 771 bfloat16
// 34 -> 24 and 62 -> 44.)
template <bool VEC>
__device__ __forceinline__ void move_cut(int c, int cols, float v[8]) {
    const int s = c - (cols - 8);                     // 1 .. 7 in the cut group
    if (VEC) return;
#pragma unroll
    for (int b = 1; b < 8; b <<= 1) {
        const bool move = s > 0 && (s & b);
#pragma unroll
        for (int e = 0; e + b < 8; ++e) v[e] = move ? v[e + b] : v[e];
    }
}

// group c of a row p; LAST: it may be cut or empty (VEC: empty)
template <typename T, bool VEC, bool LAST>
__device__ __forceinline__ void load_group(const T* p, int c, int cols, Raw<T>& r) {
    if (!LAST || VEC || cols >= 8) {
        load_raw<T, VEC>(p + (LAST ? min(c, cols - 8) : c), 8, r);
    } else {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = p[min(e, cols - 1)];
        __builtin_memcpy(&r, t, sizeof(t));
    }
}

template <typename T, bool VEC, bool LAST>
__device__ __forceinline__ void unpack_group(const Raw<T>& r, int c, int cols, float v[8]) {
    unpack<T>(r, v);
    if (LAST && cols >= 8) move_cut<VEC>(c, cols, v);
}

// a group of weights; any of them past the row's end
template <bool VEC, bool LAST>
__device__ __forceinline__ void load_w(const void* p, int c, int cols, int bf, float v[8]) {
    if (bf) {
        Raw<bf16_t> r;
        load_group<bf16_t, false, LAST>((const bf16_t*)p, c, cols, r);
        unpack_group<bf16_t, VEC, LAST>(r, c, cols, v);
    } else {
        Raw<float> r;
        load_group<float, false, LAST>((const float*)p, c, cols, r);
        unpack_group<float, VEC, LAST>(r, c, cols, v);
    }
}

// f(group, whether it is the last): the second is a constant
template <int NG, typename F>
__device__ __forceinline__ void groups(const F& f) {
#pragma unroll
    for (int i = 0; i < NG - 1; ++i) f(i, std::false_type{});
    f(NG - 1, std::true_type{});
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float((u32)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}

// sum over the LPR lanes of a row (half a wave, or the whole workgroup of 256), in every lane
template <int LPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* lds) {
    a += dpp<0xB1>(a);      // lane ^ 1
    b += dpp<0xB1>(b);
    a += dpp<0x4E>(a);      // lane ^ 2
    b += dpp<0x4E>(b);
    a += dpp<0x141>(a);     // 7 - lane of 8
    b += dpp<0x141>(b);
    a += dpp<0x140>(a);     // 15 - lane of 16
    b += dpp<0x140>(b);
#pragma unroll
    for (int o = 16; o < (LPR < 64 ? LPR : 64); o <<= 1) {
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

// One tensor's row as it is stored, this lane's groups; loaded a row ahead of its use
template <typename T, bool VEC, int LPR, int NG>
struct RowLoad {
    Raw<T> r[NG];
    __device__ __forceinline__ void load(const void* base, long long row, int cols, int l) {
        const T* p = (const T*)base + row * cols;
        groups<NG>([&](int i, auto last) { load_group<T, VEC, last.value>(p, (i * LPR + l) * 8, cols, r[i]); });
    }
    template <bool LAST>
    __device__ __forceinline__ void get(int i, int cols, int l, float v[8]) const {
        unpack_group<T, VEC, LAST>(r[i], (i * LPR + l) * 8, cols, v);
    }
};

// z of this lane's groups, zeros past the row's end; keep[i] holds the kept bits of group i
template <typename T, bool VEC, int LPR, int NG>
__device__ __forceinline__ void make_z(const NormArgs& a, const RowLoad<T, VEC, LPR, NG>& x, const RowLoad<T, VEC, LPR, NG>& res,
                                       long long row, int l, u32 k0, u32 k1, float z[NG][8], u32 keep[NG]) {
    groups<NG>([&](int i, auto last) {
        const int c = (i * LPR + l) * 8;
        x.template get<last.value>(i, a.cols, l, z[i]);
        if (a.drop.thr) {
            keep[i] = keep8((u32)(c >> 3), (u32)row, a.drop, k0, k1);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = (keep[i] >> e) & 1u ? z[i][e] : 0.0f;
        }
        // written out as one fma, as are the sums below: a row's bits do not depend on how it is aligned
        if (a.residual) {
            float r[8];
            res.template get<last.value>(i, a.cols, l, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = fmaf(z[i][e], a.drop.scale, r[e]);
        } else if (a.drop.thr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] *= a.drop.scale;
        }
        if (last.value) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = c + (VEC ? 0 : e) < a.cols ? z[i][e] : 0.0f;
        }
    });
}

// a group of a row to memory
template <typename T, bool VEC, bool LAST>
__device__ __forceinline__ void store_group(void* base, long long row, int c, int cols, const float v[8]) {
    T* p = (T*)base + row * cols + c;
    if (!LAST)
        store8<T, VEC>(p, 8, v);
    else if (c < cols)
        store8<T, VEC>(p, cols - c, v);
}

struct Seed2 {
    u32 k0 = 0, k1 = 0;
    __device__ __forceinline__ explicit Seed2(const DropArgs& d) {
        if (d.thr) {
            const u64 seed = (u64)*d.seed;
            k0 = (u32)seed;
            k1 = (u32)(seed >> 32);
        }
    }
};

// mean, then the sum of (z - mean)^2 of the same registers (no cancellation of E z^2 - mean^2): one read of x and the residual,
// one write, bound by memory.  A row is held by half a wave (up to 1024 columns: two rows a wave, no LDS) or by the workgroup;
// weight and bias stay in registers over the rows and the next row is loaded while this one is summed.
// 65536 x 768 bfloat16 with residual and dropout: 49 us = 6.1 TB/s; 4097 x 771 float32, one row a half-wave: 9 us (2.7 TB/s,
// the latency of one load, two sums and one store; 4097 x 768: 7).
template <typename T, bool VEC, int LPR, int NG>
__global__ __launch_bounds__(256) void ln_fwd_kernel(NormArgs a) {
    __shared__ float lds[8];
    constexpr int RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const Seed2 k(a.drop);
    const float inv = 1.0f / (float)a.cols;
    const long long step = (long long)gridDim.x * RPB;
    long long r0 = (long long)blockIdx.x * RPB;
    RowLoad<T, VEC, LPR, NG> x, res;
    x.load(a.x, min(r0 + slot, a.rows - 1), a.cols, l);
    if (a.residual) res.load(a.residual, min(r0 + slot, a.rows - 1), a.cols, l);
    float w[NG][8], b[NG][8];
    groups<NG>([&](int i, auto last) {
        load_w<VEC, last.value>(a.weight, (i * LPR + l) * 8, a.cols, a.wbf16, w[i]);
        load_w<VEC, last.value>(a.bias, (i * LPR + l) * 8, a.cols, a.wbf16, b[i]);
    });
    for (; r0 < a.rows; r0 += step) {
        const bool in = r0 + slot < a.rows;       // a half-wave past the end repeats the last row and stores nothing
        const long long row = in ? r0 + slot : a.rows - 1;
        float z[NG][8];
        u32 keep[NG];
        make_z<T, VEC, LPR, NG>(a, x, res, row, l, k.k0, k.k1, z, keep);
        if (r0 + step < a.rows) {
            const long long next = min(r0 + step + slot, a.rows - 1);
            x.load(a.x, next, a.cols, l);
            if (a.residual) res.load(a.residual, next, a.cols, l);
        }
        float s = 0.0f, dummy = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += z[i][e];
        row_sum2<LPR>(s, dummy, lds);
        const float mean = s / (float)a.cols;
        float v = 0.0f;
        groups<NG>([&](int i, auto last) {
            const int c = (i * LPR + l) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = z[i][e] - mean;
                z[i][e] = d;
                v = fmaf(d, !last.value || c + (VEC ? 0 : e) < a.cols ? d : 0.0f, v);
            }
        });
        row_sum2<LPR>(v, dummy, lds);
        const float rstd = 1.0f / sqrtf(fmaf(v, inv, a.eps));
        if (!in) continue;
        if (l == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        groups<NG>([&](int i, auto last) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(z[i][e] * rstd, w[i][e], b[i][e]);
            store_group<T, VEC, last.value>(a.y, row, (i * LPR + l) * 8, a.cols, o);
        });
    }
}

// dx, dresidual and this workgroup's part of dg and db in one read of dy, x and the residual: dg and db gather in the registers
// of the lanes that hold the columns, over all rows of the workgroup, and leave as one row of partial sums.
// 65536 x 768 bfloat16 with residual and dropout: 95 us = 5.3 TB/s, and 5 us for ln_wgrad_kernel.
template <typename T, bool VEC, int LPR, int NG>
__global__ __launch_bounds__(256) void ln_bwd_kernel(NormArgs a) {
    __shared__ float lds[8];
    __shared__ float red[LPR == 256 ? 1 : 256 * 8];
    constexpr int RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const Seed2 k(a.drop);
    const float inv = 1.0f / (float)a.cols;
    const long long step = (long long)gridDim.x * RPB;
    long long r0 = (long long)blockIdx.x * RPB;
    RowLoad<T, VEC, LPR, NG> x, res, g;
    float mean, rstd;
    auto fetch = [&](long long r) {
        const long long row = min(r + slot, a.rows - 1);
        x.load(a.x, row, a.cols, l);
        if (a.residual) res.load(a.residual, row, a.cols, l);
        g.load(a.dy, row, a.cols, l);
        mean = a.mean[row];
        rstd = a.rstd[row];
    };
    fetch(r0);
    float dw[NG][8], db[NG][8], w[NG][8];
    groups<NG>([&](int i, auto last) {
        load_w<VEC, last.value>(a.weight, (i * LPR + l) * 8, a.cols, a.wbf16, w[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = db[i][e] = 0.0f;
    });
    for (; r0 < a.rows; r0 += step) {
        const bool in = r0 + slot < a.rows;
        const long long row = in ? r0 + slot : a.rows - 1;
        float z[NG][8], dy[NG][8];
        u32 keep[NG];
        make_z<T, VEC, LPR, NG>(a, x, res, row, l, k.k0, k.k1, z, keep);
        const float mu = mean, rs = rstd;
        float s1 = 0.0f, s2 = 0.0f;
        groups<NG>([&](int i, auto last) {
            const int c = (i * LPR + l) * 8;
            g.template get<last.value>(i, a.cols, l, dy[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) dy[i][e] = in && (!last.value || c + (VEC ? 0 : e) < a.cols) ? dy[i][e] : 0.0f;
        });
        if (r0 + step < a.rows) fetch(r0 + step);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float xh = (z[i][e] - mu) * rs;
                z[i][e] = xh;
                dw[i][e] = fmaf(dy[i][e], xh, dw[i][e]);
                db[i][e] += dy[i][e];
                dy[i][e] *= w[i][e];              // a = dy g (0 past the row's end)
                s1 += dy[i][e];
                s2 = fmaf(dy[i][e], xh, s2);
            }
        row_sum2<LPR>(s1, s2, lds);
        if (!in) continue;
        const float m1 = s1 * inv, m2 = s2 * inv;
        groups<NG>([&](int i, auto last) {
            const int c = (i * LPR + l) * 8;
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = rs * fmaf(-z[i][e], m2, dy[i][e] - m1);
            if (a.dresidual) store_group<T, VEC, last.value>(a.dresidual, row, c, a.cols, o);
            if (a.drop.thr) apply_keep(o, keep[i], a.drop.scale);
            store_group<T, VEC, last.value>(a.dx, row, c, a.cols, o);
        });
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
                for (int q = 0; q < RPB; ++q) s += red[(q * 8 + e) * LPR + l];
                if (c + e < a.cols) out[t * a.cols + c + e] = s;
            }
        }
}

// out[c] = sum over the P partial rows, in a fixed order (atomics would not keep the bits): 16 columns x 64 row lanes a
// workgroup.  512 x 1536 sums: 4.2 us, the latency of eight dependent loads and a launch.
__global__ __launch_bounds__(1024) void ln_wgrad_kernel(const float* part, int P, int cols, void* dw, void* db, int wbf16) {
    __shared__ float red[16][17];
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + cl;               // column of [dw | db]
    float s = 0.0f;
    if (c < 2 * cols) {
#pragma unroll 4
        for (int p = rl; p < P; p += 64) s += part[(size_t)p * 2 * cols + c];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][cl] = s;
    __syncthreads();
    if (rl == 0 && c < 2 * cols) {
        float t = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; ++q) t += red[q][cl];
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

// workgroups: as many as are resident together at 768 columns of bfloat16 (65536 rows: the forward pass 50.6 us with 768, 52.5
// with 1024; the backward pass, whose every workgroup leaves a row of partial sums, 101.5 with 512, 102.7 with 1024).  Where a lane
// holds more (backward: four groups, from 769 columns on, and three of float32, from 513) the registers leave one wave a SIMD and
// half of these run at a time: float32 with the weights' sums 2000 x 771 12 us, 4097 x 771 20, 8192 x 771 28.
int norm_grid(long long rows, int cols, bool bwd) {
    const long long need = (rows + rows_per_block(cols) - 1) / rows_per_block(cols), most = bwd ? 512 : 768;
    return (int)(need < most ? need : most);
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
    launch_norm_any<false>(a, dtype, vec, norm_grid(rows, cols, false), (hipStream_t)stream);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int64_t otter_layernorm_backward_workspace(int64_t rows, int cols) {
    if (rows < 0 || cols < 1 || cols > LN_MAX_COLS)
        return set_err(OTTER_EINVAL, "layernorm_backward_workspace: bad rows=%lld cols=%d", (long long)rows, cols);
    return (int64_t)norm_grid(rows, cols, true) * 2 * cols * (int64_t)sizeof(float);
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
    const int grid = norm_grid(rows, cols, true);
    if (rows > 0) {
        const bool vec = cols % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(residual) && aligned16(dresidual);
        launch_norm_any<true>(a, dtype, vec, grid, st);
        OTTER_HIP_TRY(hipGetLastError());
    }
    ln_wgrad_kernel<<<(2 * cols + 15) / 16, 1024, 0, st>>>(a.part, grid, cols, dweight, dbias, a.wbf16);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
