// attention.hip — attention of the training path on gfx950: forward with the row statistics, backward that makes the
// probabilities again.  Bidirectional, head dimension 64, dense batches with a key mask or packed sequences.
//
//   S = scale Q K^T (masked keys left out),  P = softmax(S),  Z = keep / (1 - p),  O = (P Z) V,  lse = log sum exp S
//   D_i = sum_d dO_id O_id,  dS = P (Z (dO V^T) - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = (P Z)^T dO
//
// A sequence whose mask leaves nothing attends to all its L keys evenly (P = 1 / L, the encoder's rule); no gradient
// reaches its queries and keys.  What masked keys hold reaches nothing: they enter the products as zeros.
//
// Both operands of a product come from 16-byte fragments of 64-element rows; a score tile leaves the matrix unit with one
// of its two indices on the lane and sixteen of the other in the registers, which is the layout the next product's right
// operand needs ("accumulator tile as the next operand").  So the tile is made with the QUERY on the lane where the
// contraction runs over keys (O, dQ) and with the KEY on the lane where it runs over queries (dK, dV): no probability
// ever goes through memory.
#include "otter_common.h"
#include "otter_philox.h"

namespace otter {
int make_drop(const char* what, float p, const int64_t* seed, uint32_t call, DropArgs* out);
}

namespace {
using namespace otter;

constexpr int DH = 64;         // head dimension
constexpr int TR = 64;         // rows of a streamed tile
constexpr int OWN = 128;       // rows a workgroup owns: 4 waves x 32

struct View {                  // element strides of a [batch, token, head, 64] tensor (batch stride unused when packed)
    void* p;
    long long sb, st, sh;
};

struct AttnTrainArgs {
    View q, k, v, o, dout, dq, dk, dv;
    float* lse;                // dense [B][heads][L], packed [heads][T]
    float* delta;              // like lse
    const long long* mask;     // dense: [B][L], non-zero = attend; null: every key
    const int* cu;             // packed: [B + 1] row offsets; null: dense
    long long T;               // packed: rows of the tensors
    int B, L, heads, nblk;     // L: tokens (dense) / longest sequence (packed); nblk: workgroups a (sequence, head)
    float scale, c2;           // c2 = scale * log2 e
    DropArgs drop;
};

struct Seq {
    int b, h, blk;
    long long row0;            // first row of the sequence, counted over the whole tensor (packed) or 0 (dense)
    int len;
    long long stat;            // index of its first row in lse / delta
};

__device__ __forceinline__ Seq find_seq(const AttnTrainArgs& a, int item) {
    Seq s;
    s.blk = item % a.nblk;
    const int bh = item / a.nblk;
    s.h = bh % a.heads;
    s.b = bh / a.heads;
    if (a.cu) {
        const long long lo = min((long long)max(a.cu[s.b], 0), a.T), hi = min((long long)max(a.cu[s.b + 1], 0), a.T);
        s.row0 = lo;
        s.len = (int)max(hi - lo, 0ll);
        s.stat = (long long)s.h * a.T + lo;
    } else {
        s.row0 = 0;
        s.len = a.L;
        s.stat = ((long long)s.b * a.heads + s.h) * a.L;
    }
    return s;
}

template <typename T>
__device__ __forceinline__ T* head_ptr(const AttnTrainArgs& a, const View& v, const Seq& s) {
    return (T*)v.p + (a.cu ? s.row0 * v.st : (long long)s.b * v.sb) + (long long)s.h * v.sh;
}

// rows of a packed tensor that belong to no sequence: [0, cu[0]) and [cu[B], T), set to zero by the workgroups behind the
// last item (one a head)
template <typename T>
__device__ __forceinline__ void zero_outside(const AttnTrainArgs& a, int h, const View& v, float* stat) {
    const long long lo = min((long long)max(a.cu[0], 0), a.T), hi = min((long long)max(a.cu[a.B], 0), a.T);
    const long long n = lo + (a.T - hi);
    for (long long e = threadIdx.x; e < n * DH; e += blockDim.x) {
        const long long r = e / DH, row = r < lo ? r : hi + (r - lo);
        ((T*)v.p)[row * v.st + (long long)h * v.sh + (e & (DH - 1))] = from_f<T>(0.0f);
        if (stat && (e & (DH - 1)) == 0) stat[(long long)h * a.T + row] = 0.0f;
    }
}

// ------------------------------------------------------------------ tiles
template <typename T>
struct Tile {
    static constexpr int ROWB = DH * (int)sizeof(T);   // bytes a row
    static constexpr int CH = ROWB / 16;               // 16-byte chunks a row
    static constexpr int NF = CH / 2;                  // fragment chunks a lane
    static constexpr int EPC = 16 / (int)sizeof(T);
    static constexpr int BYTES = TR * ROWB;
    // chunk c of row r lies at chunk c ^ swz(r): the 32 rows a fragment read touches spread over the banks
    static __device__ __forceinline__ int swz(int r) { return CH == 16 ? (r & 15) : ((r >> 1) & 7); }
    static __device__ __forceinline__ float4 frag(const char* t, int row, int c) {
        return *reinterpret_cast<const float4*>(t + row * ROWB + ((c ^ swz(row)) << 4));
    }
};

// rows row0 .. row0 + 63 into LDS; rows that `keep` leaves out (bit per row) become zeros and are not read
template <typename T>
__device__ __forceinline__ void stage(char* lds, const T* base, long long st, int row0, u64 keep) {
    using X = Tile<T>;
    for (int c = threadIdx.x; c < TR * X::CH; c += blockDim.x) {
        const int r = c / X::CH, p = c % X::CH;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if ((keep >> r) & 1) v = *reinterpret_cast<const float4*>(base + (long long)(row0 + r) * st + p * X::EPC);
        *reinterpret_cast<float4*>(lds + r * X::ROWB + ((p ^ X::swz(r)) << 4)) = v;
    }
}

template <typename T>
__device__ __forceinline__ void mma(f32x16& acc, const float4& a, const float4& b) {
    if constexpr (sizeof(T) == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    } else {
        const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(av[e], bv[e], acc, 0, 0, 0);
    }
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}

// row of a 32 x 32 accumulator tile that register r of lane half h holds
__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// acc[rows of the tile][own rows on the lane] = tile rows (row0 .. row0 + 31) x own fragments
template <typename T>
__device__ __forceinline__ f32x16 row_product(const char* t, int row0, const float4 (&own)[Tile<T>::NF], int l31, int h) {
    f32x16 acc = zero16();
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j) mma<T>(acc, Tile<T>::frag(t, row0 + l31, 2 * j + h), own[j]);
    return acc;
}

// o[d half] += X^T w: X = tile rows row0 .. row0 + 31, w = an accumulator tile with X's row on the registers.
// bf16: w is rounded here, the one rounding between the two products (2^-9 of each weight; sums stay in float32).
template <typename T>
__device__ __forceinline__ void col_product(f32x16 (&o)[2], const char* t, int row0, const f32x16& w, int lane) {
    using X = Tile<T>;
    const int h = lane >> 5, l31 = lane & 31;
    if constexpr (sizeof(T) == 2) {
        const int i16 = lane & 15, qq = i16 >> 2, pp = i16 & 3, g = (lane >> 4) & 1;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            bf16x8 wb;
#pragma unroll
            for (int j = 0; j < 8; ++j) wb[j] = (__bf16)w[8 * s2 + j];
            const int r0 = row0 + s2 * 16 + 4 * h + qq;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                // X^T[d][row], rows 16 s2 + 8 (j >> 2) + 4 h + (j & 3): two transposed reads of 4 rows x 16 columns
                const int byte = (d * 32 + 16 * g + 4 * pp) * 2, c = byte >> 4, in = byte & 15;
                const char* p0 = t + r0 * X::ROWB + ((c ^ X::swz(r0)) << 4) + in;
                const char* p1 = t + (r0 + 8) * X::ROWB + ((c ^ X::swz(r0 + 8)) << 4) + in;
                const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)p0);
                const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)p1);
                const short va[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, va), wb, o[d], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = row0 + acc_row(r, h);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int col = d * 32 + l31;
                const float x = *reinterpret_cast<const float*>(t + row * X::ROWB + (((col >> 2) ^ X::swz(row)) << 4) + (col & 3) * 4);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, w[r], o[d], 0, 0, 0);
            }
        }
    }
}

// this lane's row (index `row`, clamped by the caller), chunks 2 j + h
template <typename T>
__device__ __forceinline__ void load_own(float4 (&f)[Tile<T>::NF], const T* base, long long st, int row, int h) {
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j)
        f[j] = *reinterpret_cast<const float4*>(base + (long long)row * st + (2 * j + h) * Tile<T>::EPC);
}

// store o[2] (head dimension on the registers, row on the lane) times f
template <typename T>
__device__ __forceinline__ void store_own(T* dst, const f32x16 (&o)[2], float f, int h) {
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            T* p = dst + d * 32 + 8 * g + 4 * h;
            if constexpr (sizeof(T) == 2) {
                const u32 w0 = (u32)f2bf(o[d][4 * g] * f) | ((u32)f2bf(o[d][4 * g + 1] * f) << 16);
                const u32 w1 = (u32)f2bf(o[d][4 * g + 2] * f) | ((u32)f2bf(o[d][4 * g + 3] * f) << 16);
                *reinterpret_cast<uint2*>(p) = make_uint2(w0, w1);
            } else {
                *reinterpret_cast<float4*>(p) = make_float4(o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
            }
        }
}

// ------------------------------------------------------------------ keys that count
// How far keys count in this sequence (last one + 1), and whether none does (then all do, evenly).
__device__ __forceinline__ int key_end(const AttnTrainArgs& a, const Seq& s, bool& even) {
    even = false;
    if (!a.mask || s.len == 0) return s.len;
    const long long* m = a.mask + (long long)s.b * a.L;
    for (int c = (s.len - 1) >> 6; c >= 0; --c) {
        const int j = c * 64 + (threadIdx.x & 63);
        const u64 bal = __ballot(j < s.len && m[j] != 0);
        if (bal) return c * 64 + 64 - __builtin_clzll(bal);
    }
    even = true;
    return s.len;
}

// bit r: key j0 + r counts
__device__ __forceinline__ u64 key_bits(const AttnTrainArgs& a, const Seq& s, int j0, bool even) {
    const int j = j0 + (threadIdx.x & 63);
    return __ballot(j < s.len && (even || !a.mask || a.mask[(long long)s.b * a.L + j] != 0));
}

// bits of rows j0 .. j0 + 63 below n
__device__ __forceinline__ u64 row_bits(int j0, int n) { return n - j0 >= 64 ? ~0ull : (1ull << max(n - j0, 0)) - 1ull; }

// ------------------------------------------------------------------ draws
// bit r: the value in register r is kept.  QL: the query is on the lane (row i) and keys j0 + acc_row(r, h) on the
// registers; otherwise the key is on the lane (row j) and queries i0 + acc_row(r, h) on the registers.
template <bool QL>
__device__ __forceinline__ u32 keep16(const DropArgs& d, u32 k0, u32 k1, u32 bh, int own, int t0, int h) {
    u32 keep = 0;
    if constexpr (QL) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const Philox4 w = philox7((u32)(t0 + 8 * g + 4 * h) >> 2, (u32)own >> 1, bh, d.call, k0, k1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u32 draw = own & 1 ? w.w[e] >> 16 : w.w[e] & 0xFFFFu;
                keep |= (u32)(draw >= d.thr) << (4 * g + e);
            }
        }
    } else {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const Philox4 w = philox7((u32)own >> 2, (u32)(t0 + 8 * g + 4 * h + 2 * e) >> 1, bh, d.call, k0, k1);
                const u32 x = own & 2 ? (own & 1 ? w.w[3] : w.w[2]) : (own & 1 ? w.w[1] : w.w[0]);
                keep |= (u32)((x & 0xFFFFu) >= d.thr) << (4 * g + 2 * e);
                keep |= (u32)((x >> 16) >= d.thr) << (4 * g + 2 * e + 1);
            }
    }
    return keep;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------------ forward
template <typename T>
__global__ __launch_bounds__(256) void attn_fwd_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    __shared__ __attribute__((aligned(16))) char sK[X::BYTES];
    __shared__ __attribute__((aligned(16))) char sV[X::BYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) return zero_outside<T>(a, blockIdx.x - items, a.o, a.lse);
    const Seq s = find_seq(a, xcd_remap(blockIdx.x, items));
    bool even;
    const int kend = key_end(a, s, even);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    T* O = head_ptr<T>(a, a.o, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    u32 k0 = 0, k1 = 0;
    if (a.drop.thr) {
        const u64 seed = (u64)*a.drop.seed;
        k0 = (u32)seed;
        k1 = (u32)(seed >> 32);
    }
    for (int q0 = s.blk * OWN; q0 < s.len; q0 += a.nblk * OWN) {
        const int i = q0 + wave * 32 + l31;
        float4 qf[X::NF];
        load_own<T>(qf, Q, a.q.st, min(i, s.len - 1), h);
        f32x16 o[2] = {zero16(), zero16()};
        float m = -INFINITY, l = 0.0f;
        for (int j0 = 0; j0 < kend; j0 += TR) {
            const u64 bits = key_bits(a, s, j0, even);
            if (bits == 0) continue;
            __syncthreads();
            stage<T>(sK, K, a.k.st, j0, bits);
            stage<T>(sV, V, a.v.st, j0, bits);
            __syncthreads();
            f32x16 sc[2];
            float mx = -INFINITY;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                sc[sub] = row_product<T>(sK, sub * 32, qf, l31, h);
                const u32 kb = (u32)(bits >> (32 * sub)) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = even ? 0.0f : sc[sub][r] * a.c2;
                    v = (kb >> acc_row(r, 0)) & 1u ? v : -INFINITY;
                    sc[sub][r] = v;
                    mx = fmaxf(mx, v);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mnew = fmaxf(m, mx), base = mnew == -INFINITY ? 0.0f : mnew;
            const float alpha = exp2_(m - base);
            m = mnew;
            float sum = 0.0f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const u32 keep = a.drop.thr ? keep16<true>(a.drop, k0, k1, bh, i, j0 + 32 * sub, h) : 0xFFFFu;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_(sc[sub][r] - base);
                    sum += p;                                        // the softmax's sum is over all keys, dropped or not
                    sc[sub][r] = (keep >> r) & 1u ? p : 0.0f;
                }
            }
            l = l * alpha + sum + __shfl_xor(sum, 32);
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) col_product<T>(o, sV, sub * 32, sc[sub], lane);
        }
        if (i < s.len) {
            store_own<T>(O + (long long)i * a.o.st, o, a.drop.scale / l, h);
            if (h == 0) a.lse[s.stat + i] = (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
        }
    }
}

// ------------------------------------------------------------------ backward: dQ (and D)
template <typename T>
__global__ __launch_bounds__(256) void attn_dq_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    __shared__ __attribute__((aligned(16))) char sK[X::BYTES];
    __shared__ __attribute__((aligned(16))) char sV[X::BYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) return zero_outside<T>(a, blockIdx.x - items, a.dq, nullptr);
    const Seq s = find_seq(a, xcd_remap(blockIdx.x, items));
    bool even;
    const int kend = key_end(a, s, even);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    const T *O = head_ptr<T>(a, a.o, s), *dO = head_ptr<T>(a, a.dout, s);
    T* dQ = head_ptr<T>(a, a.dq, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    u32 k0 = 0, k1 = 0;
    if (a.drop.thr) {
        const u64 seed = (u64)*a.drop.seed;
        k0 = (u32)seed;
        k1 = (u32)(seed >> 32);
    }
    for (int q0 = s.blk * OWN; q0 < s.len; q0 += a.nblk * OWN) {
        const int i = q0 + wave * 32 + l31, ic = min(i, s.len - 1);
        float4 qf[X::NF], df[X::NF];
        load_own<T>(qf, O, a.o.st, ic, h);
        load_own<T>(df, dO, a.dout.st, ic, h);
        float D = 0.0f;
#pragma unroll
        for (int j = 0; j < X::NF; ++j) {
            const T *x = reinterpret_cast<const T*>(&qf[j]), *y = reinterpret_cast<const T*>(&df[j]);
#pragma unroll
            for (int e = 0; e < X::EPC; ++e) D += to_f<T>(x[e]) * to_f<T>(y[e]);
        }
        D += __shfl_xor(D, 32);
        if (i < s.len && h == 0) a.delta[s.stat + i] = D;
        load_own<T>(qf, Q, a.q.st, ic, h);
        const float lse2 = a.lse[s.stat + ic] * 1.4426950408889634f;
        f32x16 o[2] = {zero16(), zero16()};
        if (!even)                                  // even: dS = 0
            for (int j0 = 0; j0 < kend; j0 += TR) {
                const u64 bits = key_bits(a, s, j0, even);
                if (bits == 0) continue;
                __syncthreads();
                stage<T>(sK, K, a.k.st, j0, bits);
                stage<T>(sV, V, a.v.st, j0, bits);
                __syncthreads();
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    f32x16 sc = row_product<T>(sK, sub * 32, qf, l31, h);
                    const f32x16 dp = row_product<T>(sV, sub * 32, df, l31, h);
                    const u32 kb = (u32)(bits >> (32 * sub)) >> (4 * h);
                    const u32 keep = a.drop.thr ? keep16<true>(a.drop, k0, k1, bh, i, j0 + 32 * sub, h) : 0xFFFFu;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = exp2_(fmaf(sc[r], a.c2, -lse2));
                        const float g = ((keep >> r) & 1u ? dp[r] * a.drop.scale : 0.0f) - D;
                        sc[r] = (kb >> acc_row(r, 0)) & 1u ? p * g : 0.0f;
                    }
                    col_product<T>(o, sK, sub * 32, sc, lane);
                }
            }
        if (i < s.len) store_own<T>(dQ + (long long)i * a.dq.st, o, a.scale, h);
    }
}

// ------------------------------------------------------------------ backward: dK, dV
template <typename T>
__global__ __launch_bounds__(256) void attn_dkv_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    __shared__ __attribute__((aligned(16))) char sQ[X::BYTES];
    __shared__ __attribute__((aligned(16))) char sO[X::BYTES];
    __shared__ float sL[TR], sD[TR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, l31 = lane & 31;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) {
        zero_outside<T>(a, blockIdx.x - items, a.dk, nullptr);
        return zero_outside<T>(a, blockIdx.x - items, a.dv, nullptr);
    }
    const Seq s = find_seq(a, xcd_remap(blockIdx.x, items));
    bool even;
    const int kend = key_end(a, s, even);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    const T* dO = head_ptr<T>(a, a.dout, s);
    T *dK = head_ptr<T>(a, a.dk, s), *dV = head_ptr<T>(a, a.dv, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    u32 k0 = 0, k1 = 0;
    if (a.drop.thr) {
        const u64 seed = (u64)*a.drop.seed;
        k0 = (u32)seed;
        k1 = (u32)(seed >> 32);
    }
    for (int n0 = s.blk * OWN; n0 < s.len; n0 += a.nblk * OWN) {
        const int j = n0 + wave * 32 + l31, jc = min(j, s.len - 1);
        const bool counts = j < kend && (even || !a.mask || a.mask[(long long)s.b * a.L + jc] != 0);
        float4 kf[X::NF], vf[X::NF];
        load_own<T>(kf, K, a.k.st, jc, h);
        load_own<T>(vf, V, a.v.st, jc, h);
        f32x16 ok[2] = {zero16(), zero16()}, ov[2] = {zero16(), zero16()};
        if (n0 < kend)
            for (int i0 = 0; i0 < s.len; i0 += TR) {
                const u64 bits = row_bits(i0, s.len);
                __syncthreads();
                stage<T>(sQ, Q, a.q.st, i0, bits);
                stage<T>(sO, dO, a.dout.st, i0, bits);
                if (threadIdx.x < TR) {
                    const int i = i0 + threadIdx.x;
                    // rows past the end: exp2(0 - inf) = 0
                    sL[threadIdx.x] = i < s.len ? a.lse[s.stat + i] * 1.4426950408889634f : INFINITY;
                    sD[threadIdx.x] = i < s.len ? a.delta[s.stat + i] : 0.0f;
                }
                __syncthreads();
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    f32x16 sc = row_product<T>(sQ, sub * 32, kf, l31, h);
                    f32x16 dp = row_product<T>(sO, sub * 32, vf, l31, h);
                    const u32 keep = a.drop.thr ? keep16<false>(a.drop, k0, k1, bh, j, i0 + 32 * sub, h) : 0xFFFFu;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int row = sub * 32 + acc_row(r, h);
                        float p = exp2_((even ? 0.0f : sc[r] * a.c2) - sL[row]);
                        p = counts ? p : 0.0f;
                        const bool kept = (keep >> r) & 1u;
                        const float g = (kept ? dp[r] * a.drop.scale : 0.0f) - sD[row];
                        sc[r] = kept ? p : 0.0f;
                        dp[r] = counts && !even ? p * g : 0.0f;
                    }
                    col_product<T>(ov, sO, sub * 32, sc, lane);
                    col_product<T>(ok, sQ, sub * 32, dp, lane);
                }
            }
        if (j < s.len) {
            store_own<T>(dK + (long long)j * a.dk.st, ok, a.scale, h);
            store_own<T>(dV + (long long)j * a.dv.st, ov, a.drop.scale, h);
        }
    }
}

// ------------------------------------------------------------------ host side
bool bad_view(const otter_view& v, size_t size) {
    const long long step = 16 / (long long)size;
    return !v.data || ((uintptr_t)v.data & 15) || v.stride_batch % step || v.stride_token % step || v.stride_head % step;
}

int set_view(const char* what, const char* name, const otter_view& v, size_t size, View* out) {
    if (bad_view(v, size))
        return set_err(OTTER_EINVAL, "%s: %s must be non-NULL, 16-byte aligned, its strides multiples of 16 bytes", what, name);
    *out = View{v.data, v.stride_batch, v.stride_token, v.stride_head};
    return OTTER_OK;
}

int fill(const char* what, const otter_attention_args* x, AttnTrainArgs* a, long long* rows) {
    if (!x) return set_err(OTTER_EINVAL, "%s: NULL arguments", what);
    if (x->dtype != OTTER_F32 && x->dtype != OTTER_BF16) return set_err(OTTER_EINVAL, "%s: dtype must be float32 or bfloat16", what);
    if (x->head_dim != DH) return set_err(OTTER_ENOTIMPL, "%s: head dimension %d (only 64 is built)", what, x->head_dim);
    if (x->batch < 0 || x->tokens < 0 || x->heads < 1 || x->total < 0)
        return set_err(OTTER_EINVAL, "%s: bad batch=%d tokens=%d heads=%d total=%lld", what, x->batch, x->tokens, x->heads,
                       (long long)x->total);
    if (x->cu_seqlens && x->mask) return set_err(OTTER_EINVAL, "%s: a key mask and packed sequences exclude each other", what);
    if (x->total > 0x7FFFFFFFll) return set_err(OTTER_EINVAL, "%s: total=%lld exceeds 2^31 - 1", what, (long long)x->total);
    if (!(x->scale == x->scale)) return set_err(OTTER_EINVAL, "%s: scale is not a number", what);
    int rc = make_drop(what, x->dropout_p, x->seed, x->call, &a->drop);
    if (rc) return rc;
    a->B = x->batch;
    a->L = x->tokens;
    a->heads = x->heads;
    a->T = x->total;
    a->mask = (const long long*)x->mask;
    a->cu = x->cu_seqlens;
    a->scale = x->scale;
    a->c2 = x->scale * 1.4426950408889634f;
    a->lse = x->lse;
    a->nblk = x->tokens > OWN ? (x->tokens + OWN - 1) / OWN : 1;
    *rows = x->cu_seqlens ? x->total : (long long)x->batch * x->tokens;
    if ((long long)a->nblk * a->heads * a->B + a->heads > 0x7FFFFFFFll || (long long)a->B * a->heads > 0x7FFFFFFFll)
        return set_err(OTTER_EINVAL, "%s: batch x heads x tokens is too large for one launch", what);
    return OTTER_OK;
}

}  // namespace

extern "C" {

int otter_attention_forward(int device, const otter_attention_args* x, void* stream) {
    AttnTrainArgs a = {};
    long long rows = 0;
    int rc = fill("attention_forward", x, &a, &rows);
    if (rc) return rc;
    if (rows == 0) return OTTER_OK;
    const size_t size = x->dtype == OTTER_BF16 ? 2 : 4;
    if ((rc = set_view("attention_forward", "q", x->q, size, &a.q)) || (rc = set_view("attention_forward", "k", x->k, size, &a.k)) ||
        (rc = set_view("attention_forward", "v", x->v, size, &a.v)) || (rc = set_view("attention_forward", "out", x->out, size, &a.o)))
        return rc;
    if (!a.lse) return set_err(OTTER_EINVAL, "attention_forward: NULL lse");
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "attention_forward: hipSetDevice(%d) failed", device);
    const int grid = a.nblk * a.heads * a.B + (a.cu ? a.heads : 0);
    hipStream_t st = (hipStream_t)stream;
    if (size == 2)
        attn_fwd_kernel<bf16_t><<<grid, 256, 0, st>>>(a);
    else
        attn_fwd_kernel<float><<<grid, 256, 0, st>>>(a);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int64_t otter_attention_backward_workspace(const otter_attention_args* x) {
    AttnTrainArgs a = {};
    long long rows = 0;
    int rc = fill("attention_backward_workspace", x, &a, &rows);
    if (rc) return rc;
    return rows * a.heads * (int64_t)sizeof(float);
}

int otter_attention_backward(int device, const otter_attention_args* x, void* stream) {
    AttnTrainArgs a = {};
    long long rows = 0;
    int rc = fill("attention_backward", x, &a, &rows);
    if (rc) return rc;
    if (rows == 0) return OTTER_OK;
    const size_t size = x->dtype == OTTER_BF16 ? 2 : 4;
    const struct {
        const char* name;
        const otter_view* v;
        View* out;
    } views[] = {{"q", &x->q, &a.q},       {"k", &x->k, &a.k},    {"v", &x->v, &a.v},    {"out", &x->out, &a.o},
                 {"dout", &x->dout, &a.dout}, {"dq", &x->dq, &a.dq}, {"dk", &x->dk, &a.dk}, {"dv", &x->dv, &a.dv}};
    for (const auto& v : views)
        if ((rc = set_view("attention_backward", v.name, *v.v, size, v.out))) return rc;
    if (!a.lse || !x->workspace) return set_err(OTTER_EINVAL, "attention_backward: NULL lse or workspace");
    const int64_t need = rows * a.heads * (int64_t)sizeof(float);
    if (x->workspace_bytes < need)
        return set_err(OTTER_EINVAL, "attention_backward: workspace of %lld bytes, needs %lld", (long long)x->workspace_bytes,
                       (long long)need);
    a.delta = (float*)x->workspace;
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "attention_backward: hipSetDevice(%d) failed", device);
    const int grid = a.nblk * a.heads * a.B + (a.cu ? a.heads : 0);
    hipStream_t st = (hipStream_t)stream;
    if (size == 2) {
        attn_dq_kernel<bf16_t><<<grid, 256, 0, st>>>(a);
        attn_dkv_kernel<bf16_t><<<grid, 256, 0, st>>>(a);
    } else {
        attn_dq_kernel<float><<<grid, 256, 0, st>>>(a);
        attn_dkv_kernel<float><<<grid, 256, 0, st>>>(a);
    }
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
