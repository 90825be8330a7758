// attention.hip — attention of the training path on gfx950: forward with the row statistics, backward that makes the
// probabilities again.  Bidirectional, head dimension 64, dense batches with a key mask or packed sequences.
//
//   S = scale Q K^T (masked keys left out),  P = softmax(S),  Z = keep / (1 - p),  O = (P Z) V,  lse = log sum exp S
//   D_i = sum_d dO_id O_id,  dS = P (Z (dO V^T) - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = (P Z)^T dO
//
// A sequence whose mask leaves nothing attends to all its L keys evenly (P = 1 / L, the encoder's rule); no gradient
// reaches its queries and keys, as where one key counts (P = 1).  What masked keys hold reaches nothing: they enter the
// products as zeros.
//
// Both operands of a product come from 16-byte fragments of 64-element rows; a score tile leaves the matrix unit with one
// of its two indices on the lane and sixteen of the other in the registers, which is the layout the next product's right
// operand needs ("accumulator tile as the next operand").  So the tile is made with the QUERY on the lane where the
// contraction runs over keys (O, dQ) and with the KEY on the lane where it runs over queries (dK, dV): no probability
// ever goes through memory.
//
// Roundings.  float32: none but float32's own.  bfloat16: scores, softmax, their sums and all accumulators are float32, but the
// matrix unit takes bfloat16, so that P Z (in front of P V and of dV) and dS (in front of dQ and dK) are rounded to it, half a step
// (2^-8) of each weight; and D comes from the stored, rounded O, except where 64 keys hold a whole sequence (two passes; one
// pass of batches up to 128 tokens), whose O is as large as its terms.  Off from 64 bits by 2.4e-3 of the outputs' size, where
// rounding the outputs alone costs 1.7e-3; splitting P and dS in two parts would double those products.
#include "otter_common.h"
#include "otter_philox.h"

namespace otter {
int make_drop(const char* what, float p, const int64_t* seed, uint32_t call, DropArgs* out);
}

namespace {
using namespace otter;

constexpr int DH = 64;         // head dimension
constexpr int TR = 64;         // rows of a streamed tile
constexpr int CUS = 256;       // compute units of the chip
constexpr int OUTSIDE = CUS;   // workgroups for the rows of no sequence, at most
constexpr int OWN = 128;       // rows a workgroup owns: 4 waves x 32; 64 where two waves share 32 rows (HALF)

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
    int group;                 // (sequence, head) pairs whose workgroups are dealt out in turn
    int outside;               // packed: workgroups behind the last item, for the rows of no sequence
    float scale, c2;           // c2 = scale * log2 e
    DropArgs drop;
};

struct Seq {
    int b, h, blk;
    long long row0;            // first row of the sequence, counted over the whole tensor (packed) or 0 (dense)
    int len;
    long long stat;            // index of its first row in lse / delta
};

// Workgroups b, b + 8, ... share an XCD and its L2.  The workgroups of one (sequence, head), which read the same rows, go to
// one XCD; (sequence, head) pairs go round the XCDs one by one, so that every XCD gets its share of long and short sequences.
// An XCD takes `group` pairs at a time, first every pair's first rows, then the next: the workgroups that have nothing to do (rows
// past a short sequence's end) come after the others and not between them, where the round robin over the CUs would give
// some CUs all the work if a pair's workgroups divide their number.
__device__ __forceinline__ Seq find_seq(const AttnTrainArgs& a, int bid, int pair = -1) {
    Seq s;
    int bh = pair;
    s.blk = 0;
    if (pair < 0) {
        const int pairs = a.B * a.heads, whole = pairs & ~7, end = whole * a.nblk;   // the last pairs, fewer than 8, as they come
        const int idx = bid < end ? bid >> 3 : bid - end, n = bid < end ? whole >> 3 : pairs - whole;
        const int first = idx / (a.group * a.nblk) * a.group, size = min(a.group, n - first), r = idx - first * a.nblk;
        s.blk = r / size;
        bh = first + r - s.blk * size;
        bh = bid < end ? bh * 8 + (bid & 7) : whole + bh;
    }
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

// Rows of a packed tensor that belong to no sequence, [0, cu[0]) and [cu[B], T), are set to zero by the `outside` workgroups
// behind the last item, this one the part-th, 16 bytes a store.  (One a head and 2 bytes a store had made them the most of a
// call: 36864 rows of 65536 used, 12 heads, bfloat16, 681 us forward and 895 backward, now 120 and 296.)
template <typename T>
__device__ __forceinline__ void zero_outside(const AttnTrainArgs& a, int part, const View& v, float* stat) {
    constexpr int CH = DH * (int)sizeof(T) / 16;
    const long long lo = min((long long)max(a.cu[0], 0), a.T), hi = min((long long)max(a.cu[a.B], 0), a.T);
    const long long n = lo + (a.T - hi);
    const int per = a.heads * CH, at = max((int)blockDim.x / per, 1);      // chunks a row; rows at a time
    const int mine = (int)threadIdx.x / per, c0 = (int)threadIdx.x - mine * per;
    if (mine >= at) return;
    for (long long r = (long long)part * at + mine; r < n; r += (long long)a.outside * at) {
        const long long row = r < lo ? r : hi + (r - lo);
        for (int c = c0; c < per; c += blockDim.x) {
            const int h = c / CH, k = c - h * CH;
            *reinterpret_cast<uint4*>((T*)v.p + row * v.st + (long long)h * v.sh + k * (16 / (int)sizeof(T))) = make_uint4(0, 0, 0, 0);
            if (stat && k == 0) stat[(long long)h * a.T + row] = 0.0f;
        }
    }
}

// ------------------------------------------------------------------ tiles
// A tile in LDS: 64 rows of 64 elements, 16 bytes of padding a row.  With that pitch (36 / 68 words) neither the 16-byte
// reads down a column of rows nor the transposed 8-byte reads conflict, and every address is one of two lane constants plus
// an immediate (an XOR swizzle needs a register for each of its chunks: 60 more, one wave less a SIMD).
template <typename T>
struct Tile {
    static constexpr int PITCH = DH * (int)sizeof(T) + 16;
    static constexpr int CH = DH * (int)sizeof(T) / 16;   // 16-byte chunks a row
    static constexpr int NF = CH / 2;                     // fragment chunks a lane: 2 j + lane half
    static constexpr int EPC = 16 / (int)sizeof(T);
    static constexpr int BYTES = TR * PITCH;
};

// HALF: waves w and w + 2 own the same 32 rows; each takes its half of every streamed tile, and what they gathered is added up
// through LDS at the end.  x: n registers of waves 2 and 3 to those of waves 0 and 1, one slot of 64 lanes x N floats a wave.
template <int N>
struct Handover {
    float* p;
    __device__ __forceinline__ Handover(char* lds) : p(reinterpret_cast<float*>(lds) + (threadIdx.x >> 6 & 1) * N * 64 + (threadIdx.x & 63)) {}
    __device__ __forceinline__ void put(int i, float x) const { p[i * 64] = x; }
    __device__ __forceinline__ void put(int i, const f32x16 (&o)[2]) const {
#pragma unroll
        for (int e = 0; e < 32; ++e) put(i + e, o[e >> 4][e & 15]);
    }
    __device__ __forceinline__ float get(int i) const { return p[i * 64]; }
    __device__ __forceinline__ void add(int i, f32x16 (&o)[2]) const {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e >> 4][e & 15] += get(i + e);
    }
};

struct Lane {
    int lane, wave, h, l31;
    __device__ __forceinline__ Lane() : lane(threadIdx.x & 63), wave(threadIdx.x >> 6), h((threadIdx.x >> 5) & 1), l31(threadIdx.x & 31) {}
    template <typename T>
    __device__ __forceinline__ int frag() const { return l31 * Tile<T>::PITCH + h * 16; }
    // bf16: the corner of this lane's 4 x 16 block for the transposed reads; float: row 4 h, column l31
    template <typename T>
    __device__ __forceinline__ int col() const {
        return sizeof(T) == 2 ? (4 * h + ((lane & 15) >> 2)) * Tile<T>::PITCH + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2
                              : 4 * h * Tile<T>::PITCH + l31 * 4;
    }
};

// A tile on its way: 64 rows through the registers of the workgroup's 256 threads, loaded while the tile before it is
// multiplied.  Rows that `keep` leaves out (a bit per row) become zeros.
template <typename T>
struct Stage {
    using X = Tile<T>;
    static constexpr int N = TR * X::CH / 256, STEP = 256 / X::CH;   // loads a thread, rows between them
    float4 v[N];
    u64 keep;
    const T* p;                 // this thread's chunk of row 0
    long long st;
    int row, last;              // this thread's first row of the next tile, the sequence's last row
    __device__ __forceinline__ Stage(const T* base, long long stride, int len)
        : p(base + (threadIdx.x % X::CH) * X::EPC), st(stride), row(threadIdx.x / X::CH), last(len - 1) {}
    // No lane is switched off (a load inside a branch makes the compiler wait for the ones before it): rows past the end
    // are read from the last one, and what `keep` leaves out is cleared on its way to LDS.
    __device__ __forceinline__ void load(u64 bits) {
        keep = bits;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = *reinterpret_cast<const float4*>(p + min(row + i * STEP, last) * st);
        row += TR;
    }
    __device__ __forceinline__ void store(char* lds) {
        if (~keep != 0) {
            const u64 mine = keep >> (threadIdx.x / X::CH);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (!((mine >> (i * STEP)) & 1)) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        char* d = lds + (threadIdx.x / X::CH) * X::PITCH + (threadIdx.x % X::CH) * 16;
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<float4*>(d + i * STEP * X::PITCH) = v[i];
    }
};

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
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// acc[rows of the tile][own rows on the lane] = tile rows (32 from t on) x own fragments; t: the tile + Lane::frag
template <typename T>
__device__ __forceinline__ f32x16 row_product(const char* t, const float4 (&own)[Tile<T>::NF]) {
    f32x16 acc = zero16();
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j) mma<T>(acc, *reinterpret_cast<const float4*>(t + j * 32), own[j]);
    return acc;
}

// two of them side by side: neither waits for its own last step
template <typename T>
__device__ __forceinline__ void row_products(f32x16& x, f32x16& y, const char* tx, const float4 (&ox)[Tile<T>::NF], const char* ty,
                                             const float4 (&oy)[Tile<T>::NF]) {
    x = zero16();
    y = zero16();
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j) {
        mma<T>(x, *reinterpret_cast<const float4*>(tx + j * 32), ox[j]);
        mma<T>(y, *reinterpret_cast<const float4*>(ty + j * 32), oy[j]);
    }
}

// o[d half] += X^T w: X = tile rows (32 from t on), w = an accumulator tile with X's row on the registers; t: the tile +
// Lane::col.  bf16: w is rounded here, the one rounding between the two products (2^-8 of each weight at most; the sums
// stay in float32).
__device__ __forceinline__ void col_product_b(f32x16 (&o)[2], const char* t, const bf16x8 (&wb)[2]) {
    constexpr int P = Tile<bf16_t>::PITCH;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            // X^T[d][row], rows 16 s2 + 8 (j >> 2) + 4 h + (j & 3): two transposed reads of 4 rows x 16 columns
            const char* p0 = t + s2 * 16 * P + d * 64;
            const s16x4 v[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)p0),
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)(p0 + 8 * P))};
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), wb[s2], o[d], 0, 0, 0);
        }
}

template <typename T>
__device__ __forceinline__ void col_product(f32x16 (&o)[2], const char* t, const f32x16& w) {
    constexpr int P = Tile<T>::PITCH;
    if constexpr (sizeof(T) == 2) {
        bf16x8 wb[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) wb[r >> 3][r & 7] = (__bf16)w[r];
        col_product_b(o, t, wb);
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int d = 0; d < 2; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(t + acc_row(r, 0) * P + d * 128), w[r], o[d], 0, 0, 0);
    }
}

// this lane's row (index `row`, clamped by the caller), chunks 2 j + h
template <typename T>
__device__ __forceinline__ void load_own(float4 (&f)[Tile<T>::NF], const T* base, long long st, int row, int h) {
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j)
        f[j] = *reinterpret_cast<const float4*>(base + (long long)row * st + (2 * j + h) * Tile<T>::EPC);
}

template <typename T>
__device__ __forceinline__ void negate(float4 (&f)[Tile<T>::NF]) {
    constexpr u32 sign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j) {
        u32* w = reinterpret_cast<u32*>(&f[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] ^= sign;
    }
}

template <typename T>
__device__ __forceinline__ void zero_frags(float4 (&f)[Tile<T>::NF]) {
#pragma unroll
    for (int j = 0; j < Tile<T>::NF; ++j) f[j] = make_float4(0.f, 0.f, 0.f, 0.f);
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
// How far keys count in this sequence (last one + 1), whether none does (`even`: then all do, evenly), and whether the
// probabilities are what they are whatever q and k hold (`flat`: evenly, or one key has them all): no gradient reaches those.
__device__ __forceinline__ int key_end(const AttnTrainArgs& a, const Seq& s, bool& even, bool& flat) {
    even = false;
    flat = s.len == 1;
    if (!a.mask || s.len == 0) return s.len;
    const long long* m = a.mask + (long long)s.b * a.L;
    int end = 0;
    // four chunks of 64 at a time: a short sequence in a long row costs a latency for every 256 keys it leaves out; past the
    // last key that counts the walk goes on only as long as no other is found
    for (int c = (s.len - 1) >> 6; c >= 0; c -= 4) {
        long long v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = m[min(max(c - e, 0) * 64 + (int)(threadIdx.x & 63), s.len - 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const u64 bal = __ballot(c >= e && (c - e) * 64 + (int)(threadIdx.x & 63) < s.len && v[e] != 0);
            if (!bal) continue;
            if (end || (bal & (bal - 1))) {            // a second key
                flat = false;
                return end ? end : (c - e) * 64 + 64 - __builtin_clzll(bal);
            }
            end = (c - e) * 64 + 64 - __builtin_clzll(bal);
        }
    }
    even = end == 0;
    flat = true;
    return even ? s.len : end;
}

// bit r: key j0 + r counts.  The mask's value of this lane's key is loaded a tile before it is needed.
struct KeyBits {
    const long long* m;        // the sequence's mask, or null: every key below len counts
    int len;
    long long v;
    __device__ __forceinline__ KeyBits(const AttnTrainArgs& a, const Seq& s, bool even)
        : m(a.mask && !even ? a.mask + (long long)s.b * a.L : nullptr), len(s.len), v(1) {}
    __device__ __forceinline__ void fetch(int j0) {
        const int j = j0 + (threadIdx.x & 63);
        if (m && j < len) v = m[j];
    }
    __device__ __forceinline__ u64 bits(int j0) const { return __ballot(j0 + (int)(threadIdx.x & 63) < len && v != 0); }
};

// bits of rows j0 .. j0 + 63 below n
__device__ __forceinline__ u64 row_bits(int j0, int n) { return n - j0 >= 64 ? ~0ull : (1ull << max(n - j0, 0)) - 1ull; }

// ------------------------------------------------------------------ draws
template <int CTRL>
__device__ __forceinline__ u32 quad(u32 x) { return (u32)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true); }

// Draws of a 32 x 32 score tile.  x[8]: two draws of 16 bits each; kept(r) tests the one of register r.
// A counter's eight draws (2 queries x 4 keys) belong to a pair of lanes where the query is on the lane and to four lanes
// where the key is; each of them makes its share of the counters and they hand the words around inside the quad (DPP), so no
// draw is made twice: two counters a lane for sixteen values.
struct Draws {
    u32 x[8];
    u32 thr, thrhi;
    // query on the lane: keys j0 + acc_row(r, h) of query i.  The even query's lane makes groups 0 and 1 of four keys, the
    // odd one's 2 and 3; of every word the even query takes the low half, the odd one the high half.
    __device__ __forceinline__ void queries(const DropArgs& d, u32 k0, u32 k1, u32 bh, int i, int j0, int h) {
        thr = d.thr;
        thrhi = d.thr << 16;
        const u32 odd = (u32)i & 1u, sel = odd ? 0x03020706u : 0x05040100u;     // bytes 0-3: own word, 4-7: the partner's
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const Philox4 w = philox7((u32)((j0 + 4 * h) >> 2) + 2 * g + 4 * odd, (u32)i >> 1, bh, d.call, k0, k1);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = __builtin_amdgcn_perm(quad<0xB1>(w.w[e]), w.w[e], sel);
        }
    }
    // low half of x[4 g + e]: group g, high half: group g + 2
    __device__ __forceinline__ bool kept_q(int r) const {
        return r < 8 ? (unsigned short)x[r] >= (unsigned short)thr : x[r - 8] >= thrhi;
    }
    // key on the lane: queries i0 + acc_row(r, h) of key j.  Lane t of the quad makes the counters of query pairs t and t + 4
    // (of the eight pairs its half holds) and takes word t of every counter: a 4 x 4 transpose of words, twice.
    __device__ __forceinline__ void keys(const DropArgs& d, u32 k0, u32 k1, u32 bh, int j, int i0, int h) {
        thr = d.thr;
        thrhi = d.thr << 16;
        const u32 t = (u32)j & 3u;
        const bool o1 = t & 1u, o2 = t & 2u;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            // pair p = 2 g + e: queries i0 + 8 g + 4 h + 2 e and the next; here p = t + 4 c
            const Philox4 w = philox7((u32)j >> 2, (u32)(i0 >> 1) + 8 * c + 4 * (t >> 1) + 2 * h + (t & 1u), bh, d.call, k0, k1);
            // every lane runs every move: a move inside a conditional's arm would read lanes that are switched off
            const u32 n0 = quad<0xB1>(w.w[0]), n1 = quad<0xB1>(w.w[1]), n2 = quad<0xB1>(w.w[2]), n3 = quad<0xB1>(w.w[3]);
            const u32 a0 = o1 ? n1 : w.w[0], a1 = o1 ? w.w[1] : n0, a2 = o1 ? n3 : w.w[2], a3 = o1 ? w.w[3] : n2;
            const u32 m0 = quad<0x4E>(a0), m1 = quad<0x4E>(a1), m2 = quad<0x4E>(a2), m3 = quad<0x4E>(a3);
            x[4 * c] = o2 ? m2 : a0;
            x[4 * c + 1] = o2 ? m3 : a1;
            x[4 * c + 2] = o2 ? a2 : m0;
            x[4 * c + 3] = o2 ? a3 : m1;
        }
    }
    // x[p]: low half query 2 p of the half's, high half the next
    __device__ __forceinline__ bool kept_k(int r) const {
        return r & 1 ? x[r >> 1] >= thrhi : (unsigned short)x[r >> 1] >= (unsigned short)thr;
    }
};

struct Key2 {
    u32 k0 = 0, k1 = 0;
    __device__ __forceinline__ explicit Key2(const DropArgs& d) {
        if (d.thr) {
            const u64 seed = (u64)*d.seed;
            k0 = (u32)__builtin_amdgcn_readfirstlane((int)(u32)seed);         // the round keys made of it stay scalar
            k1 = (u32)__builtin_amdgcn_readfirstlane((int)(u32)(seed >> 32));
        }
    }
};

// the larger one, a NaN if there is one (fmaxf would first quiet both operands, two instructions more)
__device__ __forceinline__ float max_(float x, float y) { return __builtin_elementwise_maximum(x, y); }
// x, made before it is rounded: the compiler otherwise rounds in front of a select, each value for itself (two conversions and
// a permutation for a pair instead of one)
__device__ __forceinline__ float made(float x) {
    asm("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------------ forward
// A workgroup owns 128 queries, a wave 32 (one on each lane of a half), and streams the keys in tiles of 64.
// The running maximum is let stand while no score passes it by more than 2^8 (in base 2 exponents: the sums and the
// probabilities then stay below 2^8 times their final size, harmless in float32 and for bfloat16's relative rounding), so
// that the accumulators are rescaled once or twice a row and not at every tile.
// Bound by the vector unit beside the matrix unit: 2 x 4001 tokens keep a SIMD's vector unit busy 58 % of its cycles (exp2, the
// conversion to bfloat16) and the matrix unit 32 %, one after the other within a wave; packed with dropout 60 % and 15 %.  bfloat16: 2 x 4001 tokens, 12 heads, no dropout 131 us
// = 0.75 PFLOP/s (a large matrix product: 1.15); 128 packed of up to 512 with dropout 124 us, without 91; 16 x 512 ragged 28 us.
// float32, 8 x 512 ragged: 64 us, 57 TFLOP/s on the 32x32x2 products (a large product: 154).
template <typename T, bool DROP, bool HALF>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    constexpr int ROWS = HALF ? OWN / 2 : OWN, NS = HALF ? 1 : 2;   // rows of the workgroup; halves of a tile a wave takes
    __shared__ __attribute__((aligned(16))) char sK[2][X::BYTES];
    __shared__ __attribute__((aligned(16))) char sV[2][X::BYTES];
    const Lane ln;
    const int h = ln.h, l31 = ln.l31, wave = HALF ? ln.wave & 1 : ln.wave, sub0 = HALF ? ln.wave >> 1 : 0;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) return zero_outside<T>(a, blockIdx.x - items, a.o, a.lse);
    const Seq s = find_seq(a, blockIdx.x);
    bool even, flat;
    const int kend = key_end(a, s, even, flat);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    T* O = head_ptr<T>(a, a.o, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    const Key2 key(a.drop);
    const float c2 = fmaxf(fabsf(a.c2), 1e-30f);   // not 0: a left-out key's -inf has to stay one
    for (int q0 = s.blk * ROWS; q0 < s.len; q0 += a.nblk * ROWS) {
        const int i = q0 + wave * 32 + l31;
        float4 qf[X::NF];
        load_own<T>(qf, Q, a.q.st, min(i, s.len - 1), h);
        if (a.c2 < 0.0f) negate<T>(qf);
        if (even) zero_frags<T>(qf);       // and zero keys below: every score is 0
        f32x16 o[2] = {zero16(), zero16()};
        float m = -INFINITY, base = 0.0f, l = 0.0f;   // base: m, or 0 while no score is above -inf
        KeyBits kb(a, s, even);
        Stage<T> rk(K, a.k.st, s.len), rv(V, a.v.st, s.len);
        kb.fetch(0);
        u64 next = kb.bits(0);
        rk.load(even ? 0 : next);
        rv.load(next);
        kb.fetch(TR);
        for (int j0 = 0, buf = 0; j0 < kend; j0 += TR, buf ^= 1) {
            const u64 bits = next;
            rk.store(sK[buf]);
            rv.store(sV[buf]);
            __syncthreads();               // everyone is done with the other buffer, too
            if (j0 + TR < kend) {
                next = kb.bits(j0 + TR);
                rk.load(even ? 0 : next);
                rv.load(next);
                kb.fetch(j0 + 2 * TR);
            }
            if (bits == 0) continue;
            f32x16 sc[NS];
#pragma unroll
            for (int sub = 0; sub < NS; ++sub) sc[sub] = row_product<T>(sK[buf] + (sub0 + sub) * 32 * X::PITCH + ln.frag<T>(), qf);
            if (~bits != 0) {
#pragma unroll
                for (int sub = 0; sub < NS; ++sub) {
                    const u32 kb32 = (u32)(bits >> (32 * (sub0 + sub))) >> (4 * h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[sub][r] = (kb32 >> acc_row(r, 0)) & 1u ? sc[sub][r] : -INFINITY;
                }
            }
            float mx = max_(sc[0][0], sc[NS - 1][0]);
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = max_(max_(sc[0][r], sc[NS - 1][r]), mx);
            mx = max_(mx, __shfl_xor(mx, 32)) * c2;
            // mx > m + 8 or a NaN: move the maximum
            if (__any(!(mx <= m + 8.0f))) {
                const float mnew = max_(m, mx);
                base = mnew == -INFINITY ? 0.0f : mnew;
                const float alpha = exp2_(m - base);
                m = mnew;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
            }
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int sub = 0; sub < NS; ++sub) {
                Draws w;
                if constexpr (DROP) w.queries(a.drop, key.k0, key.k1, bh, i, j0 + 32 * (sub0 + sub), h);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_(fmaf(sc[sub][r], c2, -base));
                    sum[r & 1] += p;                                 // the softmax's sum is over all keys, dropped or not
                    sc[sub][r] = DROP ? made(w.kept_q(r) ? p : 0.0f) : p;
                }
                col_product<T>(o, sV[buf] + (sub0 + sub) * 32 * X::PITCH + ln.col<T>(), sc[sub]);
            }
            l += sum[0] + sum[1];
        }
        if constexpr (HALF) {
            static_assert(2 * 34 * 64 * sizeof(float) <= sizeof(sK));
            const Handover<34> to(sK[0]);
            __syncthreads();               // the last tile is read
            if (sub0) {
                to.put(0, o);
                to.put(32, m);
                to.put(33, l);
            }
            __syncthreads();
            if (!sub0) {
                const float m2 = to.get(32), mnew = max_(m, m2);
                base = mnew == -INFINITY ? 0.0f : mnew;
                const float alpha = exp2_(m - base), beta = exp2_(m2 - base);
                l = l * alpha + to.get(33) * beta;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e >> 4][e & 15] = o[e >> 4][e & 15] * alpha + to.get(e) * beta;
            }
        }
        l += __shfl_xor(l, 32);
        if (i < s.len && (!HALF || !sub0)) {
            store_own<T>(O + (long long)i * a.o.st, o, a.drop.scale / l, h);
            if (h == 0) a.lse[s.stat + i] = (base + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
        }
        __syncthreads();                   // the buffers are free for the next rows
    }
}

// ------------------------------------------------------------------ backward: dQ (and D)
// The forward kernel's walk again: queries on the lanes, dS^T is the right operand of dQ^T = K^T dS^T.  Three products a score
// against the four of attn_dkv_kernel; float32, 8 x 512 ragged, 12 heads: 83 us and 118 us.
template <typename T, bool DROP, bool HALF>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    constexpr int ROWS = HALF ? OWN / 2 : OWN, NS = HALF ? 1 : 2;
    constexpr int UNROLL = DROP ? 2 : 1;      // the draws of one half fill the waits of the other (packed, dropout: 440 -> 416 us)
    __shared__ __attribute__((aligned(16))) char sK[2][X::BYTES];
    __shared__ __attribute__((aligned(16))) char sV[2][X::BYTES];
    const Lane ln;
    const int h = ln.h, l31 = ln.l31, wave = HALF ? ln.wave & 1 : ln.wave, sub0 = HALF ? ln.wave >> 1 : 0;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) return zero_outside<T>(a, blockIdx.x - items, a.dq, nullptr);
    const Seq s = find_seq(a, blockIdx.x);
    bool even, flat;
    const int kend = key_end(a, s, even, flat);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    const T *O = head_ptr<T>(a, a.o, s), *dO = head_ptr<T>(a, a.dout, s);
    T* dQ = head_ptr<T>(a, a.dq, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    const Key2 key(a.drop);
    for (int q0 = s.blk * ROWS; q0 < s.len; q0 += a.nblk * ROWS) {
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
        load_own<T>(qf, Q, a.q.st, ic, h);
        const float lse2 = a.lse[s.stat + ic] * 1.4426950408889634f;
        f32x16 o[2] = {zero16(), zero16()};
        if (!flat) {                                // dS = 0 otherwise, not what is left of P (Z dP - D)
            KeyBits kb(a, s, even);
            Stage<T> rk(K, a.k.st, s.len), rv(V, a.v.st, s.len);
            kb.fetch(0);
            u64 next = kb.bits(0);
            rk.load(next);
            rv.load(next);
            kb.fetch(TR);
            for (int j0 = 0, buf = 0; j0 < kend; j0 += TR, buf ^= 1) {
                const u64 bits = next;
                rk.store(sK[buf]);
                rv.store(sV[buf]);
                __syncthreads();
                if (j0 + TR < kend) {
                    next = kb.bits(j0 + TR);
                    rk.load(next);
                    rv.load(next);
                    kb.fetch(j0 + 2 * TR);
                }
                if (bits == 0) continue;
                // D = sum dO O from the stored O carries O's rounding into every dS of the row.  Of short rows, whose O is not
                // small, that is as much as dS's own rounding (8 keys: dQ off by 2.7e-3 instead of 2.4e-3); where one tile
                // holds all keys D is had without it, as sum_j P_ij Z_ij dP_ij.
                if (sizeof(T) == 2 && kend <= TR) {
                    D = 0.0f;
#pragma unroll 1
                    for (int sub = 0; sub < 2; ++sub) {
                        const f32x16 sc = row_product<T>(sK[buf] + sub * 32 * X::PITCH + ln.frag<T>(), qf);
                        const f32x16 dp = row_product<T>(sV[buf] + sub * 32 * X::PITCH + ln.frag<T>(), df);
                        Draws w;
                        if constexpr (DROP) w.queries(a.drop, key.k0, key.k1, bh, i, j0 + 32 * sub, h);
                        const u32 kb32 = (u32)(bits >> (32 * sub)) >> (4 * h);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const bool counts = ((kb32 >> acc_row(r, 0)) & 1u) && (!DROP || w.kept_q(r));
                            D += counts ? exp2_(fmaf(sc[r], a.c2, -lse2)) * dp[r] * a.drop.scale : 0.0f;
                        }
                    }
                    D += __shfl_xor(D, 32);
                }
#pragma unroll UNROLL
                for (int sub = sub0; sub < sub0 + NS; ++sub) {
                    f32x16 sc = row_product<T>(sK[buf] + sub * 32 * X::PITCH + ln.frag<T>(), qf);
                    const f32x16 dp = row_product<T>(sV[buf] + sub * 32 * X::PITCH + ln.frag<T>(), df);
                    Draws w;
                    if constexpr (DROP) w.queries(a.drop, key.k0, key.k1, bh, i, j0 + 32 * sub, h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = exp2_(fmaf(sc[r], a.c2, -lse2));
                        const float g = !DROP ? dp[r] - D : fmaf(w.kept_q(r) ? dp[r] : 0.0f, a.drop.scale, -D);
                        sc[r] = p * g;
                    }
                    if (~bits != 0) {
                        const u32 kb32 = (u32)(bits >> (32 * sub)) >> (4 * h);
#pragma unroll
                        for (int r = 0; r < 16; ++r) sc[r] = (kb32 >> acc_row(r, 0)) & 1u ? sc[r] : 0.0f;
                    }
                    col_product<T>(o, sK[buf] + sub * 32 * X::PITCH + ln.col<T>(), sc);
                }
            }
            __syncthreads();
        }
        if constexpr (HALF) {
            static_assert(2 * 32 * 64 * sizeof(float) <= sizeof(sK));
            const Handover<32> to(sK[0]);  // free: the walk ended with a barrier
            if (sub0) to.put(0, o);
            __syncthreads();
            if (!sub0) to.add(0, o);
            __syncthreads();
            if (sub0) continue;
        }
        if (i < s.len && h == 0) a.delta[s.stat + i] = D;
        if (i < s.len) store_own<T>(dQ + (long long)i * a.dq.st, o, a.scale, h);
    }
}

// ------------------------------------------------------------------ backward: dK, dV
// A workgroup owns 128 keys, a wave 32 (one on each lane of a half), and streams the queries in tiles of 64.  P and dS are right
// operands as they stand; lse and D of a tile's queries lie in LDS, four of them a read.
template <typename T, bool DROP, bool HALF>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(AttnTrainArgs a) {
    using X = Tile<T>;
    constexpr int ROWS = HALF ? OWN / 2 : OWN, NS = HALF ? 1 : 2;
    constexpr int UNROLL = DROP ? 2 : 1;      // the draws of one half fill the waits of the other (packed, dropout: 440 -> 416 us)
    __shared__ __attribute__((aligned(16))) char sQ[2][X::BYTES];
    __shared__ __attribute__((aligned(16))) char sO[2][X::BYTES];
    __shared__ __attribute__((aligned(16))) float sL[2][TR], sD[2][TR];
    const Lane ln;
    const int h = ln.h, l31 = ln.l31, wave = HALF ? ln.wave & 1 : ln.wave, sub0 = HALF ? ln.wave >> 1 : 0;
    const int items = a.nblk * a.heads * a.B;
    if ((int)blockIdx.x >= items) {
        zero_outside<T>(a, blockIdx.x - items, a.dk, nullptr);
        return zero_outside<T>(a, blockIdx.x - items, a.dv, nullptr);
    }
    const Seq s = find_seq(a, blockIdx.x);
    bool even, flat;
    const int kend = key_end(a, s, even, flat);
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    const T* dO = head_ptr<T>(a, a.dout, s);
    T *dK = head_ptr<T>(a, a.dk, s), *dV = head_ptr<T>(a, a.dv, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    const Key2 key(a.drop);
    for (int n0 = s.blk * ROWS; n0 < s.len; n0 += a.nblk * ROWS) {
        const int j = n0 + wave * 32 + l31, jc = min(j, s.len - 1);
        const bool counts = j < kend && (even || !a.mask || a.mask[(long long)s.b * a.L + jc] != 0);
        f32x16 ok[2] = {zero16(), zero16()}, ov[2] = {zero16(), zero16()};
        if (n0 < kend) {
            float4 kf[X::NF], vf[X::NF];
            load_own<T>(kf, K, a.k.st, jc, h);
            load_own<T>(vf, V, a.v.st, jc, h);
            if (even) zero_frags<T>(kf);       // and zero queries below: every score is 0
            Stage<T> rq(Q, a.q.st, s.len), ro(dO, a.dout.st, s.len);
            float rl, rd;
            int ri;
            auto fetch = [&](int i0) {
                const u64 rows = row_bits(i0, s.len);
                rq.load(even ? 0 : rows);
                ro.load(rows);
                ri = i0 + (int)threadIdx.x % TR;
                rl = a.lse[s.stat + min(ri, s.len - 1)];
                rd = a.delta[s.stat + min(ri, s.len - 1)];
            };
            fetch(0);
            for (int i0 = 0, buf = 0; i0 < s.len; i0 += TR, buf ^= 1) {
                rq.store(sQ[buf]);
                ro.store(sO[buf]);
                if (threadIdx.x < TR) {        // rows past the end: exp2(0 - inf) = 0
                    sL[buf][threadIdx.x] = ri < s.len ? rl * 1.4426950408889634f : INFINITY;
                    sD[buf][threadIdx.x] = ri < s.len ? rd : 0.0f;
                }
                __syncthreads();
                if (i0 + TR < s.len) fetch(i0 + TR);
#pragma unroll UNROLL
                for (int sub = sub0; sub < sub0 + NS; ++sub) {
                    f32x16 sc, dp;
                    row_products<T>(sc, dp, sQ[buf] + sub * 32 * X::PITCH + ln.frag<T>(), kf, sO[buf] + sub * 32 * X::PITCH + ln.frag<T>(), vf);
                    Draws w;
                    if constexpr (DROP) w.keys(a.drop, key.k0, key.k1, bh, j, i0 + 32 * sub, h);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 L4 = *reinterpret_cast<const float4*>(&sL[buf][sub * 32 + 8 * g + 4 * h]);
                        const float4 D4 = *reinterpret_cast<const float4*>(&sD[buf][sub * 32 + 8 * g + 4 * h]);
                        const float lv[4] = {L4.x, L4.y, L4.z, L4.w}, dv[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = 4 * g + e;
                            const float p = exp2_(fmaf(sc[r], a.c2, -lv[e]));
                            const bool kept = !DROP || w.kept_k(r);
                            const float gr = !DROP ? dp[r] - dv[e] : fmaf(kept ? dp[r] : 0.0f, a.drop.scale, -dv[e]);
                            sc[r] = DROP ? made(kept ? p : 0.0f) : p;
                            dp[r] = p * gr;
                        }
                    }
                    col_product<T>(ov, sO[buf] + sub * 32 * X::PITCH + ln.col<T>(), sc);
                    col_product<T>(ok, sQ[buf] + sub * 32 * X::PITCH + ln.col<T>(), dp);
                }
            }
            __syncthreads();
        }
        if constexpr (HALF) {
            static_assert(2 * 32 * 64 * sizeof(float) <= sizeof(sQ));
            const Handover<32> tk(sQ[0]), tv(sO[0]);   // free: the walk ended with a barrier
            if (sub0) {
                tk.put(0, ok);
                tv.put(0, ov);
            }
            __syncthreads();
            if (!sub0) {
                tk.add(0, ok);
                tv.add(0, ov);
            }
            __syncthreads();
            if (sub0) continue;
        }
        // a key's gradients are sums in its own lanes: what a key that does not count gathered is dropped here
        if (!counts || flat) {
            ok[0] = ok[1] = zero16();
            if (!counts) ov[0] = ov[1] = zero16();
        }
        if (j < s.len) {
            store_own<T>(dK + (long long)j * a.dk.st, ok, a.scale, h);
            store_own<T>(dV + (long long)j * a.dv.st, ov, a.drop.scale, h);
        }
    }
}

// ------------------------------------------------------------------ backward in one pass
// bfloat16.  A workgroup of 8 waves owns a (sequence, head); it takes its keys 256 at a time, a wave 32 (one on each lane of a
// half), and streams the queries in tiles of 32.  Every score tile is made ONCE: probabilities and dS go from the registers
// into dV and dK as in attn_dkv_kernel, dS also goes to LDS (64 bytes a key), from where all waves together make the tile's
// dQ, a block of 16 queries x 16 elements each, K read transposed from LDS.  dQ of more than 256 keys is
// carried in a float32 buffer that the same thread writes and reads.  One barrier a tile; D comes out of the staging.
// Bound by the workgroup that a CU holds (93 KB of LDS): eight waves that meet at a barrier for every tile, 2.6 to 3.4 us a tile of
// 32 x 256, whose five products take 1.2 us at a large matrix product's rate.  128 packed sequences of up to 512, 12 heads, dropout: 318
// to 365 us by the order of their lengths (0.26 PFLOP/s), without dropout 285; of a SIMD's cycles the matrix unit is busy 14 %, the
// vector unit 32 %, neither for the rest.  Tiles of 64 queries, half the barriers, measured
// no better (337 us), nor did orders of the instructions pinned by hand.
// SHORT: batches of short sequences, see D below (in a batch of long ones it would cost 64 x 200 tokens 70 -> 96 us).
constexpr int FK = 256, FQ = 32;      // keys at a time, rows of a streamed tile
constexpr int SPITCH = FQ * 2 + 8;    // bytes a key of dS^T in LDS

__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

template <int CTRL>
__device__ __forceinline__ float dppf(float x) {
    return __uint_as_float(quad<CTRL>(__float_as_uint(x)));
}

// The sums of sixteen values over the 32 lanes of a half, one a lane: lane l gets that of value lane_value(l).  A step halves the
// values and the lanes that hold each (15 moves and one shuffle; a butterfly for every value took 64 and 16).
__device__ __forceinline__ int lane_value(int l31) { return (l31 & 1) * 8 + (l31 >> 1 & 1) * 4 + (l31 >> 2 & 1) * 2 + (l31 >> 3 & 1); }
__device__ __forceinline__ float lane_sums(float (&v)[16], int l31) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float keep = l31 & 1 ? v[8 + k] : v[k], give = l31 & 1 ? v[k] : v[8 + k];
        v[k] = keep + dppf<0xB1>(give);                 // lane ^ 1
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float keep = l31 & 2 ? v[4 + k] : v[k], give = l31 & 2 ? v[k] : v[4 + k];
        v[k] = keep + dppf<0x4E>(give);                 // lane ^ 2
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float keep = l31 & 4 ? v[2 + k] : v[k], give = l31 & 4 ? v[k] : v[2 + k];
        v[k] = keep + dppf<0x141>(dppf<0x1B>(give));    // lane ^ 7 of lane ^ 3
    }
    const float keep = l31 & 8 ? v[1] : v[0], give = l31 & 8 ? v[0] : v[1];
    const float x = keep + dppf<0x128>(give);           // lane ^ 8
    return x + __shfl_xor(x, 16);
}

template <bool DROP, bool SHORT>
__global__ __launch_bounds__(512, 2) void attn_bwd_kernel(AttnTrainArgs a) {
    typedef bf16_t T;
    using X = Tile<T>;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) char sQ[2][FQ * X::PITCH];
    __shared__ __attribute__((aligned(16))) char sO[2][FQ * X::PITCH];
    __shared__ __attribute__((aligned(16))) char sS[2][FK * SPITCH];        // dS^T of a tile, two of them in turn
    __shared__ __attribute__((aligned(16))) float sL[2][FQ], sD[2][FQ];
    __shared__ __attribute__((aligned(16))) char sK[FK * X::PITCH];
    __shared__ float sE[SHORT ? 2 : 1][FQ];
    const Lane ln;
    const int lane = ln.lane, wave = ln.wave, h = ln.h, l31 = ln.l31, tid = threadIdx.x;
    const int items = a.heads * a.B;
    if ((int)blockIdx.x >= items) {
        zero_outside<T>(a, blockIdx.x - items, a.dq, nullptr);
        zero_outside<T>(a, blockIdx.x - items, a.dk, nullptr);
        return zero_outside<T>(a, blockIdx.x - items, a.dv, nullptr);
    }
    // nothing is shared between workgroups here: an XCD takes the heads of a sequence together (packed, 128 sequences: 323 us,
    // 366 with the pairs going round)
    const Seq s = find_seq(a, blockIdx.x, xcd_remap(blockIdx.x, items));
    if (s.len == 0) return;
    const T *Q = head_ptr<T>(a, a.q, s), *K = head_ptr<T>(a, a.k, s), *V = head_ptr<T>(a, a.v, s);
    const T *O = head_ptr<T>(a, a.o, s), *dO = head_ptr<T>(a, a.dout, s);
    // the first keys are on their way before the mask is looked at, and the first queries before the keys are stored
    float4 kf[X::NF], vf[X::NF];
    load_own<T>(kf, K, a.k.st, min(wave * 32 + l31, s.len - 1), h);
    load_own<T>(vf, V, a.v.st, min(wave * 32 + l31, s.len - 1), h);
    bool even, flat;
    const int kend = key_end(a, s, even, flat);
    T *dQ = head_ptr<T>(a, a.dq, s), *dK = head_ptr<T>(a, a.dk, s), *dV = head_ptr<T>(a, a.dv, s);
    const u32 bh = (u32)(s.b * a.heads + s.h);
    const Key2 key(a.drop);
    const long long* mask = a.mask && !even ? a.mask + (long long)s.b * a.L : nullptr;
    // staging: threads 0-255 a chunk of Q, 256-511 the same chunk of dO and of O (their product is D)
    const int sr = (tid & 255) >> 3, sc8 = tid & 7;
    const bool isq = tid < 256;
    const T* src = (isq ? Q : dO) + sc8 * X::EPC;
    const long long sst = isq ? a.q.st : a.dout.st;
    // dQ: this wave's block, this lane's query and four elements
    const int dcol = 16 * (wave & 3), qhalf = 16 * (wave >> 2), g4 = lane >> 4, i16 = lane & 15;
    const long long prow = (a.cu ? s.row0 : (long long)s.b * a.L);

    for (int n0 = 0; n0 < s.len; n0 += FK) {
        const int nk = min(FK, kend - n0);                 // keys that may count here
        const int j = n0 + wave * 32 + l31, jc = min(j, s.len - 1);
        bool counts = j < kend;
        if (mask) counts &= mask[jc] != 0;
        const bool all = __all(counts);
        f32x16 ok[2] = {zero16(), zero16()}, ov[2] = {zero16(), zero16()};
        if (nk > 0) {
            const bool first = n0 == 0, last = n0 + FK >= kend, busy = wave * 32 < nk;
            if (!first) {
                load_own<T>(kf, K, a.k.st, jc, h);
                load_own<T>(vf, V, a.v.st, jc, h);
            }
            if (even) zero_frags<T>(kf);
            float4 rv, ro = make_float4(0.f, 0.f, 0.f, 0.f);
            float rl = 0.0f;
            auto fetch = [&](int i0) {
                const long long row = min(i0 + sr, s.len - 1);
                rv = *reinterpret_cast<const float4*>(src + row * sst);
                if (!isq) ro = *reinterpret_cast<const float4*>(O + row * a.o.st + sc8 * X::EPC);
                rl = a.lse[s.stat + min(i0 + (tid & (FQ - 1)), s.len - 1)];
            };
            auto store = [&](int i0, int buf) {
                const bool in = i0 + sr < s.len;
                if (!in || (even && isq)) rv = make_float4(0.f, 0.f, 0.f, 0.f);
                *reinterpret_cast<float4*>((isq ? sQ[buf] : sO[buf]) + sr * X::PITCH + sc8 * 16) = rv;
                if (!isq) {
                    const T *x = reinterpret_cast<const T*>(&rv), *y = reinterpret_cast<const T*>(&ro);
                    float d = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d += to_f<T>(x[e]) * to_f<T>(y[e]);
                    d += dppf<0xB1>(d);
                    d += dppf<0x4E>(d);
                    d += dppf<0x141>(d);
                    if (sc8 == 0) sD[buf][sr] = in ? d : 0.0f;
                }
                // rows past the end: exp2(0 - inf) = 0
                if (tid < FQ) sL[buf][tid] = i0 + tid < s.len ? rl * 1.4426950408889634f : INFINITY;
            };
            fetch(0);
            __syncthreads();                               // the keys before these are done with
            float4 kt[4];
            bool kc[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int jj = n0 + e * 64 + (tid >> 3), jr = min(jj, s.len - 1);
                kt[e] = *reinterpret_cast<const float4*>(K + (long long)jr * a.k.st + sc8 * X::EPC);
                kc[e] = !even && jj < kend;
                if (mask) kc[e] &= mask[jr] != 0;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4*>(sK + (e * 64 + (tid >> 3)) * X::PITCH + sc8 * 16) = kc[e] ? kt[e] : make_float4(0.f, 0.f, 0.f, 0.f);
            __syncthreads();
            store(0, 0);
            if (FQ < s.len) fetch(FQ);
            __syncthreads();                               // K and tile 0 are there
            if (!busy)                                     // keys nobody has: their dS is zero once and for all
                for (int e = lane; e < 32 * SPITCH / 4; e += 64) {
                    reinterpret_cast<u32*>(sS[0] + wave * 32 * SPITCH)[e] = 0;
                    reinterpret_cast<u32*>(sS[1] + wave * 32 * SPITCH)[e] = 0;
                }
            for (int i0 = 0, buf = 0; i0 < s.len; i0 += FQ, buf ^= 1) {
                const int qi = i0 + qhalf + i16;
                float* part = a.delta + ((prow + min(qi, s.len - 1)) * a.heads + s.h) * DH + dcol + 4 * g4;
                f32x4 dq = {0.f, 0.f, 0.f, 0.f};
                if (!first) dq = *reinterpret_cast<const f32x4*>(part);
                if (SHORT && kend <= 2 * 32 && !even) {    // D of short rows without O's rounding, as in attn_dq_kernel
                    if (busy) {
                        f32x16 sc, dp;
                        row_products<T>(sc, dp, sQ[buf] + ln.frag<T>(), kf, sO[buf] + ln.frag<T>(), vf);
                        Draws w;
                        if constexpr (DROP) w.keys(a.drop, key.k0, key.k1, bh, j, i0, h);
                        float e[16];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float4 L4 = *reinterpret_cast<const float4*>(&sL[buf][8 * g + 4 * h]);
                            const float lv[4] = {L4.x, L4.y, L4.z, L4.w};
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const int r = 4 * g + t;
                                e[r] = counts && (!DROP || w.kept_k(r)) ? exp2_(fmaf(sc[r], a.c2, -lv[t])) * dp[r] * a.drop.scale : 0.0f;
                            }
                        }
                        const float d = lane_sums(e, l31);
                        if (l31 < 16) sE[wave & (SHORT ? 1 : 0)][acc_row(lane_value(l31), h)] = d;
                    }
                    __syncthreads();
                    if (tid < FQ) sD[buf][tid] = sE[0][tid] + (kend > 32 ? sE[SHORT ? 1 : 0][tid] : 0.0f);
                    __syncthreads();
                }
                if (busy) {
                    f32x16 sc, dp;
                    row_products<T>(sc, dp, sQ[buf] + ln.frag<T>(), kf, sO[buf] + ln.frag<T>(), vf);
                    Draws w;
                    if constexpr (DROP) w.keys(a.drop, key.k0, key.k1, bh, j, i0, h);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 L4 = *reinterpret_cast<const float4*>(&sL[buf][8 * g + 4 * h]);
                        const float4 D4 = *reinterpret_cast<const float4*>(&sD[buf][8 * g + 4 * h]);
                        const float lv[4] = {L4.x, L4.y, L4.z, L4.w}, dv[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = 4 * g + e;
                            const float p = exp2_(fmaf(sc[r], a.c2, -lv[e]));
                            const bool kept = !DROP || w.kept_k(r);
                            const float gr = !DROP ? dp[r] - dv[e] : fmaf(kept ? dp[r] : 0.0f, a.drop.scale, -dv[e]);
                            sc[r] = DROP ? made(kept ? p : 0.0f) : p;
                            dp[r] = p * gr;
                        }
                    }
                    if (!all || flat) {                    // what a key that does not count adds to dQ
#pragma unroll
                        for (int r = 0; r < 16; ++r) dp[r] = counts && !flat ? dp[r] : 0.0f;
                    }
                    bf16x8 ds[2];
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r >> 3][r & 7] = (__bf16)dp[r];
                    char* d = sS[buf] + (wave * 32 + l31) * SPITCH + 8 * h;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        typedef short s16x4a __attribute__((ext_vector_type(4)));
                        const s16x4a v = reinterpret_cast<const s16x4a*>(&ds[g >> 1])[g & 1];
                        *reinterpret_cast<s16x4a*>(d + 16 * g) = v;
                    }
                    col_product<T>(ov, sO[buf] + ln.col<T>(), sc);
                    col_product_b(ok, sQ[buf] + ln.col<T>(), ds);
                }
                if (i0 + FQ < s.len) {
                    store(i0 + FQ, buf ^ 1);
                    if (i0 + 2 * FQ < s.len) fetch(i0 + 2 * FQ);
                }
                __syncthreads();
                f32x4 dq2 = {0.f, 0.f, 0.f, 0.f};
                const char* ps = sS[buf] + (8 * g4 + (i16 >> 2)) * SPITCH + (qhalf + 4 * (i16 & 3)) * 2;
                const char* pk = sK + (8 * g4 + (i16 >> 2)) * X::PITCH + (dcol + 4 * (i16 & 3)) * 2;
#pragma unroll
                for (int k4 = 0; k4 < 8; k4 += 4) {
                    s16x4 sb[4][2], kt[4][2];
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            sb[ks][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)(ps + (32 * (k4 + ks) + 4 * e) * SPITCH));
                            kt[ks][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((OTTER_AS3 s16x4*)(pk + (32 * (k4 + ks) + 4 * e) * X::PITCH));
                        }
                    pin();
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        f32x4& acc = ks & 1 ? dq2 : dq;
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kt[ks]), __builtin_bit_cast(bf16x8, sb[ks]), acc, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) dq[e] += dq2[e];
                if (qi < s.len) {
                    if (last) {
                        const u32 w0 = (u32)f2bf(dq[0] * a.scale) | ((u32)f2bf(dq[1] * a.scale) << 16);
                        const u32 w1 = (u32)f2bf(dq[2] * a.scale) | ((u32)f2bf(dq[3] * a.scale) << 16);
                        *reinterpret_cast<uint2*>(dQ + (long long)qi * a.dq.st + dcol + 4 * g4) = make_uint2(w0, w1);
                    } else {
                        *reinterpret_cast<f32x4*>(part) = dq;
                    }
                }
            }
        }
        if (!counts || flat) {
            ok[0] = ok[1] = zero16();
            if (!counts) ov[0] = ov[1] = zero16();
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
    a->nblk = x->tokens > OWN ? (x->tokens + OWN - 1) / OWN : 1;     // own_half() may double it
    // Pairs one by one or eight at a time (find_seq), us, lengths from an eighth on, forward / two-pass backward.  Packed bfloat16:
    // two workgroups a pair 256 x 256 92 / 295 -> 81 / 263, four 128 x 512 134 / 420 -> 117 / 364, 64 x 512 with 8 heads 54 / 148 -> 48 / 137;
    // but three 170 x 384 100 / 306 -> 106 / 321, five 102 x 640 137 / 398 -> 151 / 449, eight 20 x 1024 77 / 200 -> 80 / 215, sixteen 16 x
    // 2048 188 / 496 -> 244 / 656.  float32, four: packed 128 x 512 622 / 1974 -> 550 / 1723, with a mask 642 / 2520 -> 675 / 2178
    a->group = a->nblk == 2 || a->nblk == 4 ? 8 : 1;
    // how many rows are of no sequence only the GPU knows: as many workgroups as all of them could keep busy (32 KB each)
    const long long most = x->total * x->heads * DH * (x->dtype == OTTER_BF16 ? 2 : 4) >> 15;
    a->outside = x->cu_seqlens ? (int)(most < 1 ? 1 : most < OUTSIDE ? most : OUTSIDE) : 0;
    *rows = x->cu_seqlens ? x->total : (long long)x->batch * x->tokens;
    // a launch has fewer than 2^32 threads: 256 an item, 512 where the backward pass takes a pair of two items and more at once
    if ((long long)a->B * a->heads > 0xFFFFFF || (long long)a->nblk * a->heads * a->B + (x->cu_seqlens ? 2 * OUTSIDE : 0) > 0xFFFFFF)
        return set_err(OTTER_EINVAL, "%s: batch x heads x tokens is too large for one launch", what);
    return OTTER_OK;
}

// Two waves share their rows (HALF): twice the workgroups, each half as long, for twice the staging of tiles.  Sequences of up
// to 64 rows leave no wave idle that way and stage no more (64 x 64 tokens, 12 heads, float32: 22.8 -> 17.7 us forward, 75 -> 59
// backward).  Longer ones take it where there are few workgroups; us forward / backward in two passes, 12 heads, dropout, no mask:
//   bfloat16  192 workgroups (1 x 2048) 50 / 117 -> 46 / 108, 288 (6 x 512) 23 / 57 -> 21 / 57, 384 (8 x 512) 23.5 / 57.6 -> 21.3 / 57.4,
//             4 x 1024 40 / 95 -> 35 / 94, 2 x 2048 72 / 171 -> 64 / 161; but 396 (11 x 300) 16.7 / 41 -> 15.2 / 45, 432 (9 x 512)
//             23.6 / 58 -> 26.4 / 68, 480 (5 x 1024) 41 / 98 -> 45 / 114
//   float32   288 (6 x 512) 82 / 257 -> 73 / 212, 384 (8 x 512) 83 / 258 -> 75 / 214, 4 x 1024 157 / 491 -> 136 / 400; 432 (12 x 300) 56 / 171 ->
//             49 / 143 but 9 x 512 82 / 260 -> 91 / 274, 504 (14 x 300) 57 / 174 -> 62 / 181
// Between 65 and 128 rows it gains nothing (16 x 128 float32 15.8 / 50 -> 16.7 / 52).
bool own_half(AttnTrainArgs& a) {
    if (a.L > OWN / 2 && (a.L <= OWN || (long long)a.nblk * a.heads * a.B > CUS * 3 / 2)) return false;
    a.nblk = a.L > OWN / 2 ? (a.L + OWN / 2 - 1) / (OWN / 2) : 1;
    a.group = 1;      // eight pairs at a time, packed: float32 8 x 512 51 / 150 -> 62 / 187, 2 x 1024 59 / 169 -> 86 / 266, bfloat16 8 x 512 18 / 47 -> 18 / 49
    return true;
}

int grid_of(const AttnTrainArgs& a) { return a.nblk * a.heads * a.B + a.outside; }

template <typename T, bool DROP>
void launch_fwd(AttnTrainArgs& a, hipStream_t st) {
    if (own_half(a))
        attn_fwd_kernel<T, DROP, true><<<grid_of(a), 256, 0, st>>>(a);
    else
        attn_fwd_kernel<T, DROP, false><<<grid_of(a), 256, 0, st>>>(a);
}

// One pass over the scores (bfloat16) or two, one for dQ and one for dK and dV.  One pass makes each score tile once and is one
// launch, but it is one workgroup a (sequence, head) of which a CU holds one, it needs FK keys to fill its waves, and a long
// sequence among short ones keeps one CU busy when the others are done: how full a batch is, rows over batch x longest, decides with
// the number of rounds of workgroups.  The host knows it of a packed batch and of a dense one without a mask; dense ones with
// a mask count as ragged.  Measured (kernels alone, us, one pass and two, 12 heads, dropout; ragged: lengths from an eighth on):
//   up to OWN tokens  16 x 70: 15 and 18, 21 x 128: 16.4 and 21, ragged 20.5 and 21.7; 32 x 70: 20.5 and 23, ragged 28 and 24, 32 x 33: 19
//                     and 17 -> while the CUs hold all pairs
//   up to FK          16 x 200: 25 and 41, 64 x 200: 73 and 97, ragged 72 and 87, 6 x 200: 23 and 26, ragged 24 and 25; 4 x 256: 26 and
//                     20, 4 x 129: 17 and 17 -> beyond a quarter of the CUs
//   up to 2 FK        full: 10 x 512 81 and 63, 12 x 512 81 and 85, 20 x 512 89 and 109, 14 x 300 47 and 46, 16 x 300 48 and 57 -> when
//   (one round)       two passes no longer hold all their workgroups at once; with a mask 13 x 512 82 and 79, 14 x 512 83 and 85, 20 x
//                     512 84 and 98, 14 x 300 49 and 44, 18 x 300 50 and 53 -> from three quarters of the CUs on; packed ragged 16 x
//                     512 80 and 80, 20 x 300 46 and 42 -> two passes
//   (more rounds)     22 x 512 159 and 132, 32 x 512 163 and 163, 36 x 512 170 and 181, ragged 161 and 157, 42 x 512 181 and 210, ragged
//                     170 and 174, packed 151 and 140, 128 packed 318 and 379 -> where the last round is not mostly empty
//   longer            full: 21 x 700 169 and 211, 40 x 1500 1307 and 1447, 64 x 2000 3675 and 3998; 16 x 1500 615 and 578; beyond 8 FK the
//                     carried dQ, 64 times the workspace, brings no more: 64 x 3000 8695 and 8766, 21 x 4096 5255 and 5298; with a mask 40 x 700
//                     305 and 279, 40 x 1500 1219 and 995, 64 x 700 413 and 450, 64 x 1000 738 and 793, 64 x 1500 1555 and 1554, 64 x 2000 2858
//                     and 2574 -> full ones where the last round is not mostly empty, with a mask from three rounds on and
//                     up to 6 FK; packed by how full, 40 x 700: 0.70 299 and 253, 0.80 303 and 297, 0.90 313 and 349; 64 x 1000: 0.56 601
//                     and 577, 0.70 674 and 729; 64 x 1500: 0.56 1274 and 1102, 0.70 1441 and 1446, 0.80 1632 and 1744
// Several workgroups a pair, whose parts of dQ another launch adds up, did not help (16 x 512: 97).
bool one_pass(const AttnTrainArgs& a, int dtype) {
    const long long pairs = (long long)a.B * a.heads, rounds = (pairs + CUS - 1) / CUS;
    if (dtype != OTTER_BF16) return false;
    if (a.L <= OWN) return pairs <= CUS;
    if (a.L <= FK) return pairs > CUS / 4;
    const bool last = 5 * pairs >= 4 * rounds * CUS;           // the last round is not mostly empty
    const bool full = a.cu ? 15 * a.T >= (rounds >= 3 ? 10 : 12) * (long long)a.B * a.L : !a.mask;
    if (a.L > 2 * FK) return last && (full ? a.L <= 8 * FK : !a.cu && rounds >= 3 && a.L <= 6 * FK);
    if (rounds > 1) return last;
    return full ? a.nblk * pairs > 2 * CUS : !a.cu && 4 * pairs >= 3 * CUS;
}

template <bool DROP>
void launch_one_pass(const AttnTrainArgs& a, hipStream_t st) {
    if (a.L <= OWN)
        attn_bwd_kernel<DROP, true><<<grid_of(a), 512, 0, st>>>(a);
    else
        attn_bwd_kernel<DROP, false><<<grid_of(a), 512, 0, st>>>(a);
}

template <typename T, bool DROP>
void launch_bwd(AttnTrainArgs& a, hipStream_t st) {
    if (own_half(a)) {
        attn_dq_kernel<T, DROP, true><<<grid_of(a), 256, 0, st>>>(a);
        attn_dkv_kernel<T, DROP, true><<<grid_of(a), 256, 0, st>>>(a);
    } else {
        attn_dq_kernel<T, DROP, false><<<grid_of(a), 256, 0, st>>>(a);
        attn_dkv_kernel<T, DROP, false><<<grid_of(a), 256, 0, st>>>(a);
    }
}

// D of every row and head; in one pass the float32 dQ of sequences of more than FK keys (packed ones may be longer than `tokens`)
int64_t backward_bytes(const AttnTrainArgs& a, int dtype, long long rows) {
    const int64_t n = rows * a.heads * (int64_t)sizeof(float);
    return one_pass(a, dtype) ? (a.cu || a.L > FK ? n * DH : 0) : n;
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
    hipStream_t st = (hipStream_t)stream;
    if (size == 2)
        a.drop.thr ? launch_fwd<bf16_t, true>(a, st) : launch_fwd<bf16_t, false>(a, st);
    else
        a.drop.thr ? launch_fwd<float, true>(a, st) : launch_fwd<float, false>(a, st);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

int64_t otter_attention_backward_workspace(const otter_attention_args* x) {
    AttnTrainArgs a = {};
    long long rows = 0;
    int rc = fill("attention_backward_workspace", x, &a, &rows);
    if (rc) return rc;
    return backward_bytes(a, x->dtype, rows);
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
    if (!a.lse) return set_err(OTTER_EINVAL, "attention_backward: NULL lse");
    const int64_t need = backward_bytes(a, x->dtype, rows);
    if (need > 0 && (!x->workspace || x->workspace_bytes < need || ((uintptr_t)x->workspace & 15)))
        return set_err(OTTER_EINVAL, "attention_backward: workspace of %lld bytes, needs %lld, 16-byte aligned",
                       (long long)x->workspace_bytes, (long long)need);
    a.delta = (float*)x->workspace;
    DeviceGuard g(device);
    if (!g.ok) return set_err(OTTER_EHIP, "attention_backward: hipSetDevice(%d) failed", device);
    hipStream_t st = (hipStream_t)stream;
    if (one_pass(a, x->dtype)) {
        a.nblk = 1;
        a.drop.thr ? launch_one_pass<true>(a, st) : launch_one_pass<false>(a, st);
        OTTER_HIP_TRY(hipGetLastError());
        return OTTER_OK;
    }
    if (size == 2)
        a.drop.thr ? launch_bwd<bf16_t, true>(a, st) : launch_bwd<bf16_t, false>(a, st);
    else
        a.drop.thr ? launch_bwd<float, true>(a, st) : launch_bwd<float, false>(a, st);
    OTTER_HIP_TRY(hipGetLastError());
    return OTTER_OK;
}

}  // extern "C"
