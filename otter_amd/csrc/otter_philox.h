// otter_philox.h — the counter-based random numbers of the training operators.
#pragma once
#include "otter_device.h"

namespace otter {

// Philox4x32 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): 4 words of
// output for a 4-word counter under a 64-bit key; a round is two 32 x 32 -> 64 bit products.  Seven rounds, the fewest the
// paper lists as passing its statistical tests (ten, its default, cost 43 % more of what bounds the attention kernels).
// One call makes EIGHT draws of 16 bits, low half of a word first: a probability is then a multiple of 2^-16, which the
// scale 65536 / (65536 - T) accounts for exactly.
//   rows (dropout, layer norm):  counter (col >> 3, row, 0xFFFFFFFF, call); draw of col: word (col & 7) >> 1, half col & 1
//   attention:                   counter (j >> 2, i >> 1, b * heads + h, call); draw of query i, key j: word j & 3, half i & 1
struct Philox4 {
    u32 w[4];
};

__device__ __forceinline__ u32 xor3(u32 a, u32 b, u32 c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

__device__ __forceinline__ Philox4 philox7(u32 c0, u32 c1, u32 c2, u32 c3, u32 k0, u32 k1) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const u64 p0 = (u64)c0 * 0xD2511F53u, p1 = (u64)c2 * 0xCD9E8D57u;
        c0 = xor3((u32)(p1 >> 32), c1, k0);
        c1 = (u32)p1;
        c2 = xor3((u32)(p0 >> 32), c3, k1);
        c3 = (u32)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Philox4{{c0, c1, c2, c3}};
}

// a value is dropped where its 16-bit draw is below `thr`; thr = 0: nothing is dropped and no number is drawn
struct DropArgs {
    u32 thr = 0;
    u32 call = 0;
    float scale = 1.0f;
    const long long* seed = nullptr;   // device: the 64-bit key
};

}  // namespace otter
