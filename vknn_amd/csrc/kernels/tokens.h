// Shared by the token operators (group norm, packed attention, the 8-bit cache): element types,
// 16-byte rows, and the search for the sequence that a work item belongs to.
#pragma once
#include "common.h"

namespace vkhip {

    typedef __bf16   bf16_t;
    typedef __bf16   bf8 __attribute__((ext_vector_type(8)));
    typedef __bf16   bf4 __attribute__((ext_vector_type(4)));
    typedef uint32_t tk_u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t tk_u32x4 __attribute__((ext_vector_type(4)));

    // exp2 of a difference to a running maximum: the hardware instruction (1 ulp), arguments <= 0 or NaN.
    // Below -126 it gives 0 for what would be subnormal: weights under 2^-126 of the largest one.
    __device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

    struct SeqTile {
        int b, tile; // b = -1: past the last one
    };
    // Work items are numbered sequence by sequence, count(b) of them for sequence b. Every wave finds its
    // own by a prefix sum over 64 sequences at a time; the result is the same in every lane.
    template <typename Count>
    __device__ __forceinline__ SeqTile find_tile(int item, int batch, Count count) {
        const int lane = threadIdx.x & 63;
        for (int b0 = 0; b0 < batch; b0 += 64) {
            const int b = b0 + lane, n = b < batch ? count(b) : 0;
            int       incl = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int t = __shfl_up(incl, o);
                if (lane >= o) incl += t;
            }
            const uint64_t hit = __ballot(item < incl);
            if (hit) {
                const int first = __ffsll((unsigned long long) hit) - 1;
                return {b0 + first, item - __builtin_amdgcn_readlane(incl - n, first)};
            }
            item -= __builtin_amdgcn_readlane(incl, 63);
        }
        return {-1, 0};
    }

    __device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

    inline bool misaligned16(const void *p) { return ((uintptr_t) p) % 16 != 0; }

} // namespace vkhip
