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

    // exp2 of a difference to a running reference: the hardware instruction (1 ulp), arguments up to 16 or NaN.
    // Below -126 it gives 0 for what would be subnormal: weights under 2^-126, where the largest is 2^-1 or more.
    __device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

    // Sums over the lanes up to each, and over all 64 (row shifts within 16 lanes, then the rows' last lanes).
    template <int CTRL, int ROWS>
    __device__ __forceinline__ int dpp_add_int(int x) {
        return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
    }
    __device__ __forceinline__ int wave_prefix_sum(int x) {
        x = dpp_add_int<0x111, 0xF>(x); // row_shr 1, 2, 4, 8
        x = dpp_add_int<0x112, 0xF>(x);
        x = dpp_add_int<0x114, 0xF>(x);
        x = dpp_add_int<0x118, 0xF>(x);
        x = dpp_add_int<0x142, 0xA>(x); // row_bcast 15 into rows 1 and 3
        return dpp_add_int<0x143, 0xC>(x); // row_bcast 31 into rows 2 and 3
    }
    __device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_prefix_sum(x), 63); }

    struct SeqTile {
        int b, tile; // b = -1: past the last one
    };
    // Work items are numbered sequence by sequence, count(b) of them for sequence b. Every wave finds its own by a
    // prefix sum over its lanes, a sequence each or, past 64, four neighbouring ones; the result is the same in
    // every lane.
    template <typename Count>
    __device__ __forceinline__ SeqTile find_tile(int item, int batch, Count count) {
        const int lane = threadIdx.x & 63;
        if (batch <= 64) {
            const int      n = lane < batch ? max(0, count(lane)) : 0, incl = wave_prefix_sum(n);
            const uint64_t hit = __ballot(item < incl);
            if (!hit) return {-1, 0};
            const int first = __ffsll((unsigned long long) hit) - 1;
            return {first, item - __builtin_amdgcn_readlane(incl - n, first)};
        }
        for (int b0 = 0; b0 < batch; b0 += 256) {
            int n[4], all = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = b0 + lane * 4 + i;
                n[i]        = b < batch ? max(0, count(b)) : 0;
                all += n[i];
            }
            const int      incl = wave_prefix_sum(all);
            const uint64_t hit = __ballot(item < incl);
            if (hit) {
                const int first = __ffsll((unsigned long long) hit) - 1;
                item -= __builtin_amdgcn_readlane(incl - all, first);
                int i = 0;
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const int c = __builtin_amdgcn_readlane(n[k], first);
                    if (i == k && item >= c) item -= c, ++i;
                }
                return {b0 + first * 4 + i, item};
            }
            item -= __builtin_amdgcn_readlane(incl, 63);
        }
        return {-1, 0};
    }
    // The same for up to 64 sequences with their last tiles first: all sequences' tiles are numbered by falling tile
    // index, sequences of the same index in order. C(t) = sum max(0, count - t) items have an index of t or more.
    // Sequences of equal counts go one after the other, so that neighbouring items share a sequence.
    template <typename Count>
    __device__ __forceinline__ SeqTile find_tile_falling(int item, int batch, Count count) {
        const int lane = threadIdx.x & 63, n = lane < batch ? max(0, count(lane)) : 0;
        if (item >= wave_total(n)) return {-1, 0};
        const int n0 = __builtin_amdgcn_readfirstlane(n);
        if (!__any(lane < batch && n != n0)) return {item / n0, n0 - 1 - item % n0};
        int lo = 0, hi = n; // item < C(lo), item >= C(hi)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) hi = max(hi, __shfl_xor(hi, o));
        hi = __builtin_amdgcn_readfirstlane(hi);
        while (hi - lo > 1) {
            const int t = (lo + hi) / 2;
            if (item < wave_total(max(0, n - t))) lo = t;
            else hi = t;
        }
        const uint64_t there = __ballot(n > lo);
        const int      rank = item - wave_total(max(0, n - hi)); // among the sequences that have this index
        const int      before = __builtin_amdgcn_mbcnt_hi((unsigned) (there >> 32), __builtin_amdgcn_mbcnt_lo((unsigned) there, 0));
        const uint64_t mine = __ballot((there >> lane & 1) && before == rank);
        return {__ffsll((unsigned long long) mine) - 1, lo};
    }

    __device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

    // Whether an output's first two rows or heads of `dim` values share memory (strides in elements).
    inline bool rows_overlap(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t dim) {
        return (rows > 1 && row < dim) || (heads > 1 && head < dim) || (rows > 1 && heads > 1 && row - head < dim && head - row < dim);
    }

    inline bool misaligned16(const void *p) { return ((uintptr_t) p) % 16 != 0; }

} // namespace vkhip
