// Attention over the 8-bit cache, shared by its kernels: arguments, bytes to 16-bit values, groups of sequences.
#pragma once
#include "kv_cache.h"

namespace vkhip {

    struct KvAttnArgs {
        KvArgs         c;
        const void    *q;
        void          *o;
        const int32_t *lens;
        float         *part_o, *part_s; // [batch][head][row][split]: products [head_dim]; (reference, sum)
        float          scale;
        int            group, rows, q_tokens; // query heads per kv head; rows = group * q_tokens
        int            blocks;                // blocks of 16 * RT rows
        int            max_len, span, splits; // tokens per workgroup
        int            waves;                 // of a workgroup
        int64_t        q_row, q_head, o_row, o_head;
        // sequences that share their first tokens' pages
        const int32_t *cu, *prefix;           // groups of neighbouring sequences, tokens that each shares
        int            groups, max_prefix;
        int            shared_span, shared_splits, shared_blocks; // tokens a workgroup, splits (the first of a row's), blocks of rows
        int            prefix_blocks;                             // workgroups of the prefixes, in blocks of 32 rows
        int            wide;                                      // blocks of 1 or 2 times kWideRows rows; 0: of 32
    };

    // Tokens that group g shares, as every kernel counts them: whole pages.
    __device__ __forceinline__ int prefix_of(const KvAttnArgs &a, int g) { return clampi(a.prefix[g], 0, a.max_prefix) >> a.c.page_shift << a.c.page_shift; }

    // Tokens that sequence b shares with its group, 0 outside every group; the same in every lane.
    __device__ __forceinline__ int prefix_at(const KvAttnArgs &a, int b) {
        const int lane = threadIdx.x & 63;
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            const int      g = g0 + lane, in = min(g, a.groups - 1), from = clampi(a.cu[in], 0, a.c.batch), end = clampi(a.cu[in + 1], 0, a.c.batch);
            const uint64_t hit = __ballot(g < a.groups && from <= b && b < end);
            if (hit) return prefix_of(a, g0 + __ffsll((unsigned long long) hit) - 1);
        }
        return 0;
    }

    constexpr int kWeightBits = 14; // weights are up to 2^14, values b 2^-14

    // 4 int8 (as bits) -> 4 fp16 b 2^-DOWN, exactly: the byte with its sign flipped is the low byte of
    // (1024 + (b + 128)) 2^-DOWN, whose high byte is 0x64 less 4 for each power of two.
    template <int DOWN>
    __device__ __forceinline__ void i8_to_h4(unsigned b, half2v &lo, half2v &hi) {
        b ^= 0x80808080u;
        constexpr unsigned high = (0x64u - 4 * DOWN) * 0x01010101u;
        constexpr float    zero = 1152.f / (1 << DOWN);
        const half2v       off  = {(half_t) zero, (half_t) zero};
        lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(high, b, 0x04010400u)) - off;
        hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(high, b, 0x04030402u)) - off;
    }
    template <int DOWN>
    __device__ __forceinline__ half8 i8_to_h8(unsigned a, unsigned b) {
        half2v x, y, z, w;
        i8_to_h4<DOWN>(a, x, y);
        i8_to_h4<DOWN>(b, z, w);
        return half8 {x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
    }

    constexpr int kStep = 64; // tokens a wave takes at a time

    constexpr int kWideRows = 128, kWideUnits = 256; // tiles of 64 tokens, or of smaller pages, that a workgroup takes
    int kv_wide_run(const KvAttnArgs &a, bool bf16, hipStream_t s); // the prefixes, in blocks of `wide` kWideRows

} // namespace vkhip
