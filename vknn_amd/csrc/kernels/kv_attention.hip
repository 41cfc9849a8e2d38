// Attention of a few query tokens per sequence over the 8-bit cache.
//
// Bound by the cache's bytes, so every byte is read once, straight into the registers that feed the matrix
// cores, and all query heads and tokens that share a key/value head are rows of one product:
//   S^T = K Q^T (16x16x32 tiles: 16 tokens x 16 rows), softmax per row with a running maximum, O^T += V^T P^T.
// A token tile's output registers are the other product's operand as they are: which token sits in which
// contraction slot is free as long as both operands agree, so K's rows are taken in the order that leaves each
// lane with the tokens whose values its V load brings (16 tokens of one channel, side by side in the page).
// int8 becomes fp16 exactly; a page's key scale multiplies its scores, its value scale the fp32 product of the
// page. Weights are rounded to fp16, whose smallest step is 2^-24: a row's reference is 14 below its largest exponent,
// so that its largest weight is 2^14 and what is lost lies under 2^-39 of it (a row of many small weights beside one
// large one keeps them), and values come as multiples of 2^-14 in return, at no cost. This rounding is the largest beside
// that of the output, half a step of fp16 a weight: 64 sequences on 4096 shared tokens are off by 2.6e-4 (norm of the error
// to the result's) in fp16, where fp32 weights leave 2.1e-4; 256 on 32768 in bf16 by 1.67e-3, and 1.66e-3. Both products in
// fp32 would run at a sixteenth of the matrix units' rate, a second product for the weights' rest at half of it.
// The tokens of a sequence are split over workgroups and a workgroup's four waves; partial results
// (reference, sum, product) join in LDS and, across workgroups, in a second kernel.
//
// Measured, fp16, 32 heads on 8, D = 128: 8 x 131072 tokens 330 us (6.5 TB/s), 64 x 2048 44 us (6.2), 64 ragged
// sequences up to 4000 56 us (4.8, the join 5 of it), 8 x 300 7.5 us. Head dims between the two widths read the wider
// one's values: 64 x 2048 at D = 64, 80, 96, 128 27, 44, 43, 43 us. Loading the next step's keys and values while this
// one's are multiplied gained nothing: it costs the registers of a third wave a SIMD, which does the same.
#include "kv_attention.h"
#include <type_traits>

namespace vkhip {

    // DJ = row / 64 channels, RT tiles of 16 rows, P32: pages of 32 tokens (two to a step), NW waves.
    // Two row tiles of 64 channels are compiled for two waves a SIMD: 16 x 5000 tokens, 32 rows, 31.7 -> 29.1 us; of 128
    // channels that costs more than it gives (4 x 40000, 64 rows, 132 -> 160 us), one row tile gains nothing.
    // MODE: a sequence's tokens (kAll), those behind the prefix that it shares (kTail), or a group's prefix (kPrefix), whose
    // rows are those of all its sequences; the last two leave parts for the join.
    enum { kAll, kTail, kPrefix };
    template <int DJ, int RT, int NW>
    struct KvAttnLds {
        static constexpr int NL = NW < 4 ? NW : 4; // waves whose products lie here at a time
        float wave_m[NW][RT * 16], wave_l[NW][RT * 16];
        float acc[NL][16][DJ * 64 + 4];
    };
    // x, y, z: the workgroup's place in a grid of heads x blocks of rows, sequences and splits, or heads, splits and blocks
    // of the groups' rows (kPrefix).
    template <typename T, int DJ, int RT, bool P32, int NW, int MODE>
    __device__ __forceinline__ void kv_attention_body(const KvAttnArgs &a, int bx, int by, int bz, KvAttnLds<DJ, RT, NW> &lds) {
        constexpr int Dp = DJ * 64, DT = DJ * 4, NL = KvAttnLds<DJ, RT, NW>::NL;
        auto &wave_m = lds.wave_m, &wave_l = lds.wave_l;
        auto &acc_lds = lds.acc;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, nn = lane & 15;
        // heads, then sequences, then splits: workgroups go to the 8 XCDs in turn, and with splits first the later ones,
        // which short sequences do not have, would all meet on some of them
        const int head = MODE == kPrefix ? bx : bx / a.blocks, split = MODE == kPrefix ? by : bz;
        const int P   = a.c.page_tokens, D = a.c.head_dim;
        int       b = by, row0 = bx % a.blocks * (16 * RT), rows = a.rows, len, t0, t1; // kPrefix: b is the group's first sequence
        if constexpr (MODE == kPrefix) {
            const auto    bound = [&](int i) { return clampi(a.cu[i], 0, a.c.batch); };
            const SeqTile w = find_tile(bz, a.groups, [&](int g) { return prefix_of(a, g) > 0 ? (max(0, bound(g + 1) - bound(g)) * a.rows + 16 * RT - 1) / (16 * RT) : 0; });
            if (w.b < 0) return;
            const int g = __builtin_amdgcn_readfirstlane(w.b);
            b = bound(g), rows = (bound(g + 1) - b) * a.rows, row0 = __builtin_amdgcn_readfirstlane(w.tile) * (16 * RT);
            len = prefix_of(a, g), t0 = split * a.shared_span, t1 = min(len, t0 + a.shared_span);
            if (t0 >= len) return;
        } else {
            len = clampi(a.lens[b], 0, min(a.max_len, a.c.max_blocks * P));
            t0 = split * a.span, t1 = min(len, t0 + a.span);
            if constexpr (MODE == kTail) {
                const int prefix = prefix_at(a, b);
                t0 += prefix, t1 = split == a.splits - 1 ? len : min(len, t1 + prefix);
                if (t0 >= len) return;
            }
            if (t0 >= len && split > 0) return; // split 0 also answers for a sequence without tokens
        }

        // queries: lane holds row nn, channels 64 j + 16 g + 8 e .. + 7; bf16 rows are brought into fp16's range by
        // a power of two each (their 8 bits fit its 11; what falls below 2^-24 of a row's largest is lost)
        half8 qf[RT][DJ][2];
        int   limit[RT]; // tokens below it are seen
        float c2[RT];    // factor from a score to the exponent of 2
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            int        row = row0 + rt * 16 + nn, seq = b;
            const bool in  = row < rows;
            if constexpr (MODE == kPrefix) seq += row / a.rows, row %= a.rows;
            const int t = row / a.group, h = head * a.group + row % a.group;
            limit[rt]   = in ? len - a.q_tokens + t + 1 : 0;
            if constexpr (MODE == kPrefix)
                if (in) limit[rt] = min(len, clampi(a.lens[seq], 0, min(a.max_len, a.c.max_blocks * P)) - a.q_tokens + t + 1);
            const T *src = (const T *) a.q + ((int64_t) seq * a.q_tokens + t) * a.q_row + h * a.q_head;
            float    v[DJ][2][8], big = 0.f;
#pragma unroll
            for (int j = 0; j < DJ; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 64 * j + 16 * g + 8 * e;
                    typedef T V __attribute__((ext_vector_type(8)));
                    V         x;
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = (T) 0.f;
                    if (in && d < D) x = *reinterpret_cast<const V *>(src + d);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        v[j][e][k] = (float) x[k];
                        big        = fmaxf(big, fabsf(v[j][e][k]));
                    }
                }
            float mul = 1.f;
            c2[rt]    = a.scale * 1.44269504088896f;
            if constexpr (!__is_same(T, half_t)) {
                big          = fmaxf(big, __shfl_xor(big, 16));
                big          = fmaxf(big, __shfl_xor(big, 32));
                const int ex = clampi((int) (__float_as_uint(big) >> 23), 7, 247);
                if (big > 0.f && big < __builtin_inff()) {
                    mul = __uint_as_float((unsigned) (254 - ex) << 23);
                    c2[rt] *= __uint_as_float((unsigned) ex << 23);
                }
            }
#pragma unroll
            for (int j = 0; j < DJ; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int k = 0; k < 8; ++k) qf[rt][j][e][k] = (half_t) (v[j][e][k] * mul);
        }

        float4v acc[RT][DT];
        float   m[RT], l[RT]; // reference of the exponents, sum of the weights
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[rt][d] = float4v {0.f, 0.f, 0.f, 0.f};
        }

        const int32_t *table = a.c.table + (int64_t) b * a.c.max_blocks;
        const int64_t  page_bytes = (int64_t) P * Dp;
        for (int tok = t0 + wave * kStep; tok < t1; tok += NW * kStep) {
            // the step's page, or its two; a block without memory is a page that no query sees
            const unsigned char *kp[2], *vp[2];
            float                ks[2], vs[2];
            bool                 has[2];
#pragma unroll
            for (int u = 0; u < (P32 ? 2 : 1); ++u) {
                const int at = tok + 32 * u, id = at < t1 ? table[at >> a.c.page_shift] : -1;
                has[u]       = id >= 0 && id < a.c.pages;
                const int64_t hp = (int64_t) (has[u] ? id : 0) * a.c.heads + head;
                kp[u] = a.c.k + hp * page_bytes + (int64_t) (at & (P - 1)) * Dp;
                vp[u] = a.c.v + hp * page_bytes + (at & (P - 1));
                ks[u] = has[u] ? a.c.k_scale[hp] : 0.f;
                vs[u] = has[u] ? a.c.v_scale[hp] : 0.f;
            }
            if (!has[0] && !(P32 && has[1])) continue;
            tk_u32x4 kr[4][DJ], vr[DT];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < DJ; ++j) {
                    // row nn = 4 (nn / 4) + i of tile t is the token that lane group nn / 4 multiplies
                    const int r = P32 ? 8 * (nn >> 2) + 4 * (t & 1) + (nn & 3) : 16 * (nn >> 2) + 4 * t + (nn & 3);
                    kr[t][j]    = *reinterpret_cast<const tk_u32x4 *>(kp[P32 ? t >> 1 : 0] + r * Dp + 64 * j + 16 * g);
                }
            // Values pass the caches: 8 x 131072 tokens 369 -> 330 us, 64 x 2048 48 -> 44. Keys too: 335 and 44, and four
            // workgroups that share a cache (64 rows of 128 channels, 4 x 40000) 130 -> 157 us instead of 134.
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if constexpr (P32) {
                    const tk_u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const tk_u32x2 *>(vp[0] + (int64_t) (16 * d + nn) * P + 8 * g));
                    const tk_u32x2 y = __builtin_nontemporal_load(reinterpret_cast<const tk_u32x2 *>(vp[1] + (int64_t) (16 * d + nn) * P + 8 * g));
                    vr[d]            = tk_u32x4 {x[0], x[1], y[0], y[1]};
                } else {
                    vr[d] = __builtin_nontemporal_load(reinterpret_cast<const tk_u32x4 *>(vp[0] + (int64_t) (16 * d + nn) * P + 16 * g));
                }
            }
            float4v s[RT][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][t] = float4v {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < DJ; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const half8 kf = i8_to_h8<0>(kr[t][j][2 * e], kr[t][j][2 * e + 1]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][j][e], s[rt][t], 0, 0, 0);
                    }
            }
            half8 pf[RT][2];
            float alpha[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float top = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float f = ks[P32 ? t >> 1 : 0] * c2[rt];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = tok + (P32 ? 32 * (t >> 1) + 8 * g + 4 * (t & 1) + i : 16 * g + 4 * t + i);
                        float     x  = s[rt][t][i] * f;
                        x            = at < limit[rt] && has[P32 ? t >> 1 : 0] ? x : -__builtin_inff();
                        s[rt][t][i]  = x;
                        top          = fmaxf(top, x);
                    }
                }
                top               = fmaxf(top, __shfl_xor(top, 16));
                top               = fmaxf(top, __shfl_xor(top, 32));
                float up          = top - kWeightBits;
                if (top - up > 15.f) up = top; // exponents from 2^25 on, 4 or more apart: not rounded to where 2^16 would be a weight
                const float to    = fmaxf(m[rt], up), base = to == -__builtin_inff() ? 0.f : to;
                alpha[rt]         = exp2_hw(m[rt] - base);
                m[rt]             = to;
                float sum         = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = exp2_hw(s[rt][t][i] - base);
                        sum += p;
                        pf[rt][t >> 1][(t & 1) * 4 + i] = (half_t) p;
                    }
                l[rt] = l[rt] * alpha[rt] + sum;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const half8   v0 = i8_to_h8<kWeightBits>(vr[d][0], vr[d][1]), v1 = i8_to_h8<kWeightBits>(vr[d][2], vr[d][3]);
                const float4v zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float4v x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[rt][0], zero, 0, 0, 0);
                    // a row that sees nothing of a page takes nothing from it, whatever its scale
                    const float f0 = limit[rt] > tok ? vs[0] : 0.f;
                    if constexpr (P32) {
                        const float4v y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[rt][1], zero, 0, 0, 0);
                        const float   f1 = limit[rt] > tok + 32 ? vs[1] : 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[rt][d][i] = acc[rt][d][i] * alpha[rt] + (x[i] * f0 + y[i] * f1);
                    } else {
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[rt][1], x, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[rt][d][i] = acc[rt][d][i] * alpha[rt] + x[i] * f0;
                    }
                }
            }
        }

        // join the waves, a tile of rows at a time
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            l[rt] += __shfl_xor(l[rt], 16);
            l[rt] += __shfl_xor(l[rt], 32);
            l[rt] *= 1.f / (1 << kWeightBits); // the products have it in their values
            if (g == 0) wave_m[wave][rt * 16 + nn] = m[rt], wave_l[wave][rt * 16 + nn] = l[rt];
        }
        __syncthreads();
        const auto row_max = [&](int r) {
            float top = wave_m[0][r];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, wave_m[w][r]);
            return top;
        };
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float top = row_max(rt * 16 + nn), f = exp2_hw(m[rt] - (top == -__builtin_inff() ? 0.f : top));
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[rt][d][i] *= f;
            if constexpr (NW > NL) { // the upper waves' products into the lower ones' registers
                if (wave >= NL)
#pragma unroll
                    for (int d = 0; d < DT; ++d) *reinterpret_cast<float4v *>(&acc_lds[wave - NL][nn][16 * d + 4 * g]) = acc[rt][d];
                __syncthreads();
                if (wave < NL)
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[rt][d] += *reinterpret_cast<const float4v *>(&acc_lds[wave][nn][16 * d + 4 * g]);
                __syncthreads();
            }
            if (wave < NL)
#pragma unroll
                for (int d = 0; d < DT; ++d) *reinterpret_cast<float4v *>(&acc_lds[wave][nn][16 * d + 4 * g]) = acc[rt][d];
            __syncthreads();
            // VPT neighbouring channels of one row a thread
            constexpr int VPT = Dp / (4 * NW);
            const int     n = threadIdx.x / (4 * NW), d0 = threadIdx.x % (4 * NW) * VPT, q = rt * 16 + n;
            int           row = row0 + q, seq = b;
            if (row < rows && d0 < D) {
                const float tm = row_max(q), tb = tm == -__builtin_inff() ? 0.f : tm;
                float       sum = 0.f, x[VPT];
#pragma unroll
                for (int w = 0; w < NW; ++w) sum += wave_l[w][q] * exp2_hw(wave_m[w][q] - tb);
#pragma unroll
                for (int i = 0; i < VPT; ++i) {
                    x[i] = 0.f;
#pragma unroll
                    for (int w = 0; w < NL; ++w) x[i] += acc_lds[w][n][d0 + i];
                }
                if constexpr (MODE == kPrefix) seq += row / a.rows, row %= a.rows;
                if (MODE == kAll && a.splits == 1) {
                    const int   t = row / a.group, h = head * a.group + row % a.group;
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    T          *o = (T *) a.o + ((int64_t) b * a.q_tokens + t) * a.o_row + h * a.o_head + d0;
#pragma unroll
                    for (int i = 0; i < VPT; ++i)
                        if (d0 + i < D) o[i] = (T) (x[i] * inv);
                } else {
                    const int     shared = MODE == kAll ? 0 : a.shared_splits;
                    const int64_t at = (((int64_t) seq * a.c.heads + head) * a.rows + row) * (shared + a.splits) + (MODE == kTail ? shared : 0) + split;
#pragma unroll
                    for (int i = 0; i < VPT; ++i)
                        if (d0 + i < D) a.part_o[at * D + d0 + i] = x[i];
                    if (d0 == 0) *reinterpret_cast<float2 *>(a.part_s + at * 2) = make_float2(tm, sum);
                }
            }
            if (rt + 1 < RT) __syncthreads();
        }
    }

    template <typename T, int DJ, int RT, bool P32, int NW, int MODE>
    __global__ __launch_bounds__(NW * 64, DJ == 1 && RT == 2 ? 2 : 1) void kv_attention_kernel(KvAttnArgs a) {
        __shared__ KvAttnLds<DJ, RT, NW> lds;
        kv_attention_body<T, DJ, RT, P32, NW, MODE>(a, blockIdx.x, blockIdx.y, blockIdx.z, lds);
    }
    // Prefixes, in blocks of 32 rows, and tails side by side: the first a.prefix_blocks workgroups take the prefixes. 4 sequences
    // behind 1024 tokens 9.1 us, 8.3 and 5.2 in two launches; 64 behind 4096 34.3, 21.6 and 14.3.
    template <typename T, int DJ, int RT, bool P32>
    __global__ __launch_bounds__(256, DJ == 1 ? 2 : 1) void kv_shared_kernel(KvAttnArgs a) {
        __shared__ union {
            KvAttnLds<DJ, 2, 4>  prefix;
            KvAttnLds<DJ, RT, 4> tail;
        } lds;
        const int id = (int) (blockIdx.y * gridDim.x + blockIdx.x), i = id - a.prefix_blocks, x = a.c.heads * a.blocks;
        if (i < 0) kv_attention_body<T, DJ, 2, P32, 4, kPrefix>(a, id % a.c.heads, id / a.c.heads % a.shared_splits, id / a.c.heads / a.shared_splits, lds.prefix);
        else if (i / x < a.c.batch * a.splits) kv_attention_body<T, DJ, RT, P32, 4, kTail>(a, i % x, i / x % a.c.batch, i / x / a.c.batch, lds.tail);
    }

    // Joins the splits of a row: WPR waves each, two channels a lane; the splits' weights are formed a lane each, so
    // that the products' loads wait for nothing.
    template <typename T, int WPR, bool SHARED>
    __global__ __launch_bounds__(256) void kv_join_kernel(KvAttnArgs a) {
        __shared__ float2 half[4][64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.c.head_dim, d = lane * 2;
        const int row = blockIdx.x * (4 / WPR) + wave / WPR, head = blockIdx.y, b = blockIdx.z, part = wave % WPR;
        const int len = clampi(a.lens[b], 0, min(a.max_len, a.c.max_blocks * a.c.page_tokens));
        int       n   = row < a.rows ? max(1, (len + a.span - 1) / a.span) : 0, shared = 0; // parts: of the prefix, which go first, and all
        if constexpr (SHARED) {
            const int prefix = prefix_at(a, b), tail = max(0, len - prefix);
            shared = (prefix + a.shared_span - 1) / a.shared_span;
            n      = row < a.rows ? shared + min(a.splits, (tail + a.span - 1) / a.span) : 0;
        }
        const int     skip = SHARED ? a.shared_splits - shared : 0; // slots of longer prefixes
        const int64_t at   = (((int64_t) b * a.c.heads + head) * a.rows + row) * ((SHARED ? a.shared_splits : 0) + a.splits);
        const auto    slot = [&](int k) { return at + (SHARED && k >= shared ? k + skip : k); };
        float top = -__builtin_inff(), sum = 0.f;
        for (int k = lane; k < n; k += 64) top = fmaxf(top, a.part_s[slot(k) * 2]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float base = top == -__builtin_inff() ? 0.f : top;
        float2      x = make_float2(0.f, 0.f);
        for (int k0 = 0; k0 < n; k0 += 64) {
            const int    k = k0 + lane;
            const float2 s = k < n ? *reinterpret_cast<const float2 *>(a.part_s + slot(k) * 2) : make_float2(-__builtin_inff(), 0.f);
            const float  f = exp2_hw(s.x - base);
            sum += s.y * f;
            const int end = min(64, n - k0);
            if constexpr (SHARED) {
                // eight loads under way, of a rest four, the last ones of parts that are there already (5 parts of 720 rows 10.2 us with a
                // loop's rest, 5.0; 28 of 2352 13.9, 9.0)
                const auto some = [&](int i, auto n_c) __attribute__((always_inline)) {
                    constexpr int SOME = decltype(n_c)::value;
                    float2        y[SOME];
#pragma unroll
                    for (int j = 0; j < SOME; ++j) y[j] = *reinterpret_cast<const float2 *>(a.part_o + slot(k0 + min(i + j * WPR, end - 1)) * D + min(d, D - 2));
#pragma unroll
                    for (int j = 0; j < SOME; ++j) {
                        const int   k = i + j * WPR;
                        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(k, end - 1)));
                        if (k < end) x.x += y[j].x * w, x.y += y[j].y * w;
                    }
                };
                int i = part;
                for (; i + 7 * WPR < end; i += 8 * WPR) some(i, std::integral_constant<int, 8>());
                for (; i < end; i += 4 * WPR) some(i, std::integral_constant<int, 4>());
            } else {
                for (int i = part; i < end; i += WPR) {
                    const float  w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i));
                    const float2 y = *reinterpret_cast<const float2 *>(a.part_o + slot(k0 + i) * D + min(d, D - 2));
                    x.x += y.x * w, x.y += y.y * w;
                }
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
        if constexpr (WPR > 1) {
            half[wave][lane] = x;
            __syncthreads();
            if (part) return;
#pragma unroll
            for (int w = 1; w < WPR; ++w) x.x += half[wave + w][lane].x, x.y += half[wave + w][lane].y;
        }
        if (row >= a.rows || d >= D) return;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T          *o = (T *) a.o + ((int64_t) b * a.q_tokens + row / a.group) * a.o_row + (head * a.group + row % a.group) * a.o_head + d;
        o[0] = (T) (x.x * inv), o[1] = (T) (x.y * inv);
    }

    // Tiles of 16 rows a wave multiplies with what it has read. Four would read the cache once for 64 rows, but leave
    // registers for one wave a SIMD and nothing to read while it computes: 16 x 5000 tokens, 64 rows, 63 us with four,
    // 46 with two, 56 with one.
    static int row_tiles(int rows) { return rows <= 16 ? 1 : 2; }

    static const char *kv_attention_refusal(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c) {
        if (const char *why = kv_refusal(c)) return why;
        if (!d || d->q_heads <= 0 || d->q_heads % c->kv_heads) return "q_heads is not a multiple of kv_heads";
        if (d->q_tokens < 1 || d->q_tokens > 64) return "q_tokens is not 1 .. 64";
        if (d->q_heads > 65535) return "q_heads over 65535";
        if (d->dtype != VKHIP_DT_F16 && d->dtype != VKHIP_DT_BF16) return "q and o are F16 or BF16";
        if (!(d->scale > 0.f) || d->scale > 1e30f || d->max_len < 0) return "scale is not positive or max_len negative";
        if (d->q_row < 0 || d->q_head < 0 || d->o_row < 0 || d->o_head < 0 || (d->q_row | d->q_head | d->o_row | d->o_head) % 8) return "strides are not multiples of 8";
        if (rows_overlap((int64_t) c->batch * d->q_tokens, d->o_row, d->q_heads, d->o_head, c->head_dim)) return "rows of o share memory";
        return nullptr;
    }

    // How the call is cut: rows into blocks of up to 32, tokens into spans of whole rounds of a workgroup's waves.
    static KvAttnArgs kv_attention_cut(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c) {
        KvAttnArgs a {};
        a.c        = kv_args(c);
        a.group    = d->q_heads / c->kv_heads;
        a.q_tokens = d->q_tokens;
        a.rows     = a.group * d->q_tokens;
        a.blocks   = (int) ceil_div(a.rows, 16 * row_tiles(a.rows));
        const int64_t most = (int64_t) c->max_blocks * c->page_tokens;
        a.max_len  = (int) (d->max_len > 0 && d->max_len < most ? d->max_len : most);
        const int64_t len = a.max_len > 0 ? a.max_len : 1, base = (int64_t) c->batch * c->kv_heads * a.blocks;
        // Waves of a workgroup: two where no sequence has more steps, eight and no split where one workgroup takes a
        // sequence in few rounds (a second launch costs about 3 us), four otherwise. How many are few: one, as a round is
        // 128 KB for a compute unit alone, two of 64 channels, and more where the workgroups nearly fill the card. Split /
        // not, 128 and 64 channels: 1 x 1000 tokens 8.1 / 9.9, 7.4 / 6.9 us; 8 x 700 9.2 / 10.4, 8.3 / 7.0; 16 x 1500
        // 15.3 / 16.1 (three rounds), 12.6 / 11.7; 32 x 1500 22.2 / 19.8, 16.0 / 12.8.
        const int64_t once = (c->head_dim <= 64 ? 2 : 1) + base / 128;
        const bool    few  = base <= 256 && len <= once * 8 * kStep && row_tiles(a.rows) == 1;
        a.waves        = len <= 2 * kStep ? 2 : (few ? 8 : 4);
        // Splits: two workgroups a compute unit, which all run at once; where that leaves more than 8 rounds to one,
        // which would wait for the longest sequence, spans of 8 rounds or 2048 workgroups. In between, workgroups that
        // nearly all run at once leave some for a second turn (before values passed the caches 8 x 131072 tokens 362 us
        // with 512, 404 with 1024, 370 with 2048; 64 ragged sequences up to 4000 71 us unsplit, 61 in two; since then 64 x
        // 2048 44 us, 53 with spans of four rounds).
        const int64_t rounds = ceil_div(len, a.waves * kStep);
        int64_t       splits = few || base >= 512 || base == 0 ? 1 : 512 / base;
        if (base > 0 && rounds > 8 * splits) {
            const int64_t more = rounds / 8 < 2048 / base ? rounds / 8 : 2048 / base;
            if (more > splits) splits = more;
        }
        if (splits > rounds) splits = rounds;
        a.span   = (int) (ceil_div(rounds, splits) * a.waves * kStep);
        a.splits = (int) ceil_div(len, a.span);
        return a;
    }

    template <typename T, int DJ, int RT, bool P32>
    static void kv_attention_launch(const KvAttnArgs &a, hipStream_t s) {
        const dim3 grid((unsigned) (a.c.heads * a.blocks), (unsigned) a.c.batch, (unsigned) a.splits);
        if (a.waves == 2) kv_attention_kernel<T, DJ, RT, P32, 2, kAll><<<grid, 128, 0, s>>>(a);
        else if (a.waves == 4) kv_attention_kernel<T, DJ, RT, P32, 4, kAll><<<grid, 256, 0, s>>>(a);
        else if constexpr (RT == 1) kv_attention_kernel<T, DJ, RT, P32, 8, kAll><<<grid, 512, 0, s>>>(a);
    }
    template <typename T, int DJ>
    static void kv_attention_tiles(const KvAttnArgs &a, hipStream_t s) {
        const int  rt  = row_tiles(a.rows);
        const bool p32 = a.c.page_tokens == 32;
        if (rt == 1) p32 ? kv_attention_launch<T, DJ, 1, true>(a, s) : kv_attention_launch<T, DJ, 1, false>(a, s);
        else p32 ? kv_attention_launch<T, DJ, 2, true>(a, s) : kv_attention_launch<T, DJ, 2, false>(a, s);
    }
    template <typename T>
    static int kv_attention_run(const KvAttnArgs &a, hipStream_t s) {
        if (a.c.row == 64) kv_attention_tiles<T, 1>(a, s);
        else kv_attention_tiles<T, 2>(a, s);
        int rc = check_launch("kv_attention");
        if (rc || a.splits == 1) return rc;
        const bool wide = a.splits > 8; // below, a row's products are few loads of one wave
        const dim3 grid((unsigned) (wide ? a.rows : ceil_div(a.rows, 4)), (unsigned) a.c.heads, (unsigned) a.c.batch);
        if (wide) kv_join_kernel<T, 4, false><<<grid, 256, 0, s>>>(a);
        else kv_join_kernel<T, 1, false><<<grid, 256, 0, s>>>(a);
        return check_launch("kv_attention join");
    }

    constexpr int kWideLeast = 4; // tiles of a workgroup, if the prefix has them

    // A prefix takes tiles of 128 or 256 rows (kv_prefix.hip) where groups have more than kWideGroup rows a head on average and
    // heads x rows x tokens are more than this; below, the start of a wide tile's workgroup, about 10 us, is what counts, and
    // of 64 channels narrow tiles run twice as many at a time. Whole calls, us, 32-row tiles / wide ones:
    //   128 channels: 8 x 256 x 4096 (2^23) 39.5 / 39.9, 1 x 400 x 16384 29 / 35 (2^22.6), 8 x 512 x 4096 (2^24) 57 / 54
    //   64 channels:  4 x 768 x 8192 (2^24.6) 37 / 46, x 16384 (3 * 2^24) 55.2 / 55.5, 4 x (256 sequences of 12) x 4096 65 / 64,
    //                 1 x 12288 x 8192 (3 * 2^25) 112 / 79
    // The host knows the groups' mean alone, and counts sequences outside every group to it: a large group beside many small
    // ones takes 32-row tiles too (256 sequences on 8192 tokens 71 us, with 40 pairs beside them 140).
    constexpr int64_t kWideGroup = 64, kWideWork128 = 1 << 23, kWideWork64 = 3 << 24;
    // 256 rows instead of 128, with 128 channels: 8 x 256 x 4096 42.5 / 39.9, 8 x 512 x 4096 54.1 / 53.6, 8 x 1024 x 32768 157 / 166
    // (prefixes alone).
    constexpr int64_t kWideTallGroup = 192, kWideTallWork = 1 << 24;

    // Groups of sequences: the prefixes for all rows of a group and every sequence's tail, then the join.
    template <typename T, int DJ, int RT, bool P32>
    static int kv_shared_launch(const KvAttnArgs &a, hipStream_t s) {
        if (a.wide) {
            if (int rc = kv_wide_run(a, !__is_same(T, half_t), s)) return rc;
            kv_attention_kernel<T, DJ, RT, P32, 4, kTail><<<dim3((unsigned) (a.c.heads * a.blocks), (unsigned) a.c.batch, (unsigned) a.splits), 256, 0, s>>>(a);
        } else {
            const int64_t all = a.prefix_blocks + (int64_t) a.c.heads * a.blocks * a.c.batch * a.splits, layers = ceil_div(all, 0xFFFFFF);
            kv_shared_kernel<T, DJ, RT, P32><<<dim3((unsigned) ceil_div(all, layers), (unsigned) layers), 256, 0, s>>>(a);
        }
        return check_launch("kv_attention_shared");
    }
    template <typename T, int DJ>
    static int kv_shared_tiles(const KvAttnArgs &a, hipStream_t s) {
        const bool p32 = a.c.page_tokens == 32;
        if (row_tiles(a.rows) == 1) return p32 ? kv_shared_launch<T, DJ, 1, true>(a, s) : kv_shared_launch<T, DJ, 1, false>(a, s);
        return p32 ? kv_shared_launch<T, DJ, 2, true>(a, s) : kv_shared_launch<T, DJ, 2, false>(a, s);
    }
    template <typename T>
    static int kv_shared_run(const KvAttnArgs &a, hipStream_t s) {
        if (int rc = a.c.row == 64 ? kv_shared_tiles<T, 1>(a, s) : kv_shared_tiles<T, 2>(a, s)) return rc;
        const bool wide = a.shared_splits + a.splits > 32;
        const dim3 grid((unsigned) (wide ? a.rows : ceil_div(a.rows, 4)), (unsigned) a.c.heads, (unsigned) a.c.batch);
        if (wide) kv_join_kernel<T, 4, true><<<grid, 256, 0, s>>>(a);
        else kv_join_kernel<T, 1, true><<<grid, 256, 0, s>>>(a);
        return check_launch("kv_attention_shared join");
    }

    static const char *kv_shared_refusal(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c, const vkhip_kv_prefix *p) {
        if (const char *why = kv_attention_refusal(d, c)) return why;
        if (!p || p->groups < 0 || p->groups > 65535) return "groups are not 0 .. 65535";
        if (p->max_tokens < 0 || p->max_tail < 0) return "max_tokens or max_tail negative";
        return nullptr;
    }

    // Whether a call has nothing to share, and the cut of its prefixes and tails where it has. Tails are cut like whole
    // sequences of the longest tail.
    static KvAttnArgs kv_shared_cut(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c, const vkhip_kv_prefix *p) {
        const KvAttnArgs whole = kv_attention_cut(d, c);
        vkhip_kv_attention_desc tail = *d;
        tail.max_len = p->max_tail > 0 && p->max_tail < whole.max_len ? p->max_tail : whole.max_len;
        KvAttnArgs a = kv_attention_cut(&tail, c);
        a.waves = 4; // spans are whole rounds of 2, 4 or 8
        // Tails are joined in any case, so that two workgroups a sequence cost no launch where four fit a compute unit, as with 64
        // channels (124 sequences of 4 heads, up to 800 tokens, 15.4 / 11.6 us; of 128 channels two fit: 35 x 8 of 40 rows 19.5 / 22.1).
        const int64_t tail_rounds = ceil_div(a.max_len, 4 * kStep), tail_base = (int64_t) c->batch * c->kv_heads * a.blocks;
        const int64_t more = tail_base == 0 || a.c.row != 64 ? 1 : 1024 / tail_base < tail_rounds ? 1024 / tail_base : tail_rounds;
        if (more > a.splits) {
            a.span   = (int) (ceil_div(tail_rounds, more) * 4 * kStep);
            a.splits = (int) ceil_div(a.max_len, a.span);
        }
        a.max_len    = whole.max_len;
        a.groups     = p->groups;
        a.max_prefix = p->max_tokens > 0 && p->max_tokens < whole.max_len ? p->max_tokens : whole.max_len;
        const int64_t each = p->groups > 0 ? (int64_t) c->batch * a.rows / p->groups : 0; // rows of a group
        const int64_t work = (int64_t) c->kv_heads * c->batch * a.rows * a.max_prefix;
        const bool    tall = a.c.row == 128 && each > kWideTallGroup && work > kWideTallWork;
        a.wide             = each <= kWideGroup || work <= (a.c.row == 64 ? kWideWork64 : kWideWork128) ? 0 : tall ? 2 : 1;
        const auto blocks = [&](int height) { return (int64_t) c->batch * a.rows / height + p->groups; };
        if (a.wide && blocks(a.wide * kWideRows) > 65535) a.wide = 0; // more than the third dimension of their grid; the narrow ones' has one
        const int height  = a.wide ? a.wide * kWideRows : 32;
        a.shared_blocks   = (int) blocks(height);
        const int wide_tiles = kWideUnits / (c->page_tokens == 32 ? 2 : 1);
        if (a.wide && a.max_prefix > 4096 * wide_tiles * kStep) a.max_prefix = 4096 * wide_tiles * kStep; // 4096 splits; the rest with the tails
        const int     round = (a.wide ? 1 : 4) * kStep; // tokens that a workgroup takes at a time
        const int64_t rounds = ceil_div(a.max_prefix > 0 ? a.max_prefix : 1, round), full = ceil_div((int64_t) c->batch * a.rows, height);
        const int64_t base = (full > p->groups ? full : p->groups) * c->kv_heads; // blocks, if groups fill theirs
        // blocks of uneven groups outnumber that, and two workgroups a compute unit make good for each other's ends, if not for
        // every size: of 12 drawn sets of 3 to 12 groups of 1 to 54 sequences 7 take the same splits with 512, 640 and 768 places; the
        // others, whole calls: 82, 92, 85 us; 119, 92, 107; 94, 84, 78; 56, 54, 50; 78, 68, 75. One group of 128 sequences, 512 and
        // 640: 27, 29.
        const int64_t places = a.wide == 2 ? 256 : a.wide == 1 && p->groups > 1 ? 640 : 512;
        int64_t       splits = base >= places || base == 0 ? 1 : places / base;
        const int64_t most = a.wide ? rounds / kWideLeast : rounds;
        if (splits > most) splits = most > 0 ? most : 1;
        if (a.wide && splits < ceil_div(rounds, wide_tiles)) splits = ceil_div(rounds, wide_tiles);
        a.shared_span   = (int) (ceil_div(rounds, splits) * round);
        a.shared_splits = (int) ceil_div(a.max_prefix > 0 ? a.max_prefix : 1, a.shared_span);
        const int64_t prefixes = (int64_t) c->kv_heads * a.shared_splits * blocks(height), tails = (int64_t) c->kv_heads * a.blocks * c->batch * a.splits;
        a.prefix_blocks = a.wide ? 0 : prefixes + tails < 0x7FFF0000 ? (int) prefixes : -1; // -1: more than a launch numbers
        return a;
    }
    // What no launch holds, nor the rows of a group 31 bits.
    static const char *kv_shared_too_many(const KvAttnArgs &a) {
        return (int64_t) a.c.heads * a.blocks > 65535 || (int64_t) a.c.batch * a.rows > 0x7FFFFF00 || a.prefix_blocks < 0 ? "too many heads, sequences and query tokens" : nullptr;
    }
    static bool kv_nothing_shared(const KvAttnArgs &a) { return a.groups == 0 || a.max_prefix < a.c.page_tokens; }

} // namespace vkhip

using namespace vkhip;

extern "C" {

size_t vkhip_kv_attention_workspace_bytes(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c) {
    if (kv_attention_refusal(d, c)) return 0;
    const KvAttnArgs a = kv_attention_cut(d, c);
    return a.splits == 1 ? 0 : (size_t) c->batch * c->kv_heads * a.rows * a.splits * (c->head_dim + 2) * sizeof(float);
}

int vkhip_kv_attention(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c, const void *q, const int32_t *lens, void *o, void *workspace,
                       vkhip_stream_t s) {
    if (const char *why = kv_attention_refusal(d, c)) return set_error(VKHIP_ERR_INVALID, "kv_attention: %s", why);
    if (c->batch == 0) return VKHIP_OK;
    if (const char *why = kv_bad_pointers(c)) return set_error(VKHIP_ERR_INVALID, "kv_attention: %s", why);
    KvAttnArgs a = kv_attention_cut(d, c);
    if (!q || !lens || !o || (a.splits > 1 && !workspace)) return set_error(VKHIP_ERR_INVALID, "kv_attention: null pointer");
    if (misaligned16(q) || misaligned16(o) || misaligned16(workspace) || ((uintptr_t) lens) % 4) return set_error(VKHIP_ERR_INVALID, "kv_attention: misaligned pointer");
    if ((int64_t) c->kv_heads * a.blocks > 65535) return set_error(VKHIP_ERR_INVALID, "kv_attention: too many heads and query tokens");
    if (c->pages == 0) a.max_len = 0; // no block has memory: every query gives zeros
    a.q = q, a.o = o, a.lens = lens, a.part_o = (float *) workspace, a.scale = d->scale;
    a.part_s = a.part_o + (size_t) c->batch * c->kv_heads * a.rows * a.splits * c->head_dim;
    a.q_row = d->q_row, a.q_head = d->q_head, a.o_row = d->o_row, a.o_head = d->o_head;
    return d->dtype == VKHIP_DT_F16 ? kv_attention_run<half_t>(a, resolve_stream(s)) : kv_attention_run<bf16_t>(a, resolve_stream(s));
}

size_t vkhip_kv_attention_shared_workspace_bytes(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c, const vkhip_kv_prefix *p) {
    if (kv_shared_refusal(d, c, p)) return 0;
    const KvAttnArgs a = kv_shared_cut(d, c, p);
    if (kv_nothing_shared(a)) return vkhip_kv_attention_workspace_bytes(d, c);
    if (kv_shared_too_many(a)) return 0;
    return (size_t) c->batch * c->kv_heads * a.rows * (a.shared_splits + a.splits) * (c->head_dim + 2) * sizeof(float);
}

int vkhip_kv_attention_shared(const vkhip_kv_attention_desc *d, const vkhip_kv_cache *c, const vkhip_kv_prefix *p, const void *q, const int32_t *lens, void *o,
                              void *workspace, vkhip_stream_t s) {
    const char *what = "kv_attention_shared: %s";
    if (const char *why = kv_shared_refusal(d, c, p)) return set_error(VKHIP_ERR_INVALID, what, why);
    if (c->batch == 0) return VKHIP_OK;
    if (const char *why = kv_bad_pointers(c)) return set_error(VKHIP_ERR_INVALID, what, why);
    KvAttnArgs a = kv_shared_cut(d, c, p);
    if (p->groups && (!p->cu || !p->tokens)) return set_error(VKHIP_ERR_INVALID, what, "null pointer");
    if (((uintptr_t) p->cu | (uintptr_t) p->tokens) % 4) return set_error(VKHIP_ERR_INVALID, what, "misaligned pointer");
    if (!q || !lens || !o) return set_error(VKHIP_ERR_INVALID, what, "null pointer");
    if (misaligned16(q) || misaligned16(o) || misaligned16(workspace) || ((uintptr_t) lens) % 4) return set_error(VKHIP_ERR_INVALID, what, "misaligned pointer");
    if (kv_nothing_shared(a)) return vkhip_kv_attention(d, c, q, lens, o, workspace, s);
    if (const char *why = kv_shared_too_many(a)) return set_error(VKHIP_ERR_INVALID, what, why);
    if (c->pages == 0) a.max_len = a.max_prefix = 0; // no block has memory: every query gives zeros
    if (!workspace) return set_error(VKHIP_ERR_INVALID, what, "null pointer");
    a.q = q, a.o = o, a.lens = lens, a.part_o = (float *) workspace, a.scale = d->scale, a.cu = p->cu, a.prefix = p->tokens;
    a.part_s = a.part_o + (size_t) c->batch * c->kv_heads * a.rows * (a.shared_splits + a.splits) * c->head_dim;
    a.q_row = d->q_row, a.q_head = d->q_head, a.o_row = d->o_row, a.o_head = d->o_head;
    return d->dtype == VKHIP_DT_F16 ? kv_shared_run<half_t>(a, resolve_stream(s)) : kv_shared_run<bf16_t>(a, resolve_stream(s));
}

} // extern "C"
