// A prefix of the 8-bit cache that many rows share (sequences x query heads x tokens): scores and values as products of
// whole tiles.
//
// A wave owns 32 rows, a workgroup 128. As in the attention over packed sequences, scores come out transposed (S^T = K Q^T,
// 32x32x16) and the exponentials are, as they lie in the registers, the operand of O^T += V^T P^T; the cache keeps the
// values by channel, so V^T needs no turning, only its tokens in the order in which a lane holds their weights: of each 16,
// 0-3 8-11 | 4-7 12-15. Bytes become fp16 once for the four waves, on their way from memory through registers into LDS,
// a tile of 64 tokens ahead.
// Weights are up to 2^15, as they are in the attention of one sequence, and rescaled where a row's maximum grows by more
// than 2; a page's value scale goes into its weights' exponents, relative to the largest one so far, so that the products
// of all pages add up in place (a page under 2^-8 of that, or not finite, takes a product of its own).
#include "kv_attention.h"
#include <type_traits>

namespace vkhip {

    __device__ __forceinline__ float wide_max_halves(float x) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }

    // A value that the compiler does not know to be the same each time: what follows from it is computed where it is used,
    // not kept in registers through the loop.
    __device__ __forceinline__ int again(int x) {
        __asm__ volatile("" : "+v"(x));
        return x;
    }

    // NW: waves of a workgroup, 4 or, where a group has the rows, 8, which share what is converted.
    template <typename T, int DP, bool P32, int NW>
    __global__ __launch_bounds__(NW * 64, 2) void kv_wide_kernel(KvAttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int KS = DP / 16, DB = DP / 32, ROW = DP * 2, PIECES = DP / 8; // contraction steps of a score, output blocks, bytes and pieces of a row of K
        constexpr int LOADS = DP / (16 * NW);                                    // 16-byte loads of K, and of V, per thread and tile
        constexpr int AHEAD = 6, ROWS = 32 * NW; // operands read in front of their products; rows of a workgroup
        constexpr int UNIT  = P32 ? 32 : kStep;                                  // tokens of one page, as many as a tile takes
        __shared__ __attribute__((aligned(1024))) unsigned char sm_k[2][kStep * ROW], sm_v[2][kStep * ROW];
        __shared__ float4v unit[256]; // of a unit's page: key scale; vref to its unit (0: zeros, NaN: no number); log2 of its value scale to that, and back
        __shared__ int     unit_id[256];
        __shared__ float   wave_vs[NW];
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31, tid = threadIdx.x;
        const int head = blockIdx.x, split = blockIdx.y, P = a.c.page_tokens, D = a.c.head_dim;
        const auto    bound = [&](int i) { return clampi(a.cu[i], 0, a.c.batch); };
        const SeqTile w = find_tile(blockIdx.z, a.groups, [&](int g) { return prefix_of(a, g) > 0 ? (max(0, bound(g + 1) - bound(g)) * a.rows + ROWS - 1) / ROWS : 0; });
        if (w.b < 0) return;
        const int g = __builtin_amdgcn_readfirstlane(w.b), first = bound(g), rows = (bound(g + 1) - first) * a.rows;
        const int prefix = prefix_of(a, g), t0 = split * a.shared_span, t1 = min(prefix, t0 + a.shared_span);
        if (t0 >= t1) return;
        const int32_t *table = a.c.table + (int64_t) first * a.c.max_blocks;

        // this lane's row: queries of channels 16 c + 8 h .. + 7; bf16 rows are brought into fp16's range by a power of two
        const int  block_row = __builtin_amdgcn_readfirstlane(w.tile) * ROWS + wave * 32;
        const auto row_of    = [&](int lane) {
            const int row = block_row + (lane & 31);
            return make_int3(first + row / a.rows, row % a.rows, row < rows); // sequence, row of it, whether there is one
        };
        // What the loop needs of pages it finds in LDS, for 256 units of tokens at a time (a tile, or half of one where pages
        // are smaller): a scalar load would make every wait for LDS a wait for memory.
        float vref = 0x1p-126f; // the scale that O is in units of: a power of two, no page's so far was larger
        float16v acc[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
        int   unit_page = -1; // this thread's unit
        float unit_ks = 0.f, unit_vs = 0.f;
        const auto page_of = [&](int tok) { // -1: no memory, or nothing there
            const int id = tok < t1 ? table[tok >> a.c.page_shift] : -1;
            return id < a.c.pages ? id : -1;
        };
        const auto ask = [&](int from) {
            unit_page = tid < 256 ? page_of(from + tid * UNIT) : -1, unit_ks = unit_vs = 0.f;
            if (unit_page >= 0) {
                const int64_t hp = (int64_t) unit_page * a.c.heads + head;
                unit_ks = a.c.k_scale[hp], unit_vs = a.c.v_scale[hp];
            }
        };
        const auto settle = [&] {
            const float ks = unit_ks, vs = unit_vs;
            float       larger = vs <= 0x1p126f ? vs : 0.f;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) larger = fmaxf(larger, __shfl_xor(larger, o));
            if (lane == 0) wave_vs[wave] = larger;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) larger = fmaxf(larger, wave_vs[i]);
            if (larger > vref) {
                const float to = __uint_as_float((__float_as_uint(larger) + 0x7FFFFFu) & 0x7F800000u), less = vref / to;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= less;
                vref = to;
            }
            // a page far below the largest has a unit of its own, a power of two under vref that O takes for its tile; a page
            // of zeros or of a scale that is no number is dealt with there too
            const bool none = vs == 0.f, lost = !(vs <= vref), plain = none || lost || vs >= vref * 0x1p-8f;
            const float up = __uint_as_float((__float_as_uint(vs) + 0x7FFFFFu) & 0x7F800000u), under = plain ? 1.f : fminf(vref / up, 0x1p64f);
            const float ratio = none || lost ? 1.f : vs / (vref / under);
            if (tid >= 256) return;
            unit_id[tid] = unit_page < 0 ? -1 : none || lost || !plain || !(ks > 0.f) ? unit_page | 0x40000000 : unit_page;
            unit[tid]    = float4v {ks, none ? 0.f : lost ? __builtin_nanf("") : under, __builtin_amdgcn_logf(ratio), 1.f / ratio};
        };
        // the names of a tile's pages, the same in every lane; from: the first token of the units in LDS
        const auto names = [&](int tok, int from) {
            const int i = (tok - from) / UNIT;
            return make_int2(__builtin_amdgcn_readfirstlane(unit_id[i]), P32 ? __builtin_amdgcn_readfirstlane(unit_id[i + 1]) : 0);
        };

        const auto first_names = [&](int tok) { return make_int2(page_of(tok), P32 ? page_of(tok + UNIT) : 0); }; // before they are in LDS
        // a tile's bytes: piece p of K is token p / (DP / 16), 16 channels from p % (DP / 16) on; of V channel p / 4, 16 tokens
        // from p % 4 on
        tk_u32x4      kr[LOADS], vr[LOADS];
        const int64_t page_bytes = (int64_t) P * DP;
        const auto    fetch = [&](int tok, int2 n) __attribute__((always_inline)) {
            const unsigned char *kp[2], *vp[2];
#pragma unroll
            for (int u = 0; u < (P32 ? 2 : 1); ++u) {
                const int     id = u ? n.y : n.x, at = P32 ? 0 : tok & (P - 1);
                const int64_t hp = (int64_t) (id < 0 ? 0 : id & 0x3FFFFFFF) * a.c.heads + head;
                kp[u] = a.c.k + hp * page_bytes + at * DP, vp[u] = a.c.v + hp * page_bytes + at;
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = i * (NW * 64) + tid, kt = p / (DP / 16), kc = p % (DP / 16) * 16, vc = p / 4, vt = p % 4 * 16;
                if constexpr (P32) {
                    kr[i] = *reinterpret_cast<const tk_u32x4 *>((kt >> 5 ? kp[1] : kp[0]) + (unsigned) ((kt & 31) * DP + kc));
                    vr[i] = *reinterpret_cast<const tk_u32x4 *>((vt >> 5 ? vp[1] : vp[0]) + (unsigned) (vc * P + (vt & 31)));
                } else {
                    kr[i] = *reinterpret_cast<const tk_u32x4 *>(kp[0] + (unsigned) (kt * DP + kc));
                    vr[i] = *reinterpret_cast<const tk_u32x4 *>(vp[0] + (unsigned) (vc * P + vt));
                }
            }
        };
        // the first tile's bytes and the pages' scales are on their way while the queries are
        int from = t0;
        ask(from);
        fetch(from, first_names(from));

        int        limit = t1; // tokens below it are seen
        half8      qf[KS];
        float      c2 = a.scale * 1.44269504088896f;
        {
            const int3 me = row_of(lane);
            const int  seq = me.x, t = me.y / a.group, hq = head * a.group + me.y % a.group;
            const bool in = me.z;
            const T  *src = (const T *) a.q + (in ? ((int64_t) seq * a.q_tokens + t) * a.q_row + hq * a.q_head : 0);
            typedef T V __attribute__((ext_vector_type(8)));
            V         x[KS];
            float     big = 0.f;
            const int len = a.lens[in ? seq : first];
#pragma unroll
            for (int c = 0; c < KS; ++c) x[c] = *reinterpret_cast<const V *>(src + (16 * c + 8 * h < D ? 16 * c + 8 * h : 0));
#pragma unroll
            for (int c = 0; c < KS; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] = in && 16 * c + 8 * h < D ? x[c][j] : (T) 0.f;
            if (in) limit = min(t1, clampi(len, 0, min(a.max_len, a.c.max_blocks * P)) - a.q_tokens + t + 1);
            float mul = 1.f;
            if constexpr (!__is_same(T, half_t)) {
#pragma unroll
                for (int c = 0; c < KS; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf((float) x[c][j]));
                big          = wide_max_halves(big);
                const int ex = clampi((int) (__float_as_uint(big) >> 23), 7, 247);
                if (big > 0.f && big < __builtin_inff()) {
                    mul = __uint_as_float((unsigned) (254 - ex) << 23);
                    c2 *= __uint_as_float((unsigned) ex << 23);
                }
            }
#pragma unroll
            for (int c = 0; c < KS; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) qf[c][j] = (half_t) ((float) x[c][j] * mul);
        }
        // tiles that end before `seen_by_all` need no mask in this wave
        int seen_by_all = limit;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) seen_by_all = min(seen_by_all, __shfl_xor(seen_by_all, o));
        seen_by_all = __builtin_amdgcn_readfirstlane(seen_by_all);

        // 16-byte pieces are permuted by their row so that the rows of a read meet no bank twice
        const auto k_at = [](int token, int piece) { return token * ROW + ((piece ^ (DP == 128 ? token & 15 : token >> 1 & 7)) << 4); };
        const auto v_at = [](int channel, int piece) { return channel * (kStep * 2) + ((piece ^ (channel >> 1 & 7)) << 4); };
        unsigned   ka[KS], va[4]; // where a lane's operands lie
#pragma unroll
        for (int c = 0; c < KS; ++c) ka[c] = k_at(col, 2 * c + h);
#pragma unroll
        for (int k = 0; k < 4; ++k) va[k] = v_at(col, 2 * k + h);
        const auto stage = [&](auto odd_c) __attribute__((always_inline)) {
            unsigned char *sk = sm_k[decltype(odd_c)::value], *sv = sm_v[decltype(odd_c)::value];
            const int      kt = tid / (DP / 16), kc = tid % (DP / 16) * 2, vc = tid / 4, vt = tid % 4 * 2;
            const unsigned kw[2] = {(unsigned) k_at(kt, kc), (unsigned) k_at(kt, kc + 1)}, vw[2] = {(unsigned) v_at(vc, vt), (unsigned) v_at(vc, vt + 1)};
#pragma unroll
            for (int i = 0; i < LOADS; ++i) { // 256 pieces on are 32 tokens or 64 channels: rows of the same permutation
                *reinterpret_cast<half8 *>(sk + kw[0] + i * 8192) = i8_to_h8<0>(kr[i][0], kr[i][1]);
                *reinterpret_cast<half8 *>(sk + kw[1] + i * 8192) = i8_to_h8<0>(kr[i][2], kr[i][3]);
                *reinterpret_cast<half8 *>(sv + vw[0] + i * 8192) = i8_to_h8<kWeightBits>(vr[i][0], vr[i][2]);
                *reinterpret_cast<half8 *>(sv + vw[1] + i * 8192) = i8_to_h8<kWeightBits>(vr[i][1], vr[i][3]);
            }
        };

        float m = -__builtin_inff(), l = 0.f;
        bool  far = false;

        const auto tile = [&](int tok, int from, int2 n, auto odd_c, auto other_c) __attribute__((always_inline)) {
            const unsigned char *sk = sm_k[decltype(odd_c)::value], *sv = sm_v[decltype(odd_c)::value];
            const int            ui = (tok - from) / UNIT;
            const float4v        u0 = unit[ui], u1 = unit[P32 ? ui + 1 : ui];
            float16v             s[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kk][r] = 0.f;
#pragma unroll
            for (int c = 0; c < KS; ++c)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    s[kk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sk + ka[c] + kk * 32 * ROW), qf[c], s[kk], 0, 0, 0);
            // reads stay AHEAD operands in front of their products
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 1);
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
            }
            const bool odd = n.x < 0 || n.x >= 0x40000000 || (P32 && (n.y < 0 || n.y >= 0x40000000));
            float      f[2] = {u0[0] * c2, u1[0] * c2};
            if (odd || tok + kStep > seen_by_all) {
                int upto = limit;
                __asm__ volatile("" : "+v"(upto), "+v"(f[0]), "+v"(f[1])); // a branch, not selects in every tile
                // what is not seen first, since its product with a scale of zero would be NaN; what is seen of a page whose
                // value scale is no number is none
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const bool  none = (P32 && kk ? n.y : n.x) < 0;
                    const float poison = (kk ? u1 : u0)[1] * 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[kk][r] = none || tok + 32 * kk + 8 * (r >> 2) + 4 * h + (r & 3) >= upto ? -__builtin_inff() : __builtin_fmaf(s[kk][r], f[kk], poison);
                    f[kk] = 1.f;
                }
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                float x = s[kk][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) x = fmaxf(x, s[kk][r]);
                top = fmaxf(top, x * f[kk]);
            }
            top = wide_max_halves(top);
            if (__any(top - m > kWeightBits + 1.f)) {
                float up = top - kWeightBits;
                if (top - up > kWeightBits + 1.f) up = top; // exponents from 2^25 on, 4 or more apart
                const float to = fmaxf(m, up), alpha = exp2_hw(m - (to == -__builtin_inff() ? 0.f : to));
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
                m   = to;
                far = __any(fabsf(m) >= 0x1p20f && m > -__builtin_inff());
            }
            float base = m == -__builtin_inff() ? 0.f : m;
            if (far) { // products rounded as the maximum's was
#pragma clang fp contract(off)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kk][r] = s[kk][r] * f[kk] - base;
                    f[kk] = 1.f;
                }
                base = 0.f;
            }
            half8 pf[4];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const float away = base - (kk ? u1 : u0)[2];
                float       sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    typedef float F2 __attribute__((ext_vector_type(2)));
                    const F2     p = {exp2_hw(__builtin_fmaf(s[kk][r], f[kk], -away)), exp2_hw(__builtin_fmaf(s[kk][r + 1], f[kk], -away))};
                    const half2v x = __builtin_convertvector(p, half2v);
                    sum += p[0];
                    sum += p[1];
                    pf[kk * 2 + (r >> 3)][r & 7] = x[0], pf[kk * 2 + (r >> 3)][(r & 7) + 1] = x[1];
                }
                l = __builtin_fmaf(sum, (kk ? u1 : u0)[3], l);
            }
            const auto v_frag = [&](int d, int k) { return *reinterpret_cast<const half8 *>(sv + va[k] + d * (32 * kStep * 2)); };
            const auto in_units = [&](float by) __attribute__((always_inline)) {
                __asm__ volatile("" : "+v"(by));
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= by;
            };
            const float of0 = u0[1] > 0.f ? u0[1] : 1.f, of1 = u1[1] > 0.f ? u1[1] : 1.f;
            if (odd) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if ((k >> 1 ? u1 : u0)[1] == 0.f)
#pragma unroll
                        for (int j = 0; j < 8; ++j) pf[k][j] = (half_t) 0.f; // whatever the bytes of a page of zeros are
                in_units(of0);
            }
            // the next tile's bytes become halves beside the products, or nobody's do
            stage(other_c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (P32 && k == 2 && odd) in_units(of1 / of0);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_frag(d, k), pf[k], acc[d], 0, 0, 0);
            }
            if constexpr (!P32) {
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                for (int i = 0; i < 4 * DB; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // a product, a read, conversions, a write
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
                    if (i & 1) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
                }
            }
            if (odd) in_units(1.f / of1);
        };

        const std::integral_constant<int, 0> even;
        const std::integral_constant<int, 1> odd;
        for (;;) {
            settle();
            stage(even);
            __syncthreads();
            const int end = min(t1, from + 256 * UNIT);
            int2      n0 = names(from, from), n1 = n0;
            for (int tok = from; tok < end; tok += 2 * kStep) {
                const bool second = tok + kStep < end, third = tok + 2 * kStep < end;
                if (second) {
                    n1 = names(tok + kStep, from);
                    fetch(tok + kStep, n1);
                }
                tile(tok, from, n0, even, odd);
                __syncthreads();
                if (!second) break;
                if (third) {
                    n0 = names(tok + 2 * kStep, from);
                    fetch(tok + 2 * kStep, n0);
                }
                tile(tok + kStep, from, n1, odd, even);
                __syncthreads();
            }
            from += 256 * UNIT;
            if (from >= t1) break;
            ask(from);
            fetch(from, first_names(from));
        }

        l += __shfl_xor(l, 32);
        l *= 1.f / (1 << kWeightBits); // the products have it in their values
        const int3 me = row_of(again(lane));
        const int  seq = me.x, r0 = me.y;
        if (!me.z) return;
        const int64_t at = (((int64_t) seq * a.c.heads + head) * a.rows + r0) * (a.shared_splits + a.splits) + split;
        float        *o = a.part_o + at * D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int ch = 32 * d + 2 * r + 4 * h;
                if (ch < D) *reinterpret_cast<float4v *>(o + ch) = float4v {acc[d][r] * vref, acc[d][r + 1] * vref, acc[d][r + 2] * vref, acc[d][r + 3] * vref};
            }
        if (h == 0) *reinterpret_cast<float2 *>(a.part_s + at * 2) = make_float2(m, l);
#endif
    }

    template <typename T, int DP, bool P32>
    static void kv_wide_waves(const KvAttnArgs &a, dim3 grid, hipStream_t s) {
        if constexpr (DP == 128)
            if (a.wide == 2) return kv_wide_kernel<T, DP, P32, 8><<<grid, 512, 0, s>>>(a);
        kv_wide_kernel<T, DP, P32, 4><<<grid, 256, 0, s>>>(a);
    }
    template <typename T, int DP>
    static void kv_wide_pages(const KvAttnArgs &a, dim3 grid, hipStream_t s) {
        if (a.c.page_tokens == 32) kv_wide_waves<T, DP, true>(a, grid, s);
        else kv_wide_waves<T, DP, false>(a, grid, s);
    }
    int kv_wide_run(const KvAttnArgs &a, bool bf16, hipStream_t s) {
        // blocks last: those past the last group's, which find nothing to do, then wait for no place
        const dim3 grid((unsigned) a.c.heads, (unsigned) a.shared_splits, (unsigned) a.shared_blocks);
        if (a.c.row == 64) bf16 ? kv_wide_pages<bf16_t, 64>(a, grid, s) : kv_wide_pages<half_t, 64>(a, grid, s);
        else bf16 ? kv_wide_pages<bf16_t, 128>(a, grid, s) : kv_wide_pages<half_t, 128>(a, grid, s);
        return check_launch("kv_attention_shared prefix");
    }

} // namespace vkhip
