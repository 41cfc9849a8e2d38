// A prefix of the 8-bit cache that many rows share (sequences x query heads x tokens): scores and values as products of
// whole tiles.
//
// A wave owns 32 rows, a workgroup 128 (four waves) or 256 (eight). As in the attention over packed sequences, scores come out transposed (S^T = K Q^T,
// 32x32x16) and the exponentials are, as they lie in the registers, the operand of O^T += V^T P^T; the cache keeps the
// values by channel, so V^T needs no turning, only its tokens in the order in which a lane holds their weights: of each 16,
// 0-3 8-11 | 4-7 12-15. Bytes become fp16 once for all waves, on their way from memory through registers into LDS,
// a tile of 64 tokens ahead.
// Weights are up to 2^15, as they are in the attention of one sequence, and rescaled where a row's maximum grows by more
// than 2; a page's value scale goes into its weights' exponents, relative to a power of two at or above the largest of the
// workgroup's span (2^10 at most, which scales of fp16 rows stay under), so that the products of all pages add up in place. A
// page under 2^-8 of that, or above it, takes products of its own, which are multiplied by its scale in fp32. Weights of a
// page are thus lost from 2^-30 of a row's largest on where its scale is 2^-8 of the span's, from 2^-38 on otherwise.
//
// Bound by instruction issue beside the products: 1024 rows behind 32768 tokens, 8 heads of 128, 157 to 168 us by the card, up to
// 875 TFLOP/s (a library product of 16384^3 1340); matrix units busy 41% of the time, vector units 46%, two waves a SIMD; start
// and end of a workgroup, queries in and parts out, take about 10 us of it. Value scales are 0 or more, as kv_append makes them:
// of a negative one the weights' exponents have no logarithm.
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

    // NW: waves of a workgroup, 4 (two such a compute unit, with 64 channels three) or, where a group has the rows, 8, which share what
    // is converted.
    template <typename T, int DP, bool P32, int NW>
    __global__ __launch_bounds__(NW * 64, 2) void kv_wide_kernel(KvAttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int KS = DP / 16, DB = DP / 32, ROW = DP * 2, PIECES = DP / 8; // contraction steps of a score, output blocks, bytes and pieces of a row of K
        constexpr int LOADS = DP / (16 * NW);                                    // 16-byte loads of K, and of V, per thread and tile
        constexpr int AHEAD = 6, ROWS = 32 * NW; // operands read in front of their products; rows of a workgroup
        constexpr int UNIT  = P32 ? 32 : kStep;                                  // tokens of one page, as many as a tile takes
        __shared__ __attribute__((aligned(1024))) unsigned char sm_k[2][kStep * ROW], sm_v[2][kStep * ROW];
        __shared__ float4v unit[256]; // of a unit's page: key scale; factor of its products (NaN: its value scale is no number); log2 of the one of its weights, and back
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
        float vref = 0x1p-126f; // the scale that O is in units of, a power of two
        float16v acc[DB];
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
            const bool  number = vs >= 0.f && vs < __builtin_inff();
            float       larger = number ? vs : 0.f;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) larger = fmaxf(larger, __shfl_xor(larger, o));
            if (lane == 0) wave_vs[wave] = larger;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) larger = fmaxf(larger, wave_vs[i]);
            vref = fminf(fmaxf(__uint_as_float((__float_as_uint(larger) + 0x7FFFFFu) & 0x7F800000u), 0x1p-126f), 0x1p10f);
            // a page near it has its share in its weights, any other beside its products: vref is no more than 2^10, so that this
            // factor is as good as the scale itself, however large the scale of a page is that some rows do not see
            const float ratio = vs / vref;
            const bool  near  = ratio >= 0x1p-8f && ratio <= 1.f;
            if (tid >= 256) return;
            unit_id[tid] = unit_page < 0 ? -1 : near && ks > 0.f ? unit_page : unit_page | 0x40000000;
            unit[tid]    = float4v {ks, near ? 1.f : number ? ratio : __builtin_nanf(""), near ? __builtin_amdgcn_logf(ratio) : 0.f, near ? 1.f / ratio : 1.f};
        };
        // the names of the pages of tile i of those in LDS, the same in every lane
        const auto names = [&](int i) {
            return make_int2(__builtin_amdgcn_readfirstlane(unit_id[i * (kStep / UNIT)]), P32 ? __builtin_amdgcn_readfirstlane(unit_id[i * 2 + 1]) : 0);
        };
        const auto page = [](int id) { return id < 0 ? 0 : id & 0x3FFFFFFF; }; // one without memory is read elsewhere and masked
        const auto odd_page = [](int2 n) { return n.x < 0 || n.x >= 0x40000000 || (P32 && (n.y < 0 || n.y >= 0x40000000)); };

        const auto first_names = [&](int tok) { return make_int2(page_of(tok), P32 ? page_of(tok + UNIT) : 0); }; // before they are in LDS
        // a tile's bytes: piece p of K is token p / (DP / 16), 16 channels from p % (DP / 16) on; of V channel p / 4, 16 tokens
        // from p % 4 on
        tk_u32x4      kr[LOADS], vr[LOADS];
        const int64_t page_bytes = (int64_t) P * DP;
        const auto    fetch_k = [&](int tok, int2 n, tk_u32x4 (&to)[LOADS]) __attribute__((always_inline)) {
            const unsigned char *kp[2];
#pragma unroll
            for (int u = 0; u < (P32 ? 2 : 1); ++u) kp[u] = a.c.k + ((int64_t) page(u ? n.y : n.x) * a.c.heads + head) * page_bytes + (P32 ? 0 : tok & (P - 1)) * DP;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = i * (NW * 64) + tid, kt = p / (DP / 16), kc = p % (DP / 16) * 16;
                if constexpr (P32) to[i] = *reinterpret_cast<const tk_u32x4 *>((kt >> 5 ? kp[1] : kp[0]) + (unsigned) ((kt & 31) * DP + kc));
                else to[i] = *reinterpret_cast<const tk_u32x4 *>(kp[0] + (unsigned) (kt * DP + kc));
            }
        };
        const auto fetch_v = [&](int tok, int2 n) __attribute__((always_inline)) {
            const unsigned char *vp[2];
#pragma unroll
            for (int u = 0; u < (P32 ? 2 : 1); ++u) vp[u] = a.c.v + ((int64_t) page(u ? n.y : n.x) * a.c.heads + head) * page_bytes + (P32 ? 0 : tok & (P - 1));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = i * (NW * 64) + tid, vc = p / 4, vt = p % 4 * 16;
                if constexpr (P32) vr[i] = *reinterpret_cast<const tk_u32x4 *>((vt >> 5 ? vp[1] : vp[0]) + (unsigned) (vc * P + (vt & 31)));
                else vr[i] = *reinterpret_cast<const tk_u32x4 *>(vp[0] + (unsigned) (vc * P + vt));
            }
        };
        // the first tile's bytes and the pages' scales are on their way while the queries are
        // (K of a tile is needed one round before its V)
        const int from = t0;
        tk_u32x4 k0[LOADS];
        const auto begin = [&]() __attribute__((always_inline)) {
            ask(from);
            const int2 n0 = first_names(from), n1 = first_names(from + kStep);
            fetch_k(from, n0, k0);
            fetch_k(from + kStep, n1, kr);
            fetch_v(from, n0);
        };
        begin();

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
        // where a lane's first operands lie, and this thread's pieces go: c pieces on is an xor of bits from 5 on
        const unsigned ka = k_at(col, h), va = v_at(col, h), kw = k_at(tid / (DP / 16), tid % (DP / 16) * 2), vw = v_at(tid / 4, tid % 4 * 2);
        const auto stage_k = [&](unsigned char *sk, tk_u32x4 (&x)[LOADS]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) { // 32 tokens on: rows of the same permutation
                *reinterpret_cast<half8 *>(sk + kw + i * 8192)        = i8_to_h8<0>(x[i][0], x[i][1]);
                *reinterpret_cast<half8 *>(sk + (kw ^ 16) + i * 8192) = i8_to_h8<0>(x[i][2], x[i][3]);
            }
        };
        const auto stage_v = [&](unsigned char *sv) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) { // 64 channels on
                *reinterpret_cast<half8 *>(sv + vw + i * 8192)        = i8_to_h8<kWeightBits>(vr[i][0], vr[i][2]);
                *reinterpret_cast<half8 *>(sv + (vw ^ 16) + i * 8192) = i8_to_h8<kWeightBits>(vr[i][1], vr[i][3]);
            }
        };

        float    m = -__builtin_inff(), l = 0.f;
        bool     far = false;
        float16v s[2];
        half8    pf[4];

        // Round i of a wave: the products O += V P of tile i - 1 and S = K Q of tile i, beside them K of tile i + 1 and V of
        // tile i into LDS, whose places tiles i - 1 and i - 2 have left; then the exponentials of tile i, and a barrier.
        const auto values = [&](int i, int2 n, int place) __attribute__((always_inline)) {
            const unsigned at = va + place * (kStep * 2 * DP);
            const auto     product = [&](int k) __attribute__((always_inline)) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sm_v[0] + (at ^ k << 5) + d * (32 * kStep * 2)), pf[k], acc[d], 0, 0, 0);
            };
            if (odd_page(n)) { // page by page, and nothing of them left for the others; a row that sees one of no number has weights of none
#pragma unroll
                for (int u = 0; u < (P32 ? 2 : 1); ++u) {
                    const float scale = unit[again(P32 ? i * 2 + u : i)][1], f = scale > 0.f ? scale : 0.f;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        float16v x;
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
                        for (int k = P32 ? 2 * u : 0; k < (P32 ? 2 * u + 2 : 4); ++k)
                            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sm_v[0] + (at ^ k << 5) + d * (32 * kStep * 2)), pf[k], x, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[d][r] = __builtin_fmaf(x[r], f, acc[d][r]);
                        __builtin_amdgcn_sched_barrier(0); // one product's registers at a time
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < 8; ++j) pf[k][j] = (half_t) 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) product(k);
        };
        const auto scores = [&](int place) __attribute__((always_inline)) {
            const unsigned at = ka + place * (kStep * ROW);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kk][r] = 0.f;
#pragma unroll
            for (int c = 0; c < KS; ++c)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    s[kk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(sm_k[0] + (at ^ c << 5) + kk * 32 * ROW), qf[c], s[kk], 0, 0, 0);
        };
        // the order of the products and what is beside them: reads AHEAD of their products, and after each a read, a few
        // conversions, every other time a write
        const auto beside = [&](auto products) __attribute__((always_inline)) {
            constexpr int N = decltype(products)::value, EACH = (80 * LOADS / 2 + N - 1) / N + 1;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, EACH, 0);
                if (i & 1) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            }
        };
        const auto weights = [&](int i, int2 n) __attribute__((always_inline)) {
            const int     tok = from + i * kStep;
            const float4v u0 = unit[i * (kStep / UNIT)], u1 = unit[P32 ? i * 2 + 1 : i];
            float         f[2] = {u0[0] * c2, u1[0] * c2};
            if (odd_page(n) || tok + kStep > seen_by_all) {
                int upto = limit;
                __asm__ volatile("" : "+v"(upto), "+v"(f[0]), "+v"(f[1])); // a branch, not selects in every tile
                // what is not seen first, since its product with a scale of zero would be NaN; what is seen of a page whose
                // value scale is no number is none
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int   seen = (P32 && kk ? n.y : n.x) < 0 ? 0 : upto - tok - 32 * kk - 4 * h; // of the block's tokens, from 4 h on
                    const float poison = (kk ? u1 : u0)[1] * 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[kk][r] = 8 * (r >> 2) + (r & 3) >= seen ? -__builtin_inff() : __builtin_fmaf(s[kk][r], f[kk], poison);
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
        };
        // loads stay under way across these
        const auto barrier = [] __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): this wave's writes
            __asm__ volatile("s_barrier" ::: "memory");
        };
        {
            settle();
            stage_k(sm_k[0], k0);
            __syncthreads();
            const int tiles = (t1 - t0 + 2 * kStep - 1) / (2 * kStep) * 2; // an even number: one without pages behind an odd one
            int2      before, now = names(0), next = names(min(1, tiles - 1)); // tiles i - 1, i, i + 1
            const auto ahead = [&](int i) __attribute__((always_inline)) {  // K of tile i + 2, V of tile i + 1; the last ones again behind them
                const int v = min(i + 1, tiles - 1), k = min(i + 2, tiles - 1);
                before = now, now = next, next = names(k);
                fetch_v(from + v * kStep, now);
                fetch_k(from + k * kStep, next, kr);
            };
            scores(0);
            stage_k(sm_k[1], kr), stage_v(sm_v[0]);
            ahead(0);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
            const auto round = [&](int i, auto odd_c) __attribute__((always_inline)) {
                constexpr int ODD = decltype(odd_c)::value;
                weights(i, before);
                barrier();
                values(i, before, ODD);
                scores(ODD ^ 1); // behind the last tile its scores are formed again, for nobody
                stage_k(sm_k[ODD], kr), stage_v(sm_v[ODD ^ 1]);
                beside(std::integral_constant<int, 4 * DB + 2 * KS>());
                ahead(i + 1);
            };
#pragma unroll 1
            for (int i = 0; i < tiles; i += 2) {
                round(i, std::integral_constant<int, 0>());
                round(i + 1, std::integral_constant<int, 1>());
            }
        }

        l += __shfl_xor(l, 32);
        l *= 1.f / (1 << kWeightBits); // the products have it in their values
        const int3 me = row_of(again(lane));
        // 64 bits: a wide table alone makes 2^31 parts, however few of them a call has
        const int64_t at = me.z ? (((int64_t) me.x * a.c.heads + head) * a.rows + me.y) * (a.shared_splits + a.splits) + split : -1;
        if (h == 0 && at >= 0) *reinterpret_cast<float2 *>(a.part_s + at * 2) = make_float2(m, l);
        // through LDS, 64 channels at a time, so that rows leave in whole lines (4 of 11 us for a call of 4 tiles otherwise)
        __syncthreads();
        unsigned char *own = (wave < NW / 2 ? sm_k[0] : sm_v[0]) + wave % (NW / 2) * 8192;
#pragma unroll
        for (int e = 0; e < DP / 64; ++e) {
#pragma unroll
            for (int d = 2 * e; d < 2 * e + 2; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) // channels 32 d + 2 r + 4 h .. + 3
                    *reinterpret_cast<float4v *>(own + col * 256 + ((8 * (d & 1) + r / 2 + h ^ (col & 15)) << 4)) =
                        float4v {acc[d][r] * vref, acc[d][r + 1] * vref, acc[d][r + 2] * vref, acc[d][r + 3] * vref};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int     row = 4 * i + (lane >> 4), piece = lane & 15, ch = 64 * e + 4 * piece;
                const float4v x = *reinterpret_cast<const float4v *>(own + row * 256 + ((piece ^ (row & 15)) << 4));
                const int64_t to = __shfl((long long) at, row);
                if (to >= 0 && ch < D) *reinterpret_cast<float4v *>(a.part_o + to * D + ch) = x;
            }
        }
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
