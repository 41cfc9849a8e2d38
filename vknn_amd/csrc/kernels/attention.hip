// Attention over packed sequences (whole prompts, images as tokens): one pass over the keys per tile of 128
// queries with a running maximum and sum.
//
// A wave owns 32 queries. Scores come out transposed, S^T = K Q^T (32x32x16 tiles: a lane holds one query and 16
// keys of each 32), so maximum and sum of a row are sums within a lane and one exchange between the wave's
// halves, and the exponentials are, as they lie in the registers, the operand of O^T += V^T P^T: which key sits in
// which contraction slot is free as long as V's side agrees, and the transposing LDS read (ds_read_b64_tr_b16)
// brings V's columns four keys at a time, in that order. O stays in registers.
// K and V tiles of 64 keys go from memory into LDS without passing registers, one tile ahead; rows are stored
// with their 16-byte pieces permuted (xor with the row) so that neither read pattern meets a bank twice.
//
// The weights are rounded to the type of V, since both operands of a product have one type: an error of 2^-11
// (fp16) or 2^-8 (bf16) of each term, where the output itself is rounded by as much. Their sum stays fp32. fp16
// weights are raised by 2^7 to 2^15, so that many small ones beside a large one are not lost.
//
// Bound by the matrix and vector units together, and by power: 16384 causal queries, 32 heads on 8, D = 128, fp16
// 2.06 to 2.17 ms by the card's clock (1067 to 1014 TFLOP/s; a 16384^3 library product 1246), 1.65 to 1.5 GHz, matrix
// units busy 61% of it, vector units 51%, no bank conflicts. 4 x 4096 not causal 1031, D = 64 bf16 954 TFLOP/s. Head dims
// other than 64 and 128 take the next width's products: 4 x 4096 causal, fp16, TFLOP/s of D's own products at D = 32,
// 64, 80, 96, 112, 128: 422, 820, 674, 780, 855, 951. A tile of 128 queries of one head is mostly padding where queries
// are few, and each head reads the keys again: 200 queries behind 50000 keys 96 us, 16 behind 9000 (32 heads) 30.
// Two workgroups a compute unit (LDS 72 KB, up to 256 registers) overlap one's exponentials with the other's
// products; raising a wave's priority around its products or loading V's first fragments earlier changed nothing.
#include "tokens.h"
#include <type_traits>

namespace vkhip {

    struct AttnArgs {
        const void    *q, *k, *v;
        void          *o;
        const int32_t *cu_q, *cu_k;
        int            batch, q_heads, kv_heads, head_dim, total_q, total_k, causal;
        float          c2; // scale * log2(e)
        int            splits;          // of a tile's keys
        float         *part_o, *part_s; // per split, query and head: O before its division, and (reference, sum)
        int64_t        q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    };

    template <typename T>
    struct AttnType;
    template <>
    struct AttnType<half_t> {
        typedef half8 V8;
        typedef half4 V4;
        static constexpr unsigned kExp = 0x7C00u; // bits of infinity
        // The exponents' reference lies this far below a maximum when it is set, and up to 8 further as the maximum grows:
        // fp16 weights from 2^7 up to 2^15 for the largest, whose smallest step, 2^-24, is then 2^-31 of it or less.
        static constexpr float kUp = 7.f;
        static __device__ __forceinline__ float16v mfma(V8 a, V8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    };
    template <>
    struct AttnType<bf16_t> {
        typedef bf8 V8;
        typedef bf4 V4;
        static constexpr unsigned kExp = 0x7F80u;
        static constexpr float    kUp  = 0.f; // fp32's range
        static __device__ __forceinline__ float16v mfma(V8 a, V8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    };

    constexpr int kAttnQ = 128, kAttnK = 64;

    // Which 16-byte piece of a tile's LDS row `row` holds the row's piece `piece`. K is read by 32 rows at one piece,
    // V by 8 rows at 4 neighbouring ones.
    template <int DP>
    __device__ __forceinline__ int k_swizzle(int row) { return DP == 128 ? row & 15 : row >> 1 & 7; }
    template <int DP>
    __device__ __forceinline__ int v_swizzle(int row) { return DP == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2; }

    // The larger of a lane's value and that of lane ^ 32.
    __device__ __forceinline__ float max_halves(float x) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }

#if defined(__HIP_DEVICE_COMPILE__) // the host pass knows neither the LDS address space of these nor the reads
    typedef __attribute__((address_space(3))) unsigned char *LdsPtr;
    typedef short attn_s4 __attribute__((ext_vector_type(4)));

    // 4 x 16 values of 16 bits per 16 lanes, transposed: lane i of the 16 points at 4 values of row i / 4 (columns
    // 4 (i % 4) ..) and gets column i, rows 0 .. 3.
    __device__ __forceinline__ tk_u32x2 lds_read_tr(LdsPtr p) {
        return __builtin_bit_cast(tk_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn_s4 *) p));
    }
    __device__ __forceinline__ tk_u32x4 lds_read16(LdsPtr p) { return *(__attribute__((address_space(3))) const tk_u32x4 *) p; }

#endif

    template <typename T, int DP>
    __global__ __launch_bounds__(256, 2) void attn_packed_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
        using A              = AttnType<T>;
        using V8             = typename A::V8;
        constexpr int PIECES = DP / 8;            // 16-byte pieces of a row
        constexpr int ROW    = DP * 2;            // bytes of a row
        constexpr int TILE   = kAttnK * ROW;      // bytes of a K or V tile
        constexpr int LOADS  = TILE / 1024 / 4;   // wave loads of 1 KB per wave and tile
        constexpr int KS = DP / 16, DB = DP / 32; // contraction steps of a score, 32-channel blocks of the output
        // arrays of their own for K and V of even and odd tiles: the compiler then knows that a read of one does not
        // have to wait for the copies into the others
        __shared__ __attribute__((aligned(1024))) unsigned char sm_k0[TILE], sm_v0[TILE], sm_k1[TILE], sm_v1[TILE];
        __shared__ __attribute__((aligned(16))) unsigned char   sm_w[4 * kAttnK * 32]; // the waves' weights of 32 keys
        __shared__ unsigned                                     found[8];
        const auto k_tile = [&](auto odd_c) { return odd_c ? (LdsPtr) sm_k1 : (LdsPtr) sm_k0; };
        const auto v_tile = [&](auto odd_c) { return odd_c ? (LdsPtr) sm_v1 : (LdsPtr) sm_v0; };

        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
        // heads of one key/value head next to each other in the grid: workgroups go to the 8 XCDs in turn; then splits, and
        // tiles over the other dimensions
        const int head_kv = blockIdx.x % a.kv_heads, group = a.q_heads / a.kv_heads;
        const int head_q = head_kv * group + blockIdx.x / a.kv_heads % group, split = blockIdx.x / a.q_heads;
        const int item   = (int) (blockIdx.z * gridDim.y + blockIdx.y);
        // the most work first, where that is known: with causal a sequence's last queries see the most keys
        const auto count = [&](int b) { return (clampi(a.cu_q[b + 1], 0, a.total_q) - clampi(a.cu_q[b], 0, a.total_q) + kAttnQ - 1) / kAttnQ; };
        SeqTile w = a.causal && a.batch <= 64 ? find_tile_falling(item, a.batch, count) : find_tile(item, a.batch, count);
        if (a.causal && a.batch > 64 && w.b >= 0) w.tile = count(w.b) - 1 - w.tile;
        if (w.b < 0) return;
        const int b  = __builtin_amdgcn_readfirstlane(w.b);
        const int q0 = clampi(a.cu_q[b], 0, a.total_q), nq = clampi(a.cu_q[b + 1], 0, a.total_q) - q0;
        const int k0 = clampi(a.cu_k[b], 0, a.total_k), nk = max(0, clampi(a.cu_k[b + 1], 0, a.total_k) - k0);
        const int i0 = __builtin_amdgcn_readfirstlane(w.tile) * kAttnQ;
        const int shift = nk - nq;
        const int D     = a.head_dim;

        // keys below `limit` are seen; queries past the last one compute something that is not stored
        const int qi    = i0 + wave * 32 + col;
        const int limit = a.causal ? min(nk, qi + shift + 1) : nk;
        const int k_end = max(0, a.causal ? min(nk, min(i0 + kAttnQ, nq) + shift) : nk);
        const int all = (k_end + kAttnK - 1) / kAttnK, per = ((all + a.splits - 1) / a.splits + 1) & ~1;
        const int first = min(all, split * per), tiles = min(all, first + per); // this split's tiles
        // the first tiles, an even number, are seen whole by every query of the workgroup (an odd one goes with the masked)
        const int plain = min(tiles, max(0, a.causal ? min(nk, i0 + shift + 1) : nk) / kAttnK) & ~1;
        // and this wave has no use for tiles from `used` on
        const int w_first = i0 + wave * 32;
        const int used    = w_first < nq ? (max(0, a.causal ? min(nk, min(w_first + 32, nq) + shift) : nk) + kAttnK - 1) / kAttnK : 0;

        V8 qf[KS];
        {
            const T *src = (const T *) a.q + (int64_t) (q0 + qi) * a.q_row + (int64_t) head_q * a.q_head;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 16 * s + 8 * h;
#pragma unroll
                for (int j = 0; j < 8; ++j) qf[s][j] = (T) 0.f;
                if (qi < nq && d < D) qf[s] = *reinterpret_cast<const V8 *>(src + d);
            }
        }

        const char *kb = (const char *) ((const T *) a.k + (int64_t) (k0 + first * kAttnK) * a.k_row + (int64_t) head_kv * a.k_head);
        const char *vb = (const char *) ((const T *) a.v + (int64_t) (k0 + first * kAttnK) * a.v_row + (int64_t) head_kv * a.v_head);
        const int   k_bytes = (int) a.k_row * 2, v_bytes = (int) a.v_row * 2;
        // this lane's source offsets: piece p of the LDS image is row p / PIECES, piece (p % PIECES) ^ swizzle(row)
        unsigned off_k[LOADS], off_v[LOADS];
#pragma unroll
        for (int r = 0; r < LOADS; ++r) {
            const int p = (wave * LOADS + r) * 64 + lane, row = p / PIECES, at = p % PIECES;
            const int ck = at ^ k_swizzle<DP>(row), cv = at ^ v_swizzle<DP>(row);
            off_k[r]     = ck * 8 < D ? (unsigned) (row * k_bytes + ck * 16) : 0x80000000u;
            off_v[r]     = cv * 8 < D ? (unsigned) (row * v_bytes + cv * 16) : 0x80000000u;
        }
        // past the sequence's last row, where the resource ends, and past the head's channels the copy writes zeros
        auto issue = [&](int t, auto odd_c) __attribute__((always_inline)) {
            const int rows = min(kAttnK, nk - t * kAttnK) - 1;
            const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void *) kb, (short) 0, rows * k_bytes + D * 2, 0x00020000);
            const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void *) vb, (short) 0, rows * v_bytes + D * 2, 0x00020000);
            kb += (int64_t) kAttnK * k_bytes, vb += (int64_t) kAttnK * v_bytes;
            const LdsPtr kd = k_tile(odd_c) + wave * (LOADS * 1024), vd = v_tile(odd_c) + wave * (LOADS * 1024);
#pragma unroll
            for (int r = 0; r < LOADS; ++r) __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, kd + r * 1024, 16, off_k[r], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < LOADS; ++r) __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, vd + r * 1024, 16, off_v[r], 0, 0, 0);
        };

        // fragment offsets in a tile: K row col, piece 2 c + h; V rows 4 h + (lane % 16) / 4 (+ 8), pieces 4 d + pp.
        // The swizzle is an xor of disjoint bits, so that rows further on are constant offsets.
        unsigned ka[KS], va[DB][2];
#pragma unroll
        for (int c = 0; c < KS; ++c) ka[c] = col * ROW + (((2 * c + h) ^ k_swizzle<DP>(col)) << 4);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 4 * h + ((lane & 15) >> 2) + 8 * e, piece = 4 * d + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
                va[d][e]      = row * ROW + ((piece ^ v_swizzle<DP>(row)) << 4) + (lane & 1) * 8;
            }

        float16v acc[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
        // sign bits of the two values whose exponent is all ones: a carry goes there
        const auto not_finite = [](unsigned two) { return ((two & (A::kExp * 0x10001u)) + (0x8000u - A::kExp) * 0x10001u) & 0x80008000u; };
        // the reference of the exponents, kUp to kUp + 8 below the largest one seen: weights up to 2^8 times as large cost
        // no digits, and O is rescaled only where a maximum grows by more than that
        float m = -__builtin_inff(), l = 0.f;
        bool  far = false; // a reference of the wave is 2^20 or more, either way

        // A weight of zero does not keep a NaN or an infinity of V out of a product. Where something is masked, each wave
        // looks through the piece of V that it copied and clears what it finds (`spoiled`: something was); what the
        // queries do see of it is then added key by key, read from memory again.
        auto tile = [&](int t, auto odd_c, auto masked_c, bool spoiled) __attribute__((always_inline)) {
            const LdsPtr   kt = k_tile(odd_c), vt = v_tile(odd_c);
            constexpr bool MASKED = decltype(masked_c)::value;
            const int      key0   = t * kAttnK;
            const auto     seen   = [&](int k, int j) { return key0 + 16 * k + 8 * (j >> 2) + 4 * h + (j & 3) < limit; };
            float16v       s[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kk][r] = 0.f;
#pragma unroll
                for (int c = 0; c < KS; ++c) s[kk] = A::mfma(__builtin_bit_cast(V8, lds_read16(kt + ka[c] + kk * 32 * ROW)), qf[c], s[kk]);
            }
            if constexpr (MASKED) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!seen(2 * kk + (r >> 3), r & 7)) s[kk][r] = -__builtin_inff();
            }
            float top = s[0][0];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kk][r]);
            top = max_halves(top) * a.c2;
            if (__any(top - m > 8.f + A::kUp)) {
                const float to    = fmaxf(m, top - A::kUp);
                const float alpha = exp2_hw(m - (to == -__builtin_inff() ? 0.f : to));
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
                m   = to;
                far = __any(fabsf(m) >= 0x1p20f && m > -__builtin_inff());
            }
            float base = m == -__builtin_inff() ? 0.f : m, mul = a.c2;
            if (far) {
                // fp32 is 1/8 or coarser there: the products are rounded as the maximum's was, which one rounding of
                // product and difference together would miss by up to half a step, any power of two. The branch costs
                // up to 1% (4 x 4096 causal 570 -> 576 us).
#pragma clang fp contract(off)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kk][r] = s[kk][r] * a.c2 - base;
                mul = 1.f, base = 0.f;
            }
            V8 pf[4];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    typedef float F2 __attribute__((ext_vector_type(2)));
                    typedef T     T2 __attribute__((ext_vector_type(2)));
                    const F2      p = {exp2_hw(__builtin_fmaf(s[kk][r], mul, -base)), exp2_hw(__builtin_fmaf(s[kk][r + 1], mul, -base))};
                    l += p[0];
                    l += p[1];
                    const T2 x = __builtin_convertvector(p, T2);
                    pf[kk * 2 + (r >> 3)][r & 7]       = x[0];
                    pf[kk * 2 + (r >> 3)][(r & 7) + 1] = x[1];
                }
            const auto v_frag = [&](int d, int k) __attribute__((always_inline)) {
                const tk_u32x2 x = lds_read_tr(vt + va[d][0] + k * 16 * ROW), y = lds_read_tr(vt + va[d][1] + k * 16 * ROW);
                return tk_u32x4 {x[0], x[1], y[0], y[1]};
            };
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    acc[d] = A::mfma(__builtin_bit_cast(V8, v_frag(d, k)), pf[k], acc[d]);
                }
            if (MASKED && spoiled) {
                __attribute__((address_space(3))) T *w = (__attribute__((address_space(3))) T *) ((LdsPtr) sm_w + wave * (kAttnK * 32));
                const T *rows = (const T *) a.v + (int64_t) (k0 + key0) * a.v_row + (int64_t) head_kv * a.v_head;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) { // 32 keys at a time, their weights in LDS
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const V8 p = half ? pf[2 + k] : pf[k];
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[(16 * k + 8 * (j >> 2) + 4 * h + (j & 3)) * 32 + col] = p[j];
                    }
                    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): the wave's own weights
#pragma unroll 1
                    for (int key = half * 32; key < min(half * 32 + 32, nk - key0); ++key) {
                        const float p = (float) w[(key & 31) * 32 + col];
                        const T    *v = rows + (int64_t) key * a.v_row + 4 * h;
#pragma unroll
                        for (int d = 0; d < DB; ++d)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if (32 * d + 8 * r + 4 * h >= D) continue;
                                const typename A::V4 x = *reinterpret_cast<const typename A::V4 *>(v + 32 * d + 8 * r);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float y = (float) x[j];
                                    if (key0 + key < limit && !(fabsf(y) < __builtin_inff())) acc[d][4 * r + j] += p * y;
                                }
                            }
                    }
                    __builtin_amdgcn_s_waitcnt(0xC07F); // read before the next half is written
                }
            }
        };

        // tile t has landed (every wave's pieces), and nobody reads tile t - 1 any more
        const auto landed = [] __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(7 << 4); // vmcnt(0), lgkmcnt(0)
            __asm__ volatile("s_barrier" ::: "memory");
        };
        const std::integral_constant<int, 0> even;
        const std::integral_constant<int, 1> odd;
        if (tiles > first) issue(first, even);
        int t = first;
        for (; t < plain; t += 2) {
            landed();
            issue(t + 1, odd);
            if (used) tile(t, even, std::false_type(), false);
            landed();
            if (t + 2 < tiles) issue(t + 2, even);
            if (used) tile(t + 1, odd, std::false_type(), false);
        }
        for (; t < tiles; ++t) {
            const int parity = t & 1;
            __builtin_amdgcn_s_waitcnt(7 << 4); // vmcnt(0), lgkmcnt(0)
            unsigned any = 0;
#pragma unroll
            for (int r = 0; r < LOADS; ++r) {
                LdsPtr   at = v_tile(parity) + (wave * LOADS + r) * 1024 + lane * 16;
                tk_u32x4 v  = lds_read16(at);
                unsigned hit = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned bad = not_finite(v[j]);
                    hit |= bad;
                    v[j] &= ~((bad >> 15) * 0xFFFFu);
                }
                if (hit) *(__attribute__((address_space(3))) tk_u32x4 *) at = v;
                any |= hit;
            }
            const bool mine = __any(any != 0);
            if (lane == 0) found[parity * 4 + wave] = mine;
            __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0)
            __asm__ volatile("s_barrier" ::: "memory");
            if (t + 1 < tiles) issue(t + 1, t + 1 & 1);
            if (t < used) tile(t, parity, std::true_type(), __builtin_amdgcn_readfirstlane(found[parity * 4] | found[parity * 4 + 1] | found[parity * 4 + 2] | found[parity * 4 + 3]) != 0);
        }

        l += __shfl_xor(l, 32);
        if (qi >= nq) return;
        if (a.splits > 1) {
            const int64_t at = ((int64_t) split * a.total_q + q0 + qi) * a.q_heads + head_q;
            if (h == 0) *reinterpret_cast<float2 *>(a.part_s + at * 2) = make_float2(m, l);
            if (first >= tiles) return;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (32 * d + 8 * r + 4 * h < D)
                        *reinterpret_cast<float4v *>(a.part_o + at * D + 32 * d + 8 * r + 4 * h) =
                            float4v {acc[d][4 * r], acc[d][4 * r + 1], acc[d][4 * r + 2], acc[d][4 * r + 3]};
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T          *dst = (T *) a.o + (int64_t) (q0 + qi) * a.o_row + (int64_t) head_q * a.o_head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = 32 * d + 8 * r + 4 * h;
                if (at >= D) continue;
                typename A::V4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (T) (acc[d][4 * r + j] * inv);
                *reinterpret_cast<typename A::V4 *>(dst + at) = x;
            }
#endif
    }

    // Joins the splits of a query and head: a wave each, two channels a lane. Queries in front of the first sequence or
    // behind the last have no partial results, and their rows of o are not this call's.
    template <typename T>
    __global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
        const int64_t rows = (int64_t) a.total_q * a.q_heads, at = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
        if (at >= rows) return;
        const int lane = threadIdx.x & 63, D = a.head_dim, d = lane * 2, q = (int) (at / a.q_heads);
        if (q < a.cu_q[0] || q >= a.cu_q[a.batch]) return;
        float     top = -__builtin_inff(), sum = 0.f, x0 = 0.f, x1 = 0.f;
        for (int k = 0; k < a.splits; ++k) top = fmaxf(top, a.part_s[(k * rows + at) * 2]);
        const float base = top == -__builtin_inff() ? 0.f : top;
        for (int k = 0; k < a.splits; ++k) {
            const float2 s = *reinterpret_cast<const float2 *>(a.part_s + (k * rows + at) * 2);
            if (s.y == 0.f) continue; // nothing seen, perhaps nothing written
            const float f = exp2_hw(s.x - base);
            sum += s.y * f;
            if (d < D) {
                const float2 x = *reinterpret_cast<const float2 *>(a.part_o + (k * rows + at) * D + d);
                x0 += x.x * f, x1 += x.y * f;
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (d >= D) return;
        T *o = (T *) a.o + q * a.o_row + at % a.q_heads * a.o_head + d;
        o[0] = (T) (x0 * inv), o[1] = (T) (x1 * inv);
    }

    // Splits of the keys: where the tiles of queries and heads leave compute units idle (two workgroups fit each), down
    // to 1024 keys. Measured without / with, D = 128: 8192 causal, 4 heads 151 / 115 us; 200 queries behind 50000 keys, 8
    // heads 833 / 98; 16 queries behind 9000, 32 heads 146 / 34.
    static int attn_splits(const vkhip_attention_desc *d) {
        if (d->batch == 0 || d->total_q == 0) return 1;
        const int64_t wgs = (ceil_div(d->total_q, (int64_t) kAttnQ * d->batch) * d->batch) * d->q_heads, keys = ceil_div(d->total_k, d->batch);
        if (wgs >= 512) return 1;
        int64_t n = ceil_div(1024, wgs);
        if (n > keys / 1024) n = keys / 1024;
        return (int) (n < 1 ? 1 : (n > 32 ? 32 : n));
    }

    static const char *attn_refusal(const vkhip_attention_desc *d) {
        if (!d || d->batch < 0 || d->q_heads <= 0 || d->kv_heads <= 0 || d->total_q < 0 || d->total_k < 0) return "bad sizes";
        if (d->q_heads % d->kv_heads) return "q_heads is not a multiple of kv_heads";
        if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8) return "head_dim is not a multiple of 8 up to 128";
        if (d->dtype != VKHIP_DT_F16 && d->dtype != VKHIP_DT_BF16) return "q, k, v and o are F16 or BF16";
        if (!(d->scale > 0.f) || d->scale > 1e30f) return "scale is not positive";
        const int64_t st[8] = {d->q_row, d->q_head, d->k_row, d->k_head, d->v_row, d->v_head, d->o_row, d->o_head};
        for (int64_t v: st)
            if (v < 0 || v % 8) return "strides are not multiples of 8";
        if (d->k_row < d->head_dim || d->v_row < d->head_dim || d->k_row > (1 << 23) || d->v_row > (1 << 23)) return "k_row or v_row under head_dim or over 2^23";
        if (rows_overlap(d->total_q, d->o_row, d->q_heads, d->o_head, d->head_dim)) return "rows of o share memory";
        // a dimension of a launch has fewer than 2^32 threads, 256 of them a head
        if ((ceil_div(d->total_q, kAttnQ) + d->batch) * (int64_t) d->q_heads > 0x3FFFFFF || d->q_heads > 0xFFFFFF) return "too many queries and heads";
        return nullptr;
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

size_t vkhip_attention_workspace_bytes(const vkhip_attention_desc *d) {
    if (attn_refusal(d)) return 0;
    const int n = attn_splits(d);
    return n == 1 ? 0 : (size_t) n * d->total_q * d->q_heads * (d->head_dim + 2) * sizeof(float);
}

int vkhip_attention_packed(const vkhip_attention_desc *d, const void *q, const void *k, const void *v, const int32_t *cu_q, const int32_t *cu_k,
                           void *o, void *workspace, vkhip_stream_t s) {
    if (const char *why = attn_refusal(d)) return set_error(VKHIP_ERR_INVALID, "attention_packed: %s", why);
    if (d->batch == 0 || d->total_q == 0) return VKHIP_OK;
    const int splits = attn_splits(d);
    if (!q || !o || !cu_q || !cu_k || (d->total_k > 0 && (!k || !v)) || (splits > 1 && !workspace)) return set_error(VKHIP_ERR_INVALID, "attention_packed: null pointer");
    if (misaligned16(q) || misaligned16(k) || misaligned16(v) || misaligned16(o) || misaligned16(workspace) || ((uintptr_t) cu_q | (uintptr_t) cu_k) % 4)
        return set_error(VKHIP_ERR_INVALID, "attention_packed: misaligned pointer");
    AttnArgs a {};
    a.q = q, a.k = k, a.v = v, a.o = o, a.cu_q = cu_q, a.cu_k = cu_k;
    a.batch = d->batch, a.q_heads = d->q_heads, a.kv_heads = d->kv_heads, a.head_dim = d->head_dim, a.total_q = d->total_q, a.total_k = d->total_k;
    a.causal = d->causal != 0, a.c2 = d->scale * 1.44269504088896f;
    a.q_row = d->q_row, a.q_head = d->q_head, a.k_row = d->k_row, a.k_head = d->k_head;
    a.v_row = d->v_row, a.v_head = d->v_head, a.o_row = d->o_row, a.o_head = d->o_head;
    a.splits = splits, a.part_o = (float *) workspace, a.part_s = a.part_o + (size_t) splits * d->total_q * d->q_heads * d->head_dim;
    // sequences have fewer than total_q / 128 + batch tiles together
    int64_t tiles = d->total_q / kAttnQ + d->batch;
    if (tiles > d->total_q) tiles = d->total_q;
    const int64_t layers = ceil_div(tiles, 65535); // the second dimension's limit
    const dim3  grid((unsigned) (d->q_heads * splits), (unsigned) ceil_div(tiles, layers), (unsigned) layers);
    hipStream_t st = resolve_stream(s);
    if (d->dtype == VKHIP_DT_F16) {
        if (d->head_dim <= 64) attn_packed_kernel<half_t, 64><<<grid, 256, 0, st>>>(a);
        else attn_packed_kernel<half_t, 128><<<grid, 256, 0, st>>>(a);
    } else {
        if (d->head_dim <= 64) attn_packed_kernel<bf16_t, 64><<<grid, 256, 0, st>>>(a);
        else attn_packed_kernel<bf16_t, 128><<<grid, 256, 0, st>>>(a);
    }
    int rc = check_launch("attention_packed");
    if (rc || splits == 1) return rc;
    const dim3 join((unsigned) ceil_div((int64_t) d->total_q * d->q_heads, 4));
    if (d->dtype == VKHIP_DT_F16) attn_join_kernel<half_t><<<join, 256, 0, st>>>(a);
    else attn_join_kernel<bf16_t><<<join, 256, 0, st>>>(a);
    return check_launch("attention_packed join");
}

} // extern "C"
