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
#include "tokens.h"

namespace vkhip {

    struct AttnArgs {
        const void    *q, *k, *v;
        void          *o;
        const int32_t *cu_q, *cu_k;
        int            batch, q_heads, kv_heads, head_dim, total_q, total_k, causal;
        float          c2; // scale * log2(e)
        int64_t        q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    };

    template <typename T>
    struct AttnType;
    template <>
    struct AttnType<half_t> {
        typedef half8 V8;
        typedef half4 V4;
        static constexpr unsigned kExp = 0x7C00u;
        static __device__ __forceinline__ float16v mfma(V8 a, V8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    };
    template <>
    struct AttnType<bf16_t> {
        typedef bf8 V8;
        typedef bf4 V4;
        static constexpr unsigned kExp = 0x7F80u;
        static __device__ __forceinline__ float16v mfma(V8 a, V8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    };

    constexpr int kAttnQ = 128, kAttnK = 64;

    typedef short attn_s4 __attribute__((ext_vector_type(4)));
    // 4 x 16 values of 16 bits per 16 lanes, transposed: lane i of the 16 points at 4 values of row i / 4 (columns
    // 4 (i % 4) ..) and gets column i, rows 0 .. 3.
    __device__ __forceinline__ uint2 lds_read_tr(const unsigned char *p) {
#if defined(__HIP_DEVICE_COMPILE__) // the host pass rejects a generic pointer's cast to the LDS space
        const attn_s4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn_s4 *) (p));
        return __builtin_bit_cast(uint2, t);
#else
        return {};
#endif
    }
    // 16 bytes a lane from `off` past the resource's base to `dst` + 16 * lane
    __device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t r, unsigned char *dst, unsigned off) {
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *) dst, 16, off, 0, 0, 0);
#endif
    }

    // Where a 16-byte piece of a row lies in a tile's LDS image. K is read by 32 rows at one piece, V by 8 rows at 4.
    template <int DP>
    __device__ __forceinline__ int k_swizzle(int row) { return DP == 128 ? row & 15 : row >> 1 & 7; }
    template <int DP>
    __device__ __forceinline__ int v_swizzle(int row) { return DP == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2; }

    template <typename T, int DP>
    __global__ __launch_bounds__(256, 2) void attn_packed_kernel(AttnArgs a) {
        using A              = AttnType<T>;
        constexpr int PIECES = DP / 8;            // 16-byte pieces of a row
        constexpr int TILE   = kAttnK * DP * 2;   // bytes of a K or V tile
        constexpr int LOADS  = TILE / 1024 / 4;   // wave loads of 1 KB per wave and tile
        constexpr int KS = DP / 16, DB = DP / 32; // contraction steps of a score, 32-channel blocks of the output
        __shared__ __attribute__((aligned(1024))) unsigned char sm[2][2][TILE];

        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
        // heads of one key/value head next to each other in the grid: workgroups go to the 8 XCDs in turn
        const int head_kv = blockIdx.x % a.kv_heads, group = a.q_heads / a.kv_heads;
        const int head_q = head_kv * group + blockIdx.x / a.kv_heads % group;
        const SeqTile w = find_tile((int) (blockIdx.x / a.q_heads), a.batch, [&](int b) {
            return (clampi(a.cu_q[b + 1], 0, a.total_q) - clampi(a.cu_q[b], 0, a.total_q) + kAttnQ - 1) / kAttnQ;
        });
        if (w.b < 0) return;
        const int b  = __builtin_amdgcn_readfirstlane(w.b);
        const int q0 = clampi(a.cu_q[b], 0, a.total_q), nq = clampi(a.cu_q[b + 1], 0, a.total_q) - q0;
        const int k0 = clampi(a.cu_k[b], 0, a.total_k), nk = max(0, clampi(a.cu_k[b + 1], 0, a.total_k) - k0);
        // long tiles first: the last queries of a sequence see the most keys
        const int i0 = ((nq + kAttnQ - 1) / kAttnQ - 1 - __builtin_amdgcn_readfirstlane(w.tile)) * kAttnQ;
        const int shift = nk - nq;
        const int D     = a.head_dim;

        const int qi    = i0 + wave * 32 + col;
        const int limit = qi < nq ? (a.causal ? qi + shift + 1 : nk) : 0; // keys below it are seen
        const int i_last = min(i0 + kAttnQ, nq) - 1;
        const int k_end  = max(0, a.causal ? min(nk, i_last + shift + 1) : nk);
        // the wave's own range: all its queries see keys below `low`, none sees any from `high`
        const int w_first = i0 + wave * 32, w_last = min(w_first + 32, nq) - 1;
        const int low = w_first + 31 < nq ? (a.causal ? w_first + shift + 1 : nk) : 0;
        const int high = w_first < nq ? (a.causal ? min(nk, w_last + shift + 1) : nk) : 0;

        typename A::V8 qf[KS];
        {
            const T *src = (const T *) a.q + (int64_t) (q0 + qi) * a.q_row + (int64_t) head_q * a.q_head;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 16 * s + 8 * h;
#pragma unroll
                for (int j = 0; j < 8; ++j) qf[s][j] = (T) 0.f;
                if (qi < nq && d < D) qf[s] = *reinterpret_cast<const typename A::V8 *>(src + d);
            }
        }

        const T *kb = (const T *) a.k + (int64_t) k0 * a.k_row + (int64_t) head_kv * a.k_head;
        const T *vb = (const T *) a.v + (int64_t) k0 * a.v_row + (int64_t) head_kv * a.v_head;
        // this lane's source offsets: piece p of the LDS image is row p / PIECES, piece (p % PIECES) ^ swizzle(row)
        unsigned off_k[LOADS], off_v[LOADS];
        int      row_of[LOADS];
#pragma unroll
        for (int r = 0; r < LOADS; ++r) {
            const int p = (wave * LOADS + r) * 64 + lane, row = p / PIECES, at = p % PIECES;
            const int ck = at ^ k_swizzle<DP>(row), cv = at ^ v_swizzle<DP>(row);
            row_of[r]    = row;
            off_k[r]     = ck * 8 < D ? (unsigned) (row * a.k_row * 2 + ck * 16) : 0x80000000u;
            off_v[r]     = cv * 8 < D ? (unsigned) (row * a.v_row * 2 + cv * 16) : 0x80000000u;
        }
        // past the last row of the sequence, and past the head's channels, the copy writes zeros
        auto issue = [&](int t) __attribute__((always_inline)) {
            const int valid = min(kAttnK, nk - t * kAttnK);
            const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void *) (kb + (int64_t) t * kAttnK * a.k_row), (short) 0, 0x7FFFFFFF, 0x00020000);
            const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void *) (vb + (int64_t) t * kAttnK * a.v_row), (short) 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
            for (int r = 0; r < LOADS; ++r) {
                const bool in = row_of[r] < valid;
                copy_to_lds(kr, sm[t & 1][0] + (wave * LOADS + r) * 1024, in ? off_k[r] : 0x80000000u);
                copy_to_lds(vr, sm[t & 1][1] + (wave * LOADS + r) * 1024, in ? off_v[r] : 0x80000000u);
            }
        };

        float16v acc[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
        float m = -__builtin_inff(), l = 0.f;

        const int tiles = (k_end + kAttnK - 1) / kAttnK;
        if (tiles > 0) issue(0);
        for (int t = 0; t < tiles; ++t) {
            __builtin_amdgcn_s_waitcnt(7 << 4);         // vmcnt(0), lgkmcnt(0): its pieces of tile t have landed, its reads of t - 1 too
            __asm__ volatile("s_barrier" ::: "memory");       // everybody's have, and nobody reads tile t - 1 any more
            if (t + 1 < tiles) issue(t + 1);
            const int key0 = t * kAttnK;
            if (key0 >= high) continue;
            const unsigned char *kt = sm[t & 1][0], *vt = sm[t & 1][1];

            float16v s[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kk][r] = 0.f;
                const int row = kk * 32 + col;
#pragma unroll
                for (int c = 0; c < KS; ++c) {
                    const typename A::V8 kf = *reinterpret_cast<const typename A::V8 *>(kt + row * DP * 2 + (((2 * c + h) ^ k_swizzle<DP>(row)) << 4));
                    s[kk]                   = A::mfma(kf, qf[c], s[kk]);
                }
            }
            const bool masked = key0 + kAttnK > low;
            if (masked) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (key0 + kk * 32 + 8 * (r >> 2) + 4 * h + (r & 3) >= limit) s[kk][r] = -__builtin_inff();
            }
            float top = s[0][0];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kk][r]);
            top              = fmaxf(top, __shfl_xor(top, 32));
            const float to   = fmaxf(m, top), base = to == -__builtin_inff() ? 0.f : to * a.c2;
            if (__any(to > m)) {
                const float alpha = exp2_hw(m * a.c2 - base);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
                m = to;
            }
            typename A::V8 pf[4];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_hw(__builtin_fmaf(s[kk][r], a.c2, -base));
                    l += p;
                    pf[kk * 2 + (r >> 3)][r & 7] = (T) p;
                }
            // V: rows 16 k + 4 h + {0 .. 3} and 8 further, channels 32 d + lane % 32
            const auto v_frag = [&](int d, int k) __attribute__((always_inline)) {
                const int   row = 16 * k + 4 * h + ((lane & 15) >> 2), piece = 4 * d + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
                const uint2 x = lds_read_tr(vt + row * DP * 2 + ((piece ^ v_swizzle<DP>(row)) << 4) + (lane & 1) * 8);
                const uint2 y = lds_read_tr(vt + (row + 8) * DP * 2 + ((piece ^ v_swizzle<DP>(row + 8)) << 4) + (lane & 1) * 8);
                return tk_u32x4 {x.x, x.y, y.x, y.y};
            };
            if (masked) {
                // a weight of zero does not keep a NaN or an infinity of V out of a product: look for them where
                // something is masked
                unsigned odd = 0;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const tk_u32x4 f = v_frag(d, k);
#pragma unroll
                        for (int j = 0; j < 4; ++j) odd |= (f[j] & (A::kExp * 0x10001u)) + (0x8000u - A::kExp) * 0x10001u;
                    }
                if (__any((odd & 0x80008000u) != 0)) {
                    // finite values as usual; then NaN, +inf and -inf each by a product that counts the seen ones
                    for (int kind = 0; kind < 4; ++kind) {
                        typename A::V8 wf[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int key = key0 + 16 * k + 8 * (j >> 2) + 4 * h + (j & 3);
                                wf[k][j]      = kind ? (T) (key < limit ? 1.f : 0.f) : pf[k][j];
                            }
                        for (int d = 0; d < DB; ++d) {
                            float16v x;
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[r] = 0.f;
                            if (kind == 0) {
#pragma unroll
                                for (int dd = 0; dd < DB; ++dd)
                                    if (dd == d) x = acc[dd];
                            }
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                tk_u32x4 f = v_frag(d, k);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    unsigned out = 0;
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const unsigned u = f[j] >> (16 * e) & 0xFFFFu, mag = u & 0x7FFFu;
                                        const bool     hit = kind == 1 ? mag > A::kExp : mag == A::kExp && (u >> 15) == (unsigned) (kind - 2);
                                        const unsigned one = __builtin_bit_cast(uint16_t, (T) 1.f);
                                        out |= (kind == 0 ? (mag >= A::kExp ? 0u : u) : (hit ? one : 0u)) << (16 * e);
                                    }
                                    f[j] = out;
                                }
                                x = A::mfma(__builtin_bit_cast(typename A::V8, f), wf[k], x);
                            }
                            const float special = kind == 1 ? __builtin_nanf("") : (kind == 2 ? __builtin_inff() : -__builtin_inff());
#pragma unroll
                            for (int dd = 0; dd < DB; ++dd)
                                if (dd == d)
#pragma unroll
                                    for (int r = 0; r < 16; ++r) acc[dd][r] = kind == 0 ? x[r] : (x[r] > 0.f ? acc[dd][r] + special : acc[dd][r]);
                        }
                    }
                    continue;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = A::mfma(__builtin_bit_cast(typename A::V8, v_frag(d, k)), pf[k], acc[d]);
        }

        l += __shfl_xor(l, 32);
        if (qi >= nq) return;
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
        if (d->k_row > (1 << 23) || d->v_row > (1 << 23)) return "k_row or v_row over 2^23";
        if ((ceil_div(d->total_q, kAttnQ) + d->batch) * (int64_t) d->q_heads > 0x7FFFFFFF) return "too many queries and heads";
        return nullptr;
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

size_t vkhip_attention_workspace_bytes(const vkhip_attention_desc *) { return 0; }

int vkhip_attention_packed(const vkhip_attention_desc *d, const void *q, const void *k, const void *v, const int32_t *cu_q, const int32_t *cu_k,
                           void *o, void *, vkhip_stream_t s) {
    if (const char *why = attn_refusal(d)) return set_error(VKHIP_ERR_INVALID, "attention_packed: %s", why);
    if (d->batch == 0 || d->total_q == 0) return VKHIP_OK;
    if (!q || !o || !cu_q || !cu_k || (d->total_k > 0 && (!k || !v))) return set_error(VKHIP_ERR_INVALID, "attention_packed: null pointer");
    if (misaligned16(q) || misaligned16(k) || misaligned16(v) || misaligned16(o) || ((uintptr_t) cu_q | (uintptr_t) cu_k) % 4)
        return set_error(VKHIP_ERR_INVALID, "attention_packed: misaligned pointer");
    AttnArgs a {};
    a.q = q, a.k = k, a.v = v, a.o = o, a.cu_q = cu_q, a.cu_k = cu_k;
    a.batch = d->batch, a.q_heads = d->q_heads, a.kv_heads = d->kv_heads, a.head_dim = d->head_dim, a.total_q = d->total_q, a.total_k = d->total_k;
    a.causal = d->causal != 0, a.c2 = d->scale * 1.44269504088896f;
    a.q_row = d->q_row, a.q_head = d->q_head, a.k_row = d->k_row, a.k_head = d->k_head;
    a.v_row = d->v_row, a.v_head = d->v_head, a.o_row = d->o_row, a.o_head = d->o_head;
    // sequences have fewer than total_q / 128 + batch tiles together
    int64_t tiles = d->total_q / kAttnQ + d->batch;
    if (tiles > d->total_q) tiles = d->total_q;
    const dim3  grid((unsigned) (tiles * d->q_heads));
    hipStream_t st = resolve_stream(s);
    if (d->dtype == VKHIP_DT_F16) {
        if (d->head_dim <= 64) attn_packed_kernel<half_t, 64><<<grid, 256, 0, st>>>(a);
        else attn_packed_kernel<half_t, 128><<<grid, 256, 0, st>>>(a);
    } else {
        if (d->head_dim <= 64) attn_packed_kernel<bf16_t, 64><<<grid, 256, 0, st>>>(a);
        else attn_packed_kernel<bf16_t, 128><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("attention_packed");
}

} // extern "C"
