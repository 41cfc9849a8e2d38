// The 8-bit key/value cache: rows into its pages (quantising, one scale per page and head) and back.
//
// Bound by memory: 2 bytes in and 1 out a value, and the other way round. A workgroup takes a page, head, and keys or
// values, so that the largest magnitude is found and used without leaving it; the rows stay in registers
// between. 8 x 4096 rows, 8 heads, D = 128: 40 us in (201 MB, 5.0 TB/s), 38 us back.
// Rows in both directions and whole pages pass the caches (44 and 44 us otherwise; pages as they are read back are
// better left to them: 15 thousand ragged rows 20 us, 23 past them).
#include "kv_cache.h"

namespace vkhip {

    struct KvRowArgs {
        KvArgs         c;
        const int32_t *cu, *at; // at: tokens held before (append), first token (read)
        void          *k, *v;   // rows; append only reads them
        int64_t        k_row, k_head, v_row, v_head;
        int            total;
    };

    // x / s to the nearest whole number, as the low byte of the result's bits (1.5 * 2^23 added: the sum's last place
    // is 1). |x| is at most 127 s but for roundings. r = 1 / s: one remainder step makes x * r the correctly
    // rounded quotient (but for rare last places). A scale so small that r or the remainder could leave the normal
    // range (bf16 rows near its smallest numbers) takes the division itself.
    __device__ __forceinline__ unsigned quantise(float x, float s, float r) {
        float q;
        if (s < 1e-30f) {
            q = s > 0.f ? x / s : 0.f;
        } else {
            q = x * r;
            q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
        }
        return __float_as_uint(q + 12582912.f);
    }
    __device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
        const unsigned ab = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), cd = __builtin_amdgcn_perm(d, c, 0x0C0C0400u);
        return ab | cd << 16;
    }

    // The largest magnitude of 8 values of 16 bits and a pair so far: without the sign their bits are ordered as they
    // are, a NaN above infinity.
    typedef unsigned short KvPair __attribute__((ext_vector_type(2)));
    template <typename V>
    __device__ __forceinline__ KvPair magnitude(KvPair m, V x) {
        const tk_u32x4 b = __builtin_bit_cast(tk_u32x4, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(KvPair, b[j] & 0x7FFF7FFFu));
        return m;
    }
    template <typename T>
    __device__ __forceinline__ float as_float(unsigned bits) {
        return (float) __builtin_bit_cast(T, (unsigned short) bits);
    }

    // Blocks go over the grid's first dimension, which holds 2^24 workgroups of 256 threads, and on over its third, whose
    // lowest bit says keys or values. Sequence, block of page_tokens tokens, and the rows of the call that lie in it.
    struct KvSpan {
        int     b, n0, n; // tokens of the block before the call's rows (append) or in front of them (read), rows
        int     row, page;
    };
    __device__ __forceinline__ KvSpan kv_span(const KvRowArgs &a) {
        const int P = a.c.page_tokens, most = a.c.max_blocks * P;
        const auto range = [&](int b, int &from, int &len, int &row) {
            row  = clampi(a.cu[b], 0, a.total);
            from = clampi(a.at[b], 0, most);
            len  = min(clampi(a.cu[b + 1], 0, a.total) - row, most - from);
        };
        const SeqTile t = find_tile((int) ((blockIdx.z >> 1) * gridDim.x + blockIdx.x), a.c.batch, [&](int b) {
            int from, len, row;
            range(b, from, len, row);
            return len > 0 ? ((from + len - 1) >> a.c.page_shift) - (from >> a.c.page_shift) + 1 : 0;
        });
        if (t.b < 0) return {-1, 0, 0, 0, -1};
        int from, len, row;
        range(t.b, from, len, row);
        const int block = (from >> a.c.page_shift) + t.tile, lo = max(from, block * P), hi = min(from + len, (block + 1) * P);
        const int id    = a.c.table[(int64_t) t.b * a.c.max_blocks + block];
        return {t.b, lo - block * P, hi - lo, row + lo - from, id >= 0 && id < a.c.pages ? id : -1};
    }

    // Both kernels cut a block into patches of 4 tokens and 8 channels, a patch (or R of them) a thread: four rows'
    // vectors of 16 bytes on one side; on the other four times 8 bytes of keys, or eight words of 4 tokens of values,
    // which are turned through LDS (rows of a channel, an odd number of words apart).
    struct Patch {
        int token, channel; // the first ones; token is a multiple of 4
    };
    template <int THREADS>
    __device__ __forceinline__ Patch patch_of(int r, int first_quad, int dv) {
        const int i = (int) threadIdx.x + r * THREADS;
        return {(first_quad + i / dv) * 4, i % dv * 8};
    }

    // One workgroup per block that gets rows, head, and keys or values. First the largest magnitude, as
    // integers (a NaN is larger than infinity, infinity than every number), then the scale, then the bytes.
    template <typename T, int THREADS, int R, bool VALUES>
    __device__ void append_block(const KvRowArgs &a, const KvSpan &w, int head, unsigned *words, unsigned *red) {
        typedef T      V __attribute__((ext_vector_type(8)));
        const int      P = a.c.page_tokens, D = a.c.head_dim, Dp = a.c.row, dv = D / 8, tid = threadIdx.x, end = w.n0 + w.n, quad0 = w.n0 / 4;
        const int64_t  stride = VALUES ? a.v_row : a.k_row;
        const T       *rows   = (const T *) (VALUES ? a.v : a.k) + (int64_t) (w.row - w.n0) * stride + (int64_t) head * (VALUES ? a.v_head : a.k_head);
        const int64_t  at     = (int64_t) w.page * a.c.heads + head;
        float         *scale  = (VALUES ? a.c.v_scale : a.c.k_scale) + at;
        unsigned char *page   = (VALUES ? a.c.v : a.c.k) + at * P * Dp;

        V      x[R][4];
        KvPair most = {0, 0};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Patch p = patch_of<THREADS>(r, quad0, dv);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = p.token + k;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[r][k][j] = (T) 0.f;
                if (t >= w.n0 && t < end) x[r][k] = __builtin_nontemporal_load(reinterpret_cast<const V *>(rows + t * stride + p.channel));
            }
        }
        const float s0 = w.n0 ? *scale : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                most = magnitude(most, x[r][k]);
        unsigned big = max((unsigned) most[0], (unsigned) most[1]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) big = max(big, (unsigned) __shfl_xor((int) big, o));
        if ((tid & 63) == 0) red[tid >> 6] = big;
        __syncthreads(); // also: every thread has read the old scale
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) big = max(big, red[i]);
        const float largest = as_float<T>(big);
        const bool  bad = !(largest < __builtin_inff()) || s0 != s0;
        const float s = bad ? __builtin_nanf("") : fmaxf(s0, largest / 127.f), inv = 1.f / s;
        if (tid == 0) *scale = s;
        const bool  grown = !bad && s > s0 && w.n0 > 0;
        const float ratio = grown ? s0 / s : 1.f;
        const auto  again = [&](int q) { return (unsigned) (unsigned char) (int) rintf((float) (signed char) q * ratio); };
        const auto  again4 = [&](unsigned t) { return again(t & 255) | again(t >> 8 & 255) << 8 | again(t >> 16 & 255) << 16 | again(t >> 24) << 24; };
        const auto  four  = [&](T v0, T v1, T v2, T v3) {
            return bad ? 0u : low_bytes(quantise((float) v0, s, inv), quantise((float) v1, s, inv), quantise((float) v2, s, inv), quantise((float) v3, s, inv));
        };

        if (!VALUES) {
            if (grown) {
                uint4 *old = reinterpret_cast<uint4 *>(page);
#pragma unroll 4
                for (int i = tid; i < w.n0 * Dp / 16; i += THREADS) {
                    const uint4 t = old[i];
                    old[i]        = make_uint4(again4(t.x), again4(t.y), again4(t.z), again4(t.w));
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const Patch p = patch_of<THREADS>(r, quad0, dv);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const V v = x[r][k];
                    if (p.token + k >= w.n0 && p.token + k < end)
                        __builtin_nontemporal_store((tk_u32x2) {four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7])}, reinterpret_cast<tk_u32x2 *>(page + (p.token + k) * Dp + p.channel));
                }
            }
            return;
        }
        const int pitch = P / 4 + 1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Patch p = patch_of<THREADS>(r, quad0, dv);
            if (p.token >= end) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                words[(p.channel + j) * pitch + p.token / 4] = four(x[r][0][j], x[r][1][j], x[r][2][j], x[r][3][j]);
        }
        __syncthreads();
        if (w.n == P) { // a whole page: 16 tokens of a channel at a time
            for (int i = tid; i < D * (P / 16); i += THREADS) {
                const int       d = i / (P / 16), c = i % (P / 16);
                const unsigned *q = words + d * pitch + c * 4;
                __builtin_nontemporal_store((tk_u32x4) {q[0], q[1], q[2], q[3]}, reinterpret_cast<tk_u32x4 *>(page + d * P + c * 16));
            }
            return;
        }
        // words of 4 tokens: old tokens kept or rounded again, the call's rows, what lies behind them kept
        const int w0 = grown ? 0 : quad0, count = (end + 3) / 4 - w0;
        for (int i = tid; i < D * count; i += THREADS) {
            const int d = i / count, t0 = (w0 + i % count) * 4;
            unsigned *p = reinterpret_cast<unsigned *>(page + d * P + t0), was = 0;
            if (t0 < w.n0 || t0 + 4 > end) was = *p;
            const unsigned old = grown ? again4(was) : was, fresh = t0 + 4 > w.n0 ? words[d * pitch + t0 / 4] : 0;
            unsigned       now = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) now |= (t0 + j < w.n0 ? old : (t0 + j < end ? fresh : was)) & 255u << (8 * j);
            *p = now;
        }
    }

    template <typename T, int THREADS, int R>
    __global__ __launch_bounds__(THREADS) void kv_append_kernel(KvRowArgs a) {
        extern __shared__ unsigned words[];
        __shared__ unsigned        red[THREADS / 64];
        const KvSpan w = kv_span(a);
        if (w.b < 0 || w.page < 0) return;
        if (blockIdx.z & 1) append_block<T, THREADS, R, true>(a, w, blockIdx.y, words, red);
        else append_block<T, THREADS, R, false>(a, w, blockIdx.y, words, red);
    }

    template <typename T, int THREADS>
    __global__ __launch_bounds__(THREADS) void kv_read_kernel(KvRowArgs a) {
        extern __shared__ unsigned words[];
        typedef T    V __attribute__((ext_vector_type(8)));
        const KvSpan w = kv_span(a);
        if (w.b < 0) return;
        const int     P = a.c.page_tokens, D = a.c.head_dim, Dp = a.c.row, dv = D / 8, tid = threadIdx.x, head = blockIdx.y, end = w.n0 + w.n, quad0 = w.n0 / 4;
        const bool    values = blockIdx.z & 1, none = w.page < 0;
        const int64_t stride = values ? a.v_row : a.k_row, at = (int64_t) (none ? 0 : w.page) * a.c.heads + head;
        T            *rows   = (T *) (values ? a.v : a.k) + (int64_t) (w.row - w.n0) * stride + (int64_t) head * (values ? a.v_head : a.k_head);
        const float   s      = none ? 0.f : (values ? a.c.v_scale : a.c.k_scale)[at];
        const unsigned char *page  = (values ? a.c.v : a.c.k) + at * P * Dp;
        const int            pitch = P / 4 + 1;
        if (values && !none) {
            const int c0 = w.n0 / 16, count = (end + 15) / 16 - c0;
            for (int i = tid; i < D * count; i += THREADS) {
                const int   d = i / count, c = c0 + i % count;
                const uint4 q = *reinterpret_cast<const uint4 *>(page + d * P + c * 16);
                unsigned   *o = words + d * pitch + c * 4;
                o[0] = q.x, o[1] = q.y, o[2] = q.z, o[3] = q.w;
            }
            __syncthreads();
        }
        const int patches = ((end + 3) / 4 - quad0) * dv;
        for (int r = 0; r * THREADS + tid < patches; ++r) {
            const Patch p = patch_of<THREADS>(r, quad0, dv);
            unsigned    q[4][2], by_channel[8]; // a token's 8 bytes; values: a channel's 4
            if (none) {
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k][0] = q[k][1] = 0;
            } else if (values) {
#pragma unroll
                for (int j = 0; j < 8; ++j) by_channel[j] = words[(p.channel + j) * pitch + p.token / 4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        q[k][i] = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) q[k][i] |= (by_channel[4 * i + j] >> (8 * k) & 255) << (8 * j);
                    }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) { // a page holds whole quads
                    const uint2 t = *reinterpret_cast<const uint2 *>(page + (p.token + k) * Dp + p.channel);
                    q[k][0] = t.x, q[k][1] = t.y;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                V o;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = (T) ((float) (signed char) (q[k][j >> 2] >> (8 * (j & 3))) * s);
                if (p.token + k >= w.n0 && p.token + k < end) __builtin_nontemporal_store(o, reinterpret_cast<V *>(rows + (p.token + k) * stride + p.channel));
            }
        }
    }

    // The same for a few rows, a wave per block, head, and keys or values: a lane a vector of 8 channels, the rows
    // read twice where there are more than 64, values stored byte by byte.
    template <typename T>
    __global__ __launch_bounds__(256) void kv_append_few_kernel(KvRowArgs a) {
        typedef T    V __attribute__((ext_vector_type(8)));
        const KvSpan w = kv_span(a);
        const int    part = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), head = part >> 1, lane = threadIdx.x & 63;
        if (w.b < 0 || w.page < 0 || head >= a.c.heads) return;
        const bool     values = part & 1;
        const int      P = a.c.page_tokens, D = a.c.head_dim, Dp = a.c.row, dv = D / 8, vectors = w.n * dv;
        const int64_t  stride = values ? a.v_row : a.k_row, at = (int64_t) w.page * a.c.heads + head;
        const T       *rows   = (const T *) (values ? a.v : a.k) + (int64_t) w.row * stride + (int64_t) head * (values ? a.v_head : a.k_head);
        float         *scale  = (values ? a.c.v_scale : a.c.k_scale) + at;
        unsigned char *page   = (values ? a.c.v : a.c.k) + at * P * Dp;
        const float    s0     = w.n0 ? *scale : 0.f;

        V      x {};
        KvPair most = {0, 0};
        for (int i = lane; i < vectors; i += 64) {
            x    = *reinterpret_cast<const V *>(rows + i / dv * stride + i % dv * 8);
            most = magnitude(most, x);
        }
        unsigned big = max((unsigned) most[0], (unsigned) most[1]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) big = max(big, (unsigned) __shfl_xor((int) big, o));
        const float largest = as_float<T>(big);
        const bool  bad = !(largest < __builtin_inff()) || s0 != s0;
        const float s = bad ? __builtin_nanf("") : fmaxf(s0, largest / 127.f), inv = 1.f / s;
        if (lane == 0) *scale = s;
        if (!bad && s > s0 && w.n0 > 0) {
            // the page's old tokens; what lies behind them in a word is rewritten below or of no use
            const float ratio = s0 / s;
            const int   whole = (w.n0 + 15) / 16, count = values ? D * whole : w.n0 * Dp / 16;
            const auto  again = [&](unsigned t) {
                unsigned o = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) o |= (unsigned) (unsigned char) (int) rintf((float) (signed char) (t >> (8 * j)) * ratio) << (8 * j);
                return o;
            };
#pragma unroll 4
            for (int i = lane; i < count; i += 64) {
                uint4      *p = reinterpret_cast<uint4 *>(page + (values ? i / whole * P + i % whole * 16 : i * 16));
                const uint4 t = *p;
                *p            = make_uint4(again(t.x), again(t.y), again(t.z), again(t.w));
            }
            // these are written before the new bytes of the same words are
            __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); // vmcnt(0)
            __asm__ volatile("" ::: "memory");
        }
        for (int i = lane; i < vectors; i += 64) {
            const int t = w.n0 + i / dv, d = i % dv * 8;
            if (vectors > 64) x = *reinterpret_cast<const V *>(rows + i / dv * stride + d);
            unsigned o[2] = {0, 0};
            if (!bad)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    o[j] = low_bytes(quantise((float) x[4 * j], s, inv), quantise((float) x[4 * j + 1], s, inv), quantise((float) x[4 * j + 2], s, inv), quantise((float) x[4 * j + 3], s, inv));
            if (values) {
#pragma unroll
                for (int j = 0; j < 8; ++j) page[(d + j) * P + t] = (unsigned char) (o[j / 4] >> (j % 4 * 8));
            } else {
                *reinterpret_cast<uint2 *>(page + t * Dp + d) = make_uint2(o[0], o[1]);
            }
        }
    }

    template <typename T>
    static void kv_append_launch(const KvRowArgs &a, dim3 grid, size_t lds, hipStream_t s) {
        // A wave a block where the call brings four rows a sequence or fewer (256 sequences of one row, 8 heads: 8.3 us
        // against 22 with workgroups that turn a page through LDS; 8 x 4096 rows: 177 against 46).
        if (a.total <= 4 * (int64_t) a.c.batch) {
            grid.y = (unsigned) ceil_div(2 * (int64_t) a.c.heads, 4), grid.z = 1;
            kv_append_few_kernel<T><<<grid, 256, 0, s>>>(a);
            return;
        }
        const int patches = a.c.page_tokens / 4 * (a.c.head_dim / 8);
        if (patches <= 128) kv_append_kernel<T, 128, 1><<<grid, 128, lds, s>>>(a);
        else if (patches <= 256) kv_append_kernel<T, 256, 1><<<grid, 256, lds, s>>>(a);
        else if (patches <= 512) kv_append_kernel<T, 256, 2><<<grid, 256, lds, s>>>(a);
        else kv_append_kernel<T, 256, 4><<<grid, 256, lds, s>>>(a);
    }
    template <typename T>
    static void kv_read_launch(const KvRowArgs &a, dim3 grid, size_t lds, hipStream_t s) {
        if (a.c.page_tokens / 4 * (a.c.head_dim / 8) <= 128) kv_read_kernel<T, 128><<<grid, 128, lds, s>>>(a);
        else kv_read_kernel<T, 256><<<grid, 256, lds, s>>>(a);
    }

    const char *kv_refusal(const vkhip_kv_cache *c) {
        if (!c || c->pages < 0 || c->batch < 0 || c->max_blocks < 0 || c->kv_heads <= 0) return "bad sizes";
        if (!vkhip_kv_row(c->head_dim)) return "head_dim is not a multiple of 8 up to 128";
        if (c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128 && c->page_tokens != 256) return "page_tokens is not 32, 64, 128 or 256";
        if (c->batch > 65535 || c->kv_heads > 65535 || (int64_t) c->max_blocks * c->page_tokens > 0x40000000) return "batch or kv_heads over 65535 or over 2^30 tokens a sequence";
        return nullptr;
    }
    const char *kv_bad_pointers(const vkhip_kv_cache *c) {
        if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table) return "null cache pointer";
        if (misaligned16(c->k) || misaligned16(c->v) || ((uintptr_t) c->k_scale | (uintptr_t) c->v_scale | (uintptr_t) c->table) % 4) return "misaligned cache pointer";
        return nullptr;
    }
    KvArgs kv_args(const vkhip_kv_cache *c) {
        KvArgs a {};
        a.k = (unsigned char *) c->k, a.v = (unsigned char *) c->v, a.k_scale = c->k_scale, a.v_scale = c->v_scale, a.table = c->table;
        a.pages = c->pages, a.page_tokens = c->page_tokens, a.page_shift = __builtin_ctz((unsigned) c->page_tokens), a.heads = c->kv_heads, a.head_dim = c->head_dim, a.row = vkhip_kv_row(c->head_dim);
        a.batch = c->batch, a.max_blocks = c->max_blocks;
        return a;
    }

    static int kv_rows(const char *what, bool append, const vkhip_kv_cache *c, const vkhip_kv_rows *r, void *k, void *v, const int32_t *cu, const int32_t *at,
                       vkhip_stream_t s) {
        if (const char *why = kv_refusal(c)) return set_error(VKHIP_ERR_INVALID, "%s: %s", what, why);
        if (!r || r->total < 0) return set_error(VKHIP_ERR_INVALID, "%s: bad rows", what);
        if (r->dtype != VKHIP_DT_F16 && r->dtype != VKHIP_DT_BF16) return set_error(VKHIP_ERR_INVALID, "%s: rows are F16 or BF16", what);
        if (r->k_row < 0 || r->v_row < 0 || r->k_head < 0 || r->v_head < 0 || (r->k_row | r->v_row | r->k_head | r->v_head) % 8)
            return set_error(VKHIP_ERR_INVALID, "%s: strides are not multiples of 8", what);
        if (!append && (rows_overlap(r->total, r->k_row, c->kv_heads, r->k_head, c->head_dim) || rows_overlap(r->total, r->v_row, c->kv_heads, r->v_head, c->head_dim)))
            return set_error(VKHIP_ERR_INVALID, "%s: rows share memory", what);
        if (r->total == 0 || c->batch == 0 || c->max_blocks == 0) return VKHIP_OK;
        if (!k || !v || !cu || !at) return set_error(VKHIP_ERR_INVALID, "%s: null pointer", what);
        if (misaligned16(k) || misaligned16(v) || ((uintptr_t) cu | (uintptr_t) at) % 4) return set_error(VKHIP_ERR_INVALID, "%s: misaligned pointer", what);
        if (const char *why = kv_bad_pointers(c)) return set_error(VKHIP_ERR_INVALID, "%s: %s", what, why);
        KvRowArgs a {};
        a.c = kv_args(c), a.cu = cu, a.at = at, a.k = k, a.v = v, a.total = r->total;
        a.k_row = r->k_row, a.k_head = r->k_head, a.v_row = r->v_row, a.v_head = r->v_head;
        // n rows touch fewer than n / page_tokens + 2 blocks and no more than n
        int64_t tiles = (int64_t) r->total / c->page_tokens + 2 * (int64_t) c->batch;
        if (tiles > r->total) tiles = r->total;
        const int64_t layers = ceil_div(tiles, 0xFFFFFF);
        const dim3   grid((unsigned) ceil_div(tiles, layers), (unsigned) c->kv_heads, (unsigned) (2 * layers));
        const size_t lds = (size_t) a.c.head_dim * (c->page_tokens / 4 + 1) * 4;
        hipStream_t  q   = resolve_stream(s);
        if (append) {
            if (r->dtype == VKHIP_DT_F16) kv_append_launch<half_t>(a, grid, lds, q);
            else kv_append_launch<bf16_t>(a, grid, lds, q);
        } else {
            if (r->dtype == VKHIP_DT_F16) kv_read_launch<half_t>(a, grid, lds, q);
            else kv_read_launch<bf16_t>(a, grid, lds, q);
        }
        return check_launch(what);
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

int32_t vkhip_kv_row(int32_t head_dim) { return head_dim < 8 || head_dim > 128 || head_dim % 8 ? 0 : (head_dim <= 64 ? 64 : 128); }

int vkhip_kv_append(const vkhip_kv_cache *c, const vkhip_kv_rows *r, const void *k, const void *v, const int32_t *cu, const int32_t *lens,
                    vkhip_stream_t s) {
    return kv_rows("kv_append", true, c, r, const_cast<void *>(k), const_cast<void *>(v), cu, lens, s);
}

int vkhip_kv_read(const vkhip_kv_cache *c, const vkhip_kv_rows *r, const int32_t *start, const int32_t *cu, void *k, void *v, vkhip_stream_t s) {
    return kv_rows("kv_read", false, c, r, k, v, cu, start, s);
}

} // extern "C"
