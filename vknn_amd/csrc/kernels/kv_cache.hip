// The 8-bit key/value cache: rows into its pages (quantising, one scale per page and head) and back.
#include "kv_cache.h"

namespace vkhip {

    struct KvRowArgs {
        KvArgs         c;
        const int32_t *cu, *at; // at: tokens held before (append), first token (read)
        void          *k, *v;   // rows; append only reads them
        int64_t        k_row, k_head, v_row, v_head;
        int            total;
    };

    // fp32 bits of 8 row elements
    template <typename T>
    __device__ __forceinline__ void row8(const T *s, float *v) {
        typedef T V __attribute__((ext_vector_type(8)));
        const V t = *reinterpret_cast<const V *>(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float) t[j];
    }

    // x / s to the nearest whole number. r = 1 / s: one remainder step makes x * r the correctly rounded
    // quotient (but for rare last places). A scale so small that r or the remainder could leave the normal
    // range (bf16 rows near its smallest numbers) takes the division itself.
    __device__ __forceinline__ int quantise(float x, float s, float r) {
        float q;
        if (s < 1e-30f) {
            q = s > 0.f ? x / s : 0.f;
        } else {
            q = x * r;
            q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
        }
        return clampi((int) rintf(q), -127, 127);
    }

    // Sequence, block of page_tokens tokens, and the rows of the call that lie in it.
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
        const SeqTile t = find_tile((int) blockIdx.x, a.c.batch, [&](int b) {
            int from, len, row;
            range(b, from, len, row);
            return len > 0 ? (from + len - 1) / P - from / P + 1 : 0;
        });
        if (t.b < 0) return {-1, 0, 0, 0, -1};
        int from, len, row;
        range(t.b, from, len, row);
        const int block = from / P + t.tile, lo = max(from, block * P), hi = min(from + len, (block + 1) * P);
        const int id    = a.c.table[(int64_t) t.b * a.c.max_blocks + block];
        return {t.b, lo - block * P, hi - lo, row + lo - from, id >= 0 && id < a.c.pages ? id : -1};
    }

    // One workgroup per block that gets rows, head, and keys or values. First the largest magnitude, as
    // integers (a NaN is larger than infinity, infinity than every number), then the scale, then the bytes.
    template <typename T, bool VALUES>
    __device__ void append_block(const KvRowArgs &a, const KvSpan &w, int head, unsigned char *tile, unsigned *red) {
        const int      P = a.c.page_tokens, D = a.c.head_dim, Dp = a.c.row, dv = D / 8, tid = threadIdx.x;
        const int64_t  stride = VALUES ? a.v_row : a.k_row;
        const T       *rows   = (const T *) (VALUES ? a.v : a.k) + (int64_t) w.row * stride + (int64_t) head * (VALUES ? a.v_head : a.k_head);
        const int64_t  at     = (int64_t) w.page * a.c.heads + head;
        float         *scale  = (VALUES ? a.c.v_scale : a.c.k_scale) + at;
        unsigned char *page   = (VALUES ? a.c.v : a.c.k) + at * P * Dp;

        unsigned big = 0;
        for (int i = tid; i < w.n * dv; i += 256) {
            float v[8];
            row8(rows + (int64_t) (i / dv) * stride + i % dv * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) big = max(big, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) big = max(big, (unsigned) __shfl_xor((int) big, o));
        if ((tid & 63) == 0) red[tid >> 6] = big;
        const float s0 = w.n0 ? *scale : 0.f;
        __syncthreads(); // also: every thread has read the old scale
        big = max(max(red[0], red[1]), max(red[2], red[3]));
        const bool  bad = big >= 0x7F800000u || s0 != s0;
        const float s = bad ? __builtin_nanf("") : fmaxf(s0, __uint_as_float(big) / 127.f), r = 1.f / s;
        if (tid == 0) *scale = s;
        const bool  grown = !bad && s > s0 && w.n0 > 0;
        const float ratio = grown ? s0 / s : 1.f;
        const auto  again = [&](int q) { return (unsigned) (unsigned char) (int) rintf((float) (signed char) q * ratio); };

        if (!VALUES) {
            if (grown)
                for (int i = tid; i < w.n0 * Dp / 4; i += 256) {
                    unsigned *p = reinterpret_cast<unsigned *>(page) + i, t = *p;
                    *p          = again(t & 255) | again(t >> 8 & 255) << 8 | again(t >> 16 & 255) << 16 | again(t >> 24) << 24;
                }
            for (int i = tid; i < w.n * dv; i += 256) {
                float v[8];
                row8(rows + (int64_t) (i / dv) * stride + i % dv * 8, v);
                unsigned o[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j / 4] |= (unsigned) (unsigned char) (bad ? 0 : quantise(v[j], s, r)) << (j % 4 * 8);
                *reinterpret_cast<uint2 *>(page + (int64_t) (w.n0 + i / dv) * Dp + i % dv * 8) = make_uint2(o[0], o[1]);
            }
            return;
        }
        // values: [channel][token], turned through LDS (rows of page_tokens + 4 bytes)
        const int pitch = P + 4;
        for (int i = tid; i < w.n * dv; i += 256) {
            float v[8];
            row8(rows + (int64_t) (i / dv) * stride + i % dv * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[(i % dv * 8 + j) * pitch + w.n0 + i / dv] = (unsigned char) (bad ? 0 : quantise(v[j], s, r));
        }
        __syncthreads();
        // words of 4 tokens: old tokens kept or rounded again, the call's rows, what lies behind them kept
        const int w0 = grown ? 0 : w.n0 / 4, words = (w.n0 + w.n + 3) / 4 - w0;
        for (int i = tid; i < D * words; i += 256) {
            const int d = i / words, t0 = (w0 + i % words) * 4;
            unsigned *p = reinterpret_cast<unsigned *>(page + (int64_t) d * P + t0), was = 0, now = 0;
            if (t0 < w.n0 || t0 + 4 > w.n0 + w.n) was = *p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t0 + j;
                unsigned  q = was >> (8 * j) & 255;
                if (t < w.n0) q = grown ? again(q) : q;
                else if (t < w.n0 + w.n) q = tile[d * pitch + t];
                now |= q << (8 * j);
            }
            *p = now;
        }
    }

    template <typename T>
    __global__ __launch_bounds__(256) void kv_append_kernel(KvRowArgs a) {
        extern __shared__ unsigned char tile[];
        __shared__ unsigned             red[4];
        const KvSpan w = kv_span(a);
        if (w.b < 0 || w.page < 0) return;
        if (blockIdx.z) append_block<T, true>(a, w, blockIdx.y, tile, red);
        else append_block<T, false>(a, w, blockIdx.y, tile, red);
    }

    template <typename T>
    __global__ __launch_bounds__(256) void kv_read_kernel(KvRowArgs a) {
        extern __shared__ unsigned char tile[];
        typedef T    V __attribute__((ext_vector_type(8)));
        const KvSpan w = kv_span(a);
        if (w.b < 0) return;
        const int     P = a.c.page_tokens, D = a.c.head_dim, Dp = a.c.row, dv = D / 8, tid = threadIdx.x, head = blockIdx.y;
        const bool    values = blockIdx.z, none = w.page < 0;
        const int64_t stride = values ? a.v_row : a.k_row, at = (int64_t) (none ? 0 : w.page) * a.c.heads + head;
        T            *rows   = (T *) (values ? a.v : a.k) + (int64_t) w.row * stride + (int64_t) head * (values ? a.v_head : a.k_head);
        const float   s      = none ? 0.f : (values ? a.c.v_scale : a.c.k_scale)[at];
        const unsigned char *page  = (values ? a.c.v : a.c.k) + at * P * Dp;
        const int            pitch = P + 4;
        if (values && !none) {
            const int w0 = w.n0 / 4, words = (w.n0 + w.n + 3) / 4 - w0;
            for (int i = tid; i < D * words; i += 256)
                *reinterpret_cast<unsigned *>(tile + (i / words) * pitch + (w0 + i % words) * 4) =
                    *reinterpret_cast<const unsigned *>(page + (int64_t) (i / words) * P + (w0 + i % words) * 4);
            __syncthreads();
        }
        for (int i = tid; i < w.n * dv; i += 256) {
            const int t = i / dv, d = i % dv * 8;
            V         o;
            if (none) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = (T) 0.f;
            } else if (values) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = (T) ((float) (signed char) tile[(d + j) * pitch + w.n0 + t] * s);
            } else {
                const uint2 q = *reinterpret_cast<const uint2 *>(page + (int64_t) (w.n0 + t) * Dp + d);
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = (T) ((float) (signed char) ((j < 4 ? q.x : q.y) >> (8 * (j & 3))) * s);
            }
            *reinterpret_cast<V *>(rows + t * stride + d) = o;
        }
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
        a.pages = c->pages, a.page_tokens = c->page_tokens, a.heads = c->kv_heads, a.head_dim = c->head_dim, a.row = vkhip_kv_row(c->head_dim);
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
        const dim3   grid((unsigned) tiles, (unsigned) c->kv_heads, 2);
        const size_t lds = (size_t) a.c.row * (c->page_tokens + 4);
        hipStream_t  q   = resolve_stream(s);
        if (append) {
            if (r->dtype == VKHIP_DT_F16) kv_append_kernel<half_t><<<grid, 256, lds, q>>>(a);
            else kv_append_kernel<bf16_t><<<grid, 256, lds, q>>>(a);
        } else {
            if (r->dtype == VKHIP_DT_F16) kv_read_kernel<half_t><<<grid, 256, lds, q>>>(a);
            else kv_read_kernel<bf16_t><<<grid, 256, lds, q>>>(a);
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
