// What lies between two blocks of a token model: the block's output, normed, gated and scaled, joins the residual, whose
// norm, scaled and shifted, is the next block's input.
//
// Bound by memory: two values in and two out, once each. A row stays in the registers of the threads that read it, while
// its sums are formed: of squares, or first the mean and then the squared deviations from it (never E[z^2] - E[z]^2).
// Measured: 50176 rows of 2048 bf16 155 us, 5.3 TB/s; 12800 of 1100 fp16 with a gate, scale and shift an image 34 us, 3.3 TB/s
// (vector units busy 60%: rows that end inside a line, 138 of 192 threads with values); 64 of 4096 7.4 us, a launch. fp32:
// 50176 rows of 2048 317 us, 5.2 TB/s.
// Squares and their sum are fp32 as they are: a row whose sum leaves its range (values of 2^64 / sqrt(dim)) has an inverse
// deviation of 0, one whose squares vanish (under about 2^-75) has eps alone.
#include "tokens.h"

namespace vkhip {

    struct NormArgs {
        const void    *x, *r, *gate, *scale, *shift;
        const float   *post_w, *post_b, *pre_w, *pre_b;
        const int32_t *mod;
        void          *h, *y;
        int            rows, dim, post, pre, mods, mod_rows;
        bool           in_place;
        float          alpha, post_eps, pre_eps, each; // each: 1 / dim
        int64_t        x_row, r_row, h_row, y_row, mod_row;
    };

    // A lane's number and its partner's: quad_perm of 1 and of 2 apart, then the other half of 8 and of 16 lanes mirrored.
    template <int CTRL>
    __device__ __forceinline__ float add_partner(float x) {
        return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xF, 0xF, true));
    }
    // The sum over the threads of a row, in each of them.
    template <int GT>
    __device__ __forceinline__ float row_sum(float v, float *waves) {
        v = add_partner<0x141>(add_partner<0x4E>(add_partner<0xB1>(v)));
        if constexpr (GT > 8) v = add_partner<0x140>(v);
        if constexpr (GT == 32) v += __shfl_xor(v, 16);
        if constexpr (GT >= 64) {
            const auto row = [&](int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); };
            v = (row(0) + row(16)) + (row(32) + row(48));
        }
        if constexpr (GT > 64) {
            __syncthreads(); // the last sum has been read
            if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int i = 0; i < GT / 64; ++i) v += waves[i];
        }
        return v;
    }

    // GT threads a row, N vectors of VEC values each, vector i of thread t at (i GT + t) VEC. RAGGED: a row's last vector begins
    // at dim - VEC; its first values, of the vector before, count once, and are stored twice, or once in place, where its owner
    // may be a wave that has yet to read them. PAST: rows pass the caches.
    template <typename T, int VEC, int N, int GT, bool RAGGED, bool PAST>
    __global__ __launch_bounds__(GT <= 64 ? 256 : GT) void residual_norm_kernel(NormArgs a) {
        typedef T     V __attribute__((ext_vector_type(VEC), aligned(sizeof(T)))); // of any alignment: one instruction
        typedef float F __attribute__((ext_vector_type(VEC), aligned(4)));
        __shared__ float waves[GT <= 64 ? 1 : GT / 64];
        constexpr int RPB = GT <= 64 ? 256 / GT : 1; // rows of a workgroup
        const int     t = RPB > 1 ? (int) threadIdx.x % GT : (int) threadIdx.x;
        const int64_t row = ((int64_t) blockIdx.y * gridDim.x + blockIdx.x) * RPB + (RPB > 1 ? (int) threadIdx.x / GT : 0);
        if (row >= a.rows) return; // the whole group
        const int64_t m = a.mod ? clampi(a.mod[row], 0, a.mods - 1) : (a.mod_rows ? (int64_t) ((unsigned) row / (unsigned) a.mod_rows) : 0);
        const float   count = (float) a.dim;
        F             z[N];
        const auto    whole = [&](int i) { return (i * GT + t) * VEC; };
        const auto    in = [&](int i) { return whole(i) < a.dim; };
        const auto    at = [&](int i) { return RAGGED ? min(whole(i), a.dim - VEC) : whole(i); };
        const auto    own = [&](int i) { // what counts of z[i]: by a branch, which few waves take
            F c = z[i];
            if (whole(i) + VEC > a.dim)
#pragma unroll
                for (int j = 0; j < VEC; ++j) c[j] = RAGGED && j >= whole(i) - at(i) ? c[j] : 0.f;
            return c;
        };
        const auto    load = [&](const void *p, int64_t offset, int i) {
            const V v = *reinterpret_cast<const V *>((const T *) p + offset + at(i));
            return __builtin_convertvector(v, F);
        };
        const auto load_row = [&](const void *p, int64_t offset, int i) {
            if constexpr (PAST) return __builtin_convertvector(__builtin_nontemporal_load(reinterpret_cast<const V *>((const T *) p + offset + at(i))), F);
            else return load(p, offset, i);
        };
        const auto store_row = [&](void *p, int64_t offset, int i) {
            const V v = __builtin_convertvector(z[i], V);
            if (RAGGED && a.in_place && whole(i) > at(i)) {
#pragma unroll
                for (int j = 1; j < VEC; ++j)
                    if (j >= whole(i) - at(i)) ((T *) p + offset + at(i))[j] = v[j];
            } else if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<V *>((T *) p + offset + at(i)));
            else *reinterpret_cast<V *>((T *) p + offset + at(i)) = v;
        };
        const auto norm = [&](int kind, float eps, const float *w, const float *b) {
            if (kind == VKHIP_NORM_NONE) return;
            if (kind == VKHIP_NORM_LAYER) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const F c = own(i);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum += c[j];
                }
                const float mean = row_sum<GT>(sum, waves) / count; // a row of one value has it as its mean, and no variance
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) z[i][j] -= mean;
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const F c = own(i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum = __builtin_fmaf(c[j], c[j], sum);
            }
            const float rstd = 1.f / __builtin_sqrtf(__builtin_fmaf(row_sum<GT>(sum, waves), a.each, eps));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                F g, c;
#pragma unroll
                for (int j = 0; j < VEC; ++j) g[j] = 1.f, c[j] = 0.f;
                if (in(i)) {
                    if (w) g = *reinterpret_cast<const F *>(w + at(i));
                    if (b) c = *reinterpret_cast<const F *>(b + at(i));
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[i][j] = __builtin_fmaf(z[i][j] * rstd, g[j], c[j]);
            }
        };

        F r[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[i][j] = 0.f, r[i][j] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (a.x && in(i)) z[i] = load_row(a.x, row * a.x_row, i);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (a.r && in(i)) r[i] = load_row(a.r, row * a.r_row, i);
        if (a.x) {
            norm(a.post, a.post_eps, a.post_w, a.post_b);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                F g;
#pragma unroll
                for (int j = 0; j < VEC; ++j) g[j] = 1.f;
                if (a.gate && in(i)) g = load(a.gate, m * a.mod_row, i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[i][j] = __builtin_fmaf(z[i][j] * a.alpha, g[j], r[i][j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] = r[i];
        }
        if (a.h)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (in(i)) store_row(a.h, row * a.h_row, i);
        if (!a.y) return;
        norm(a.pre, a.pre_eps, a.pre_w, a.pre_b);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!in(i)) continue;
            if (a.scale) {
                const F s = load(a.scale, m * a.mod_row, i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[i][j] = __builtin_fmaf(z[i][j], s[j], z[i][j]);
            }
            if (a.shift) z[i] += load(a.shift, m * a.mod_row, i);
            store_row(a.y, row * a.y_row, i);
        }
    }

    static bool overlaps(const vkhip_residual_norm_desc *d, int64_t row) { return d->rows > 1 && row < d->dim; }

    static const char *residual_norm_refusal(const vkhip_residual_norm_desc *d) {
        if (!d || d->rows < 0 || d->dim <= 0 || d->dim > 32768) return "rows are negative or dim is not 1 .. 32768";
        if (d->dtype < VKHIP_DT_F16 || d->dtype > VKHIP_DT_F32) return "dtype is not F16, BF16 or F32";
        if (d->post < VKHIP_NORM_NONE || d->post > VKHIP_NORM_LAYER || d->pre < VKHIP_NORM_NONE || d->pre > VKHIP_NORM_LAYER) return "unknown norm";
        if (!(d->post_eps >= 0.f && d->post_eps < 1e30f) || !(d->pre_eps >= 0.f && d->pre_eps < 1e30f)) return "an eps is negative or not finite";
        if (!(d->alpha > -1e30f && d->alpha < 1e30f)) return "alpha is not finite";
        if (d->x_row < 0 || d->r_row < 0 || d->mod_row < 0 || d->mods < 0 || d->mod_rows < 0) return "a stride or count is negative";
        return nullptr;
    }

    constexpr int64_t kNormPast = (int64_t) 64 << 20; // bytes of x from which rows pass the caches (50000 of 1101 bf16 128 us, in them 139)

    template <typename T, int VEC, int N, int GT>
    static void residual_norm_start(const NormArgs &a, hipStream_t s) {
        constexpr int RPB = GT <= 64 ? 256 / GT : 1, THREADS = RPB * GT;
        const int64_t blocks = ceil_div(a.rows, RPB), layers = ceil_div(blocks, 0xFFFFFFFF / THREADS);
        const dim3    grid((unsigned) ceil_div(blocks, layers), (unsigned) layers);
        const bool    past = (int64_t) a.rows * a.dim * (int64_t) sizeof(T) >= kNormPast;
        if (a.dim % VEC) past ? residual_norm_kernel<T, VEC, N, GT, VEC != 1, true><<<grid, THREADS, 0, s>>>(a) : residual_norm_kernel<T, VEC, N, GT, VEC != 1, false><<<grid, THREADS, 0, s>>>(a);
        else past ? residual_norm_kernel<T, VEC, N, GT, false, true><<<grid, THREADS, 0, s>>>(a) : residual_norm_kernel<T, VEC, N, GT, false, false><<<grid, THREADS, 0, s>>>(a);
    }
    // Threads of a row: one for each vector of 8, in whole waves, up to 1024 threads. bf16, us with several vectors a thread, and with
    // one: 25088 rows of 2500 values 170 (four), 142 (two), 122; 12500 of 4096 104, 84, 86; 64 of 4096 6.8, 5.4, 4.6; 12800 of 1100 fp16
    // with gate, scale and shift 33.1 (three, a wave a row) and 28.5. A vector of 8 at any alignment, the last one overlapping: 12800 of
    // 1101 values 141.6 (value by value) and 30.7.
    // Several rows share a wave up to 256 values: 500000 of 88 bf16 283 a wave each, 84 in 16 threads.
    // Past 24576 values a thread's four vectors and the residual's do not fit the 128 registers of 1024 threads: 84 to 104 bytes a
    // lane go through scratch. 4096 rows bf16: of 16384 114 us (4.7 TB/s), of 24576 163 (4.9), of 28672 286 (3.3), of 32768 319 (3.4).
    template <typename T>
    static void residual_norm_threads(const NormArgs &a, hipStream_t s) {
        if (a.dim < 8) residual_norm_start<T, 1, 1, 8>(a, s);
        else if (a.dim <= 64) residual_norm_start<T, 8, 1, 8>(a, s);
        else if (a.dim <= 128) residual_norm_start<T, 8, 1, 16>(a, s);
        else if (a.dim <= 256) residual_norm_start<T, 8, 1, 32>(a, s);
        else if (a.dim <= 512) residual_norm_start<T, 8, 1, 64>(a, s);
        else if (a.dim <= 1024) residual_norm_start<T, 8, 1, 128>(a, s);
        else if (a.dim <= 1536) residual_norm_start<T, 8, 1, 192>(a, s);
        else if (a.dim <= 2048) residual_norm_start<T, 8, 1, 256>(a, s);
        else if (a.dim <= 6 * 512) residual_norm_start<T, 8, 1, 384>(a, s);
        else if (a.dim <= 4096) residual_norm_start<T, 8, 1, 512>(a, s);
        else if (a.dim <= 6144) residual_norm_start<T, 8, 1, 768>(a, s);
        else if (a.dim <= 8192) residual_norm_start<T, 8, 1, 1024>(a, s);
        else if (a.dim <= 16384) residual_norm_start<T, 8, 2, 1024>(a, s);
        else if (a.dim <= 24576) residual_norm_start<T, 8, 3, 1024>(a, s);
        else residual_norm_start<T, 8, 4, 1024>(a, s);
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

int vkhip_residual_norm(const vkhip_residual_norm_desc *d, const void *x, const void *r, const float *post_w, const float *post_b, const void *gate, const float *pre_w,
                        const float *pre_b, const void *scale, const void *shift, const int32_t *mod, void *h, void *y, vkhip_stream_t s) {
    if (const char *why = residual_norm_refusal(d)) return set_error(VKHIP_ERR_INVALID, "residual_norm: %s", why);
    if (d->rows == 0) return VKHIP_OK;
    const char *what = "residual_norm: %s";
    if ((!x && !r) || (!h && !y)) return set_error(VKHIP_ERR_INVALID, what, "null pointer");
    if (h == y) return set_error(VKHIP_ERR_INVALID, what, "h and y are one");
    if ((h && overlaps(d, d->h_row)) || (y && overlaps(d, d->y_row))) return set_error(VKHIP_ERR_INVALID, what, "rows share memory");
    for (const void *out : {(const void *) h, (const void *) y}) {
        const int64_t row = out == h ? d->h_row : d->y_row;
        if (out && ((out == x && row != d->x_row) || (out == r && row != d->r_row))) return set_error(VKHIP_ERR_INVALID, what, "in place with other strides");
    }
    const bool with_mod = gate || scale || shift;
    if (with_mod && d->mods < 1) return set_error(VKHIP_ERR_INVALID, what, "vectors without a number of them");
    if (with_mod && !mod && (d->mod_rows < 1 ? d->mods != 1 : (int64_t) d->mods * d->mod_rows < d->rows)) return set_error(VKHIP_ERR_INVALID, what, "rows without a vector");
    const uintptr_t elem = d->dtype == VKHIP_DT_F32 ? 4 : 2;
    const uintptr_t rows = (uintptr_t) x | (uintptr_t) r | (uintptr_t) h | (uintptr_t) y | (uintptr_t) gate | (uintptr_t) scale | (uintptr_t) shift;
    const uintptr_t weights = (uintptr_t) post_w | (uintptr_t) post_b | (uintptr_t) pre_w | (uintptr_t) pre_b;
    if (rows % elem || weights % 4 || (uintptr_t) mod % 4) return set_error(VKHIP_ERR_INVALID, what, "misaligned pointer");
    NormArgs a {};
    a.x = x, a.r = r, a.gate = gate, a.scale = scale, a.shift = shift, a.mod = with_mod ? mod : nullptr, a.h = h, a.y = y;
    a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w, a.pre_b = pre_b;
    a.rows = d->rows, a.dim = d->dim, a.post = d->post, a.pre = d->pre, a.mods = d->mods, a.mod_rows = with_mod ? d->mod_rows : 0;
    a.alpha = d->alpha, a.post_eps = d->post_eps, a.pre_eps = d->pre_eps, a.each = 1.f / (float) d->dim;
    a.x_row = d->x_row, a.r_row = d->r_row, a.h_row = d->h_row, a.y_row = d->y_row, a.mod_row = d->mod_row;
    a.in_place = (h && (h == x || h == r)) || (y && (y == x || y == r));
    hipStream_t st = resolve_stream(s);
    if (d->dtype == VKHIP_DT_F16) residual_norm_threads<half_t>(a, st);
    else if (d->dtype == VKHIP_DT_BF16) residual_norm_threads<bf16_t>(a, st);
    else residual_norm_threads<float>(a, st);
    return check_launch("residual_norm");
}

} // extern "C"
