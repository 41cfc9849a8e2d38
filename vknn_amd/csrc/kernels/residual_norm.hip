// What lies between two blocks of a token model: the block's output, normed, gated and scaled, joins the residual, whose
// norm, scaled and shifted, is the next block's input.
//
// Bound by memory: two values in and two out, once each. A row stays in the registers of the threads that read it, while
// its sums are formed: of squares, or first the mean and then the squared deviations from it (never E[z^2] - E[z]^2).
#include "tokens.h"

namespace vkhip {

    struct NormArgs {
        const void    *x, *r, *gate, *scale, *shift;
        const float   *post_w, *post_b, *pre_w, *pre_b;
        const int32_t *mod;
        void          *h, *y;
        int            rows, dim, post, pre, mods, mod_rows;
        float          alpha, post_eps, pre_eps;
        int64_t        x_row, r_row, h_row, y_row, mod_row;
    };

    // The sum over the threads of a row, in each of them.
    template <int GT>
    __device__ __forceinline__ float row_sum(float v, float *waves) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
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

    // GT threads a row, N vectors of VEC values each, vector i of thread t at (i GT + t) VEC. PAST: rows pass the caches.
    template <typename T, int VEC, int N, int GT, bool PAST>
    __global__ __launch_bounds__(GT < 256 ? 256 : GT) void residual_norm_kernel(NormArgs a) {
        typedef T     V __attribute__((ext_vector_type(VEC)));
        typedef float F __attribute__((ext_vector_type(VEC)));
        __shared__ float waves[GT / 64];
        constexpr int RPB = GT < 256 ? 256 / GT : 1; // rows of a workgroup
        const int     t = (int) threadIdx.x % GT;
        const int64_t row = ((int64_t) blockIdx.y * gridDim.x + blockIdx.x) * RPB + (int) threadIdx.x / GT;
        if (row >= a.rows) return; // the whole group
        const int64_t m = a.mod ? clampi(a.mod[row], 0, a.mods - 1) : (a.mod_rows ? row / a.mod_rows : 0);
        const float   count = (float) a.dim;
        F             z[N];
        const auto    at = [&](int i) { return (i * GT + t) * VEC; };
        const auto    in = [&](int i) { return at(i) < a.dim; };
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
            if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<V *>((T *) p + offset + at(i)));
            else *reinterpret_cast<V *>((T *) p + offset + at(i)) = v;
        };
        const auto norm = [&](int kind, float eps, const float *w, const float *b) {
            if (kind == VKHIP_NORM_NONE) return;
            if (kind == VKHIP_NORM_LAYER) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum += z[i][j];
                const float mean = row_sum<GT>(sum, waves) / count; // a row of one value has it as its mean, and no variance
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) z[i][j] = in(i) ? z[i][j] - mean : 0.f;
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum = __builtin_fmaf(z[i][j], z[i][j], sum);
            const float rstd = 1.f / __builtin_sqrtf(row_sum<GT>(sum, waves) / count + eps);
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
                for (int j = 0; j < VEC; ++j) z[i][j] = in(i) ? __builtin_fmaf(z[i][j] * a.alpha, g[j], r[i][j]) : 0.f;
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

    constexpr int     kNormWave = 1280, kNormWide = 4096;
    constexpr int64_t kNormPast = (int64_t) 64 << 20; // bytes of x from which rows pass the caches

    template <typename T, int VEC, int N, int GT>
    static void residual_norm_start(const NormArgs &a, hipStream_t s) {
        constexpr int RPB = GT < 256 ? 256 / GT : 1, THREADS = GT < 256 ? 256 : GT;
        const int64_t blocks = ceil_div(a.rows, RPB), layers = ceil_div(blocks, 0xFFFFFFFF / THREADS);
        const dim3    grid((unsigned) ceil_div(blocks, layers), (unsigned) layers);
        if ((int64_t) a.rows * a.dim * (int64_t) sizeof(T) >= kNormPast) residual_norm_kernel<T, VEC, N, GT, true><<<grid, THREADS, 0, s>>>(a);
        else residual_norm_kernel<T, VEC, N, GT, false><<<grid, THREADS, 0, s>>>(a);
    }
    // Vectors of a thread: as many as its row has, up to 32 values.
    template <typename T, int VEC, int GT>
    static void residual_norm_width(const NormArgs &a, hipStream_t s) {
        const int n = (int) ceil_div(a.dim, GT * VEC);
        if constexpr (VEC == 1) {
            if (n <= 8) residual_norm_start<T, VEC, 8, GT>(a, s);
            else if (n <= 16) residual_norm_start<T, VEC, 16, GT>(a, s);
            else residual_norm_start<T, VEC, 32, GT>(a, s);
        } else if (n == 1) residual_norm_start<T, VEC, 1, GT>(a, s);
        else if (n == 2) residual_norm_start<T, VEC, 2, GT>(a, s);
        else if (n == 3) residual_norm_start<T, VEC, 3, GT>(a, s);
        else if (n == 4) residual_norm_start<T, VEC, 4, GT>(a, s);
        else if constexpr (VEC == 4) {
            if (n == 5) residual_norm_start<T, VEC, 5, GT>(a, s);
            else if (n == 6) residual_norm_start<T, VEC, 6, GT>(a, s);
            else residual_norm_start<T, VEC, 8, GT>(a, s);
        }
    }
    // Threads of a row: a wave up to 1280 values, 256 threads up to 4096, 1024 above; a vector or two a thread is what keeps
    // many rows under way (bf16, us at 411 MB of rows, x, r, h and y: 2048 values in a wave 206, in 256 threads 164; 8192 in 256, 512,
    // 1024 threads 211, 196, 172; 12800 x 1100 fp16 with gate, scale and shift 35 and 38).
    template <typename T, int VEC>
    static void residual_norm_threads(const NormArgs &a, hipStream_t s) {
        if (a.dim <= kNormWave) residual_norm_width<T, VEC, 64>(a, s);
        else if (a.dim <= kNormWide) residual_norm_width<T, VEC, 256>(a, s);
        else residual_norm_width<T, VEC, 1024>(a, s);
    }
    template <typename T>
    static void residual_norm_vectors(const NormArgs &a, int vec, hipStream_t s) {
        if (vec == 8) residual_norm_threads<T, 8>(a, s);
        else if (vec == 4) residual_norm_threads<T, 4>(a, s);
        else residual_norm_threads<T, 1>(a, s);
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
    a.alpha = d->alpha, a.post_eps = d->post_eps, a.pre_eps = d->pre_eps;
    a.x_row = d->x_row, a.r_row = d->r_row, a.h_row = d->h_row, a.y_row = d->y_row, a.mod_row = d->mod_row;
    // vectors of 8 or 4 values where rows come in such
    const int64_t all = d->dim | (x ? d->x_row : 0) | (r ? d->r_row : 0) | (h ? d->h_row : 0) | (y ? d->y_row : 0) | (with_mod ? d->mod_row : 0);
    const auto    fits = [&](int vec) {
        const uintptr_t bytes = (uintptr_t) vec * elem;
        return all % vec == 0 && rows % (bytes < 16 ? bytes : 16) == 0 && weights % 16 == 0;
    };
    const int   vec = fits(8) ? 8 : fits(4) ? 4 : 1;
    hipStream_t st  = resolve_stream(s);
    if (d->dtype == VKHIP_DT_F16) residual_norm_vectors<half_t>(a, vec, st);
    else if (d->dtype == VKHIP_DT_BF16) residual_norm_vectors<bf16_t>(a, vec, st);
    else residual_norm_vectors<float>(a, vec, st);
    return check_launch("residual_norm");
}

} // extern "C"
