// Group norm with an activation, NHWC rows and NC4HW4 in any combination.
//
// The mean and variance of a group are joined from parts (Chan's update): each thread forms the exact mean
// and the squared deviations M2 of a few loaded values, and parts (n, mean, M2) merge as
//   d = mean_b - mean_a,  mean = mean_a + d n_b / n,  M2 = M2_a + M2_b + d^2 n_a n_b / n
// so a mean far from zero costs no digits of the variance, as the difference of two sums would.
#include "tokens.h"

namespace vkhip {

    struct GnArgs {
        const void  *x;
        void        *y;
        const float *gamma, *beta;
        float2      *part; // (mean, M2) per image, chunk, group
        int          N, C, CV, HW, G, Cg, chunk, chunks;
        int64_t      x_row, y_row;
        int          act;
        float        lo, hi, eps;
    };

    struct Moments {
        float n, mean, m2;
    };
    __device__ __forceinline__ Moments merge(Moments a, Moments b) {
        const float n = a.n + b.n;
        if (n == 0.f) return a;
        const float r = b.n / n, d = b.mean - a.mean;
        return {n, a.mean + d * r, a.m2 + b.m2 + d * d * a.n * r};
    }

    // `lanes` (a power of two up to 64) neighbouring lanes each hold moments: merged in all of them.
    __device__ __forceinline__ Moments merge_lanes(Moments m, int lanes) {
        for (int o = 1; o < lanes; o <<= 1) {
            const Moments t = {__shfl_xor(m.n, o), __shfl_xor(m.mean, o), __shfl_xor(m.m2, o)};
            m               = merge(m, t);
        }
        return m;
    }

    // VEC channels of one pixel. AL: whole aligned vectors; otherwise channel by channel up to C.
    template <typename T, int VEC, bool NC4, bool AL>
    struct GnIo {
        static __device__ __forceinline__ int64_t at(const GnArgs &a, int64_t row, int n, int p, int cv) {
            return NC4 ? (((int64_t) n * a.CV + cv) * a.HW + p) * 4 : ((int64_t) n * a.HW + p) * row + cv * VEC;
        }
        typedef T V __attribute__((ext_vector_type(VEC)));
        static __device__ __forceinline__ void load(const GnArgs &a, int n, int p, int cv, float *v) {
            const T *s = (const T *) a.x + at(a, a.x_row, n, p, cv);
            if constexpr (NC4 || AL) {
                const V t = *reinterpret_cast<const V *>(s);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = (float) t[j];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = cv * VEC + j < a.C ? (float) s[j] : 0.f;
            }
        }
        static __device__ __forceinline__ void store(const GnArgs &a, int n, int p, int cv, const float *v) {
            T *d = (T *) a.y + at(a, a.y_row, n, p, cv);
            if constexpr (NC4 || AL) {
                V t;
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[j] = (T) (!NC4 || cv * VEC + j < a.C ? v[j] : 0.f);
                *reinterpret_cast<V *>(d) = t;
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (cv * VEC + j < a.C) d[j] = (T) v[j];
            }
        }
    };

    constexpr int kGnThreads = 256;
    constexpr int kGnBatch   = 4; // pixels a thread has in flight

    // Threads over (channel vectors, pixels): neighbouring threads read neighbouring memory, which is the
    // channels of an NHWC row and the pixels of an NC4HW4 plane.
    struct GnLane {
        int cv, cvs, pl, pls;
    };
    template <bool NC4>
    __device__ __forceinline__ GnLane gn_lane(const GnArgs &a) {
        const int t = threadIdx.x;
        if (NC4) return {t >> 6, kGnThreads / 64, t & 63, 64};
        const int cvs = a.CV < kGnThreads ? a.CV : kGnThreads, pls = kGnThreads / cvs;
        return {t % cvs, cvs, t / cvs, pls};
    }

    template <typename T, int VEC, bool XN4, bool XAL>
    __global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(GnArgs a) {
        extern __shared__ float sm[];
        Moments *ent = reinterpret_cast<Moments *>(sm);                    // [pixel lane][channel of the pass]
        float2  *ch  = reinterpret_cast<float2 *>(sm + 3 * kGnThreads * VEC); // (mean, M2) of every channel over the chunk
        const int    n = blockIdx.y, p0 = blockIdx.x * a.chunk, np = min(a.chunk, a.HW - p0);
        const GnLane L = gn_lane<XN4>(a);
        for (int base = 0; base < a.CV; base += L.cvs) {
            const int cv = base + L.cv;
            if (L.pl < L.pls) {
                Moments m[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) m[j] = {0.f, 0.f, 0.f};
                if (cv < a.CV)
                    for (int p = L.pl; p < np; p += L.pls * kGnBatch) {
                        float v[kGnBatch][VEC];
                        int   k = 0;
#pragma unroll
                        for (int u = 0; u < kGnBatch; ++u) {
                            const bool in = p + u * L.pls < np;
                            k += in;
                            GnIo<T, VEC, XN4, XAL>::load(a, n, p0 + (in ? p + u * L.pls : p), cv, v[u]);
                        }
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            float s = 0.f, q = 0.f;
#pragma unroll
                            for (int u = 0; u < kGnBatch; ++u) s += u < k ? v[u][j] : 0.f;
                            const float mean = s / (float) k;
#pragma unroll
                            for (int u = 0; u < kGnBatch; ++u) q += u < k ? (v[u][j] - mean) * (v[u][j] - mean) : 0.f;
                            m[j] = merge(m[j], {(float) k, mean, q});
                        }
                    }
#pragma unroll
                for (int j = 0; j < VEC; ++j) ent[(L.pl * L.cvs + L.cv) * VEC + j] = m[j];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < L.cvs * VEC && base * VEC + c < a.C; c += kGnThreads) {
                Moments m = {0.f, 0.f, 0.f};
                for (int r = 0; r < L.pls; ++r) m = merge(m, ent[r * L.cvs * VEC + c]);
                ch[base * VEC + c] = make_float2(m.mean, m.m2);
            }
            __syncthreads();
        }
        int lanes = 64;
        while (lanes > 1 && lanes * a.G > kGnThreads) lanes >>= 1;
        for (int g0 = 0; g0 < a.G; g0 += kGnThreads / lanes) {
            const int g = g0 + threadIdx.x / lanes;
            Moments   m = {0.f, 0.f, 0.f};
            if (g < a.G)
                for (int c = threadIdx.x % lanes; c < a.Cg; c += lanes) m = merge(m, {(float) np, ch[g * a.Cg + c].x, ch[g * a.Cg + c].y});
            m = merge_lanes(m, lanes);
            if (g < a.G && threadIdx.x % lanes == 0) a.part[((int64_t) n * a.chunks + blockIdx.x) * a.G + g] = make_float2(m.mean, m.m2);
        }
    }

    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL>
    __global__ __launch_bounds__(kGnThreads) void gn_apply_kernel(GnArgs a) {
        extern __shared__ float sm[];
        float2   *st = reinterpret_cast<float2 *>(sm); // (mean, rstd) of every group
        const int n = blockIdx.y, p0 = blockIdx.x * a.chunk, np = min(a.chunk, a.HW - p0);
        int       lanes = 64;
        while (lanes > 1 && lanes * a.G > kGnThreads) lanes >>= 1;
        for (int g0 = 0; g0 < a.G; g0 += kGnThreads / lanes) {
            const int g = g0 + threadIdx.x / lanes;
            Moments   m = {0.f, 0.f, 0.f};
            if (g < a.G)
                for (int k = threadIdx.x % lanes; k < a.chunks; k += lanes) {
                    const float2 q = a.part[((int64_t) n * a.chunks + k) * a.G + g];
                    m              = merge(m, {(float) min(a.chunk, a.HW - k * a.chunk) * (float) a.Cg, q.x, q.y});
                }
            m = merge_lanes(m, lanes);
            if (g < a.G && threadIdx.x % lanes == 0) st[g] = make_float2(m.mean, 1.f / sqrtf(m.m2 / m.n + a.eps));
        }
        __syncthreads();
        const GnLane L = gn_lane<XN4>(a);
        if (L.pl >= L.pls) return;
        for (int cv = L.cv; cv < a.CV; cv += L.cvs) {
            float mean[VEC], mul[VEC], add[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = min(cv * VEC + j, a.C - 1), g = c / a.Cg;
                mean[j]     = st[g].x;
                mul[j]      = st[g].y * (a.gamma ? a.gamma[c] : 1.f);
                add[j]      = a.beta ? a.beta[c] : 0.f;
            }
            for (int p = L.pl; p < np; p += L.pls * kGnBatch) {
                float v[kGnBatch][VEC];
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u) GnIo<T, VEC, XN4, XAL>::load(a, n, p0 + (p + u * L.pls < np ? p + u * L.pls : p), cv, v[u]);
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u) {
                    if (p + u * L.pls >= np) break;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[u][j] = apply_act((v[u][j] - mean[j]) * mul[j] + add[j], a.act, a.lo, a.hi);
                    GnIo<T, VEC, YN4, YAL>::store(a, n, p0 + p + u * L.pls, cv, v[u]);
                }
            }
        }
    }

    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL>
    static int gn_launch(const GnArgs &a, hipStream_t s) {
        const dim3 grid((unsigned) a.chunks, (unsigned) a.N);
        gn_stats_kernel<T, VEC, XN4, XAL><<<grid, kGnThreads, (3 * kGnThreads * VEC + 2 * a.C) * sizeof(float), s>>>(a);
        int rc = check_launch("group_norm statistics");
        if (rc) return rc;
        gn_apply_kernel<T, VEC, XN4, YN4, XAL, YAL><<<grid, kGnThreads, 2 * a.G * sizeof(float), s>>>(a);
        return check_launch("group_norm");
    }

    static int gn_chunks(const vkhip_group_norm_desc *d) {
        const int64_t hw = (int64_t) d->H * d->W;
        int64_t       k  = ceil_div(1024, d->N);
        if (k > 128) k = 128;
        if (k > ceil_div(hw, 32)) k = ceil_div(hw, 32);
        const int64_t chunk = ceil_div(hw, k);
        return (int) ceil_div(hw, chunk);
    }

    static const char *gn_refusal(const vkhip_group_norm_desc *d) {
        if (!d || d->N < 0 || d->H < 0 || d->W < 0 || d->C <= 0 || d->groups <= 0) return "bad sizes";
        if (d->C % d->groups) return "channels are not a multiple of the groups";
        if ((int64_t) d->H * d->W > 0x7FFFFFF0 || d->N > 65535 || d->C > 4096) return "N <= 65535, C <= 4096 and H * W < 2^31";
        if (d->dtype < VKHIP_DT_F16 || d->dtype > VKHIP_DT_F32) return "unknown dtype";
        if ((d->x_fmt != 1 && d->x_fmt != 2) || (d->y_fmt != 1 && d->y_fmt != 2)) return "formats are 1 (NHWC) and 2 (NC4HW4)";
        if ((d->x_fmt == 2 || d->y_fmt == 2) && d->dtype != VKHIP_DT_F16) return "NC4HW4 is F16";
        if ((d->x_row && d->x_row < d->C) || (d->y_row && d->y_row < d->C)) return "rows shorter than the channels";
        if (d->act < VKHIP_ACT_NONE || d->act > VKHIP_ACT_HARDSIGMOID) return "unknown activation";
        if (!(d->eps >= 0.f)) return "eps is negative";
        return nullptr;
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

size_t vkhip_group_norm_workspace_bytes(const vkhip_group_norm_desc *d) {
    if (gn_refusal(d) || d->N == 0 || d->H == 0 || d->W == 0) return 0;
    return (size_t) d->N * gn_chunks(d) * d->groups * sizeof(float2);
}

int vkhip_group_norm(const vkhip_group_norm_desc *d, const void *x, const float *gamma, const float *beta, void *y, void *workspace,
                     vkhip_stream_t s) {
    if (const char *why = gn_refusal(d)) return set_error(VKHIP_ERR_INVALID, "group_norm: %s", why);
    if (d->N == 0 || d->H == 0 || d->W == 0) return VKHIP_OK;
    if (!x || !y || !workspace) return set_error(VKHIP_ERR_INVALID, "group_norm: null pointer");
    const int    size = d->dtype == VKHIP_DT_F32 ? 4 : 2;
    const bool   xn4 = d->x_fmt == 2, yn4 = d->y_fmt == 2;
    if (((uintptr_t) x) % (xn4 ? 8 : size) || ((uintptr_t) y) % (yn4 ? 8 : size) || misaligned16(workspace) || ((uintptr_t) gamma) % 4 || ((uintptr_t) beta) % 4)
        return set_error(VKHIP_ERR_INVALID, "group_norm: misaligned pointer");
    GnArgs a {};
    a.x = x, a.y = y, a.gamma = gamma, a.beta = beta, a.part = (float2 *) workspace;
    a.N = d->N, a.C = d->C, a.HW = d->H * d->W, a.G = d->groups, a.Cg = d->C / d->groups;
    a.x_row = d->x_row ? d->x_row : d->C, a.y_row = d->y_row ? d->y_row : d->C;
    a.act = d->act, a.lo = d->act_lo, a.hi = d->act_hi, a.eps = d->eps;
    a.chunks      = gn_chunks(d);
    a.chunk       = (int) ceil_div(a.HW, a.chunks);
    hipStream_t q = resolve_stream(s);
    // the widest vector that divides the channels and that both sides' rows start on
    const auto fits = [&](int vec, bool side_x, bool side_y) {
        const int64_t by = (int64_t) vec * size;
        return d->C % vec == 0 && (!side_x || (((uintptr_t) x) % by == 0 && a.x_row % vec == 0)) && (!side_y || (((uintptr_t) y) % by == 0 && a.y_row % vec == 0));
    };
    if (xn4 || yn4) {
        a.CV = (d->C + 3) / 4;
        if (xn4 && yn4) return gn_launch<half_t, 4, true, true, true, true>(a, q);
        const bool al = fits(4, !xn4, !yn4);
        if (xn4) return al ? gn_launch<half_t, 4, true, false, true, true>(a, q) : gn_launch<half_t, 4, true, false, true, false>(a, q);
        return al ? gn_launch<half_t, 4, false, true, true, true>(a, q) : gn_launch<half_t, 4, false, true, false, true>(a, q);
    }
    const int vec = size == 2 && fits(8, true, true) ? 8 : (fits(4, true, true) ? 4 : 1);
    a.CV          = d->C / vec;
    if (d->dtype == VKHIP_DT_F32) return vec == 4 ? gn_launch<float, 4, false, false, true, true>(a, q) : gn_launch<float, 1, false, false, true, true>(a, q);
    if (d->dtype == VKHIP_DT_BF16) {
        if (vec == 8) return gn_launch<bf16_t, 8, false, false, true, true>(a, q);
        return vec == 4 ? gn_launch<bf16_t, 4, false, false, true, true>(a, q) : gn_launch<bf16_t, 1, false, false, true, true>(a, q);
    }
    if (vec == 8) return gn_launch<half_t, 8, false, false, true, true>(a, q);
    return vec == 4 ? gn_launch<half_t, 4, false, false, true, true>(a, q) : gn_launch<half_t, 1, false, false, true, true>(a, q);
}

} // extern "C"
