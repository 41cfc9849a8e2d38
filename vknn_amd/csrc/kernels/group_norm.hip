// Group norm with an activation, NHWC rows and NC4HW4 in any combination.
//
// The mean and variance of a group are joined from parts (Chan's update): each thread forms the exact mean
// and the squared deviations M2 of a few loaded values, and parts (n, mean, M2) merge as
//   d = mean_b - mean_a,  mean = mean_a + d n_b / n,  M2 = M2_a + M2_b + d^2 n_a n_b / n
// so a mean far from zero costs no digits of the variance, as the difference of two sums would. d n_a n_b / n is
// formed before its product with d: 0 for a first part, whose d is the whole mean and whose square may leave fp32.
//
// Bound by memory. What a workgroup can hold in its registers (a group of one image) is read once, in one
// launch (gn_slab_kernel). Larger groups take two launches, statistics of chunks of pixels and the output, and
// read x twice: 64 x 256 x 56 x 56 fp16 62 us, the statistics 22 (103 MB at 4.6 TB/s) and the output 39 (206 MB
// at 5.3 TB/s, a large copy's rate); one launch of slabs takes 112 there, since 16-byte pieces of 512-byte rows cost
// whole cache lines. The smallest calls are a launch: 1 x 128 x 40 x 40 6.0 us.
#include "tokens.h"
#include <type_traits>

namespace vkhip {

    struct GnArgs {
        const void  *x;
        void        *y;
        const float *gamma, *beta;
        float2      *part; // (mean, M2) per image, chunk, group
        int          N, C, CV, HW, G, Cg, chunk, chunks;
        int64_t      x_row, y_row;
        int          kind; // of activation, see gn_act
        float        s, t, lo, hi, eps;
    };

    // Every activation is one of three forms, so that a loop over a batch branches once:
    // 0 clamp(s z + t, lo, hi), 1 z clamp(s z + t, lo, hi), 2 z sigmoid(z). NaN passes.
    template <int KIND>
    __device__ __forceinline__ float gn_act(const GnArgs &a, float z) {
        if constexpr (KIND == 2) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
        float g = __builtin_fmaf(a.s, z, a.t);
        g       = g < a.lo ? a.lo : (g > a.hi ? a.hi : g);
        return KIND ? z * g : g;
    }
    template <typename F>
    __device__ __forceinline__ void gn_by_kind(int kind, F f) {
        if (kind == 0) f(std::integral_constant<int, 0>());
        else if (kind == 1) f(std::integral_constant<int, 1>());
        else f(std::integral_constant<int, 2>());
    }

    struct Moments {
        float n, mean, m2;
    };
    __device__ __forceinline__ Moments merge(Moments a, Moments b) {
        const float n = a.n + b.n;
        if (n == 0.f) return a;
        const float r = b.n * __builtin_amdgcn_rcpf(n), d = b.mean - a.mean; // 1 ulp of the share: 1e-7 of a part's weight
        return {n, a.mean + d * r, a.m2 + b.m2 + d * (d * (a.n * r))};
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
        static __device__ __forceinline__ V raw(const GnArgs &a, int n, int p, int cv) {
            const T *s = (const T *) a.x + at(a, a.x_row, n, p, cv);
            if constexpr (NC4 || AL) return *reinterpret_cast<const V *>(s);
            V t;
#pragma unroll
            for (int j = 0; j < VEC; ++j) t[j] = cv * VEC + j < a.C ? s[j] : (T) 0.f;
            return t;
        }
        // STREAM: past the caches, for whole lines of a wave's store (from one format to the same; slabs of NC4HW4), so
        // that x stays for its second read: 64 x 256 x 56 x 56 75 -> 63 us, NC4HW4 16 x 128 x 80 x 80 19.2 -> 14.9, with
        // the next norm reading y at once 17.0 -> 15.6 (64 x 64 x 112 x 112 59.4 -> 60.8). Pieces of lines lose: to the
        // other format 30 -> 67 us, the rows of 1 x 128 x 40 x 40 5.6 -> 6.3.
        template <bool STREAM>
        static __device__ __forceinline__ void store(const GnArgs &a, int n, int p, int cv, const float *v) {
            T *d = (T *) a.y + at(a, a.y_row, n, p, cv);
            if constexpr (NC4 || AL) {
                V t;
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[j] = (T) (!NC4 || cv * VEC + j < a.C ? v[j] : 0.f);
                if constexpr (STREAM) __builtin_nontemporal_store(t, reinterpret_cast<V *>(d));
                else *reinterpret_cast<V *>(d) = t;
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (cv * VEC + j < a.C) d[j] = (T) v[j];
            }
        }
    };

    constexpr int kGnThreads = 256;
    constexpr int kGnBatch   = 8; // pixels a thread has in flight

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

    // Moments of a thread's channels over the chunk's pixels pl, pl + pls, ...: eight pixels at a time, whose
    // mean and deviations are formed in registers and merged with equal counts.
    template <typename T, int VEC, bool XN4, bool XAL>
    __device__ __forceinline__ void gn_thread_moments(const GnArgs &a, int n, int p0, int np, int cv, int pl, int pls, float (&mean)[VEC], float (&m2)[VEC]) {
        using X = GnIo<T, VEC, XN4, XAL>;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mean[j] = m2[j] = 0.f;
        float     count = 0.f;
        int       base  = 0;
        const int step  = pls * kGnBatch;
        for (; base + step <= np; base += step) {
            typename X::V v[kGnBatch];
#pragma unroll
            for (int u = 0; u < kGnBatch; ++u) v[u] = X::raw(a, n, p0 + base + pl + u * pls, cv);
            __builtin_amdgcn_sched_barrier(0); // the loads stay ahead of the first use
            const float share = kGnBatch * __builtin_amdgcn_rcpf(count + kGnBatch), cross = count * share;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float s = 0.f, q = 0.f;
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u) s += (float) v[u][j];
                s *= 1.f / kGnBatch;
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u) q = __builtin_fmaf((float) v[u][j] - s, (float) v[u][j] - s, q);
                const float d = s - mean[j];
                mean[j]       = __builtin_fmaf(d, share, mean[j]);
                m2[j] += __builtin_fmaf(d, d * cross, q);
            }
            count += kGnBatch;
        }
        const int left = (np - base - pl + pls - 1) / pls; // pixels of this thread's last, shorter batch
        if (left <= 0) return;
        typename X::V v[kGnBatch];
#pragma unroll
        for (int u = 0; u < kGnBatch; ++u) v[u] = X::raw(a, n, p0 + min(base + pl + u * pls, np - 1), cv);
        __builtin_amdgcn_sched_barrier(0);
        const float k = (float) left, share = k * __builtin_amdgcn_rcpf(count + k), cross = count * share, ik = 1.f / k;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float s = 0.f, q = 0.f;
#pragma unroll
            for (int u = 0; u < kGnBatch; ++u) s += u < left ? (float) v[u][j] : 0.f;
            s *= ik;
#pragma unroll
            for (int u = 0; u < kGnBatch; ++u) q += u < left ? ((float) v[u][j] - s) * ((float) v[u][j] - s) : 0.f;
            const float d = s - mean[j];
            mean[j]       = __builtin_fmaf(d, share, mean[j]);
            m2[j] += __builtin_fmaf(d, d * cross, q);
        }
    }
    __device__ __forceinline__ float gn_thread_count(int np, int pl, int pls) { return pl < np ? (float) ((np - pl + pls - 1) / pls) : 0.f; }

    // Statistics of a chunk of pixels into a.part: (mean, M2) of every channel from NC4HW4, where a wave is 64
    // pixels of one block of channels, and of every group from NHWC, where the threads' channels meet in LDS.
    template <typename T, int VEC, bool XN4, bool XAL>
    __global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(GnArgs a) {
        extern __shared__ float sm[];
        float2      *ent = reinterpret_cast<float2 *>(sm);
        const int    n = blockIdx.y, p0 = blockIdx.x * a.chunk, np = min(a.chunk, a.HW - p0);
        const GnLane L = gn_lane<XN4>(a);
        float        mean[VEC], m2[VEC];
        if constexpr (XN4) {
            const int cv = blockIdx.z * L.cvs + L.cv;
            if (cv >= a.CV) return;
            gn_thread_moments<T, VEC, XN4, XAL>(a, n, p0, np, cv, L.pl, L.pls, mean, m2);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Moments m = merge_lanes({gn_thread_count(np, L.pl, L.pls), mean[j], m2[j]}, 64);
                if (L.pl == 0 && cv * VEC + j < a.C) a.part[((int64_t) n * a.chunks + blockIdx.x) * a.C + cv * VEC + j] = make_float2(m.mean, m.m2);
            }
            return;
        }
        const int width = (a.CV < kGnThreads ? L.cvs : a.CV) * VEC; // channels of a row of entries
        for (int cv = L.cv; cv < a.CV; cv += L.cvs) {
            if (L.pl >= L.pls) break;
            gn_thread_moments<T, VEC, XN4, XAL>(a, n, p0, np, cv, L.pl, L.pls, mean, m2);
#pragma unroll
            for (int j = 0; j < VEC; ++j) ent[L.pl * width + cv * VEC + j] = make_float2(mean[j], m2[j]);
        }
        __syncthreads();
        const int rows = L.pls;
        int       lanes = 64;
        while (lanes > 1 && lanes * a.G > kGnThreads) lanes >>= 1;
        for (int g0 = 0; g0 < a.G; g0 += kGnThreads / lanes) {
            const int g = g0 + threadIdx.x / lanes;
            Moments   m = {0.f, 0.f, 0.f};
            if (g < a.G)
                for (int i = threadIdx.x % lanes; i < rows * a.Cg; i += lanes) {
                    const int    r = i / a.Cg, c = g * a.Cg + i - r * a.Cg;
                    const float2 e = ent[r * width + c];
                    m              = merge(m, {gn_thread_count(np, r, rows), e.x, e.y});
                }
            m = merge_lanes(m, lanes);
            if (g < a.G && threadIdx.x % lanes == 0) a.part[((int64_t) n * a.chunks + blockIdx.x) * a.G + g] = make_float2(m.mean, m.m2);
        }
    }

    // From NC4HW4 every workgroup joins the entries of all channels of its groups, chunks * Cg of each, 64 lanes a group at
    // most. That is little next to its pixels but for wide groups: 1 x 512 x 112 x 112 in 32 groups 17 us, in two 50, in one
    // 88.
    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL>
    __global__ __launch_bounds__(kGnThreads) void gn_apply_kernel(GnArgs a) {
        extern __shared__ float sm[];
        float2   *st = reinterpret_cast<float2 *>(sm); // (mean, rstd) of every group
        // last image first: what the statistics read last is still in the caches
        const int n = gridDim.y - 1 - blockIdx.y, p0 = (gridDim.x - 1 - blockIdx.x) * a.chunk, np = min(a.chunk, a.HW - p0);
        // the groups of the workgroup's channels
        const int g_first = XN4 ? blockIdx.z * (kGnThreads / 64) * VEC / a.Cg : 0;
        const int gs      = XN4 ? min(a.G - 1, (((int) blockIdx.z + 1) * (kGnThreads / 64) * VEC - 1) / a.Cg) - g_first + 1 : a.G;
        const int per = XN4 ? a.Cg : 1, row = XN4 ? a.C : a.G; // entries of a group in a chunk, of a chunk
        int       lanes = 64;
        while (lanes > 1 && lanes * gs > kGnThreads) lanes >>= 1;
        for (int g0 = 0; g0 < gs; g0 += kGnThreads / lanes) {
            const int g = g0 + threadIdx.x / lanes;
            Moments   m = {0.f, 0.f, 0.f};
            if (g < gs)
                for (int i = threadIdx.x % lanes; i < a.chunks * per; i += lanes) {
                    const int    k = i / per;
                    const float2 q = a.part[((int64_t) n * a.chunks + k) * row + (g_first + g) * per + i - k * per];
                    m              = merge(m, {(float) min(a.chunk, a.HW - k * a.chunk) * (XN4 ? 1.f : (float) a.Cg), q.x, q.y});
                }
            m = merge_lanes(m, lanes);
            if (g < gs && threadIdx.x % lanes == 0) st[g] = make_float2(m.mean, 1.f / sqrtf(m.m2 / m.n + a.eps));
        }
        __syncthreads();
        const GnLane L = gn_lane<XN4>(a);
        if (L.pl >= L.pls) return;
        for (int cv = XN4 ? blockIdx.z * L.cvs + L.cv : L.cv; cv < (XN4 ? min(a.CV, ((int) blockIdx.z + 1) * L.cvs) : a.CV); cv += L.cvs) {
            float mean[VEC], mul[VEC], add[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = min(cv * VEC + j, a.C - 1), g = c / a.Cg - g_first;
                mean[j]     = st[g].x;
                mul[j]      = st[g].y * (a.gamma ? a.gamma[c] : 1.f);
                add[j]      = a.beta ? a.beta[c] : 0.f;
            }
            gn_by_kind(a.kind, [&](auto kind) __attribute__((always_inline)) {
                using X        = GnIo<T, VEC, XN4, XAL>;
                const int step = L.pls * kGnBatch;
                const auto put = [&](const typename X::V &x, int p) __attribute__((always_inline)) {
                    float v[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] = gn_act<decltype(kind)::value>(a, ((float) x[j] - mean[j]) * mul[j] + add[j]);
                    GnIo<T, VEC, YN4, YAL>::template store<XN4 == YN4>(a, n, p0 + p, cv, v);
                };
                int base = 0;
                for (; base + step <= np; base += step) {
                    typename X::V x[kGnBatch];
#pragma unroll
                    for (int u = 0; u < kGnBatch; ++u) x[u] = X::raw(a, n, p0 + base + L.pl + u * L.pls, cv);
                    __builtin_amdgcn_sched_barrier(0); // the loads stay ahead of the first use
#pragma unroll
                    for (int u = 0; u < kGnBatch; ++u) put(x[u], base + L.pl + u * L.pls);
                }
                if (base + L.pl >= np) return;
                typename X::V x[kGnBatch]; // fewer than eight are left
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u) x[u] = X::raw(a, n, p0 + min(base + L.pl + u * L.pls, np - 1), cv);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < kGnBatch; ++u)
                    if (base + L.pl + u * L.pls < np) put(x[u], base + L.pl + u * L.pls);
            });
        }
    }

    // Sums of a wave and of a workgroup; the latter in a fixed order, the same in every thread.
    template <int CTRL>
    __device__ __forceinline__ float dpp_add(float x) {
        return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
    }
    __device__ __forceinline__ float wave_sum(float x) {
        x = dpp_add<0x111>(x); // row_shr 1, 2, 4, 8: lane 15 of each 16 has its row
        x = dpp_add<0x112>(x);
        x = dpp_add<0x114>(x);
        x = dpp_add<0x118>(x);
        x = dpp_add<0x142>(x); // row_bcast 15, 31: lane 63 has them all
        x = dpp_add<0x143>(x);
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
    }
    template <int THREADS, int GS>
    __device__ __forceinline__ void block_sums(float (&x)[GS], float (*red)[GS]) {
#pragma unroll
        for (int g = 0; g < GS; ++g) {
            x[g] = wave_sum(x[g]);
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][g] = x[g];
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < GS; ++g) {
            x[g] = red[0][g];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) x[g] += red[w][g];
        }
    }

    // One launch: a workgroup owns a slab of one image and keeps all of its pixels to itself: mean, then
    // deviations from it, then the output, x read once. A slab is a group of SV whole vectors of channels or
    // (GV > 1) a vector of GV whole groups. Every thread loads R pixels, those past its own the last one again: at 7 x 7
    // seven loads of eight. The compiler keeps x's fp32 values from the first sum to the output beside x itself. 256
    // threads hold them in registers; 1024 threads (128 registers each) hold 8 pixels of 4 channels, 16 where they are one
    // group's, and 8 pixels of 8 channels of one group (fp16: of two). The other variants of 1024 threads put up to 976
    // bytes a lane into scratch.
    // Slabs of several groups side by side, whose rows' pieces are longer, measured 34 us against 24 (64 x 256 x 28 x 28,
    // four groups), in a form that may have used scratch too: not settled.
    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL, int THREADS, int R, int GV>
    __global__ __launch_bounds__(THREADS) void gn_slab_kernel(GnArgs a, int SV, int spread) {
        using X             = GnIo<T, VEC, XN4, XAL>;
        constexpr int SHARE = VEC / GV; // channels of a vector in one group
        __shared__ float red[2][THREADS / 64][GV];
        // images over the XCDs, the slabs of one on the same: their pieces of a cache line meet in its L2
        const int n = blockIdx.y * spread + blockIdx.x % spread, slab = blockIdx.x / spread;
        if (n >= a.N) return;
        const int pls = THREADS / SV, v = XN4 ? threadIdx.x / pls : threadIdx.x % SV, pl = XN4 ? threadIdx.x % pls : threadIdx.x / SV;
        const int cv = slab * SV + v;
        // pixels of this thread; the loads of the others repeat the last pixel
        const int mine = (int) threadIdx.x < pls * SV && cv < a.CV && pl < a.HW ? (a.HW - pl + pls - 1) / pls : 0;
        typename X::V x[R];
#pragma unroll
        for (int k = 0; k < R; ++k) x[k] = X::raw(a, n, min(pl + k * pls, a.HW - 1), min(cv, a.CV - 1));
        __builtin_amdgcn_sched_barrier(0); // the loads stay ahead of the first use
        float       mean[GV], m2[GV];
        const float count = (float) a.HW * (float) a.Cg;
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            float sum[GV];
#pragma unroll
            for (int g = 0; g < GV; ++g) sum[g] = 0.f;
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int g = 0; g < GV; ++g) {
                    float part = 0.f;
#pragma unroll
                    for (int j = 0; j < SHARE; ++j) {
                        const bool  lost = XN4 && SHARE * g + j + cv * VEC >= a.C; // past the channels
                        const float d    = lost ? 0.f : (float) x[k][SHARE * g + j] - (pass ? mean[g] : 0.f);
                        part             = pass ? __builtin_fmaf(d, d, part) : part + d;
                    }
                    sum[g] += k < mine ? part : 0.f;
                }
            block_sums<THREADS, GV>(sum, red[pass]);
#pragma unroll
            for (int g = 0; g < GV; ++g) (pass ? m2 : mean)[g] = sum[g] / count;
        }
        float mul[VEC], be[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int c = min(cv * VEC + j, a.C - 1);
            mul[j]      = (a.gamma ? a.gamma[c] : 1.f) / sqrtf(m2[j / SHARE] + a.eps);
            be[j]       = a.beta ? a.beta[c] : 0.f;
        }
        gn_by_kind(a.kind, [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float o[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = gn_act<decltype(kind)::value>(a, ((float) x[k][j] - mean[j / SHARE]) * mul[j] + be[j]);
                if (k < mine) GnIo<T, VEC, YN4, YAL>::template store<XN4 && YN4>(a, n, pl + k * pls, cv, o);
            }
        });
    }

    // How the one-launch kernel cuts a norm; threads 0: two launches.
    struct GnSlab {
        int vectors, groups, threads, pixels; // SV, GV, and a thread's pixels
    };
    // Where a slab fits, it is taken from NC4HW4 always (its planes are contiguous; 8 x 108 x 75 x 75 to rows 12.2 us
    // against 18.2 with two launches, 16 x 128 x 80 x 80 15.1 against 21.3), and from NHWC by the two sides' times as
    // measured, in us: 4 and 1 + 3 / SV ns a vector and compute unit (a row's piece of SV vectors costs whole cache
    // lines), against 11.5 and three passes over the tensor at 5.5 TB/s. Measured slab / two launches:
    // 1 x 128 x 40 x 40 5.7 / 12.8, 8 x 512 x 28 x 28 6.9 / 14.6, 64 x 256 x 28 x 28 23.8 / 24.6,
    // 1 x 64 x 80 x 80 20.8 / 11.5, 64 x 256 x 56 x 56 112 / 62.
    static GnSlab gn_slab(const GnArgs &a, int vec, int size, bool planes) {
        if (a.Cg % vec && vec % a.Cg) return {0, 0, 0, 0};
        const int    sv      = a.Cg < vec ? 1 : a.Cg / vec;
        const double vectors = (double) a.HW * sv * (double) ceil_div((int64_t) a.N * ceil_div(a.CV, sv), 256);
        if (!planes && 4 + vectors * (1 + 3. / sv) * 1e-3 > 11.5 + 3. * size * a.N * a.C * (double) a.HW / 5.5e6) return {0, 0, 0, 0};
        for (int threads: {256, 1024}) {
            const int r = sv > threads ? 99 : (int) ceil_div(a.HW, threads / sv);
            if (r <= (threads == 256 ? 8 : 16)) return {sv, a.Cg < vec ? vec / a.Cg : 1, threads, r <= 8 ? 8 : 16};
        }
        return {0, 0, 0, 0};
    }

    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL, int GV>
    static int gn_slab_launch(const GnArgs &a, const GnSlab &c, hipStream_t s) {
        const int  slabs = (int) ceil_div(a.CV, c.vectors), spread = a.N >= 8 ? 8 : 1;
        const dim3 grid((unsigned) (spread * slabs), (unsigned) ceil_div(a.N, spread)); // a dimension of a launch has fewer than 2^32 threads
        if (c.threads == 256) gn_slab_kernel<T, VEC, XN4, YN4, XAL, YAL, 256, 8, GV><<<grid, 256, 0, s>>>(a, c.vectors, spread);
        else if (c.pixels == 8) gn_slab_kernel<T, VEC, XN4, YN4, XAL, YAL, 1024, 8, GV><<<grid, 1024, 0, s>>>(a, c.vectors, spread);
        else gn_slab_kernel<T, VEC, XN4, YN4, XAL, YAL, 1024, 16, GV><<<grid, 1024, 0, s>>>(a, c.vectors, spread);
        return check_launch("group_norm");
    }

    template <typename T, int VEC, bool XN4, bool YN4, bool XAL, bool YAL>
    static int gn_launch(const GnArgs &a, hipStream_t s) {
        const GnSlab c = gn_slab(a, VEC, (int) sizeof(T), XN4);
        if (c.threads) {
            if (c.groups == 1) return gn_slab_launch<T, VEC, XN4, YN4, XAL, YAL, 1>(a, c, s);
            if constexpr (VEC >= 4) {
                if (c.groups == 2) return gn_slab_launch<T, VEC, XN4, YN4, XAL, YAL, 2>(a, c, s);
                if (c.groups == 4) return gn_slab_launch<T, VEC, XN4, YN4, XAL, YAL, 4>(a, c, s);
            }
            if constexpr (VEC >= 8) return gn_slab_launch<T, VEC, XN4, YN4, XAL, YAL, 8>(a, c, s);
        }
        const dim3   grid((unsigned) a.chunks, (unsigned) a.N, XN4 ? (unsigned) ceil_div(a.CV, kGnThreads / 64) : 1u);
        const size_t lds = XN4 ? 0 : (size_t) (a.CV > kGnThreads ? a.CV : kGnThreads) * VEC; // entries
        gn_stats_kernel<T, VEC, XN4, XAL><<<grid, kGnThreads, lds * sizeof(float2), s>>>(a);
        int rc = check_launch("group_norm statistics");
        if (rc) return rc;
        gn_apply_kernel<T, VEC, XN4, YN4, XAL, YAL><<<grid, kGnThreads, 2 * a.G * sizeof(float), s>>>(a);
        return check_launch("group_norm");
    }

    // Pixels of a chunk: workgroups for every compute unit, and no more than 48 chunks, since each workgroup of the
    // second launch joins them all (1 x 64 x 80 x 80: 11.6 us, 15.0 with up to 128); then whole batches of the threads'
    // pixels where there are enough, rounded down, which makes up to 96 chunks. Rounded up there instead, rows lose (1 x
    // 64 x 150 x 150 12.2 -> 14.1 us, 1 x 512 x 60 x 60 15.1 -> 17.7) and NC4HW4 of wide groups gains (1 x 256 x 200 x 240,
    // four groups, 54 -> 35).
    static int gn_chunk(const vkhip_group_norm_desc *d) {
        const int64_t hw = (int64_t) d->H * d->W, vectors = ceil_div((int64_t) d->C * (d->dtype == VKHIP_DT_F32 ? 4 : 2), 16);
        const int64_t batch = kGnBatch * (d->x_fmt == 2 ? 64 : kGnThreads / (vectors < kGnThreads ? vectors : kGnThreads));
        int64_t       k = ceil_div(1024, d->N);
        if (k > 48) k = 48;
        const int64_t least = d->x_fmt == 2 ? batch : 32;
        if (k > ceil_div(hw, least)) k = ceil_div(hw, least);
        int64_t chunk = ceil_div(hw, k);
        if (chunk >= batch) chunk -= chunk % batch;
        else if (chunk * 2 > batch) chunk = batch;
        return (int) chunk;
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
    return (size_t) d->N * ceil_div((int64_t) d->H * d->W, gn_chunk(d)) * (d->x_fmt == 2 ? d->C : d->groups) * sizeof(float2);
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
    const float inf = __builtin_inff();
    a.kind = 0, a.s = 1.f, a.t = 0.f, a.lo = -inf, a.hi = inf, a.eps = d->eps;
    switch (d->act) {
        case VKHIP_ACT_RELU: a.lo = 0.f; break;
        case VKHIP_ACT_RELU6: a.lo = 0.f, a.hi = 6.f; break;
        case VKHIP_ACT_CLIP: a.lo = d->act_lo, a.hi = d->act_hi; break;
        case VKHIP_ACT_HARDSWISH: a.kind = 1, a.s = 1.f / 6.f, a.t = 0.5f, a.lo = 0.f, a.hi = 1.f; break;
        case VKHIP_ACT_SILU: a.kind = 2; break;
        case VKHIP_ACT_HARDSIGMOID: a.s = d->act_lo, a.t = d->act_hi, a.lo = 0.f, a.hi = 1.f; break;
        default: break;
    }
    a.chunk       = gn_chunk(d);
    a.chunks      = (int) ceil_div(a.HW, a.chunk);
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
