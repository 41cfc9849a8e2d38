// Rotary positions with several axes: pairs of channels of query and key rows turned by the row's positions.
//
// Angles are kept as fractions of a turn in 64 bits: a pair's frequency is f 2^64 / 2 pi rounded to a whole number, the
// angle its product with the position modulo 2^64, which is the fraction of the turn but for position * 2^-65: whole
// turns fall off by themselves, and no 64-bit floats are needed. The nearest quarter turn is taken off as a whole number; the
// rest, within an eighth of a turn, becomes a float from both halves of its 64 bits, so that small angles keep their digits
// (the upper half alone has 2^-32 of a turn: sines of the slowest pairs at theta 10^6 were off by 3e-4 of themselves), and
// goes into Taylor's series, the sine's up to x^11 (next term 2^-37), the cosine's up to x^10 (next 2^-33). One pair's sine
// and cosine serve all heads that a thread takes.
//
// Bound by memory where rows are many: 50176 rows of 40 heads of 128 bf16 181 us, 5.7 TB/s in and out, fp32 422 us, 4.9 TB/s;
// 45000 rows of 32 heads of 64 fp16, neighbours, 65 us, 5.7 TB/s (partly from the caches), fp32, halves, 163 us, 4.5 TB/s. 64 rows
// 8.2 us, a launch and two loads in a row.
#include "tokens.h"
#include <algorithm>
#include <math.h>

namespace vkhip {

    constexpr int     kRotaryPairs = 128, kRotaryHeads = 4; // of a head; of a thread
    constexpr int64_t kRotaryPast = (int64_t) 64 << 20; // bytes of rows from which they pass the caches

    struct RotaryArgs {
        const void    *q, *k;
        void          *qo, *ko;
        const int32_t *pos;
        int            rows, q_heads, heads, head_dim, pairs; // heads: of q and k together
        int            units, turned;   // pieces of a head; the first `turned` are pairs, the others copied
        int            slots, per;      // threads that share a row's unit, heads of each
        int            block_rows;      // rows of a workgroup, where several fit
        bool           in_place;
        int64_t        pos_axis, q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
        uint64_t       freq[kRotaryPairs]; // turns * 2^64 per position
        uint8_t        axis[kRotaryPairs];
    };

    __device__ __forceinline__ void turn_of(uint64_t freq, int pos, float &c, float &s) {
        const uint64_t turn = freq * (uint64_t) (int64_t) pos;
        const int      low = (int) (unsigned) turn; // as a number of its own, so that it takes nothing from a small high half
        const unsigned high = (unsigned) (turn >> 32) + ((unsigned) low >> 31), quarter = (high + 0x20000000u) >> 30;
        const float    x = __builtin_fmaf((float) low, 0x1.921fb6p+2f * 0x1p-64f, (float) (int) (high - (quarter << 30)) * (0x1.921fb6p+2f * 0x1p-32f)), z = x * x;
        float          sx = __builtin_fmaf(z, -1.f / 39916800, 1.f / 362880), cx = __builtin_fmaf(z, -1.f / 3628800, 1.f / 40320);
        sx = __builtin_fmaf(sx, z, -1.f / 5040);
        cx = __builtin_fmaf(cx, z, -1.f / 720);
        sx = __builtin_fmaf(sx, z, 1.f / 120);
        cx = __builtin_fmaf(cx, z, 1.f / 24);
        sx = __builtin_fmaf(sx, z, -1.f / 6);
        cx = __builtin_fmaf(cx, z, -.5f);
        sx = __builtin_fmaf(sx * z, x, x);
        cx = __builtin_fmaf(cx, z, 1.f);
        c  = quarter & 1 ? sx : cx;
        s  = quarter & 1 ? cx : sx;
        if ((quarter + 1) & 2) c = -c;
        if (quarter & 2) s = -s;
    }

    // Rows in the caches, past them in stores, or past them altogether.
    enum { kCached, kStoresPast, kPast };

    // A thread takes one unit of a row in several heads. A unit of halves is VEC pairs, two vectors of VEC channels that lie
    // half of the rotated channels apart; of neighbours VEC channels, or a pair; behind the rotated channels as many that
    // are copied. RAGGED: the last vectors begin that much earlier that they end with their channels; the channels of the
    // vector before are stored twice, or once where their owner turns them, or in place, where it may be a wave that has yet to
    // read them.
    template <typename T, int VEC, bool NEAR, bool RAGGED, int PAST>
    __global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
        typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T)))); // of any alignment: one instruction
        constexpr int  PAIRS = NEAR ? (VEC > 1 ? VEC / 2 : 1) : VEC;
        constexpr bool TWO   = !NEAR || VEC == 1; // vectors of a unit
        const int      each  = a.units * a.slots;
        const int64_t  block = (int64_t) blockIdx.y * gridDim.x + blockIdx.x;
        const int      r = (int) threadIdx.x / each;
        const int64_t  row = block * a.block_rows + r;
        if (r >= a.block_rows || row >= a.rows) return;
        const auto load = [](const T *p) {
            if constexpr (PAST == kPast) return __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
            else return *reinterpret_cast<const V *>(p);
        };
        const auto store = [&](V v, T *p, int skip, bool once) {
            if (RAGGED && skip > 0 && once) {
#pragma unroll
                for (int j = 1; j < VEC; ++j)
                    if (j >= skip) p[j] = v[j];
            } else if constexpr (PAST != kCached) __builtin_nontemporal_store(v, reinterpret_cast<V *>(p));
            else *reinterpret_cast<V *>(p) = v;
        };
        for (int i = (int) threadIdx.x - r * each; i < each; i += 256) {
            const int  unit = i % a.units, h0 = i / a.units * a.per, h1 = min(a.heads, h0 + a.per);
            const bool turned = unit < a.turned;
            // the first channel of each vector, and how many of its channels are another's
            int        c0, c1, s0 = 0, s1 = 0, p0 = unit * PAIRS;
            if (turned) {
                if constexpr (RAGGED) {
                    s0 = max(0, p0 + PAIRS - a.pairs);
                    p0 -= s0;
                    s1 = s0 = NEAR ? 2 * s0 : s0;
                }
                c0 = NEAR ? 2 * p0 : p0, c1 = NEAR ? c0 + VEC : a.pairs + p0;
            } else {
                c0 = 2 * a.pairs + (unit - a.turned) * 2 * PAIRS, c1 = c0 + VEC;
                if constexpr (RAGGED) {
                    s0 = max(0, c0 + VEC - a.head_dim), s1 = max(0, c1 + VEC - a.head_dim);
                    c0 -= s0, c1 -= s1;
                }
            }
            const bool second = TWO && s1 < VEC && c1 < a.head_dim;
            const auto place = [&](const void *q, const void *k, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int h) {
                return h < a.q_heads ? (T *) q + (row * q_row + h * q_head) : (T *) k + (row * k_row + (h - a.q_heads) * k_head);
            };
            // All heads are on their way while the angles are, but for whole heads of neighbours past the caches, which go one by one (50176
            // rows of 40 heads of 128, bf16, at once and one by one: halves 182, 192 us, neighbours 205, 185; 45000 x 32 of 40 channels,
            // fp16, 59, 81).
            constexpr bool ALL = !NEAR || PAST != kPast;
            V              u[kRotaryHeads], w[kRotaryHeads];
            const auto     head = [&](int n) {
                const T *x = place(a.q, a.k, a.q_row, a.q_head, a.k_row, a.k_head, h0 + n);
                u[n] = load(x + c0);
                if (second) w[n] = load(x + c1);
            };
            if constexpr (ALL)
#pragma unroll
                for (int n = 0; n < kRotaryHeads; ++n)
                    if (h0 + n < h1) head(n);
            float c[PAIRS], s[PAIRS];
            if (turned)
#pragma unroll
                for (int j = 0; j < PAIRS; ++j) {
                    const int p = p0 + j;
                    turn_of(a.freq[p], a.pos[a.axis[p] * a.pos_axis + row], c[j], s[j]);
                }
#pragma unroll
            for (int n = 0; n < kRotaryHeads; ++n)
                if (h0 + n < h1) {
                    if constexpr (!ALL) head(n);
                    V &v = u[n], &z = w[n];
                    if (turned)
#pragma unroll
                        for (int j = 0; j < PAIRS; ++j) {
                            const float p = (float) (TWO ? v[j] : v[2 * j]), q = (float) (TWO ? z[j] : v[2 * j + (VEC > 1)]);
                            const T     p1 = (T) __builtin_fmaf(p, c[j], -(q * s[j])), q1 = (T) __builtin_fmaf(q, c[j], p * s[j]); // the same in each of two threads
                            if constexpr (TWO) v[j] = p1, z[j] = q1;
                            else v[2 * j] = p1, v[2 * j + (VEC > 1)] = q1;
                        }
                    T *y = place(a.qo, a.ko, a.qo_row, a.qo_head, a.ko_row, a.ko_head, h0 + n);
                    store(v, y + c0, s0, a.in_place || (!turned && c0 < 2 * a.pairs));
                    if (second) store(z, y + c1, s1, a.in_place || (!turned && c1 < 2 * a.pairs));
                }
        }
    }

    // Of each pair its axis and its fraction of a turn per position, times 2^64.
    static void rotary_pairs(const vkhip_rotary_desc *d, const double *freq, RotaryArgs &a) {
        // 2 pi and what it lacks: whole turns come off a frequency without its fraction losing digits
        const long double two64 = 18446744073709551616.0L, turn = 6.28318530717958647692528676655900577L, rest = -1.0033115225336664538847901e-19L;
        int               had[4] = {0, 0, 0, 0}, axis = 0;
        long double       step[4], now[4]; // the next pair's angle per position, by axis; all pairs' in [0]
        for (int i = 0; i < 4; ++i) {
            const int n = d->spectra ? (i < d->axes ? d->sections[i] : 0) : a.pairs;
            step[i] = n > 0 && !freq ? powl((long double) d->theta, -1.0L / n) : 1.0L, now[i] = 1.0L;
        }
        for (int p = 0; p < a.pairs; ++p) {
            while (had[axis] == d->sections[axis]) axis = (axis + 1) % d->axes;
            const int   of = d->spectra ? axis : 0;
            const long double f = freq ? (long double) freq[p] : now[of];
            now[of] *= step[of];
            long double t = f * (1.0L / turn);
            if (f < 0 || f >= turn) {
                const long double n = floorl(f / turn);
                t = (fmal(-n, turn, f) - n * rest) / turn;
                t -= floorl(t); // rounding may leave it outside 0 .. 1
            }
            const long double whole = t * two64 + 0.5L;
            a.freq[p] = whole >= two64 ? 0 : (uint64_t) whole;
            a.axis[p] = (uint8_t) axis;
            ++had[axis];
            if (d->interleaved) axis = (axis + 1) % d->axes;
        }
    }

    // Frequencies that rotary_pairs takes: of 10^6 and more the whole turns would leave its digits too few of the rest.
    constexpr double kRotaryFreq = 1e6;

    // The largest frequency that theta gives: with a theta under 1 the last pair's of its axis.
    static double rotary_largest(const vkhip_rotary_desc *d) {
        int n = d->rotary_dim / 2;
        if (d->spectra) n = *std::max_element(d->sections, d->sections + d->axes);
        return d->theta >= 1.0 ? 1.0 : pow(d->theta, -(n - 1.0) / n);
    }

    static bool rotary_strides(int64_t row, int64_t head) { return row >= 0 && head >= 0 && row <= (int64_t) 1 << 31 && head <= (int64_t) 1 << 40; }

    // Whether an output's heads lie apart within its rows, or its rows within its heads.
    static bool rotary_apart(const vkhip_rotary_desc *d, int heads, int64_t row, int64_t head) {
        const int64_t dim = d->head_dim, in_row = (heads - 1) * head + dim, in_head = (d->rows - 1) * row + dim;
        const bool    one_row = d->rows <= 1, one_head = heads <= 1;
        return ((one_head || head >= dim) && (one_row || row >= in_row)) || ((one_row || row >= dim) && (one_head || head >= in_head));
    }

    static const char *rotary_refusal(const vkhip_rotary_desc *d) {
        if (!d || d->rows < 0 || d->q_heads <= 0 || d->k_heads < 0) return "bad sizes";
        if (d->q_heads > 65535 || d->k_heads > 65535) return "over 65535 heads";
        if (d->head_dim < 2 || d->head_dim > 256) return "head_dim is not 2 .. 256";
        if (d->rotary_dim < 2 || d->rotary_dim % 2 || d->rotary_dim > d->head_dim) return "rotary_dim is not even or not 2 .. head_dim";
        if (d->dtype < VKHIP_DT_F16 || d->dtype > VKHIP_DT_F32) return "dtype is not F16, BF16 or F32";
        if (d->axes < 1 || d->axes > 4) return "axes is not 1 .. 4";
        int64_t pairs = 0;
        for (int i = 0; i < d->axes; ++i) {
            if (d->sections[i] < 0) return "a section is negative";
            pairs += d->sections[i];
        }
        if (pairs != d->rotary_dim / 2) return "sections do not sum to rotary_dim / 2";
        if (d->axes > 1 && d->pos_axis < 0) return "pos_axis is negative";
        if (!rotary_strides(d->q_row, d->q_head) || !rotary_strides(d->qo_row, d->qo_head)) return "a stride of q or qo is negative or too large";
        if (!rotary_apart(d, d->q_heads, d->qo_row, d->qo_head)) return "rows of qo share memory";
        if (d->k_heads == 0) return nullptr;
        if (!rotary_strides(d->k_row, d->k_head) || !rotary_strides(d->ko_row, d->ko_head)) return "a stride of k or ko is negative or too large";
        if (!rotary_apart(d, d->k_heads, d->ko_row, d->ko_head)) return "rows of ko share memory";
        return nullptr;
    }

    template <typename T, int VEC, bool RAGGED>
    static void rotary_launch(const vkhip_rotary_desc *d, RotaryArgs &a, hipStream_t s) {
        const int pairs = d->neighbours ? (VEC > 1 ? VEC / 2 : 1) : VEC; // of a unit
        a.turned = (int) ceil_div(a.pairs, pairs);
        a.units  = a.turned + (int) ceil_div(d->head_dim - d->rotary_dim, 2 * pairs);
        // Heads of a thread: as many as leave the card full, at most 4 (50176 rows of 40 heads of 128, bf16, 2, 4, 8, 10 of them: 201,
        // 193, 197, 206 us; neighbours 210, 187, 181, 186).
        const int64_t items = (int64_t) a.rows * a.heads * a.units, fill = 256 * 2048;
        a.per   = (int) (items / fill < 1 ? 1 : items / fill > kRotaryHeads ? kRotaryHeads : items / fill);
        a.slots = (int) ceil_div(a.heads, a.per);
        const int each = a.units * a.slots;
        a.block_rows   = each >= 256 ? 1 : 256 / each;
        const int64_t blocks = ceil_div(a.rows, a.block_rows), layers = ceil_div(blocks, 0xFFFFFF);
        const dim3    grid((unsigned) ceil_div(blocks, layers), (unsigned) layers);
        // Past the caches go only heads of whole lines, and in loads only whole lines at a time. 45000 rows of 32 heads, fp16, halves, us with
        // both past, stores past, all cached: heads of 64 100, 66, 86; of 40 180, 127, 83; ragged (52 of 64) 183, 135, 93.
        const int elem = (int) sizeof(T);
        if constexpr (!RAGGED)
            if ((int64_t) a.rows * a.heads * d->head_dim * elem >= kRotaryPast && d->head_dim * elem % 128 == 0) {
                if (d->neighbours) rotary_kernel<T, VEC, true, false, kPast><<<grid, 256, 0, s>>>(a);
                else if (a.pairs * elem % 128 == 0) rotary_kernel<T, VEC, false, false, kPast><<<grid, 256, 0, s>>>(a);
                else rotary_kernel<T, VEC, false, false, kStoresPast><<<grid, 256, 0, s>>>(a);
                return;
            }
        if (d->neighbours) rotary_kernel<T, VEC, true, RAGGED, kCached><<<grid, 256, 0, s>>>(a);
        else rotary_kernel<T, VEC, false, RAGGED, kCached><<<grid, 256, 0, s>>>(a);
    }
    // Vectors of 8 channels, or of 4 where these come out even or there is no full one of 8; single ones below that. 45000 rows of 32 heads
    // of 64, fp16, halves, us: 56 turned 60 in even vectors of 4, 92 in ragged ones of 8; 52 turned 183 (single), 107 (4), 93 (8).
    template <typename T>
    static void rotary_vectors(const vkhip_rotary_desc *d, RotaryArgs &a, hipStream_t s) {
        const int turned = d->neighbours ? d->rotary_dim : a.pairs, both = turned | (d->head_dim - d->rotary_dim);
        if (turned >= 8 && both % 8 == 0) rotary_launch<T, 8, false>(d, a, s);
        else if (both % 4 == 0) rotary_launch<T, 4, false>(d, a, s);
        else if (turned >= 8) rotary_launch<T, 8, true>(d, a, s);
        else if (turned >= 4) rotary_launch<T, 4, true>(d, a, s);
        else rotary_launch<T, 1, false>(d, a, s);
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

int vkhip_rotary(const vkhip_rotary_desc *d, const int32_t *pos, const double *freq, const void *q, const void *k, void *qo, void *ko, vkhip_stream_t s) {
    if (const char *why = rotary_refusal(d)) return set_error(VKHIP_ERR_INVALID, "rotary: %s", why);
    RotaryArgs a {};
    a.pairs = d->rotary_dim / 2;
    if (!freq && !(d->theta > 0.0 && d->theta < 1e30)) return set_error(VKHIP_ERR_INVALID, "rotary: theta is not positive");
    if (!freq && !(rotary_largest(d) < kRotaryFreq)) return set_error(VKHIP_ERR_INVALID, "rotary: theta gives a frequency of 10^6 or more");
    if (freq)
        for (int i = 0; i < a.pairs; ++i)
            if (!(fabs(freq[i]) < kRotaryFreq)) return set_error(VKHIP_ERR_INVALID, "rotary: a frequency is not finite or 10^6 or more");
    if (d->rows == 0) return VKHIP_OK;
    const bool with_k = d->k_heads > 0;
    if (!pos || !q || !qo || (with_k && (!k || !ko))) return set_error(VKHIP_ERR_INVALID, "rotary: null pointer");
    const uintptr_t elem = d->dtype == VKHIP_DT_F32 ? 4 : 2, places = (uintptr_t) q | (uintptr_t) qo | (with_k ? (uintptr_t) k | (uintptr_t) ko : 0);
    if ((uintptr_t) pos % 4 || places % elem) return set_error(VKHIP_ERR_INVALID, "rotary: misaligned pointer");
    if ((q == qo && (d->q_row != d->qo_row || d->q_head != d->qo_head)) || (with_k && k == ko && (d->k_row != d->ko_row || d->k_head != d->ko_head)))
        return set_error(VKHIP_ERR_INVALID, "rotary: in place with other strides");
    a.q = q, a.k = k, a.qo = qo, a.ko = ko, a.pos = pos;
    a.rows = d->rows, a.q_heads = d->q_heads, a.heads = d->q_heads + d->k_heads, a.head_dim = d->head_dim, a.pos_axis = d->pos_axis;
    a.q_row = d->q_row, a.q_head = d->q_head, a.qo_row = d->qo_row, a.qo_head = d->qo_head;
    a.k_row = d->k_row, a.k_head = d->k_head, a.ko_row = d->ko_row, a.ko_head = d->ko_head;
    rotary_pairs(d, freq, a);
    a.in_place = q == qo || (with_k && k == ko);
    hipStream_t st = resolve_stream(s);
    if (d->dtype == VKHIP_DT_F16) rotary_vectors<half_t>(d, a, st);
    else if (d->dtype == VKHIP_DT_BF16) rotary_vectors<bf16_t>(d, a, st);
    else rotary_vectors<float>(d, a, st);
    return check_launch("rotary");
}

} // extern "C"
