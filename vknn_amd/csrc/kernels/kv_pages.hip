// Pages of the cache for a step's rows, from lengths on the device, and back: what a host program would otherwise have
// to know every length for, between two steps.
//
// Nothing to read or write that counts: a launch, the lengths, two sums over the sequences (rows; blocks that begin) and
// stores. One workgroup takes the sequences 1024 at a time with both sums; a step's few rows it writes itself, rows of
// prompts take a second launch of a workgroup a sequence. Measured: 256 sequences of a token each 4.6 us, their pages back
// 3.8; 64 prompts of up to 8000 tokens 5.7 and 5.2 us, back 6.9.
#include "kv_cache.h"

namespace vkhip {

    struct KvPageArgs {
        int32_t       *table, *free, *state;
        const int32_t *lens, *add; // add: new tokens (reserve), tokens that stay (release)
        int32_t       *cu, *now, *pos;
        int64_t       *slot;
        int            pages, page_tokens, page_shift, batch, max_blocks, capacity, total;
        bool           few; // rows are written along with the table
    };

    constexpr int kSeqs = 1024; // sequences at a time, one a thread

    __device__ __forceinline__ int blocks_of(const KvPageArgs &a, int tokens) {
        return min(a.max_blocks, (int) (((int64_t) tokens + a.page_tokens - 1) >> a.page_shift));
    }

    // Sums over the workgroup's threads up to each, and all of them; `waves` holds a number a wave.
    __device__ __forceinline__ int block_prefix_sum(int x, int *waves, int &all) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = wave_prefix_sum(x);
        __syncthreads(); // the last sums have been read
        if (lane == 63) waves[wave] = mine;
        __syncthreads();
        const int of = lane < kSeqs / 64 ? waves[lane] : 0, incl = wave_prefix_sum(of);
        all          = __builtin_amdgcn_readlane(incl, 63);
        return mine + __builtin_amdgcn_readlane(incl - of, __builtin_amdgcn_readfirstlane(wave));
    }

    // The last i below n with from[i] <= item, where from[0] <= item.
    __device__ __forceinline__ int last_at(const int *from, int n, int item) {
        int lo = 0;
#pragma unroll
        for (int step = kSeqs / 2; step; step >>= 1)
            if (lo + step < n && from[lo + step] <= item) lo += step;
        return lo;
    }

    __device__ __forceinline__ void row_out(const KvPageArgs &a, int b, int row, int at) {
        if (a.pos) a.pos[row] = at;
        if (a.slot) {
            const int block = at >> a.page_shift, id = block < a.max_blocks ? a.table[(int64_t) b * a.max_blocks + block] : -1;
            a.slot[row]     = id >= 0 && id < a.pages ? ((int64_t) id << a.page_shift) + (at & (a.page_tokens - 1)) : -1;
        }
    }

    __global__ __launch_bounds__(kSeqs) void kv_reserve_kernel(KvPageArgs a) {
        __shared__ int waves[kSeqs / 64], row_from[kSeqs], block_from[kSeqs], first_block[kSeqs], held[kSeqs];
        const int tid = threadIdx.x, most = a.max_blocks << a.page_shift;
        if (tid == 0) a.cu[0] = 0;
        if (a.batch == 0) return; // there may be no list either
        const int left = clampi(a.state[0], 0, a.capacity);
        int       rows = 0, taken = 0; // of the sequences before
        for (int b0 = 0; b0 < a.batch; b0 += kSeqs) {
            const int b = b0 + tid, n = min(kSeqs, a.batch - b0);
            // what does not fit the remaining rows is cut, here by halves, so that the sum stays within 32 bits
            const int len = b < a.batch ? clampi(a.lens[b], 0, most) : 0, want = b < a.batch ? clampi(a.add[b], 0, a.total - rows) : 0;
            int       sum, end;
            {
                int       low, high;
                const int lo = block_prefix_sum(want & 0xFFFF, waves, low), hi = block_prefix_sum(want >> 16, waves, high);
                const int64_t upto = (int64_t) hi * 65536 + lo, every = (int64_t) high * 65536 + low;
                end = (int) min(upto, (int64_t) (a.total - rows));
                sum = (int) min(every, (int64_t) (a.total - rows));
                const int begin = (int) min(upto - want, (int64_t) (a.total - rows));
                row_from[tid]   = rows + begin;
                held[tid]       = len;
                end -= begin; // rows of this sequence
            }
            const int made = end, first = blocks_of(a, len), begun = max(0, blocks_of(a, len + made) - first);
            int       blocks;
            const int upto = block_prefix_sum(begun, waves, blocks);
            block_from[tid]  = upto - begun;
            first_block[tid] = first;
            if (b < a.batch) {
                a.cu[b + 1] = row_from[tid] + made;
                if (a.now) a.now[b] = len + made;
            }
            __syncthreads();
            for (int i = tid; i < blocks; i += kSeqs) {
                const int k = last_at(block_from, n, i), at = left - 1 - taken - i;
                a.table[(int64_t) (b0 + k) * a.max_blocks + first_block[k] + (i - block_from[k])] = at >= 0 ? a.free[at] : -1;
            }
            if (a.few) {
                __syncthreads(); // the table's entries are there
                for (int i = tid; i < sum; i += kSeqs) {
                    const int k = last_at(row_from, n, rows + i);
                    row_out(a, b0 + k, rows + i, held[k] + (rows + i - row_from[k]));
                }
            }
            rows += sum, taken += blocks;
            __syncthreads(); // the lists have been read
        }
        if (tid == 0) {
            a.state[0] = max(0, left - taken);
            if (taken > left) a.state[1] += taken - left;
        }
    }

    __global__ __launch_bounds__(256) void kv_rows_kernel(KvPageArgs a) {
        const int b = blockIdx.x, from = a.cu[b], end = a.cu[b + 1], len = clampi(a.lens[b], 0, a.max_blocks << a.page_shift);
        for (int row = from + blockIdx.y * 256 + threadIdx.x; row < end; row += gridDim.y * 256) row_out(a, b, row, len + (row - from));
    }

    // Sequences and their blocks from the last to the first, so that the first block given back lies on top.
    __global__ __launch_bounds__(kSeqs) void kv_release_kernel(KvPageArgs a) {
        __shared__ int waves[kSeqs / 64], block_from[kSeqs], first_block[kSeqs];
        const int tid = threadIdx.x, most = a.max_blocks << a.page_shift;
        int       count = clampi(a.state[0], 0, a.capacity);
        for (int b0 = (a.batch - 1) / kSeqs * kSeqs; b0 >= 0; b0 -= kSeqs) {
            const int b = b0 + tid, n = min(kSeqs, a.batch - b0);
            const int first = b < a.batch ? blocks_of(a, clampi(a.add[b], 0, most)) : 0, last = b < a.batch ? blocks_of(a, clampi(a.lens[b], 0, most)) : 0;
            const int mine = max(0, last - first);
            int       blocks;
            const int upto = block_prefix_sum(mine, waves, blocks);
            block_from[tid] = upto - mine, first_block[tid] = first;
            __syncthreads();
            for (int i0 = 0; i0 < blocks; i0 += kSeqs) {
                const int item = blocks - 1 - i0 - tid;
                int       id = -1, given;
                if (item >= 0) {
                    const int k = last_at(block_from, n, item);
                    int32_t  *e = a.table + (int64_t) (b0 + k) * a.max_blocks + first_block[k] + (item - block_from[k]);
                    id          = *e;
                    *e          = -1;
                }
                const bool is = id >= 0 && id < a.pages;
                const int  rank = block_prefix_sum(is, waves, given) - 1;
                if (is && count + rank < a.capacity) a.free[count + rank] = id;
                count = min(a.capacity, count + given);
            }
            __syncthreads(); // the lists have been read
        }
        if (tid == 0) a.state[0] = count;
    }

    static const char *kv_pages_refusal(const vkhip_kv_cache *c, const vkhip_kv_pool *p, const int32_t *lens, const int32_t *add) {
        if (const char *why = kv_refusal(c)) return why;
        if (!p || p->capacity < 0) return "bad pool";
        if ((int64_t) c->batch * c->max_blocks > 0x7FFFFFFF) return "over 2^31 blocks";
        if (c->batch == 0) return nullptr;
        if ((!c->table && c->max_blocks) || !p->state || (p->capacity && !p->free) || !lens || !add) return "null pointer";
        if (((uintptr_t) c->table | (uintptr_t) p->state | (uintptr_t) p->free | (uintptr_t) lens | (uintptr_t) add) % 4) return "misaligned pointer";
        return nullptr;
    }
    static KvPageArgs kv_page_args(const vkhip_kv_cache *c, const vkhip_kv_pool *p, const int32_t *lens, const int32_t *add) {
        KvPageArgs a {};
        a.table = const_cast<int32_t *>(c->table), a.free = p->free, a.state = p->state, a.lens = lens, a.add = add;
        a.pages = c->pages, a.page_tokens = c->page_tokens, a.page_shift = __builtin_ctz((unsigned) c->page_tokens), a.batch = c->batch, a.max_blocks = c->max_blocks;
        a.capacity = p->capacity;
        return a;
    }

} // namespace vkhip

using namespace vkhip;

extern "C" {

int vkhip_kv_reserve(const vkhip_kv_cache *c, const vkhip_kv_pool *p, const int32_t *lens, const int32_t *add, int32_t total, int32_t *cu, int32_t *now,
                     int32_t *pos, int64_t *slot, vkhip_stream_t s) {
    if (const char *why = kv_pages_refusal(c, p, lens, add)) return set_error(VKHIP_ERR_INVALID, "kv_reserve: %s", why);
    if (total < 0 || total >= 1 << 30) return set_error(VKHIP_ERR_INVALID, "kv_reserve: total is not 0 .. 2^30 - 1");
    if (c->batch == 0 && !cu) return VKHIP_OK;
    if (!cu) return set_error(VKHIP_ERR_INVALID, "kv_reserve: null pointer");
    if (((uintptr_t) cu | (uintptr_t) now | (uintptr_t) pos) % 4 || (uintptr_t) slot % 8) return set_error(VKHIP_ERR_INVALID, "kv_reserve: misaligned pointer");
    if (c->batch > 0 && (now == lens || now == add || cu == lens || cu == add)) return set_error(VKHIP_ERR_INVALID, "kv_reserve: an output is an input");
    KvPageArgs a = kv_page_args(c, p, lens, add);
    a.cu = cu, a.now = now, a.pos = pos, a.slot = slot, a.total = total;
    const bool rows = (pos || slot) && total > 0 && c->batch > 0;
    a.few           = rows && total <= 8 * kSeqs;
    kv_reserve_kernel<<<1, kSeqs, 0, resolve_stream(s)>>>(a);
    int rc = check_launch("kv_reserve");
    if (rc || !rows || a.few) return rc;
    const int64_t parts = ceil_div(ceil_div(total, c->batch), 1024);
    kv_rows_kernel<<<dim3((unsigned) c->batch, (unsigned) (parts < 64 ? parts : 64)), 256, 0, resolve_stream(s)>>>(a);
    return check_launch("kv_reserve rows");
}

int vkhip_kv_release(const vkhip_kv_cache *c, const vkhip_kv_pool *p, const int32_t *lens, const int32_t *keep, vkhip_stream_t s) {
    if (const char *why = kv_pages_refusal(c, p, lens, keep)) return set_error(VKHIP_ERR_INVALID, "kv_release: %s", why);
    if (c->batch == 0 || c->max_blocks == 0) return VKHIP_OK;
    kv_release_kernel<<<1, kSeqs, 0, resolve_stream(s)>>>(kv_page_args(c, p, lens, keep));
    return check_launch("kv_release");
}

} // extern "C"
