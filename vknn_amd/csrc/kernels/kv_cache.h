// The 8-bit cache as the kernels see it, shared by its rows in and out and the attention over it.
#pragma once
#include "tokens.h"

namespace vkhip {

    struct KvArgs {
        unsigned char *k, *v; // [page][head][token][row], [page][head][row][token]
        float         *k_scale, *v_scale;
        const int32_t *table;
        int            pages, page_tokens, page_shift, heads, head_dim, row, batch, max_blocks; // page_tokens = 1 << page_shift
    };

    const char *kv_refusal(const vkhip_kv_cache *c);
    const char *kv_bad_pointers(const vkhip_kv_cache *c);
    KvArgs      kv_args(const vkhip_kv_cache *c);

} // namespace vkhip
