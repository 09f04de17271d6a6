// Copies inside paged K/V pools (see kv_rows.cu).
#pragma once
#include "common.cuh"

namespace mk {

// Pools [layers][pages][kv_heads][block_tokens][row_bytes], K and V alike.
struct KvRowsArgs {
    void *k_pool = nullptr, *v_pool = nullptr;
    int64_t layers = 0, pages = 0;
    int kv_heads = 0, block_tokens = 0, row_bytes = 0;
    // copies: [n][3] of (from page, to page, rows)
    const int32_t* copies = nullptr;
    int n = 0;
    // gathering: token keep[lane][j] of the pages in `from` becomes token first[lane] + j of the pages in `to`, j < counts[lane]
    const int32_t *from = nullptr, *to = nullptr, *keep = nullptr, *counts = nullptr, *first = nullptr;
    int64_t ld_from = 0, ld_to = 0, ld_keep = 0;
    int lanes = 0, from_width = 0, to_width = 0, keep_width = 0;
    int32_t* status = nullptr;
};
void launch_copy_pages(const KvRowsArgs& a, cudaStream_t s);
void launch_gather_tokens(const KvRowsArgs& a, cudaStream_t s);

}  // namespace mk
