// Attention of a batch whose lanes share their first pages (see shared_attention.cu).
#pragma once
#include "common.cuh"

namespace mk {

// Bits of the status word of the operators over device buffers (MK_DEV_* of the C header).
constexpr int kDevBadPage = 1;    // a page number outside the pool
constexpr int kDevWait = 2;       // a bounded wait gave up
constexpr int kDevBadRange = 4;   // a length, count or position outside its table

struct SharedAttnArgs {
    const void* q = nullptr;      // [total] rows of q_heads * d values, row stride ldq (values)
    void* out = nullptr;          // the same, row stride ldo
    int64_t ldq = 0, ldo = 0;
    const void* k_pool = nullptr; // pages [kv_heads][block_tokens][d], page_rows rows of d values apart
    const void* v_pool = nullptr;
    int64_t pool_pages = 0, page_rows = 0;
    int q_heads = 0, kv_heads = 0, d = 0, block_tokens = 0, bt_shift = 0;
    bool bf16 = false;
    const int32_t* tables = nullptr;   // [lanes][ld_table], the first `width` entries of a row count
    int64_t ld_table = 0;
    int width = 0;
    const int32_t* lengths = nullptr;  // [lanes]
    const int32_t* cu = nullptr;       // [lanes + 1] or null: lane i has rows i * rows ..
    int lanes = 0, rows = 0, total = 0;
    int shared = 0;                    // keys that all lanes have in the pages of lane 0's table
    float scale = 1.f, softcap = 0.f;
    int window = 0;
    // [parts][total][q_heads][d] unnormalised outputs and [parts][total][q_heads] (maximum as a base-2 logarithm, sum): the shared keys' parts, then the lanes'
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    int32_t* status = nullptr;         // may be null
};

// How a call is cut, from sizes alone.
struct SharedAttnPlan {
    bool alone = false;      // each lane reads the shared keys as its own
    int item_tiles = 0;      // blocks of (row, head) items of a lane and KV head
    int items = 0;           // items of such a block, a multiple of 8
    int chunk = 0, shares = 0;   // keys of a lane's share, and shares
    int item_rows = 0, row_tiles = 0, shared_parts = 0;   // shared keys: tiles of items to a CTA, CTAs along the items, shares of the keys
    bool joined = false;     // by a kernel of its own
    int64_t parts = 0;       // partial results of a row; 0: none are written
    int64_t bytes(int total, int q_heads, int d) const { return parts * total * q_heads * ((int64_t)d * 4 + 8); }
};
SharedAttnPlan shared_attention_plan(int q_heads, int kv_heads, int d, int block_tokens, int width, int lanes, int rows, int total, int shared, int window);

void launch_shared_attention(SharedAttnArgs a, const SharedAttnPlan& p, cudaStream_t s);

}  // namespace mk
