// Attention over paged caches in 4 or 8 bits (see quantized_attention.cu).
#pragma once
#include "quantized_kv.h"

namespace mk {

struct QuantAttnArgs {
    QuantPools pools;
    QuantLanes lanes;             // lanes.rows: the most rows that a lane has
    const void* q = nullptr;      // [total] rows of q_heads * d values, row stride ldq
    void* out = nullptr;          // the same, row stride ldo
    int64_t ldq = 0, ldo = 0;
    int q_heads = 0;
    float scale = 1.f, softcap = 0.f;
    int window = 0;
};

// How the lanes' keys are shared out on the device (see quantized_attention.cu).
struct QuantAttnCut {
    bool split = false;     // otherwise every lane has one share
    int least = 0;          // keys of a share, at least
    float want = 1.f;       // shares in all
    int window_keys = 0;    // keys of a lane that a window leaves, at most
};
// How a call is cut, from sizes alone.
struct QuantAttnPlan {
    int items = 0, blocks = 0;   // (row, query head) items of a lane and KV head to a CTA, and such blocks
    int slots = 0;               // shares of all lanes, at most
    QuantAttnCut cut;
    int64_t bytes = 0;           // workspace: a partial result of each slot's rows
};
QuantAttnPlan quantized_attention_plan(int q_heads, int kv_heads, int d, int bits, int block_tokens, int width, int lanes, int rows, int total, int window);
void launch_quantized_attention(const QuantAttnArgs& a, const QuantAttnPlan& p, void* workspace, cudaStream_t s);

}  // namespace mk
