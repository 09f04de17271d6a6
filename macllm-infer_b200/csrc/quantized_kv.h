// Paged caches of keys and values in 4 or 8 bits (see quantized_kv.cu).
#pragma once
#include "common.cuh"
#include "shared_attention.h"   // bits of the status word
#include <cuda_bf16.h>

namespace mk {

constexpr int kQuantGroup = 64;   // neighbouring values of a head's row that share a step and a lowest value

// One layer's pools.  Pages of codes [kv_heads][block_tokens][d * bits / 8] bytes, value i of a row in bits (i * bits) % 8 .. of byte i * bits / 8; pages of scales
// [kv_heads][block_tokens][d / 64] pairs (step, lowest value) of the rows' type.  Code c stands for lowest + step * c.
struct QuantPools {
    uint8_t *k_codes = nullptr, *v_codes = nullptr;
    uint32_t *k_scales = nullptr, *v_scales = nullptr;   // pairs
    int64_t pages = 0, codes_stride = 0, scales_stride = 0;   // between pages, in bytes and pairs
    int kv_heads = 0, d = 0, bits = 4, block_tokens = 0, bt_shift = 0;
    bool bf16 = false;
};

// Lane i has lengths[i] tokens in the pages tables[i][..], the last of which are its rows: cu[i] .. cu[i + 1] - 1, or `rows` for every lane.
struct QuantLanes {
    const int32_t* tables = nullptr;
    int64_t ld_table = 0;
    int width = 0;
    const int32_t *lengths = nullptr, *cu = nullptr;
    int lanes = 0, rows = 0, total = 0;
    int32_t* status = nullptr;   // may be null
};

struct QuantRowsArgs {
    QuantPools pools;
    QuantLanes lanes;
    void *k = nullptr, *v = nullptr;   // [total][kv_heads][d], read or written
    int64_t k_row = 0, k_head = 0, v_row = 0, v_head = 0;   // strides in values
};
void launch_quantize_rows(const QuantRowsArgs& a, cudaStream_t s);
void launch_dequantize_rows(const QuantRowsArgs& a, cudaStream_t s);

}  // namespace mk
