// C ABI, part 5: operators over the caller's device buffers.  Nothing is allocated, copied to the host or waited for; arguments are checked before the
// device is asked for, so that a refusal is the same on a machine without one.
#include "../../include/macllm_b200.h"
#include "c_api_util.h"
#include "kv_rows.h"
#include "quantized_attention.h"
#include "shared_attention.h"
#include "token_logprobs.h"
#include "verify_drafts.h"
#include <algorithm>
#include <climits>
#include <cmath>

using namespace mk;

namespace {

void need(bool ok, const char* what) {
    if (!ok) throw std::runtime_error(what);
}
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// Arrays of 32-bit numbers, and the status word; null ones are aligned.
template <typename... P>
bool words(const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) == 0; }

SharedAttnPlan checked_plan(int q_heads, int kv_heads, int d, int block_tokens, int width, int lanes, int rows, int total, int shared, int window) {
    need(window >= 0, "mk_k_shared_attention: window is not negative");
    need(d == 64 || d == 128 || d == 256, "mk_k_shared_attention: head_dim is 64, 128 or 256");
    need(kv_heads > 0 && q_heads > 0 && q_heads % kv_heads == 0, "mk_k_shared_attention: q_heads is a multiple of kv_heads");
    need(q_heads / kv_heads <= 128 && kv_heads <= 65535, "mk_k_shared_attention: at most 128 query heads share a KV head, and there are at most 65535 of those");
    need(block_tokens >= 16 && block_tokens <= 65536 && (block_tokens & (block_tokens - 1)) == 0, "mk_k_shared_attention: block_tokens is a power of two from 16 to 65536");
    need(width >= 0 && (int64_t)width * block_tokens <= INT32_MAX / 2, "mk_k_shared_attention: the tables hold at most 2^30 positions a lane");
    need(lanes >= 0 && rows >= 0 && total >= 0, "mk_k_shared_attention: negative lanes or rows");
    need((int64_t)rows * (q_heads / kv_heads) <= 65535, "mk_k_shared_attention: rows of a lane times query heads of a KV head go up to 65535");
    need((int64_t)total * q_heads <= INT32_MAX / 4, "mk_k_shared_attention: too many rows");
    need(shared >= 0 && shared % block_tokens == 0 && shared / block_tokens <= width, "mk_k_shared_attention: shared_len is whole pages of the tables");
    const SharedAttnPlan p = shared_attention_plan(q_heads, kv_heads, d, block_tokens, width, lanes, rows, total, shared, window);
    need((int64_t)lanes * p.shares * std::max(1, p.item_tiles) * kv_heads <= INT32_MAX, "mk_k_shared_attention: too many lanes");
    return p;
}

int logits_kind(int type) { return type == MK_TYPE_F32 ? 0 : (type == MK_TYPE_F16 ? 1 : 2); }
VerifyPlan checked_verify_plan(int type, int lanes, int drafts, int vocab) {
    need(type == MK_TYPE_F32 || type == MK_TYPE_F16 || type == MK_TYPE_BF16, "mk_k_verify_drafts: logits are f32, f16 or bf16");
    need(lanes >= 0 && drafts >= 0 && vocab > 0, "mk_k_verify_drafts: negative sizes");
    need(vocab <= kVerifyMaxVocab, "mk_k_verify_drafts: a vocabulary has at most 416000 tokens");
    need((int64_t)lanes * ((int64_t)drafts + 1) <= 1 << 22, "mk_k_verify_drafts: too many rows");
    return verify_plan(logits_kind(type), lanes, drafts, vocab);
}

// The pools' arguments, as all calls that take them have them.
struct PoolArgs {
    int32_t type, bits;
    const void *k_codes, *v_codes, *k_scales, *v_scales;
    int64_t pages, codes_stride, scales_stride;
    int32_t kv_heads, head_dim, block_tokens;
};
QuantPools checked_pools(const PoolArgs& c) {
    need(c.type == MK_TYPE_F16 || c.type == MK_TYPE_BF16, "mk_k_quantized: rows and scales are f16 or bf16, all of one type");
    need(c.bits == 4 || c.bits == 8, "mk_k_quantized: codes have 4 or 8 bits");
    need(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "mk_k_quantized: head_dim is 64, 128 or 256");
    need(c.kv_heads > 0 && c.kv_heads <= 65535, "mk_k_quantized: there are 1 to 65535 KV heads");
    need(c.block_tokens >= 16 && c.block_tokens <= 65536 && (c.block_tokens & (c.block_tokens - 1)) == 0, "mk_k_quantized: block_tokens is a power of two from 16 to 65536");
    const int64_t rows = (int64_t)c.kv_heads * c.block_tokens, page = rows * (c.head_dim * c.bits / 8), pairs = rows * (c.head_dim / kQuantGroup);
    need(rows <= INT32_MAX / 256, "mk_k_quantized: a page has too many rows");
    need(c.pages > 0 && c.pages <= INT32_MAX, "mk_k_quantized: there are 1 to 2^31 - 1 pages");
    need(c.codes_stride >= page && c.scales_stride >= 2 * pairs, "mk_k_quantized: pages overlap");
    need(c.codes_stride <= INT64_MAX / c.pages && c.scales_stride <= INT64_MAX / 4 / c.pages, "mk_k_quantized: pages are too far apart");
    need(c.codes_stride % 16 == 0 && c.scales_stride % 8 == 0, "mk_k_quantized: pages begin at multiples of 16 bytes");
    QuantPools p;
    p.k_codes = static_cast<uint8_t*>(const_cast<void*>(c.k_codes)); p.v_codes = static_cast<uint8_t*>(const_cast<void*>(c.v_codes));
    p.k_scales = static_cast<uint32_t*>(const_cast<void*>(c.k_scales)); p.v_scales = static_cast<uint32_t*>(const_cast<void*>(c.v_scales));
    p.pages = c.pages; p.codes_stride = c.codes_stride; p.scales_stride = c.scales_stride / 2;
    p.kv_heads = c.kv_heads; p.d = c.head_dim; p.bits = c.bits; p.block_tokens = c.block_tokens; p.bt_shift = __builtin_ctz(c.block_tokens);
    p.bf16 = c.type == MK_TYPE_BF16;
    return p;
}
void checked_pool_pointers(const QuantPools& p) {
    need(p.k_codes != nullptr && p.v_codes != nullptr && p.k_scales != nullptr && p.v_scales != nullptr, "mk_k_quantized: null pointer");
    need(aligned(p.k_codes, 16) && aligned(p.v_codes, 16) && aligned(p.k_scales, 16) && aligned(p.v_scales, 16), "mk_k_quantized: pools begin at multiples of 16 bytes");
}

void checked_lane_sizes(int block_tokens, int width, int64_t table_stride, int lanes, int total) {
    need(lanes >= 0 && total >= 0, "mk_k_quantized: negative lanes or rows");
    need(width >= 0 && (int64_t)width * block_tokens <= INT32_MAX / 2, "mk_k_quantized: the tables hold at most 2^30 positions a lane");
    need(table_stride >= width, "mk_k_quantized: table rows overlap");
}
void checked_lane_pointers(const QuantLanes& l) {
    need(l.lengths != nullptr && (l.tables != nullptr || l.width == 0), "mk_k_quantized: null pointer");
    need(words(l.tables, l.lengths, l.cu, l.status), "mk_k_quantized: tables, lengths, rows and status are words aligned to 4 bytes");
}

// What rows into pages and rows out of them have in common; false where there is nothing to do.
bool checked_rows(const PoolArgs& pools, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int32_t* tables,
                  int64_t table_stride, int table_width, const int32_t* lengths, const int32_t* cu, int lanes, int total, int32_t* status, QuantRowsArgs& a) {
    a.pools = checked_pools(pools);
    checked_lane_sizes(a.pools.block_tokens, table_width, table_stride, lanes, total);
    need(cu != nullptr || (lanes > 0 ? total % lanes == 0 : total == 0), "mk_k_quantized: without cu_seqlens every lane has the same number of rows");
    need(k_row >= 0 && k_head >= 0 && v_row >= 0 && v_head >= 0 && k_row <= INT64_MAX / INT32_MAX / 2 && v_row <= INT64_MAX / INT32_MAX / 2 && k_head <= INT64_MAX / 65536 / 4 &&
             v_head <= INT64_MAX / 65536 / 4,
         "mk_k_quantized: strides out of range");
    if (lanes == 0 || total == 0) return false;
    need(k != nullptr && v != nullptr, "mk_k_quantized: null pointer");
    need(aligned(k, 16) && aligned(v, 16) && ((k_row | k_head | v_row | v_head) & 7) == 0, "mk_k_quantized: heads of rows begin at multiples of 16 bytes");
    a.lanes.tables = tables; a.lanes.ld_table = table_stride; a.lanes.width = table_width; a.lanes.lengths = lengths; a.lanes.cu = cu;
    a.lanes.lanes = lanes; a.lanes.rows = cu == nullptr ? total / lanes : 0; a.lanes.total = total; a.lanes.status = status;
    checked_lane_pointers(a.lanes);
    checked_pool_pointers(a.pools);
    a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
    return true;
}
bool apart(int64_t row, int64_t head, int rows, int heads, int d) {   // [rows][heads][d] whose values are all different ones
    if (rows == 1) return heads == 1 || head >= d;
    if (heads == 1) return row >= d;
    return (head >= d && row >= (heads - 1) * head + d) || (row >= d && head >= (rows - 1) * row + d);
}

QuantAttnPlan checked_quantized_plan(const QuantPools& p, int q_heads, int width, int lanes, int rows, int total, int window) {
    checked_lane_sizes(p.block_tokens, width, width, lanes, total);
    need(rows >= 0, "mk_k_quantized_attention: negative lanes or rows");
    need(window >= 0, "mk_k_quantized_attention: window is not negative");
    need(q_heads > 0 && q_heads % p.kv_heads == 0, "mk_k_quantized_attention: q_heads is a multiple of kv_heads");
    need(q_heads / p.kv_heads <= 128, "mk_k_quantized_attention: at most 128 query heads share a KV head");
    need((int64_t)rows * (q_heads / p.kv_heads) <= 4 << 20 && (int64_t)total * q_heads <= INT32_MAX / 4, "mk_k_quantized_attention: too many rows");
    const QuantAttnPlan plan = quantized_attention_plan(q_heads, p.kv_heads, p.d, p.bits, p.block_tokens, width, lanes, rows, total, window);
    need(plan.slots <= INT32_MAX / p.kv_heads / plan.blocks, "mk_k_quantized_attention: too many lanes");
    return plan;
}

}  // namespace

extern "C" {

int32_t mk_k_shared_attention_workspace(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_tokens, int32_t table_width, int32_t lanes, int32_t rows,
                                        int32_t total, int32_t shared_len, int32_t window, int64_t* bytes) {
    return guarded([&] {
        need(bytes != nullptr, "mk_k_shared_attention_workspace: null pointer");
        *bytes = checked_plan(q_heads, kv_heads, head_dim, block_tokens, table_width, lanes, rows, total, shared_len, window).bytes(total, q_heads, head_dim);
    });
}

int32_t mk_k_shared_attention_dev(int32_t type, const void* q_dev, int64_t q_stride, const void* k_pool_dev, const void* v_pool_dev, int64_t pool_pages, int64_t page_stride,
                                  int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_tokens, const int32_t* tables_dev, int64_t table_stride, int32_t table_width,
                                  const int32_t* lengths_dev, const int32_t* cu_seqlens_dev, int32_t lanes, int32_t rows, int32_t total, int32_t shared_len, float scale,
                                  float softcap, int32_t window, void* out_dev, int64_t out_stride, void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev,
                                  void* cuda_stream) {
    return guarded([&] {
        need(type == MK_TYPE_F16 || type == MK_TYPE_BF16, "mk_k_shared_attention_dev: queries, pools and results are f16 or bf16, all of one type");
        const SharedAttnPlan p = checked_plan(q_heads, kv_heads, head_dim, block_tokens, table_width, lanes, rows, total, shared_len, window);
        if (lanes == 0 || total == 0 || rows == 0) return;
        need(q_dev != nullptr && k_pool_dev != nullptr && v_pool_dev != nullptr && lengths_dev != nullptr && out_dev != nullptr && (tables_dev != nullptr || table_width == 0),
             "mk_k_shared_attention_dev: null pointer");
        need(cu_seqlens_dev != nullptr || (int64_t)lanes * rows == total, "mk_k_shared_attention_dev: without cu_seqlens every lane has the same number of rows");
        need(aligned(q_dev, 16) && aligned(k_pool_dev, 16) && aligned(v_pool_dev, 16) && aligned(out_dev, 16) && q_stride % 8 == 0 && out_stride % 8 == 0,
             "mk_k_shared_attention_dev: rows and pools begin at multiples of 16 bytes");
        need(words(tables_dev, lengths_dev, cu_seqlens_dev, status_dev), "mk_k_shared_attention_dev: tables, lengths, rows and status are words aligned to 4 bytes");
        need(q_stride >= (int64_t)q_heads * head_dim && out_stride >= (int64_t)q_heads * head_dim && table_stride >= table_width, "mk_k_shared_attention_dev: rows overlap");
        need(pool_pages > 0 && page_stride % head_dim == 0 && page_stride >= (int64_t)kv_heads * block_tokens * head_dim, "mk_k_shared_attention_dev: pages overlap, or do not begin at a row");
        need(pool_pages <= INT32_MAX && page_stride / head_dim <= INT32_MAX && pool_pages * (page_stride / head_dim) <= INT32_MAX,
             "mk_k_shared_attention_dev: a pool has at most 2^31 - 1 rows of a head");
        need(scale > 0.f && std::isfinite(scale), "mk_k_shared_attention_dev: scale is positive");
        need(softcap >= 0.f && std::isfinite(softcap), "mk_k_shared_attention_dev: softcap is not negative");
        const int64_t bytes = p.bytes(total, q_heads, head_dim);
        need(bytes == 0 || (workspace_dev != nullptr && workspace_bytes >= bytes && aligned(workspace_dev, 16)), "mk_k_shared_attention_dev: the workspace is missing, too small or not aligned to 16 bytes");
        require_device();
        SharedAttnArgs a;
        a.q = q_dev; a.out = out_dev; a.ldq = q_stride; a.ldo = out_stride;
        a.k_pool = k_pool_dev; a.v_pool = v_pool_dev; a.pool_pages = pool_pages; a.page_rows = page_stride / head_dim;
        a.q_heads = q_heads; a.kv_heads = kv_heads; a.d = head_dim; a.block_tokens = block_tokens; a.bf16 = type == MK_TYPE_BF16;
        a.tables = tables_dev; a.ld_table = table_stride; a.width = table_width; a.lengths = lengths_dev; a.cu = cu_seqlens_dev;
        a.lanes = lanes; a.rows = rows; a.total = total; a.shared = shared_len;
        a.scale = scale; a.softcap = softcap; a.window = window;
        a.part_o = static_cast<float*>(workspace_dev); a.status = status_dev;
        launch_shared_attention(a, p, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_verify_drafts_workspace(int32_t type, int32_t lanes, int32_t drafts, int32_t vocab, int64_t* bytes) {
    return guarded([&] {
        need(bytes != nullptr, "mk_k_verify_drafts_workspace: null pointer");
        *bytes = checked_verify_plan(type, lanes, drafts, vocab).bytes;
    });
}

int32_t mk_k_verify_drafts_dev(int32_t type, const void* logits_dev, int64_t logits_stride, int32_t lanes, int32_t drafts, int32_t vocab, const int32_t* drafts_dev,
                               const float* draft_probs_dev, const float* u_dev, const float* temperature_dev, const int32_t* top_k_dev, const float* top_p_dev,
                               int32_t* tokens_dev, int32_t* accepted_dev, void* workspace_dev, int64_t workspace_bytes, int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        const VerifyPlan p = checked_verify_plan(type, lanes, drafts, vocab);
        need(logits_stride >= vocab, "mk_k_verify_drafts_dev: rows overlap");
        if (lanes == 0) return;
        need(aligned(logits_dev, type == MK_TYPE_F32 ? 4 : 2), "mk_k_verify_drafts_dev: logits are not aligned to their type");
        need(logits_dev != nullptr && (drafts_dev != nullptr || drafts == 0) && u_dev != nullptr && temperature_dev != nullptr && top_k_dev != nullptr && top_p_dev != nullptr &&
                 tokens_dev != nullptr && accepted_dev != nullptr,
             "mk_k_verify_drafts_dev: null pointer");
        need(words(drafts_dev, draft_probs_dev, u_dev, temperature_dev, top_k_dev, top_p_dev, tokens_dev, accepted_dev, status_dev), "mk_k_verify_drafts_dev: arrays are not aligned to 4 bytes");
        need(workspace_dev != nullptr && workspace_bytes >= p.bytes && aligned(workspace_dev, 16),
             "mk_k_verify_drafts_dev: the workspace is missing, too small or not aligned to 16 bytes");
        require_device();
        VerifyArgs a;
        a.logits = logits_dev; a.ld = logits_stride; a.type = logits_kind(type);
        a.lanes = lanes; a.n_drafts = drafts; a.vocab = vocab; a.drafts = drafts_dev; a.draft_probs = draft_probs_dev; a.u = u_dev;
        a.temperature = temperature_dev; a.top_k = top_k_dev; a.top_p = top_p_dev; a.tokens = tokens_dev; a.accepted = accepted_dev;
        a.status = status_dev;
        launch_verify_drafts(a, p, static_cast<uint8_t*>(workspace_dev), static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_copy_pages_dev(void* k_pool_dev, void* v_pool_dev, int64_t layers, int64_t pages, int32_t kv_heads, int32_t block_tokens, int32_t row_bytes,
                            const int32_t* copies_dev, int32_t n, int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        need(layers >= 0 && pages >= 0 && kv_heads > 0 && block_tokens > 0 && n >= 0, "mk_k_copy_pages_dev: negative or empty sizes");
        need(row_bytes > 0 && row_bytes % 2 == 0 && row_bytes <= 65536 && (int64_t)kv_heads * block_tokens * row_bytes <= INT32_MAX,
             "mk_k_copy_pages_dev: a row has an even number of bytes, at most 65536, and a page less than 2 GiB");
        if (n == 0 || layers == 0) return;
        need(k_pool_dev != nullptr && v_pool_dev != nullptr && copies_dev != nullptr, "mk_k_copy_pages_dev: null pointer");
        need(aligned(k_pool_dev, 2) && aligned(v_pool_dev, 2), "mk_k_copy_pages_dev: pools begin at even addresses");
        need(words(copies_dev, status_dev), "mk_k_copy_pages_dev: arrays are not aligned to 4 bytes");
        require_device();
        KvRowsArgs a;
        a.k_pool = k_pool_dev; a.v_pool = v_pool_dev; a.layers = layers; a.pages = pages; a.kv_heads = kv_heads; a.block_tokens = block_tokens; a.row_bytes = row_bytes;
        a.copies = copies_dev; a.n = n; a.status = status_dev;
        launch_copy_pages(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_gather_tokens_dev(void* k_pool_dev, void* v_pool_dev, int64_t layers, int64_t pages, int32_t kv_heads, int32_t block_tokens, int32_t row_bytes,
                               const int32_t* from_tables_dev, int64_t from_stride, int32_t from_width, const int32_t* keep_dev, int64_t keep_stride, int32_t keep_width,
                               const int32_t* counts_dev, const int32_t* to_tables_dev, int64_t to_stride, int32_t to_width, const int32_t* first_dev, int32_t lanes,
                               int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        need(layers >= 0 && pages >= 0 && kv_heads > 0 && block_tokens > 0 && lanes >= 0, "mk_k_gather_tokens_dev: negative or empty sizes");
        need(row_bytes > 0 && row_bytes % 2 == 0 && row_bytes <= 65536 && (int64_t)kv_heads * block_tokens * row_bytes <= INT32_MAX,
             "mk_k_gather_tokens_dev: a row has an even number of bytes, at most 65536, and a page less than 2 GiB");
        need(from_width >= 0 && to_width >= 0 && keep_width >= 0 && from_stride >= from_width && to_stride >= to_width && keep_stride >= keep_width, "mk_k_gather_tokens_dev: table rows overlap");
        need((int64_t)from_width * block_tokens <= INT32_MAX && (int64_t)to_width * block_tokens <= INT32_MAX && (int64_t)lanes * kv_heads <= INT32_MAX, "mk_k_gather_tokens_dev: too many positions or lanes");
        if (lanes == 0 || layers == 0 || keep_width == 0) return;
        need(k_pool_dev != nullptr && v_pool_dev != nullptr && from_tables_dev != nullptr && to_tables_dev != nullptr && keep_dev != nullptr && counts_dev != nullptr && first_dev != nullptr,
             "mk_k_gather_tokens_dev: null pointer");
        need(aligned(k_pool_dev, 2) && aligned(v_pool_dev, 2), "mk_k_gather_tokens_dev: pools begin at even addresses");
        need(words(from_tables_dev, keep_dev, counts_dev, to_tables_dev, first_dev, status_dev), "mk_k_gather_tokens_dev: arrays are not aligned to 4 bytes");
        require_device();
        KvRowsArgs a;
        a.k_pool = k_pool_dev; a.v_pool = v_pool_dev; a.layers = layers; a.pages = pages; a.kv_heads = kv_heads; a.block_tokens = block_tokens; a.row_bytes = row_bytes;
        a.from = from_tables_dev; a.to = to_tables_dev; a.keep = keep_dev; a.counts = counts_dev; a.first = first_dev;
        a.ld_from = from_stride; a.ld_to = to_stride; a.ld_keep = keep_stride;
        a.lanes = lanes; a.from_width = from_width; a.to_width = to_width; a.keep_width = keep_width; a.status = status_dev;
        launch_gather_tokens(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_quantize_rows_dev(const void* k_dev, int64_t k_row_stride, int64_t k_head_stride, const void* v_dev, int64_t v_row_stride, int64_t v_head_stride,
                               int32_t type, int32_t bits, void* k_codes_dev, void* v_codes_dev, void* k_scales_dev, void* v_scales_dev,
                               int64_t pool_pages, int64_t codes_stride, int64_t scales_stride, int32_t kv_heads, int32_t head_dim, int32_t block_tokens,
                               const int32_t* tables_dev, int64_t table_stride, int32_t table_width, const int32_t* lengths_dev, const int32_t* cu_seqlens_dev, int32_t lanes,
                               int32_t total, int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        QuantRowsArgs a;
        if (!checked_rows(PoolArgs{type, bits, k_codes_dev, v_codes_dev, k_scales_dev, v_scales_dev, pool_pages, codes_stride, scales_stride, kv_heads, head_dim, block_tokens},
                           k_dev, k_row_stride, k_head_stride, v_dev, v_row_stride, v_head_stride, tables_dev, table_stride, table_width, lengths_dev, cu_seqlens_dev, lanes,
                          total, status_dev, a))
            return;
        require_device();
        a.k = const_cast<void*>(k_dev); a.v = const_cast<void*>(v_dev);
        launch_quantize_rows(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_dequantize_rows_dev(int32_t type, int32_t bits, const void* k_codes_dev, const void* v_codes_dev, const void* k_scales_dev, const void* v_scales_dev,
                                 int64_t pool_pages, int64_t codes_stride, int64_t scales_stride, int32_t kv_heads, int32_t head_dim, int32_t block_tokens,
                                 const int32_t* tables_dev, int64_t table_stride, int32_t table_width, const int32_t* lengths_dev, const int32_t* cu_seqlens_dev, int32_t lanes,
                                 int32_t total, void* k_dev, int64_t k_row_stride, int64_t k_head_stride, void* v_dev, int64_t v_row_stride, int64_t v_head_stride,
                                 int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        QuantRowsArgs a;
        if (!checked_rows(PoolArgs{type, bits, k_codes_dev, v_codes_dev, k_scales_dev, v_scales_dev, pool_pages, codes_stride, scales_stride, kv_heads, head_dim, block_tokens},
                           k_dev, k_row_stride, k_head_stride, v_dev, v_row_stride, v_head_stride, tables_dev, table_stride, table_width, lengths_dev, cu_seqlens_dev, lanes,
                          total, status_dev, a))
            return;
        need(apart(a.k_row, a.k_head, total, a.pools.kv_heads, a.pools.d) && apart(a.v_row, a.v_head, total, a.pools.kv_heads, a.pools.d), "mk_k_dequantize_rows_dev: rows overlap");
        require_device();
        a.k = k_dev; a.v = v_dev;
        launch_dequantize_rows(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_quantized_attention_workspace(int32_t bits, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_tokens, int32_t table_width, int32_t lanes,
                                           int32_t rows, int32_t total, int32_t window, int64_t* bytes) {
    return guarded([&] {
        need(bytes != nullptr, "mk_k_quantized_attention_workspace: null pointer");
        const int64_t rows_of_page = (int64_t)std::max(kv_heads, 0) * std::max(block_tokens, 0);
        const PoolArgs pools{MK_TYPE_F16, bits, nullptr, nullptr, nullptr, nullptr, 1, rows_of_page * std::max(head_dim, 0), rows_of_page * std::max(head_dim, 0), kv_heads, head_dim, block_tokens};
        *bytes = checked_quantized_plan(checked_pools(pools), q_heads, table_width, lanes, rows, total, window).bytes;
    });
}

int32_t mk_k_quantized_attention_dev(const void* q_dev, int64_t q_stride, int32_t q_heads,
                                     int32_t type, int32_t bits, const void* k_codes_dev, const void* v_codes_dev, const void* k_scales_dev, const void* v_scales_dev,
                                     int64_t pool_pages, int64_t codes_stride, int64_t scales_stride, int32_t kv_heads, int32_t head_dim, int32_t block_tokens,
                                     const int32_t* tables_dev, int64_t table_stride, int32_t table_width, const int32_t* lengths_dev, const int32_t* cu_seqlens_dev, int32_t lanes,
                                     int32_t rows, int32_t total, float scale, float softcap, int32_t window, void* out_dev, int64_t out_stride, void* workspace_dev,
                                     int64_t workspace_bytes, int32_t* status_dev, void* cuda_stream) {
    return guarded([&] {
        QuantAttnArgs a;
        a.pools = checked_pools(PoolArgs{type, bits, k_codes_dev, v_codes_dev, k_scales_dev, v_scales_dev, pool_pages, codes_stride, scales_stride, kv_heads, head_dim, block_tokens});
        const QuantAttnPlan p = checked_quantized_plan(a.pools, q_heads, table_width, lanes, rows, total, window);
        need(table_stride >= table_width, "mk_k_quantized: table rows overlap");
        if (lanes == 0 || total == 0 || rows == 0) return;
        need(q_dev != nullptr && out_dev != nullptr, "mk_k_quantized_attention_dev: null pointer");
        need(cu_seqlens_dev != nullptr || (int64_t)lanes * rows == total, "mk_k_quantized_attention_dev: without cu_seqlens every lane has the same number of rows");
        need(aligned(q_dev, 16) && aligned(out_dev, 16) && q_stride % 8 == 0 && out_stride % 8 == 0, "mk_k_quantized_attention_dev: rows begin at multiples of 16 bytes");
        need(q_stride >= (int64_t)q_heads * a.pools.d && out_stride >= (int64_t)q_heads * a.pools.d, "mk_k_quantized_attention_dev: rows overlap");
        need(scale > 0.f && std::isfinite(scale), "mk_k_quantized_attention_dev: scale is positive");
        need(softcap >= 0.f && std::isfinite(softcap), "mk_k_quantized_attention_dev: softcap is not negative");
        a.lanes.tables = tables_dev; a.lanes.ld_table = table_stride; a.lanes.width = table_width; a.lanes.lengths = lengths_dev; a.lanes.cu = cu_seqlens_dev;
        a.lanes.lanes = lanes; a.lanes.rows = rows; a.lanes.total = total; a.lanes.status = status_dev;
        checked_lane_pointers(a.lanes);
        checked_pool_pointers(a.pools);
        need(p.bytes == 0 || (workspace_dev != nullptr && workspace_bytes >= p.bytes && aligned(workspace_dev, 16)),
             "mk_k_quantized_attention_dev: the workspace is missing, too small or not aligned to 16 bytes");
        require_device();
        a.q = q_dev; a.out = out_dev; a.ldq = q_stride; a.ldo = out_stride; a.q_heads = q_heads;
        a.scale = scale; a.softcap = softcap; a.window = window;
        launch_quantized_attention(a, p, workspace_dev, static_cast<cudaStream_t>(cuda_stream));
    });
}

int32_t mk_k_token_logprobs_dev(int32_t type, const void* logits_dev, int64_t logits_stride, int32_t rows, int32_t vocab, const int32_t* tokens_dev, int32_t top,
                                float* logprobs_dev, float* entropy_dev, int32_t* ranks_dev, int32_t* top_tokens_dev, float* top_logprobs_dev, int32_t* status_dev,
                                void* cuda_stream) {
    return guarded([&] {
        need(type == MK_TYPE_F32 || type == MK_TYPE_F16 || type == MK_TYPE_BF16, "mk_k_token_logprobs_dev: logits are f32, f16 or bf16");
        need(rows >= 0 && vocab > 0 && vocab <= 1 << 24, "mk_k_token_logprobs_dev: a vocabulary has 1 to 2^24 tokens");
        need(top >= 0 && top <= kLogprobMaxTop && top <= vocab, "mk_k_token_logprobs_dev: top is at most 64 and at most the vocabulary");
        need(rows <= 1 || logits_stride >= vocab, "mk_k_token_logprobs_dev: rows overlap");
        need(logits_stride <= INT64_MAX / 4 / std::max(rows, 1), "mk_k_token_logprobs_dev: rows are too far apart");
        if (rows == 0) return;
        need(logits_dev != nullptr && tokens_dev != nullptr && logprobs_dev != nullptr && entropy_dev != nullptr && ranks_dev != nullptr &&
                 (top == 0 || (top_tokens_dev != nullptr && top_logprobs_dev != nullptr)),
             "mk_k_token_logprobs_dev: null pointer");
        need(aligned(logits_dev, type == MK_TYPE_F32 ? 4 : 2), "mk_k_token_logprobs_dev: logits are not aligned to their type");
        need(words(tokens_dev, logprobs_dev, entropy_dev, ranks_dev, top_tokens_dev, top_logprobs_dev, status_dev), "mk_k_token_logprobs_dev: arrays are not aligned to 4 bytes");
        require_device();
        LogprobArgs a;
        a.logits = logits_dev; a.ld = logits_stride; a.kind = logits_kind(type); a.rows = rows; a.vocab = vocab; a.top = top; a.tokens = tokens_dev;
        a.logprobs = logprobs_dev; a.entropy = entropy_dev; a.ranks = ranks_dev; a.top_tokens = top_tokens_dev; a.top_logprobs = top_logprobs_dev; a.status = status_dev;
        launch_token_logprobs(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

}  // extern "C"
