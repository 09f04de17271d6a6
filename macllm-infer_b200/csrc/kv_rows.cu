// Copies inside paged K/V pools: whole or partly filled pages, and the kept tokens of a lane moved together.  Nothing is computed: what bounds them is that
// each byte is read and written once, over all layers of K and V.
#include "kv_rows.h"
#include "shared_attention.h"
#include <algorithm>

namespace mk {

namespace {

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

// A CTA per (copy, layer, K or V): the rows of all heads.
template <typename PIECE>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ KvRowsArgs a) {
    const int row_pieces = a.row_bytes / (int)sizeof(PIECE);
    const int64_t page_pieces = (int64_t)a.kv_heads * a.block_tokens * row_pieces;
    const int32_t* c = a.copies + (int64_t)blockIdx.x * 3;
    const int from = c[0], to = c[1], rows = c[2];
    if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || rows < 0 || rows > a.block_tokens) {
        if (threadIdx.x == 0) tell(a.status, kDevBadPage);
        return;
    }
    if (from == to) return;
    for (int64_t layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
        PIECE* pool = static_cast<PIECE*>(blockIdx.z == 0 ? a.k_pool : a.v_pool) + layer * a.pages * page_pieces;
        const int per_head = rows * row_pieces;
        for (int i = threadIdx.x; i < a.kv_heads * per_head; i += 256) {
            const int64_t at = (int64_t)(i / per_head) * a.block_tokens * row_pieces + i % per_head;
            pool[to * page_pieces + at] = pool[from * page_pieces + at];
        }
    }
}

// A CTA per (lane, layer, head, K or V) walks the kept tokens in their order: a chunk is read whole before it is written, and since keep ascends and
// keep[j] >= first + j, no later chunk's source has been written.
template <typename PIECE>
__global__ void __launch_bounds__(256) gather_tokens_kernel(const __grid_constant__ KvRowsArgs a) {
    constexpr int PER = 4;
    const int row_pieces = a.row_bytes / (int)sizeof(PIECE), lane = blockIdx.x / a.kv_heads, head = blockIdx.x - lane * a.kv_heads;
    const int64_t head_pieces = (int64_t)a.block_tokens * row_pieces, page_pieces = a.kv_heads * head_pieces;
    const int count = a.counts[lane], first = a.first[lane];
    if (count < 0 || count > a.keep_width || first < 0 || first > a.to_width * a.block_tokens - count) {
        if (threadIdx.x == 0) tell(a.status, kDevBadRange);
        return;
    }
    const int32_t *keep = a.keep + lane * a.ld_keep, *from = a.from + lane * a.ld_from, *to = a.to + lane * a.ld_to;
    for (int64_t layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
        PIECE* pool = static_cast<PIECE*>(blockIdx.z == 0 ? a.k_pool : a.v_pool) + layer * a.pages * page_pieces + head * head_pieces;
        for (int64_t i0 = 0; i0 < (int64_t)count * row_pieces; i0 += PER * 256) {
            PIECE v[PER];
            int64_t dst[PER];
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const int64_t i = i0 + p * 256 + threadIdx.x;
                const int j = (int)(i / row_pieces), c = (int)(i - (int64_t)j * row_pieces);
                dst[p] = -1;
                if (j >= count) continue;
                const int s = keep[j], t = first + j;
                if (s < 0 || s >= a.from_width * a.block_tokens) {
                    tell(a.status, kDevBadRange);
                    continue;
                }
                const int sp = from[s / a.block_tokens], tp = to[t / a.block_tokens];
                if (sp < 0 || sp >= a.pages || tp < 0 || tp >= a.pages) {
                    tell(a.status, kDevBadPage);
                    continue;
                }
                v[p] = pool[sp * page_pieces + (int64_t)(s % a.block_tokens) * row_pieces + c];
                dst[p] = tp * page_pieces + (int64_t)(t % a.block_tokens) * row_pieces + c;
            }
            __syncthreads();
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if (dst[p] >= 0) pool[dst[p]] = v[p];
            __syncthreads();
        }
    }
}

// The widest pieces that rows and pools allow.
template <typename F>
void with_piece(const KvRowsArgs& a, F&& f) {
    const uintptr_t low = reinterpret_cast<uintptr_t>(a.k_pool) | reinterpret_cast<uintptr_t>(a.v_pool) | (uintptr_t)a.row_bytes;
    if (low % 16 == 0) f(uint4{});
    else if (low % 4 == 0) f(uint32_t{});
    else f(uint16_t{});
}

}  // namespace

void launch_copy_pages(const KvRowsArgs& a, cudaStream_t s) {
    if (a.n <= 0 || a.layers <= 0) return;
    with_piece(a, [&](auto piece) { copy_pages_kernel<decltype(piece)><<<dim3((unsigned)a.n, (unsigned)std::min<int64_t>(a.layers, 65535), 2), 256, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

void launch_gather_tokens(const KvRowsArgs& a, cudaStream_t s) {
    if (a.lanes <= 0 || a.layers <= 0 || a.keep_width <= 0) return;
    with_piece(a, [&](auto piece) {
        gather_tokens_kernel<decltype(piece)><<<dim3((unsigned)(a.lanes * a.kv_heads), (unsigned)std::min<int64_t>(a.layers, 65535), 2), 256, 0, s>>>(a);
    });
    MK_LAUNCH_CHECK();
}

}  // namespace mk
