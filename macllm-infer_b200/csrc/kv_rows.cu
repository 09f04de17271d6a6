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

// A CTA per (copy, layer, K or V): the rows of all heads.  600 pages of 16 tokens of 36 layers of 8 heads of 128: 421 us, 6.7 TB/s read and written.
template <typename PIECE>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ KvRowsArgs a) {
    const int row_pieces = a.row_bytes / (int)sizeof(PIECE);
    const int64_t page_pieces = (int64_t)a.kv_heads * a.block_tokens * row_pieces;
    const int32_t* c = a.copies + (int64_t)blockIdx.x * 3;
    const int from = c[0], to = c[1], rows = c[2];
    const int wrong = (from < 0 || from >= a.pages || to < 0 || to >= a.pages ? kDevBadPage : 0) | (rows < 0 || rows > a.block_tokens ? kDevBadRange : 0);
    if (wrong != 0) {
        if (threadIdx.x == 0) tell(a.status, wrong);
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

// A CTA per (lane, head, K or V) and run of layers walks the kept tokens in their order.  Where 1024 of them come from and go to is looked up once for all its layers.  A chunk
// is read whole before it is written, and the one behind it is on its way by then: since keep ascends and keep[j] >= first + j, what a chunk writes is in front of what a later
// one reads, so in place is the same as apart.  9600 tokens of 36 layers of 4 heads of 128 (1.4 GB read and written): 241 us, 5.9 TB/s; with the rows looked up per 64 tokens and
// layer 325 us; 274 us with 256 threads of four pieces, which wait longer at the barrier between reading and writing; 324 us with a warp for each column, which has too few
// pieces on their way.
constexpr int kGatherThreads = 128, kGatherTokens = 1024;

template <typename PIECE>
__global__ void __launch_bounds__(kGatherThreads) gather_tokens_kernel(const __grid_constant__ KvRowsArgs a) {
    constexpr int PER = 2;
    __shared__ longlong2 rows[kGatherTokens];   // (from, to) in rows of a layer; from < 0: left out
    const int tid = threadIdx.x, row_pieces = a.row_bytes / (int)sizeof(PIECE), lane = blockIdx.x / a.kv_heads, head = blockIdx.x - lane * a.kv_heads;
    const int count = a.counts[lane], first = a.first[lane];
    if (count < 0 || count > a.keep_width || first < 0 || first > a.to_width * a.block_tokens - count) {
        if (tid == 0) tell(a.status, kDevBadRange);
        return;
    }
    const int32_t *keep = a.keep + lane * a.ld_keep, *from = a.from + lane * a.ld_from, *to = a.to + lane * a.ld_to;
    const int64_t page_rows = (int64_t)a.kv_heads * a.block_tokens, layer_pieces = a.pages * page_rows * row_pieces;
    const bool even = kGatherThreads % row_pieces == 0;   // then a thread has the same piece of every row
    const int my_row = tid / row_pieces, my_piece = tid - my_row * row_pieces, row_step = kGatherThreads / row_pieces;
    for (int j0 = 0; j0 < count; j0 += kGatherTokens) {
        const int n = min(kGatherTokens, count - j0);
        __syncthreads();
        for (int j = tid; j < n; j += kGatherThreads) {
            const int s = keep[j0 + j], t = first + j0 + j;
            longlong2 r = make_longlong2(-1, -1);
            if (s < 0 || s >= a.from_width * a.block_tokens) {
                tell(a.status, kDevBadRange);
            } else {
                const int sp = from[s / a.block_tokens], tp = to[t / a.block_tokens];
                if (sp < 0 || sp >= a.pages || tp < 0 || tp >= a.pages) tell(a.status, kDevBadPage);
                else r = make_longlong2(sp * page_rows + head * a.block_tokens + s % a.block_tokens, tp * page_rows + head * a.block_tokens + t % a.block_tokens);
            }
            rows[j] = r;
        }
        __syncthreads();
        for (int64_t layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
            PIECE* pool = static_cast<PIECE*>(blockIdx.z == 0 ? a.k_pool : a.v_pool) + layer * layer_pieces;
            PIECE now[PER], next[PER];
            int64_t to_now[PER], to_next[PER];
            auto read = [&](int chunk, PIECE (&v)[PER], int64_t (&dst)[PER]) {
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    int j, c = my_piece;
                    if (even) {
                        j = (chunk * PER + p) * row_step + my_row;
                    } else {
                        const int i = (chunk * PER + p) * kGatherThreads + tid;
                        j = i / row_pieces;
                        c = i - j * row_pieces;
                    }
                    dst[p] = -1;
                    if (j >= n) continue;
                    const longlong2 r = rows[j];
                    if (r.x < 0) continue;
                    v[p] = pool[r.x * row_pieces + c];
                    dst[p] = r.y * row_pieces + c;
                }
            };
            const int chunks = (int)(((int64_t)n * row_pieces + PER * kGatherThreads - 1) / (PER * kGatherThreads));
            read(0, now, to_now);
            for (int chunk = 0; chunk < chunks; ++chunk) {
                if (chunk + 1 < chunks) read(chunk + 1, next, to_next);
                __syncthreads();
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    if (to_now[p] >= 0) pool[to_now[p]] = now[p];
                    now[p] = next[p];
                    to_now[p] = to_next[p];
                }
            }
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
    // as many layers to a CTA as leave 32 CTAs for each SM (16: 246 us where these take 241), split evenly
    const int64_t columns = (int64_t)a.lanes * a.kv_heads * 2, most = std::min<int64_t>({a.layers, std::max<int64_t>(1, (32 * 148 + columns - 1) / columns), 65535});
    const int64_t each = (a.layers + most - 1) / most, runs = (a.layers + each - 1) / each;
    with_piece(a, [&](auto piece) { gather_tokens_kernel<decltype(piece)><<<dim3((unsigned)(a.lanes * a.kv_heads), (unsigned)runs, 2), kGatherThreads, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

}  // namespace mk
