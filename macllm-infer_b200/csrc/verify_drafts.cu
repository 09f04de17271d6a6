// Verification of drafted tokens against the target's distribution, from given random numbers.
//
// Row i of a lane holds the target's logits behind its first i drafts.  p_i = softmax(logits / temperature) over the top_k best tokens, of those the head
// that adds up to top_p (the sampler's rule); temperature 0: all on the best token.  q_i is the distribution that draft d_i came from.  Draft i is kept
// while u_i q_i(d_i) < p_i(d_i); the first that is not is replaced by a draw from max(p_i - q_i, 0), and behind the last draft one more token is drawn from
// p.  The tokens are then distributed as if drawn from the target one by one: q min(1, p / q) + (1 - sum q min(1, p / q)) max(p - q, 0) / sum max(p - q, 0) = p.
// A draw takes the first token, in the order of tokens, whose cumulative weight exceeds u_n times the whole.
//
// Every row is judged by itself, by a cluster of eight CTAs that hold it in their shared memory: it is fetched once, with bulk copies, and what needs more than
// one look at it (maximum, sum, candidates, draw) looks there.  A second kernel takes a lane's first row that ends it.
//
// Candidates of a top_k: each of the cluster's 4096 threads has the best of its own tokens, and the k-th best of those is a bound that at least k tokens reach and, since
// tokens are dealt out evenly, few more do; those are sorted.  Where too many reach it (thousands of equal logits) bisection over (value, token) finds one that
// fewer do.  Weights and sums of candidates are 64-bit.  Over the whole vocabulary a weight is a 32-bit number (ex2 of a product kept to twice 32 bits: 2^-22, and
// with no trend, so that sums over many are better), a sum of four is added up in 64 bits.
#include "verify_drafts.h"
#include "sampling_math.h"
#include "shared_attention.h"
#include "umma.cuh"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <algorithm>

namespace mk {

namespace {

namespace cg = cooperative_groups;

constexpr int kCtas = 8, kThreads = 512, kWarps = kThreads / 32, kPieces = 4;
constexpr int kCandidates = 2048;   // sorted at once; at least twice the largest top_k

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void set_low(float* x) { *x = -INFINITY; }
__device__ __forceinline__ void set_low(__half* x) { *x = __ushort_as_half(0xFC00); }
__device__ __forceinline__ void set_low(__nv_bfloat16* x) { *x = __ushort_as_bfloat16(0xFF80); }
// The values of 16 bytes.
__device__ __forceinline__ void unpack(const uint4& r, float (&v)[4], const float*) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(const uint4& r, float (&v)[8], const __half*) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const uint4& r, float (&v)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
// Larger first, the lower token first among equals; -0 counts as 0.
__device__ __forceinline__ uint64_t key_of(float x, int i) { return rank_key(x + 0.0f, (uint32_t)i); }
__device__ __forceinline__ float value_of_key(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return bits_f32((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
}

__device__ __forceinline__ double warp_scan(double v, int lane) {
    for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// Inclusive sums over the block's threads; *total: of all.
__device__ double block_scan(double v, double* red, double* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    v = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) red[w] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < w) before += red[i];
        all += red[i];
    }
    *total = all;
    return before + v;
}

// 512 E keys, the larger first: a thread has E neighbours, so that most exchanges of the bitonic network are inside a thread or a warp.
template <int E>
__device__ void sort_desc(uint64_t* keys) {
    const int tid = threadIdx.x;
    uint64_t a[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = keys[tid * E + e];
    for (int size = 2; size <= kThreads * E; size <<= 1) {
        auto exchange = [&](int stride, auto&& partner) {
            uint64_t y[E];
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = partner(e);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int at = tid * E + e;
                const bool larger = ((at & stride) == 0) == ((at & size) == 0);
                a[e] = (y[e] > a[e]) == larger ? y[e] : a[e];
            }
        };
        for (int stride = size >> 1; stride >= 32 * E; stride >>= 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) keys[tid * E + e] = a[e];
            __syncthreads();
            exchange(stride, [&](int e) { return keys[(tid * E + e) ^ stride]; });
        }
        for (int stride = min(size >> 1, 16 * E); stride >= E; stride >>= 1) exchange(stride, [&](int e) { return __shfl_xor_sync(0xffffffffu, a[e], stride / E); });
#pragma unroll
        for (int stride = E / 2; stride > 0; stride >>= 1)
            if (stride < size) exchange(stride, [&](int e) { return a[e ^ stride]; });
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) keys[tid * E + e] = a[e];
    __syncthreads();
}
__device__ void sort_desc(uint64_t* keys, int n) {   // keys behind n are there to be filled up
    const int size = n <= kThreads ? kThreads : (n <= 2 * kThreads ? 2 * kThreads : 4 * kThreads);
    for (int j = n + (int)threadIdx.x; j < size; j += kThreads) keys[j] = 0;
    __syncthreads();
    if (size == kThreads) sort_desc<1>(keys);
    else if (size == 2 * kThreads) sort_desc<2>(keys);
    else sort_desc<4>(keys);
}

// exp((x - top) / temperature) with 1 / (temperature ln 2) as the sum of two 32-bit numbers.
struct Exponential {
    float top, hi, lo;
    __device__ __forceinline__ float operator()(float x) const {
        const float y = x - top, t = y * hi, rest = fmaf(y, lo, fmaf(y, hi, -t));
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        return t > -126.f ? fmaf(e, rest * 0.69314718f, e) : 0.f;   // -inf among what is not
    }
};

template <typename T>
__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kThreads) verify_rows_kernel(const __grid_constant__ VerifyArgs a, int chunk) {
    constexpr int EPV = 16 / (int)sizeof(T);   // values of 16 bytes
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t bars[kPieces], best_of[kCtas], warp_best[kWarps];
    __shared__ double sum_of[3][kCtas], red[kWarps], region[kWarps];
    __shared__ int bad_of[kCtas], count_of[2][kCtas];
    __shared__ uint32_t thread_best[kThreads], warp_low[kWarps];
    __shared__ int s_count, s_pick, s_last, hist[256];
    __shared__ int2 s_step;
    __shared__ double s_pd;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, wl = tid & 31, rank = (int)cluster.block_rank(), index = blockIdx.x / kCtas;
    const int lane = index / (a.n_drafts + 1), i = index - lane * (a.n_drafts + 1), vocab = a.vocab;
    pdl_trigger();
    const int32_t* drafts = a.drafts + (int64_t)lane * a.n_drafts;
    const float* u = a.u + (int64_t)lane * (a.n_drafts + 1);
    const float temperature = a.temperature[lane], top_p = a.top_p[lane], u_last = u[a.n_drafts], u_mine = u[i];
    int k = a.top_k[lane], d = i < a.n_drafts ? drafts[i] : -1;
    bool gone = false;
    for (int j = wl; j < i; j += 32) gone |= drafts[j] < 0 || drafts[j] >= vocab;
    if (__any_sync(0xffffffffu, gone)) return;   // nothing gets here
    if (d >= vocab) {
        if (tid == 0) tell(a.status, kDevBadRange);
        d = -1;
    }
    const T* x = static_cast<const T*>(a.logits) + index * a.ld;
    int2* out = a.rows + index;

    // ---- this CTA's run of tokens, in 16-byte pieces of its row; places of the first and last piece that are not its hold -inf
    const int n0 = min(vocab, rank * chunk), n = min(chunk, vocab - n0);
    const uintptr_t src = reinterpret_cast<uintptr_t>(x + n0);
    const int shift = (int)(src & 15), bytes = n * (int)sizeof(T), vecs = n > 0 ? (shift + bytes + 15) / 16 : 0;
    const int v_lo = shift > 0 ? 1 : 0, v_hi = max(v_lo, (shift + bytes) / 16), per_piece = (v_hi - v_lo + kPieces - 1) / kPieces;
    const int token0 = n0 - shift / (int)sizeof(T);   // of the first place
    uint4* buf = reinterpret_cast<uint4*>(smem);
    uint16_t* list = reinterpret_cast<uint16_t*>(smem + a.list_at);
    if (tid == 0) {
        for (int p = 0; p < kPieces; ++p) umma::bar_init(&bars[p], 1);
        umma::bar_init_fence();
        s_count = 0;
        s_pick = INT_MAX;
        s_last = -1;
        s_pd = 0.0;
    }
    __syncthreads();
    if (tid == 0)
        for (int p = 0; p < kPieces; ++p) {
            const int lo = v_lo + p * per_piece, hi = min(v_hi, lo + per_piece);
            if (hi <= lo) continue;
            umma::bar_expect_tx(&bars[p], (uint32_t)(hi - lo) * 16);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(umma::smem_u32(buf + lo)), "l"(src - shift + (uintptr_t)lo * 16),
                         "r"((uint32_t)(hi - lo) * 16), "r"(umma::smem_u32(&bars[p]))
                         : "memory");
        }
    auto edge = [&](int v) {
        for (int j = tid; j < EPV; j += kThreads) {
            const int t = token0 + v * EPV + j;
            T* to = reinterpret_cast<T*>(buf + v) + j;
            if (t >= n0 && t < n0 + n) *to = x[t];
            else set_low(to);
        }
    };
    if (vecs > 0 && v_lo == 1) edge(0);
    if (vecs > v_hi && (v_hi > 0 || v_lo == 0)) edge(v_hi);
    __syncthreads();

    float mine = -INFINITY;
    bool bad = false, ok = true;
    uint64_t best = 0;
    auto look = [&](int v) {
        float f[EPV];
        unpack(buf[v], f, static_cast<const T*>(nullptr));
        float m = f[0];
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
            bad |= !(f[j] < INFINITY);
            m = fmaxf(m, f[j]);
        }
        if (m > mine || best == 0) {
            mine = m;
#pragma unroll
            for (int j = EPV - 1; j >= 0; --j)
                if (f[j] == m) best = key_of(m, token0 + v * EPV + j);
        }
    };
    if (tid == 0 && vecs > 0 && v_lo == 1) look(0);
    for (int p = 0; p < kPieces; ++p) {
        const int lo = v_lo + p * per_piece, hi = min(v_hi, lo + per_piece);
        if (hi <= lo) continue;
        ok = umma::bar_wait(&bars[p], 0) && ok;
        for (int v = lo + tid; v < hi; v += kThreads) look(v);
    }
    if (tid == kThreads - 1 && vecs > v_hi && (v_hi > 0 || v_lo == 0)) look(v_hi);
    if (best == 0) best = key_of(-INFINITY, vocab);
    thread_best[tid] = (uint32_t)(best >> 32);
    if (!ok) tell(a.status, kDevWait);
    bad = __syncthreads_or(bad || !ok);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (wl == 0) warp_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = warp_best[wl % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (wl < kCtas) {
            *cluster.map_shared_rank(&best_of[rank], wl) = best;
            *cluster.map_shared_rank(&bad_of[rank], wl) = bad;
        }
    }
    cluster.sync();
    best = best_of[0];
    bad = bad_of[0];
#pragma unroll
    for (int c = 1; c < kCtas; ++c) {
        best = best_of[c] > best ? best_of[c] : best;
        bad |= bad_of[c] != 0;
    }
    const float top = value_of_key(best);
    if (bad || top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            tell(a.status, kDevBadRow);
            *out = make_int2(0, -1);
        }
        return;
    }
    if (!(temperature > 0.f)) {
        if (rank == 0 && tid == 0) *out = make_int2(d == (int)rank_key_index(best), (int)rank_key_index(best));
        return;
    }
    if (k > kVerifyMaxTopK || (k <= 0 && top_p < 1.f)) {
        if (rank == 0 && tid == 0) tell(a.status, kDevBadRange);
        k = min(k, kVerifyMaxTopK);
    }
    k = min(k, vocab);
    const double per_t = 1.0 / (double)temperature;
    const float* q = a.draft_probs == nullptr || d < 0 ? nullptr : a.draft_probs + ((int64_t)lane * a.n_drafts + i) * vocab;
    const double u_draw = (double)u_last, kept_below = d >= 0 ? (double)u_mine * (q != nullptr ? (double)q[d] : 1.0) : 0.0;

    if (k <= 0) {
        // ---- the whole vocabulary
        const double unit = per_t * 1.4426950408889634074;
        Exponential weight;
        weight.top = top;
        weight.hi = (float)unit;
        weight.lo = (float)(unit - (double)weight.hi);
        auto block_sum_to = [&](double v, double* slot) {   // of this CTA, to the whole cluster
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            if (wl == 0) region[warp] = v;
            __syncthreads();
            if (warp == 0) {
                double s = region[wl % kWarps];
#pragma unroll
                for (int o = kWarps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (wl < kCtas) *cluster.map_shared_rank(slot + rank, wl) = s;
            }
            cluster.sync();
        };
        double part = 0.0;
        for (int v = tid; v < vecs; v += kThreads) {
            float f[EPV], s[EPV / 4];
            unpack(buf[v], f, static_cast<const T*>(nullptr));
#pragma unroll
            for (int j = 0; j < EPV; j += 4) s[j / 4] = (weight(f[j]) + weight(f[j + 1])) + (weight(f[j + 2]) + weight(f[j + 3]));
#pragma unroll
            for (int j = 0; j < EPV / 4; ++j) part += (double)s[j];
        }
        block_sum_to(part, sum_of[0]);
        double z = 0.0;
#pragma unroll
        for (int c = 0; c < kCtas; ++c) z += sum_of[0][c];
        if (d >= 0 && kept_below < exp(((double)value_of(x[d]) - (double)top) * per_t) / z) {
            if (rank == 0 && tid == 0) *out = make_int2(1, -1);
            return;
        }
        const float per_z = (float)(1.0 / z), per_z_rest = (float)(1.0 / z - (double)per_z);
        // The draw: every warp adds up a run of its own, one of them walks through the run where the target lies.
        const int run = (vecs + kWarps - 1) / kWarps, r_lo = min(vecs, warp * run), r_hi = min(vecs, r_lo + run);
        bool rest = d >= 0;
        auto load_q = [&](int v, float (&r)[EPV]) {   // what the draft's distribution has there, 0 where the row ends
            const int t0 = token0 + v * EPV;
#pragma unroll
            for (int j = 0; j < EPV; ++j) r[j] = q != nullptr ? (t0 + j >= n0 && t0 + j < n0 + n && v < vecs ? q[t0 + j] : 0.f) : (t0 + j == d ? 1.f : 0.f);
        };
        auto shares_of = [&](int v, const float (&qv)[EPV], float (&r)[EPV]) {
            unpack(buf[v], r, static_cast<const T*>(nullptr));
#pragma unroll
            for (int j = 0; j < EPV; ++j) {
                const float w = weight(r[j]);
                r[j] = rest ? fmaxf(fmaf(w, per_z, -qv[j]) + w * per_z_rest, 0.f) : w;
            }
        };
        double total = 0.0, *sums = sum_of[1];
        for (;;) {
            part = 0.0;
            constexpr int AHEAD = 16 / EPV;   // the draft's values of several pieces are on their way together
            for (int v0 = r_lo + wl; v0 < r_hi; v0 += 32 * AHEAD) {
                float qv[AHEAD][EPV];
                if (rest) {
#pragma unroll
                    for (int c = 0; c < AHEAD; ++c) load_q(v0 + 32 * c, qv[c]);
                }
#pragma unroll
                for (int c = 0; c < AHEAD; ++c) {
                    if (v0 + 32 * c >= r_hi) break;
                    float r[EPV];
                    shares_of(v0 + 32 * c, qv[c], r);
#pragma unroll
                    for (int j = 0; j < EPV; j += 4) part += (double)((r[j] + r[j + 1]) + (r[j + 2] + r[j + 3]));
                }
            }
            block_sum_to(part, sums);
            total = 0.0;
#pragma unroll
            for (int c = 0; c < kCtas; ++c) total += sums[c];
            if (total > 0.0 || !rest) break;
            rest = false;   // the draft's distribution covers the target's
            sums = sum_of[2];
        }
        const double target = u_draw * total;
        double before = 0.0;
        int at = -1;
#pragma unroll
        for (int c = 0; c < kCtas; ++c) {
            if (sums[c] > 0.0 && !(at >= 0 && before > target)) at = c;
            if (!(before > target)) before += sums[c];
        }
        if (at != rank) return;
        // at: the first CTA up to whose end the sum exceeds the target, or, where rounding left none, the last with a share; the same for its warps' runs
        before = 0.0;
        for (int c = 0; c < rank; ++c) before += sums[c];
        int w_at = -1;
        double w_before = before, upto_run = before;
        for (int w = 0; w < kWarps; ++w) {
            if (region[w] > 0.0) {
                w_at = w;
                w_before = upto_run;
            }
            upto_run += region[w];
            if (upto_run > target) break;
        }
        // the whole CTA looks through that run
        const int at_lo = min(vecs, w_at * run), at_hi = min(vecs, at_lo + run);
        for (int v0 = at_lo; v0 < at_hi; v0 += kThreads) {
            const int v = v0 + tid;
            float qv[EPV], r[EPV];
            double s = 0.0, all;
            if (v < at_hi) {
                load_q(v, qv);
                shares_of(v, qv, r);
#pragma unroll
                for (int j = 0; j < EPV; ++j) {
                    s += (double)r[j];
                    if (r[j] > 0.f) atomicMax(&s_last, token0 + v * EPV + j);
                }
            }
            double c = w_before + block_scan(s, red, &all) - s;
            if (v < at_hi && s > 0.0 && c + s > target) {
                int pick = -1;
#pragma unroll
                for (int j = 0; j < EPV; ++j) {
                    c += (double)r[j];
                    if (r[j] > 0.f && (pick < 0 || !(c - (double)r[j] > target))) pick = token0 + v * EPV + j;
                }
                atomicMin(&s_pick, pick);
            }
            w_before += all;
            __syncthreads();
            if (s_pick < INT_MAX) break;
        }
        if (tid == 0) *out = make_int2(0, s_pick < INT_MAX ? s_pick : s_last);
        return;
    }

    // ---- the k best
    uint32_t others[kCtas];
#pragma unroll
    for (int c = 0; c < kCtas; ++c) others[c] = *cluster.map_shared_rank(&thread_best[tid], c);
    uint32_t low = others[0];
#pragma unroll
    for (int c = 1; c < kCtas; ++c) low = min(low, others[c]);
    low = __reduce_min_sync(0xffffffffu, low);
    if (wl == 0) warp_low[warp] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) low = min(low, warp_low[w]);
    // low: at least k threads' best reach it (at first: all); twice, 256 steps between it and the next bound
    uint32_t high = (uint32_t)(best >> 32);
    int wanted = k;
    for (int round = 0; round < 2; ++round) {
        const int bits = max(0, 24 - __clz(high - low));   // the range is less than 256 steps of 2^bits
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kCtas; ++c)
            if (others[c] >= low && others[c] <= high) atomicAdd(&hist[(others[c] - low) >> bits], 1);
        __syncthreads();
        if (warp == 0) {   // a lane has eight steps, the first lane the highest
            int c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += c[j] = hist[255 - wl * 8 - j];
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, incl, o);
                if (wl >= o) incl += other;
            }
            int over = incl - sum;   // threads above the lane's steps
            if (over < wanted && incl >= wanted) {
                int at = 255 - wl * 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (over + c[j] >= wanted) break;
                    over += c[j];
                    --at;
                }
                s_step = make_int2(at, over);
            }
        }
        __syncthreads();
        const int2 step = s_step;
        wanted -= step.y;
        low += (uint32_t)step.x << bits;
        high = min(high, low + ((1u << bits) - 1u));
        if (bits == 0) break;
        __syncthreads();
    }
    // tokens that reach a bound, listed by their places; at least k reach `enough`, fewer reach `few`
    uint64_t enough = (uint64_t)low << 32, few = best + 1, bound = enough;
    int n_all, turn = 0;
    for (;; ++turn) {
        const uint32_t bound_value = (uint32_t)(bound >> 32);
        for (int v = tid; v < vecs; v += kThreads) {
            float f[EPV];
            unpack(buf[v], f, static_cast<const T*>(nullptr));
#pragma unroll
            for (int j = 0; j < EPV; ++j) {
                if (f32_order_key(f[j] + 0.0f) < bound_value) continue;
                const int t = token0 + v * EPV + j;
                if (key_of(f[j], t) < bound || t < n0 || t >= n0 + n) continue;
                const int at = atomicAdd(&s_count, 1);
                if (at < kCandidates) list[at] = (uint16_t)(v * EPV + j);
            }
        }
        __syncthreads();
        if (tid < kCtas) *cluster.map_shared_rank(&count_of[turn & 1][rank], tid) = s_count;
        cluster.sync();
        n_all = 0;
#pragma unroll
        for (int c = 0; c < kCtas; ++c) n_all += count_of[turn & 1][c];
        if (n_all >= k && n_all <= kCandidates) break;
        if (n_all >= k) enough = bound;
        else few = bound;
        bound = enough + (few - enough) / 2;   // keys differ, and kCandidates > k: it ends
        if (tid == 0) s_count = 0;
        __syncthreads();
    }
    static_assert(kCandidates > kVerifyMaxTopK && kCandidates % kThreads == 0, "more can be sorted than are wanted");
    // they meet where the first CTA had its tokens
    const int mine_n = count_of[turn & 1][rank];
    int first = 0;
    for (int c = 0; c < rank; ++c) first += count_of[turn & 1][c];
    uint64_t found[kCandidates / kThreads];
#pragma unroll
    for (int c = 0; c < kCandidates / kThreads; ++c)
        if (tid + c * kThreads < mine_n) {
            const int at = list[tid + c * kThreads];
            found[c] = key_of(value_of(reinterpret_cast<const T*>(smem)[at]), token0 + at);
        }
    cluster.sync();
    uint64_t* keys = reinterpret_cast<uint64_t*>(smem);
    uint64_t* there = cluster.map_shared_rank(keys, 0);
#pragma unroll
    for (int c = 0; c < kCandidates / kThreads; ++c)
        if (tid + c * kThreads < mine_n) there[first + tid + c * kThreads] = found[c];
    cluster.sync();
    if (rank != 0) return;
    const double* shares;   // of the kept candidates in the order of tokens, and those
    const int* tokens;
    double* values = reinterpret_cast<double*>(keys + kCandidates);
    int* ids = reinterpret_cast<int*>(values + kThreads);
    int n_last;
    if (n_all <= kThreads) {
        // A candidate a thread, which counts those before it in either order.
        const uint64_t key = tid < n_all ? keys[tid] : 0;
        int rank_by_value = 0, rank_by_token = 0;
        if (warp * 32 < n_all) {
            if (tid < 2) keys[n_all + tid] = 0;
        }
        __syncthreads();
        if (warp * 32 < n_all)
            for (int j = 0; j < n_all; j += 2) {
                const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(keys + j);
                rank_by_value += (int)(other.x > key) + (int)(other.y > key);
                rank_by_token += (int)((uint32_t)other.x > (uint32_t)key) + (int)((uint32_t)other.y > (uint32_t)key);
            }
        const bool among = tid < n_all && rank_by_value < k;
        const double e = among ? exp(((double)value_of_key(key) - (double)top) * per_t) : 0.0;
        bool in = among;
        double kept;
        if (top_p < 1.f) {
            values[tid] = 0.0;
            __syncthreads();
            if (among) values[rank_by_value] = e;
            __syncthreads();
            const double mine_e = values[tid];
            double z;
            const double upto = block_scan(mine_e, red, &z);
            values[tid] = upto - mine_e;
            __syncthreads();
            in = among && (rank_by_value == 0 || values[rank_by_value] / z < (double)top_p);
            __syncthreads();
        }
        const double e_in = in ? e : 0.0;
        block_scan(e_in, red, &kept);
        const int token = (int)rank_key_index(key);
        if (in && token == d) s_pd = e / kept;
        values[tid] = 0.0;
        __syncthreads();
        if (d >= 0 && kept_below < s_pd) {
            if (tid == 0) *out = make_int2(1, -1);
            return;
        }
        if (tid < n_all) {
            values[rank_by_token] = e_in / kept;
            ids[rank_by_token] = token;
        }
        __syncthreads();
        shares = values;
        tokens = ids;
        n_last = n_all;
    } else {
        // two candidates a thread: the head that adds up to top_p
        sort_desc(keys, n_all);
        const int j0 = 2 * tid;
        int token[2];
        double e[2], z, kept;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            token[j] = j0 + j < k ? (int)rank_key_index(keys[j0 + j]) : -1;
            e[j] = j0 + j < k ? exp(((double)value_of_key(keys[j0 + j]) - (double)top) * per_t) : 0.0;
        }
        const double upto_e = block_scan(e[0] + e[1], red, &z);
        bool in[2] = {j0 < k, j0 + 1 < k};
        if (top_p < 1.f) {
            in[0] = in[0] && (j0 == 0 || (upto_e - e[1] - e[0]) / z < (double)top_p);
            in[1] = in[1] && (upto_e - e[1]) / z < (double)top_p;
        }
        block_scan((in[0] ? e[0] : 0.0) + (in[1] ? e[1] : 0.0), red, &kept);
        double* weights = reinterpret_cast<double*>(keys + kVerifyMaxTopK);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (in[j] && token[j] == d) s_pd = e[j] / kept;
            weights[j0 + j] = in[j] ? e[j] / kept : 0.0;
            keys[j0 + j] = j0 + j < k ? (uint64_t)(0xFFFFFFFFu - (uint32_t)token[j]) << 32 | (uint32_t)(j0 + j) : 0;
        }
        __syncthreads();
        if (d >= 0 && kept_below < s_pd) {
            if (tid == 0) *out = make_int2(1, -1);
            return;
        }
        sort_desc(keys, k);   // by token; at most kVerifyMaxTopK, the weights lie behind
        double w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint64_t key = j0 + j < k ? keys[j0 + j] : 0;
            token[j] = (int)(0xFFFFFFFFu - (uint32_t)(key >> 32));
            w[j] = j0 + j < k ? weights[(uint32_t)key] : 0.0;
        }
        __syncthreads();
        ids = reinterpret_cast<int*>(keys);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            weights[j0 + j] = w[j];
            ids[j0 + j] = token[j];
        }
        __syncthreads();
        shares = weights;
        tokens = ids;
        n_last = k;
    }
    // the draw, two tokens a thread
    const int j0 = 2 * tid;
    int token[2];
    double p[2], r[2], total;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        token[j] = j0 + j < n_last ? tokens[j0 + j] : -1;
        p[j] = r[j] = j0 + j < n_last ? shares[j0 + j] : 0.0;
        if (d >= 0 && p[j] > 0.0) r[j] = fmax(p[j] - (q != nullptr ? (double)q[token[j]] : (token[j] == d ? 1.0 : 0.0)), 0.0);
    }
    double upto = block_scan(r[0] + r[1], red, &total);
    if (!(total > 0.0)) {   // the draft's distribution covers the target's
        r[0] = p[0];
        r[1] = p[1];
        upto = block_scan(r[0] + r[1], red, &total);
    }
    const double target = u_draw * total;
    if (r[0] > 0.0) {
        if (upto - r[1] > target) atomicMin(&s_pick, token[0]);
        atomicMax(&s_last, token[0]);
    }
    if (r[1] > 0.0) {
        if (upto > target) atomicMin(&s_pick, token[1]);
        atomicMax(&s_last, token[1]);
    }
    __syncthreads();
    if (tid == 0) *out = make_int2(0, s_pick < INT_MAX ? s_pick : s_last);
}

__global__ void __launch_bounds__(128) verify_lanes_kernel(const __grid_constant__ VerifyArgs a) {
    const int lane = blockIdx.x * 4 + (threadIdx.x >> 5), t = threadIdx.x & 31, n = a.n_drafts;
    pdl_wait();
    if (lane >= a.lanes) return;
    const int32_t* drafts = a.drafts + (int64_t)lane * n;
    const int2* rows = a.rows + (int64_t)lane * (n + 1);
    int32_t* tokens = a.tokens + (int64_t)lane * (n + 1);
    int end = 0;   // the lane's first row that ends it
    for (;; ++end)
        if (end == n || drafts[end] < 0 || drafts[end] >= a.vocab || rows[end].x == 0) break;
    for (int i = t; i <= n; i += 32) tokens[i] = i < end ? drafts[i] : (i == end ? rows[end].y : -1);
    if (t == 0) a.accepted[lane] = end;
}

}  // namespace

void launch_verify_drafts(VerifyArgs a, cudaStream_t s) {
    if (a.lanes <= 0) return;
    const int size = a.type == 0 ? 4 : 2, chunk = ((a.vocab + kCtas - 1) / kCtas + 7) / 8 * 8;
    a.list_at = std::max(chunk * size + 32, kCandidates * 8 + kThreads * 12);   // where candidates meet
    const size_t smem = (size_t)a.list_at + kCandidates * 2;
    auto* kernel = a.type == 0 ? verify_rows_kernel<float> : (a.type == 1 ? verify_rows_kernel<__half> : verify_rows_kernel<__nv_bfloat16>);
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    kernel<<<(unsigned)(a.lanes * (a.n_drafts + 1) * kCtas), kThreads, smem, s>>>(a, chunk);
    MK_LAUNCH_CHECK();
    launch_pdl(verify_lanes_kernel, dim3((unsigned)((a.lanes + 3) / 4)), dim3(128), 0, s, a);
}

}  // namespace mk
