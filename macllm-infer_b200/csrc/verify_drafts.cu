// Verification of drafted tokens against the target's distribution, from given random numbers.
//
// Row i of a lane holds the target's logits behind its first i drafts.  p_i = softmax(logits / temperature) over the top_k best tokens, of those the head
// that adds up to top_p (the sampler's rule); temperature 0: all on the best token.  q_i is the distribution that draft d_i came from.  Draft i is kept
// while u_i q_i(d_i) < p_i(d_i); the first that is not is replaced by a draw from max(p_i - q_i, 0), and behind the last draft one more token is drawn from
// p.  The tokens are then distributed as if drawn from the target one by one: q min(1, p / q) + (1 - sum q min(1, p / q)) max(p - q, 0) / sum max(p - q, 0) = p.
// A draw takes the first token, in the order of tokens, whose cumulative weight exceeds u_n times the whole.
//
// Every row is judged by itself, and a second kernel takes a lane's first row that ends it.  Sums and weights of candidates are 64-bit.
#include "verify_drafts.h"
#include "sampling_math.h"
#include "shared_attention.h"
#include <cuda_bf16.h>

namespace mk {

namespace {

constexpr int kThreads = 1024;

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
// Larger first, the lower token first among equals; -0 counts as 0.
__device__ __forceinline__ uint64_t key_of(float x, int i) { return rank_key(x + 0.0f, (uint32_t)i); }
__device__ __forceinline__ float value_of_key(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return bits_f32((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
}

// Inclusive sums over the block's threads; *total: of all.
__device__ double block_scan(double v, double* red, double* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) red[w] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int i = 0; i < nw; ++i) {
        if (i < w) before += red[i];
        all += red[i];
    }
    *total = all;
    return before + v;
}

__device__ void sort_desc(uint64_t* a) {
    for (int size = 2; size <= kThreads; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            __syncthreads();
            const int tid = threadIdx.x, partner = tid ^ stride;
            if (partner > tid) {
                const uint64_t x = a[tid], y = a[partner];
                if ((x < y) == ((tid & size) == 0)) a[tid] = y, a[partner] = x;
            }
        }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ uint64_t keys[kThreads];
    __shared__ double weight[kThreads], red[32];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_prefix, s_need, s_count;
    __shared__ int s_pick, s_last;
    __shared__ double s_pd;
    const int tid = threadIdx.x, lane = blockIdx.x / (a.n_drafts + 1), i = blockIdx.x - lane * (a.n_drafts + 1), vocab = a.vocab;
    const int32_t* drafts = a.drafts + (int64_t)lane * a.n_drafts;
    for (int j = 0; j < i; ++j)
        if (drafts[j] < 0 || drafts[j] >= vocab) return;   // nothing gets here
    int d = i < a.n_drafts ? drafts[i] : -1;
    if (d >= vocab) {
        if (tid == 0) tell(a.status, kDevBadRange);
        d = -1;
    }
    const T* x = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
    const float temperature = a.temperature[lane];
    int2* out = a.rows + blockIdx.x;

    uint64_t best = 0;
    bool bad = false;
    for (int j = tid; j < vocab; j += kThreads) {
        const float v = value_of(x[j]);
        bad |= !(v < INFINITY);
        const uint64_t k = key_of(v, j);
        best = k > best ? k : best;
    }
    bad = __syncthreads_or(bad);
    keys[tid] = best;
    __syncthreads();
    for (int s = kThreads / 2; s > 0; s >>= 1) {
        if (tid < s && keys[tid + s] > keys[tid]) keys[tid] = keys[tid + s];
        __syncthreads();
    }
    best = keys[0];
    __syncthreads();
    const float top = value_of_key(best);
    if (bad || top == -INFINITY) {
        if (tid == 0) {
            tell(a.status, kDevBadRow);
            *out = make_int2(0, -1);
        }
        return;
    }
    if (!(temperature > 0.f)) {
        if (tid == 0) *out = make_int2(d == (int)rank_key_index(best), (int)rank_key_index(best));
        return;
    }
    int k = a.top_k[lane];
    float top_p = a.top_p[lane];
    if (k > kVerifyMaxTopK || (k <= 0 && top_p < 1.f)) {
        if (tid == 0) tell(a.status, kDevBadRange);
        k = min(k, kVerifyMaxTopK);
    }
    k = min(k, vocab);
    const double per_t = 1.0 / (double)temperature;
    const float* q = a.draft_probs == nullptr || d < 0 ? nullptr : a.draft_probs + ((int64_t)lane * a.n_drafts + i) * vocab;
    const double u_keep = d >= 0 ? (double)a.u[(int64_t)lane * (a.n_drafts + 1) + i] : 0.0, u_draw = (double)a.u[(int64_t)lane * (a.n_drafts + 1) + a.n_drafts];
    const double qd = q != nullptr ? (double)q[d] : 1.0;
    if (tid == 0) s_pick = INT_MAX, s_last = -1, s_pd = 0.0;
    __syncthreads();
    auto q_at = [&](int t) { return d < 0 ? 0.0 : (q != nullptr ? (double)q[t] : (t == d ? 1.0 : 0.0)); };

    if (k <= 0) {
        // the whole vocabulary, a run of tokens per thread
        const int per = (vocab + kThreads - 1) / kThreads, lo = min(vocab, tid * per), hi = min(vocab, lo + per);
        auto weight_of = [&](int t) { return exp(((double)value_of(x[t]) - (double)top) * per_t); };
        double mine = 0.0, z, total;
        for (int t = lo; t < hi; ++t) mine += weight_of(t);
        block_scan(mine, red, &z);
        const double pd = d >= 0 ? weight_of(d) / z : 0.0;
        if (d >= 0 && u_keep * qd < pd) {
            if (tid == 0) *out = make_int2(1, -1);
            return;
        }
        bool rest = d >= 0;
        auto share_of = [&](int t) {
            const double p = weight_of(t) / z;
            return rest ? fmax(p - q_at(t), 0.0) : p;
        };
        mine = 0.0;
        for (int t = lo; t < hi; ++t) mine += share_of(t);
        double upto = block_scan(mine, red, &total);
        if (!(total > 0.0)) {   // the draft's distribution covers the target's
            rest = false;
            mine = 0.0;
            for (int t = lo; t < hi; ++t) mine += share_of(t);
            upto = block_scan(mine, red, &total);
        }
        const double target = u_draw * total;
        double c = upto - mine;
        int last = -1;
        for (int t = lo; t < hi; ++t) {
            const double r = share_of(t);
            c += r;
            if (r > 0.0) last = t;
            if (r > 0.0 && c > target) {
                atomicMin(&s_pick, t);
                break;
            }
        }
        atomicMax(&s_last, last);
        __syncthreads();
        if (tid == 0) *out = make_int2(0, s_pick < INT_MAX ? s_pick : s_last);
        return;
    }
    // the value of the k-th best token, eight bits at a time
    uint32_t prefix = 0, mask = 0, need = (uint32_t)k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < vocab; j += kThreads) {
            const uint32_t key = (uint32_t)(key_of(value_of(x[j]), j) >> 32);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t acc = 0;
            int b = 255;
            for (; b > 0 && acc + hist[b] < need; --b) acc += hist[b];
            s_prefix = prefix | (uint32_t)b << shift;
            s_need = need - acc;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        mask |= 255u << shift;
        __syncthreads();
    }
    if (tid == 0) s_count = 0;
    keys[tid] = 0;
    __syncthreads();
    const int per = (vocab + kThreads - 1) / kThreads, lo = min(vocab, tid * per), hi = min(vocab, lo + per);
    int equals = 0;
    for (int j = lo; j < hi; ++j) {
        const uint64_t key = key_of(value_of(x[j]), j);
        if ((uint32_t)(key >> 32) > prefix) keys[atomicAdd(&s_count, 1u)] = key;
        else if ((uint32_t)(key >> 32) == prefix) ++equals;
    }
    double all;
    int rank = (int)block_scan((double)equals, red, &all) - equals;
    for (int j = lo; j < hi && equals > 0 && rank < (int)need; ++j) {
        const uint64_t key = key_of(value_of(x[j]), j);
        if ((uint32_t)(key >> 32) == prefix) keys[k - (int)need + rank++] = key;
    }
    sort_desc(keys);
    // the head that adds up to top_p
    double e = tid < k ? exp(((double)value_of_key(keys[tid]) - (double)top) * per_t) : 0.0, z, kept;
    const double upto_e = block_scan(e, red, &z);
    if (tid > 0 && !((upto_e - e) / z < (double)top_p) && top_p < 1.f) e = 0.0;
    block_scan(e, red, &kept);
    const int token = tid < k ? (int)rank_key_index(keys[tid]) : -1;
    if (tid < k && token == d) s_pd = e / kept;
    weight[tid] = e / kept;
    __syncthreads();
    if (d >= 0 && u_keep * qd < s_pd) {
        if (tid == 0) *out = make_int2(1, -1);
        return;
    }
    // the draw, in the order of tokens
    keys[tid] = tid < k ? (uint64_t)(0xFFFFFFFFu - (uint32_t)token) << 32 | (uint32_t)tid : 0;
    sort_desc(keys);
    const int t = tid < k ? (int)(0xFFFFFFFFu - (uint32_t)(keys[tid] >> 32)) : -1;
    const double p = tid < k ? weight[(uint32_t)keys[tid]] : 0.0;
    double r = d >= 0 && p > 0.0 ? fmax(p - q_at(t), 0.0) : p, total;
    double upto = block_scan(r, red, &total);
    if (!(total > 0.0)) {
        r = p;
        upto = block_scan(r, red, &total);
    }
    if (r > 0.0) {
        if (upto > u_draw * total) atomicMin(&s_pick, t);
        atomicMax(&s_last, t);
    }
    __syncthreads();
    if (tid == 0) *out = make_int2(0, s_pick < INT_MAX ? s_pick : s_last);
}

__global__ void __launch_bounds__(128) verify_lanes_kernel(const __grid_constant__ VerifyArgs a) {
    const int lane = blockIdx.x * 4 + (threadIdx.x >> 5), t = threadIdx.x & 31, n = a.n_drafts;
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

void launch_verify_drafts(const VerifyArgs& a, cudaStream_t s) {
    if (a.lanes <= 0) return;
    auto* kernel = a.type == 0 ? verify_rows_kernel<float> : (a.type == 1 ? verify_rows_kernel<__half> : verify_rows_kernel<__nv_bfloat16>);
    kernel<<<(unsigned)(a.lanes * (a.n_drafts + 1)), kThreads, 0, s>>>(a);
    MK_LAUNCH_CHECK();
    verify_lanes_kernel<<<(unsigned)((a.lanes + 3) / 4), 128, 0, s>>>(a);
    MK_LAUNCH_CHECK();
}

}  // namespace mk
