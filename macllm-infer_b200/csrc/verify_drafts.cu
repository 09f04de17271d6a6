// Verification of drafted tokens against the target's distribution, from given random numbers.
//
// Row i of a lane holds the target's logits behind its first i drafts.  p_i = softmax(logits / temperature) over the top_k best tokens, of those the head
// that adds up to top_p (the sampler's rule); temperature 0: all on the best token.  q_i is the distribution that draft d_i came from.  Draft i is kept
// while u_i q_i(d_i) < p_i(d_i); the first that is not is replaced by a draw from max(p_i - q_i, 0), and behind the last draft one more token is drawn from
// p.  The tokens are then distributed as if drawn from the target one by one: q min(1, p / q) + (1 - sum q min(1, p / q)) max(p - q, 0) / sum max(p - q, 0) = p.
// A draw takes the first token, in the order of tokens, whose cumulative weight exceeds u_n times the whole.
//
// Two kernels.  The first streams every row that can be reached once, a run of tokens to a CTA and at most 32 of them to a thread, and leaves what a run amounts
// to: its best token, whether it holds what is no logit, the sum of its weights (whole vocabulary), and the best value of each thread's tokens (top_k).  What bounds it is HBM.
// The second finishes lanes, a cluster of eight CTAs to each, or fewer where there are many lanes.  Over the whole vocabulary a row's sum follows from its runs', which tells where the lane ends, and
// the cluster goes through that one row again, for the draw.  With a top_k they share out the rows: the k-th best of the threads' best values is a bound that at
// least k tokens reach and few more do, and only the tokens of threads that reach it are read again; where too many reach it (thousands of equal
// logits) bisection over (value, token) finds one that fewer do.
//
// Weights and sums of candidates are 64-bit.  Over the whole vocabulary a weight is a 32-bit number (ex2 of a product kept to twice 32 bits: 2^-22, and with no trend, so that
// sums over many are better) and sums are 64-bit; where a draw's target or remainder is so small that what 32 bits leave out may decide, its weights are 64-bit too.
#include "verify_drafts.h"
#include "sampling_math.h"
#include "shared_attention.h"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <algorithm>

namespace mk {

namespace {

namespace cg = cooperative_groups;

constexpr int kMostCtas = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kScan = 256;          // threads of the first kernel's CTAs
constexpr int kCandidates = 2048;   // sorted at once
// Candidates that are compared with one another, by four threads each; more are sorted (4 lanes with 4 drafts of 128256 in f16: 15.1 us and 21.2 sorted at top_k 40, 17.6 and 21.9 at
// 100; two threads each, for up to 256: 20.1 and 22.4 at 128, 23.5 and 23.0 at 200, and slower below).
constexpr int kCounted = 128;

struct Run {
    uint64_t best;   // key of its best token
    double sum;      // of the weights against that one, where the whole vocabulary counts
    int bad, pad_;
};

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void load4(const float* x, float (&v)[4]) {
    const float4 r = *reinterpret_cast<const float4*>(x);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
}
__device__ __forceinline__ void load4(const __half* x, float (&v)[4]) {
    const uint2 r = *reinterpret_cast<const uint2*>(x);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* x, float (&v)[4]) {
    const uint2 r = *reinterpret_cast<const uint2*>(x);
    v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xFFFF0000u); v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xFFFF0000u);
}
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
// What the block's threads before this one add up to, which no larger number is taken from again; *total: of all.
__device__ double block_before(double v, double* red, double* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    v = warp_scan(v, lane);
    const double others = __shfl_up_sync(0xffffffffu, v, 1);
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
    return lane > 0 ? before + others : before;
}

// 512 E keys, the larger first: a thread has E neighbours, so that most exchanges of the bitonic network are inside a thread or a warp.
template <int E, typename K>
__device__ void sort_desc(K* keys) {
    const int tid = threadIdx.x;
    K a[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = keys[tid * E + e];
    for (int size = 2; size <= kThreads * E; size <<= 1) {
        auto exchange = [&](int stride, auto&& partner) {
            K y[E];
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
template <typename K>
__device__ void sort_desc(K* keys, int n) {   // keys behind n are there to be filled up
    const int size = n <= kThreads ? kThreads : (n <= 2 * kThreads ? 2 * kThreads : 4 * kThreads);
    for (int j = n + (int)threadIdx.x; j < size; j += kThreads) keys[j] = 0;
    __syncthreads();
    if (size == kThreads) sort_desc<1>(keys);
    else if (size == 2 * kThreads) sort_desc<2>(keys);
    else sort_desc<4>(keys);
}

// Two 32-bit numbers in one instruction.
struct Two {
    unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void apart(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
// The larger, or NaN where there is one.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// exp((x - top) / temperature) with 1 / (temperature ln 2) as the sum of two 32-bit numbers: t = y hi rounded, what it lost and y lo come behind as a factor.  What is below 2^-126 of the
// best counts as 0 (ex2 flushes what is no normal number), -inf too: y is not followed beyond 2^-160.
struct Exponential {
    float top, hi, lo, least;
    __device__ __forceinline__ Exponential(float best, float temperature) : top(best) {
        const double unit = 1.4426950408889634074 / (double)temperature;
        hi = (float)unit;
        lo = (float)(unit - (double)hi);
        least = -160.f / hi;
    }
    __device__ __forceinline__ void operator()(float& a, float& b) const {
        float u, v;
        apart(add2(two(a, b), two(-top, -top)), u, v);
        const Two y = two(fmaxf(u, least), fmaxf(v, least)), minus_t = mul2(y, two(-hi, -hi)), lost = fma2(y, two(lo, lo), fma2(y, two(hi, hi), minus_t));
        apart(minus_t, u, v);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(u) : "f"(-u));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(-v));
        const Two e = two(u, v);
        apart(fma2(e, mul2(lost, two(0.69314718f, 0.69314718f)), e), a, b);
    }
};

// Piece v of a row, 16 bytes counted from the last boundary at or before its first value; places outside the row hold -inf.
template <typename T>
struct Row {
    static constexpr int EPV = 16 / (int)sizeof(T);
    const T* x;
    int vocab, shift;   // shift: values of the first piece that are in front of the row
    __device__ __forceinline__ Row(const T* row, int n) : x(row), vocab(n), shift((int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))) {}
    __device__ __forceinline__ int token(int v) const { return v * EPV - shift; }
    __device__ __forceinline__ void load(int v, float (&f)[EPV]) const {
        const int t0 = token(v);
        if (t0 >= 0 && t0 + EPV <= vocab) {
            unpack(*reinterpret_cast<const uint4*>(x + t0), f, static_cast<const T*>(nullptr));
        } else {
#pragma unroll
            for (int j = 0; j < EPV; ++j) f[j] = t0 + j >= 0 && t0 + j < vocab ? value_of(x[t0 + j]) : -INFINITY;
        }
    }
};

// What a warp knows of a row from its runs.
struct RowSum {
    uint64_t best;
    double z;
    bool bad;
};
__device__ __forceinline__ RowSum sum_runs(const Run* runs, int n, double unit, bool whole) {
    const int wl = threadIdx.x & 31;
    RowSum s{0, 0.0, false};
    for (int c = wl; c < n; c += 32) {
        s.best = runs[c].best > s.best ? runs[c].best : s.best;
        s.bad |= runs[c].bad != 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, s.best, o);
        s.best = other > s.best ? other : s.best;
    }
    const float top = value_of_key(s.best);
    s.bad = __any_sync(0xffffffffu, s.bad) || top == -INFINITY;
    if (whole && !s.bad) {
        for (int c = wl; c < n; c += 32) {
            const float own = value_of_key(runs[c].best);
            if (own > -INFINITY) s.z += runs[c].sum * exp(((double)own - (double)top) * unit);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
    }
    return s;
}

__device__ __forceinline__ bool is_draft(int d, int vocab) { return d >= 0 && d < vocab; }
// A lane's temperature: 0 where it is none or so low that only the best token is left, and not beyond what 32 bits turn into a factor.
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int lane) {
    const float t = a.temperature[lane];
    return t > 1e-30f ? fminf(t, 1e30f) : 0.f;
}

// 64 lanes with 4 drafts of 151936 in f32 (194 MB), whole vocabulary: 46 us, 4.2 TB/s, issue slots 61 % busy (a weight is 10 instructions for two tokens, its maximum, its sum); 16 tokens a thread
// are slower, since the ends of a CTA come twice as often.
template <typename T, int VPT>
__global__ void __launch_bounds__(kScan) scan_rows_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int EPV = 16 / (int)sizeof(T);
    __shared__ Run warp_runs[kScan / 32];
    const int tid = threadIdx.x, wl = tid & 31, warp = tid >> 5, index = blockIdx.x / a.runs, run = blockIdx.x - index * a.runs;
    const int lane = index / (a.n_drafts + 1), i = index - lane * (a.n_drafts + 1), vocab = a.vocab;
    pdl_trigger();
    const int32_t* drafts = a.drafts + (int64_t)lane * a.n_drafts;
    const float temperature = temperature_of(a, lane);
    const int k = a.top_k[lane];
    bool gone = false;
    for (int j = wl; j < i; j += 32) gone |= !is_draft(drafts[j], vocab);
    if (__any_sync(0xffffffffu, gone)) return;   // nothing gets here
    const Row<T> row(static_cast<const T*>(a.logits) + index * a.ld, vocab);
    float f[VPT][EPV];
#pragma unroll
    for (int c = 0; c < VPT; ++c) row.load((run * VPT + c) * kScan + tid, f[c]);
    float best_of[VPT];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        best_of[c] = f[c][0];
#pragma unroll
        for (int j = 1; j < EPV; ++j) best_of[c] = max_or_nan(best_of[c], f[c][j]);
    }
    float top = best_of[0];
#pragma unroll
    for (int c = 1; c < VPT; ++c) top = max_or_nan(top, best_of[c]);
    const bool bad = __any_sync(0xffffffffu, !(top < INFINITY));
    if (temperature > 0.f && k > 0) a.group_best[((int64_t)index * a.runs + run) * kScan + tid] = top;
    // warps by themselves, then the block's by one of them
    const uint32_t value = f32_order_key(top + 0.0f), warp_value = __reduce_max_sync(0xffffffffu, value);
    int at = vocab;   // which token it is: for greedy lanes
    if (!(temperature > 0.f) && value == warp_value && top > -INFINITY) {
#pragma unroll
        for (int c = VPT - 1; c >= 0; --c)
#pragma unroll
            for (int j = EPV - 1; j >= 0; --j)
                if (f[c][j] == top) at = row.token((run * VPT + c) * kScan + tid) + j;
    }
    if (!(temperature > 0.f)) at = __reduce_min_sync(0xffffffffu, at);
    Run r;
    r.best = (uint64_t)warp_value << 32 | (0xFFFFFFFFu - (uint32_t)at);
    r.sum = 0.0;
    const bool whole = temperature > 0.f && k <= 0;
    if (whole) {
        const Exponential weight(value_of_key(r.best), temperature);
#pragma unroll
        for (int c = 0; c < VPT; ++c)
#pragma unroll
            for (int j = 0; j < EPV; j += 4) {
                weight(f[c][j], f[c][j + 1]);
                weight(f[c][j + 2], f[c][j + 3]);
                r.sum += (double)((f[c][j] + f[c][j + 1]) + (f[c][j + 2] + f[c][j + 3]));
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
    }
    r.bad = bad;
    r.pad_ = 0;
    if (wl == 0) warp_runs[warp] = r;
    __syncthreads();
    if (warp != 0) return;
    const RowSum s = sum_runs(warp_runs, kScan / 32, whole ? 1.0 / (double)temperature : 0.0, whole);
    if (wl == 0) {
        r.best = s.best;
        r.sum = s.z;
        r.bad = s.bad && value_of_key(s.best) > -INFINITY;   // a run of nothing is no fault of the row's
        for (int w = 0; w < kScan / 32; ++w) r.bad |= warp_runs[w].bad;
        static_cast<Run*>(a.run_results)[(int64_t)index * a.runs + run] = r;
    }
}

__device__ __forceinline__ void put_lane(const VerifyArgs& a, int lane, int end, int token) {   // a warp
    for (int j = threadIdx.x & 31; j <= a.n_drafts; j += 32)
        a.tokens[(int64_t)lane * (a.n_drafts + 1) + j] = j < end ? a.drafts[(int64_t)lane * a.n_drafts + j] : (j == end ? token : -1);
    if ((threadIdx.x & 31) == 0) a.accepted[lane] = end;
}

// Places in a list, n of them one after the other for each thread of a warp.
__device__ __forceinline__ int list_places(int* count, int n) {
    const int wl = threadIdx.x & 31;
    int upto = n, at = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, o);
        if (wl >= o) upto += other;
    }
    if (wl == 31 && upto > 0) at = atomicAdd(count, upto);
    return __shfl_sync(0xffffffffu, at, 31) + upto - n;
}
// Sum over the block, the same in every thread.
__device__ unsigned long long block_sum(unsigned long long v, unsigned long long* red) {
    const int wl = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (wl == 0) red[warp] = v;
    __syncthreads();
    v = red[wl % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct TopShared {
    double red[kWarps], pd;
    uint64_t best;
    float warp_low[kWarps];
    int warp_live[kWarps];
    int count, groups, pick, last, bad, hist[256];
    int2 step;
};

// One row with a top_k, by a CTA: (draft kept, token drawn in its place; -1 where the row is no distribution).
template <typename T>
__device__ int2 finish_top_row(const VerifyArgs& a, TopShared& s, uint8_t* smem, int lane, int i, int d, int k, float temperature, float top_p, double u_keep, double u_draw) {
    constexpr int EPV = Row<T>::EPV;
    const int tid = threadIdx.x, warp = tid >> 5, wl = tid & 31, vocab = a.vocab, index = lane * (a.n_drafts + 1) + i, n_groups = a.runs * kScan, vpt = a.vpt;
    const double per_t = 1.0 / (double)temperature;
    const Row<T> row(static_cast<const T*>(a.logits) + index * a.ld, vocab);
    const float* q = a.draft_probs == nullptr || d < 0 ? nullptr : a.draft_probs + ((int64_t)lane * a.n_drafts + i) * vocab;
    const double kept_below = d >= 0 ? u_keep * (q != nullptr ? (double)q[d] : 1.0) : 0.0;
    float* group_best = reinterpret_cast<float*>(smem);
    uint16_t* group_list = reinterpret_cast<uint16_t*>(smem + a.list_at);
    uint64_t* keys = reinterpret_cast<uint64_t*>(smem + a.keys_at);
    __syncthreads();   // the row before is done with
    if (tid == 0) {
        s.count = s.groups = 0;
        s.pick = INT_MAX;
        s.last = -1;
        s.pd = 0.0;
    }
    if (tid < 256) s.hist[tid] = 0;
    if (warp == 0) {
        const RowSum r = sum_runs(static_cast<const Run*>(a.run_results) + (int64_t)index * a.runs, a.runs, per_t, false);
        if (wl == 0) {
            s.best = r.best;
            s.bad = r.bad;
            s.step = make_int2(-1, 0);
        }
    }
    float low = INFINITY;
    for (int j = tid; j < n_groups; j += kThreads) {
        const float b = a.group_best[(int64_t)index * n_groups + j];
        group_best[j] = b;
        if (b > -INFINITY) low = fminf(low, b);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    if (wl == 0) s.warp_low[warp] = low;
    __syncthreads();
    if (s.bad) return make_int2(0, -1);   // told of where the lane gets here
    const uint64_t best = s.best;
    const float top = value_of_key(best);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) low = fminf(low, s.warp_low[w]);
    // 256 steps of value between the groups' lowest and highest; the highest step with which at least k groups' best are counted.  Its lower end, moved down by more than
    // the roundings on the way, is a bound that at least k tokens reach.
    const float range = top - low, per_step = range > 0.f && range < INFINITY ? 256.f / range : 0.f;
    for (int j = tid; j < n_groups; j += kThreads) {
        const float b = group_best[j];
        if (b > -INFINITY) atomicAdd(&s.hist[min(255, (int)((b - low) * per_step))], 1);
    }
    __syncthreads();
    if (warp == 0) {   // a lane has eight steps, the first lane the highest
        int c[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += c[j] = s.hist[255 - wl * 8 - j];
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, incl, o);
            if (wl >= o) incl += other;
        }
        int over = incl - sum;   // groups above the lane's steps
        if (over < k && incl >= k) {
            int step = 255 - wl * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                over += c[j];
                if (over >= k) break;
                --step;
            }
            s.step = make_int2(step, over);
        }
    }
    __syncthreads();
    // tokens that reach a bound; at least k reach `enough`, fewer reach `few`
    const float bound_low = s.step.x < 0 || per_step == 0.f ? (s.step.x < 0 ? -INFINITY : low) : low + (float)s.step.x / per_step - range * 1e-5f;
    uint64_t enough = (uint64_t)f32_order_key(bound_low + 0.0f) << 32, few = (best | 0xFFFFFFFFu) + 1, bound = enough;
    int n_all;
    for (;;) {
        const float bound_value = value_of_key(bound);
        for (int j0 = tid; j0 - tid < n_groups; j0 += 32 * kThreads) {
            unsigned mine = 0;
            for (int b = 0; b < 32 && j0 + b * kThreads < n_groups; ++b)
                if (group_best[j0 + b * kThreads] >= bound_value) mine |= 1u << b;
            int at = list_places(&s.groups, __popc(mine));
            for (; mine != 0; mine &= mine - 1) group_list[at++] = (uint16_t)(j0 + (__ffs(mine) - 1) * kThreads);
        }
        __syncthreads();
        // their tokens, two pieces on their way to a thread (a place for each token by itself: twice the time)
        const int pieces = s.groups * vpt;
        for (int w0 = 0; w0 < pieces; w0 += 2 * kThreads) {
            float f[2][EPV];
            int t0[2] = {INT_MIN / 2, INT_MIN / 2};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int w = w0 + h * kThreads + tid;
#pragma unroll
                for (int j = 0; j < EPV; ++j) f[h][j] = -INFINITY;
                if (w < pieces) {
                    const int g = group_list[w / vpt], v = (g / kScan * vpt + w % vpt) * kScan + g % kScan;
                    t0[h] = row.token(v);
                    row.load(v, f[h]);
                }
            }
            unsigned mine = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < EPV; ++j)
                    if (t0[h] + j >= 0 && t0[h] + j < vocab && key_of(f[h][j], t0[h] + j) >= bound) mine |= 1u << (h * EPV + j);
            if (!__any_sync(0xffffffffu, mine != 0)) continue;
            int at = list_places(&s.count, __popc(mine));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < EPV; ++j)
                    if (mine >> (h * EPV + j) & 1) {
                        if (at < kCandidates) keys[at] = key_of(f[h][j], t0[h] + j);
                        ++at;
                    }
        }
        __syncthreads();
        n_all = s.count;
        if (n_all >= k && n_all <= kCandidates) break;
        if (n_all >= k) enough = bound;
        else few = bound;
        bound = enough + (few - enough) / 2;   // keys differ, and kCandidates > k: it ends
        __syncthreads();
        if (tid == 0) s.count = s.groups = 0;
        __syncthreads();
    }
    static_assert(kCandidates > kVerifyMaxTopK, "more can be sorted than are wanted");
    if (n_all <= kCounted) {
        // Four threads to a candidate, which compare it with every other one: who is better, and how much those weigh; later whose token is lower.  The list's order is not
        // the same in every call, so sums are of whole numbers of 2^-52.  Where the target is less than 2^-40 (u = 0, or a remainder of next to nothing) what is below a unit may decide:
        // then candidates are sorted, and their shares are 64-bit numbers.
        unsigned long long* values = reinterpret_cast<unsigned long long*>(keys + kCandidates);
        constexpr double kUnits = 0x1p52, kLeastUnits = 0x1p12;
        constexpr int parts = kThreads / kCounted;
        const int c = tid / parts, part = tid % parts;
        const uint64_t key = c < n_all ? keys[c] : 0;
        const int token = c < n_all ? (int)rank_key_index(key) : -1;
        const double e = c < n_all ? exp(((double)value_of_key(key) - (double)top) * per_t) : 0.0;
        const double qt = d >= 0 && c < n_all ? (q != nullptr ? (double)q[token] : (token == d ? 1.0 : 0.0)) : 0.0;
        const unsigned long long units = __double2ull_rn(e * kUnits);
        if (part == 0) values[c] = units;
        __syncthreads();
        int better = 0;
        unsigned long long before = 0;
        for (int j = part; j < n_all; j += parts)
            if (keys[j] > key) {
                ++better;
                before += values[j];
            }
        for (int o = 1; o < parts; o <<= 1) {
            better += __shfl_xor_sync(0xffffffffu, better, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        bool in = c < n_all && better < k;
        unsigned long long kept = block_sum(in && part == 0 ? units : 0ull, reinterpret_cast<unsigned long long*>(s.red));
        if (top_p < 1.f) {
            in = in && (better == 0 || (double)before < (double)top_p * (double)kept);
            kept = block_sum(in && part == 0 ? units : 0ull, reinterpret_cast<unsigned long long*>(s.red));
        }
        const double p = in ? e * (kUnits / (double)kept) : 0.0;
        if (in && token == d) s.pd = p;
        const unsigned long long r = __double2ull_rn((d >= 0 && in ? fmax(p - qt, 0.0) : p) * kUnits);
        if (part == 0) values[c] = r;
        __syncthreads();
        if (d >= 0 && kept_below < s.pd) return make_int2(1, -1);
        const unsigned long long total = block_sum(part == 0 ? r : 0ull, reinterpret_cast<unsigned long long*>(s.red));
        if (u_draw * (double)total >= kLeastUnits) {
            unsigned long long upto = 0;
            for (int j = part; j < n_all; j += parts)
                if ((uint32_t)keys[j] >= (uint32_t)key) upto += values[j];   // its token, or a lower one
            for (int o = 1; o < parts; o <<= 1) upto += __shfl_xor_sync(0xffffffffu, upto, o);
            if (r > 0 && part == 0) {
                if ((double)upto > u_draw * (double)total) atomicMin(&s.pick, token);
                atomicMax(&s.last, token);
            }
            __syncthreads();
            return make_int2(0, s.pick < INT_MAX ? s.pick : s.last);
        }
    }
    // More, or a draw that such units are too coarse for: sorted, two candidates a thread from then on.
    const double* shares;
    const int* tokens;
    int n_last;
    {
        int* ids;
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
        const double before_e = block_before(e[0] + e[1], s.red, &z);
        bool in[2] = {j0 < k, j0 + 1 < k};
        if (top_p < 1.f) {
            in[0] = in[0] && (j0 == 0 || before_e / z < (double)top_p);
            in[1] = in[1] && (before_e + e[0]) / z < (double)top_p;
        }
        block_before((in[0] ? e[0] : 0.0) + (in[1] ? e[1] : 0.0), s.red, &kept);
        double* weights = reinterpret_cast<double*>(keys + kVerifyMaxTopK);
        uint32_t* by_token = reinterpret_cast<uint32_t*>(keys);   // a token and where it was, in 32 bits
        constexpr uint32_t kLastToken = (1u << 22) - 1;
        static_assert(kVerifyMaxVocab <= kLastToken && kVerifyMaxTopK <= 1 << 10, "a token and a place fit 32 bits");
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (in[j] && token[j] == d) s.pd = e[j] / kept;
            weights[j0 + j] = in[j] ? e[j] / kept : 0.0;
            by_token[j0 + j] = j0 + j < k ? (kLastToken - (uint32_t)token[j]) << 10 | (uint32_t)(j0 + j) : 0;
        }
        __syncthreads();
        if (d >= 0 && kept_below < s.pd) {
            return make_int2(1, -1);
        }
        sort_desc(by_token, k);   // the weights lie behind
        double w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t key = j0 + j < k ? by_token[j0 + j] : 0;
            token[j] = (int)(kLastToken - (key >> 10));
            w[j] = j0 + j < k ? weights[key & 1023] : 0.0;
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
    // the draw
    const int j0 = 2 * tid;
    int token[2];
    double p[2], r[2], total;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        token[j] = j0 + j < n_last ? tokens[j0 + j] : -1;
        p[j] = r[j] = j0 + j < n_last ? shares[j0 + j] : 0.0;
        if (d >= 0 && p[j] > 0.0) r[j] = fmax(p[j] - (q != nullptr ? (double)q[token[j]] : (token[j] == d ? 1.0 : 0.0)), 0.0);
    }
    double before = block_before(r[0] + r[1], s.red, &total);
    if (!(total > 0.0)) {   // the draft's distribution covers the target's
        r[0] = p[0];
        r[1] = p[1];
        before = block_before(r[0] + r[1], s.red, &total);
    }
    const double target = u_draw * total;
    if (r[0] > 0.0) {
        if (before + r[0] > target) atomicMin(&s.pick, token[0]);
        atomicMax(&s.last, token[0]);
    }
    if (r[1] > 0.0) {
        if (before + (r[0] + r[1]) > target) atomicMin(&s.pick, token[1]);
        atomicMax(&s.last, token[1]);
    }
    __syncthreads();
    return make_int2(0, s.pick < INT_MAX ? s.pick : s.last);
}

// A token's share of a draw in 64 bits.  Not inlined: it is hardly ever needed, and its registers are everyone's.
__device__ __noinline__ double wide_share(float x, float top, float temperature, bool rest, double z, float q) {
    const double w = exp(((double)x - (double)top) / (double)temperature);
    return rest ? fmax(w / z - (double)q, 0.0) : w;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) finish_lanes_kernel(const __grid_constant__ VerifyArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ TopShared top_shared;
    __shared__ double sum_of[2][kMostCtas], region[kWarps], s_z;
    __shared__ uint64_t s_best;
    __shared__ int s_end, s_bad, s_pick, s_last;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, wl = tid & 31, ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = blockIdx.x / ctas, n_drafts = a.n_drafts, vocab = a.vocab;
    const int32_t* drafts = a.drafts + (int64_t)lane * n_drafts;
    const float* u = a.u + (int64_t)lane * (n_drafts + 1);
    const float temperature = temperature_of(a, lane), top_p = a.top_p[lane];
    const double u_draw = (double)u[n_drafts];
    int k = a.top_k[lane];
    int n = 0;   // drafts in front of the first that is none
    for (bool more = true; more && n < n_drafts;) {
        const unsigned none = __ballot_sync(0xffffffffu, n + wl >= n_drafts || !is_draft(drafts[n + wl], vocab));
        more = none == 0;
        n = more ? n + 32 : n + __ffs(none) - 1;
    }
    const bool hot = temperature > 0.f, whole = hot && k <= 0, unknown = hot && (k > kVerifyMaxTopK || (whole && top_p < 1.f));
    if (rank == 0 && tid == 0 && ((n < n_drafts && drafts[n] >= vocab) || unknown)) tell(a.status, kDevBadRange);
    if (rank != 0 && (!hot || unknown || (!whole && rank > n))) return;   // no row for this CTA: whom the cluster's barrier then does not wait for
    if (tid == 0) {
        s_end = INT_MAX;
        s_pick = INT_MAX;
        s_last = -1;
    }
    __syncthreads();
    pdl_wait();
    if (unknown) {   // no draw from a distribution that nobody asked for
        if (warp == 0) put_lane(a, lane, 0, -1);
        return;
    }
    if (hot && !whole) {
        // ---- rows with a top_k, shared out over the CTAs
        k = min(k, vocab);
        int2* rows = a.rows + (int64_t)lane * (n_drafts + 1);
        for (int i = rank; i <= n; i += ctas) {
            const int2 r = finish_top_row<T>(a, top_shared, smem, lane, i, i < n ? drafts[i] : -1, k, temperature, top_p, (double)u[i], u_draw);
            if (tid == 0) rows[i] = r;
        }
        cluster.sync();
        if (rank != 0 || warp != 0) return;
        int end = 0, token = -1;
        for (bool more = true; more; end += more ? 32 : 0) {
            int2 r = make_int2(0, -1);
            if (end + wl <= n) r = __ldcg(rows + end + wl);
            const unsigned ends = __ballot_sync(0xffffffffu, r.x == 0);   // the row behind the last draft keeps nothing
            more = ends == 0;
            if (!more) {
                token = __shfl_sync(0xffffffffu, r.y, __ffs(ends) - 1);
                end += __ffs(ends) - 1;
            }
        }
        if (token < 0 && wl == 0) tell(a.status, kDevBadRow);
        put_lane(a, lane, end, token);
        return;
    }
    // ---- rows that their runs tell all of
    const Run* runs = static_cast<const Run*>(a.run_results) + (int64_t)lane * (n_drafts + 1) * a.runs;
    const T* logits = static_cast<const T*>(a.logits) + (int64_t)lane * (n_drafts + 1) * a.ld;
    const float* probs = a.draft_probs == nullptr ? nullptr : a.draft_probs + (int64_t)lane * n_drafts * vocab;
    const double per_t = hot ? 1.0 / (double)temperature : 0.0;
    RowSum mine{0, 0.0, false};
    int ends = INT_MAX;
    for (int j = warp; j <= n; j += kWarps) {
        const int d = j < n ? drafts[j] : -1;
        const double below = d >= 0 && whole ? (double)u[j] * (probs != nullptr ? (double)probs[(int64_t)j * vocab + d] : 1.0) : 0.0;
        const double logit = d >= 0 && whole ? (double)value_of(logits[j * a.ld + d]) : 0.0;
        mine = sum_runs(runs + (int64_t)j * a.runs, a.runs, per_t, whole);
        const bool kept = d >= 0 && !mine.bad && (whole ? below < exp((logit - (double)value_of_key(mine.best)) * per_t) / mine.z : d == (int)rank_key_index(mine.best));
        if (!kept) {
            ends = j;
            break;
        }
    }
    if (wl == 0 && ends < INT_MAX) atomicMin(&s_end, ends);
    __syncthreads();
    const int end = s_end;
    if (ends == end && wl == 0) {
        s_best = mine.best;
        s_z = mine.z;
        s_bad = mine.bad;
    }
    __syncthreads();
    if (s_bad || !whole) {
        if (rank != 0 || warp != 0) return;
        if (s_bad && wl == 0) tell(a.status, kDevBadRow);
        put_lane(a, lane, end, s_bad ? -1 : (int)rank_key_index(s_best));
        return;
    }
    // ---- the draw: every warp adds up a run of its own, and a CTA looks through the one where the target lies
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");   // every CTA is there before one writes to another's memory
    const T* x = logits + end * a.ld;
    const int d = end < n ? drafts[end] : -1;
    const float* q = probs == nullptr || d < 0 ? nullptr : probs + (int64_t)end * vocab;
    double z = s_z;
    const Exponential weight(value_of_key(s_best), temperature);
    const float per_z = (float)(1.0 / z), per_z_rest = (float)(1.0 / z - (double)per_z);
    const int chunk = (vocab + 4 * ctas - 1) / (4 * ctas) * 4, n0 = min(vocab, rank * chunk), n1 = min(vocab, n0 + chunk);
    const int run = (n1 - n0 + 4 * kWarps - 1) / (4 * kWarps) * 4, r_lo = min(n1, n0 + warp * run), r_hi = min(n1, r_lo + run);
    const bool fours = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;   // rows begin where four values can be read at once
    bool rest = d >= 0;
    auto shares2 = [&](float& a, float& b, float qa, float qb) {   // of two tokens
        weight(a, b);
        if (rest) {
            a = fmaxf(fmaf(a, per_z, -qa) + a * per_z_rest, 0.f);
            b = fmaxf(fmaf(b, per_z, -qb) + b * per_z_rest, 0.f);
        }
    };
    auto q_at = [&](int t) { return !rest ? 0.f : (q != nullptr ? q[t] : (t == d ? 1.f : 0.f)); };
    // All the weights that 32 bits leave out are together below 2^-100 of the whole, and what they round is 2^-22 of a share of p.  Where the target is so small that the former may decide (u = 0),
    // or the remainder so small that the latter do (draft and target all but agree), weights, their sum and shares are 64-bit: one draw in 2^24, and one in 1024 that end at such a remainder, since
    // its size is how often that happens.
    constexpr double kLeastTarget = 0x1p-60, kLeastRest = 0x1p-10;
    bool wide = false, weigh = false, first = true;   // weigh: for the sum of the weights
    auto share64 = [&](int t) { return wide_share(value_of(x[t]), value_of_key(s_best), temperature, rest && !weigh, z, q_at(t)); };
    double total = 0.0, *sums = sum_of[0];
    for (;; first = false) {
        constexpr int AHEAD = 4;   // fours of tokens a thread has on their way together
        double part = 0.0;
        for (int t = r_lo + wl; wide && t < r_hi; t += 32) part += share64(t);
        for (int t0 = r_lo + wl * 4; !wide && t0 < r_hi; t0 += 128 * AHEAD) {
            float l[AHEAD][4], qv[AHEAD][4];
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) {
                const int t = t0 + 128 * c;
                if (fours && t + 4 <= r_hi) {
                    load4(x + t, l[c]);
                    if (rest && q != nullptr) load4(q + t, qv[c]);
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) qv[c][j] = q_at(t + j);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        l[c][j] = t + j < r_hi ? value_of(x[t + j]) : -INFINITY;
                        qv[c][j] = t + j < r_hi ? q_at(t + j) : 0.f;
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) {
                if (t0 + 128 * c >= r_hi) break;
                shares2(l[c][0], l[c][1], qv[c][0], qv[c][1]);
                shares2(l[c][2], l[c][3], qv[c][2], qv[c][3]);
                part += (double)((l[c][0] + l[c][1]) + (l[c][2] + l[c][3]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (wl == 0) region[warp] = part;
        if (first) asm volatile("barrier.cluster.wait;" ::: "memory");
        __syncthreads();
        if (warp == 0) {
            double s = region[wl % kWarps];
#pragma unroll
            for (int o = kWarps / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (wl < ctas) *cluster.map_shared_rank(sums + rank, wl) = s;
        }
        cluster.sync();
        total = 0.0;
        for (int c = 0; c < ctas; ++c) total += sums[c];
        if (!wide && (!(u_draw * total >= kLeastTarget) || (rest && total < kLeastRest))) {
            wide = true;
            weigh = rest;
        } else if (weigh) {
            z = total;
            weigh = false;
        } else if (rest && !(total > 0.0)) rest = false;   // the draft's distribution covers the target's
        else break;
        sums = sums == sum_of[0] ? sum_of[1] : sum_of[0];   // nobody is still at the one before the last
    }
    const double target = u_draw * total;
    // the first CTA up to whose end the sum exceeds the target, or, where rounding left none, the last with a share; the same for its warps' runs
    double upto = 0.0;
    int at = -1;
    for (int c = 0; c < ctas; ++c) {
        if (upto > target) break;
        if (sums[c] > 0.0) at = c;
        upto += sums[c];
    }
    if (at != rank) return;
    upto = 0.0;
    for (int c = 0; c < rank; ++c) upto += sums[c];
    int w_at = 0;
    double before = upto;
    for (int w = 0; w < kWarps; ++w) {
        if (region[w] > 0.0) {
            w_at = w;
            before = upto;
        }
        upto += region[w];
        if (upto > target) break;
    }
    const int at_lo = min(n1, n0 + w_at * run), at_hi = min(n1, at_lo + run);
    for (int t0 = at_lo; t0 < at_hi; t0 += kThreads) {
        const int t = t0 + tid;
        double r = 0.0, all;
        if (wide) {
            if (t < at_hi) r = share64(t);
        } else {
            float r_mine = t < at_hi ? value_of(x[t]) : -INFINITY, none = -INFINITY;
            shares2(r_mine, none, t < at_hi ? q_at(t) : 0.f, 0.f);
            r = (double)r_mine;
        }
        const double c = before + (block_before(r, top_shared.red, &all) + r);
        if (r > 0.0) {
            atomicMax(&s_last, t);
            if (c > target) atomicMin(&s_pick, t);
        }
        before += all;
        __syncthreads();
        if (s_pick < INT_MAX) break;
    }
    __syncthreads();
    if (warp == 0) put_lane(a, lane, end, s_pick < INT_MAX ? s_pick : s_last);
}

}  // namespace

VerifyPlan verify_plan(int type, int lanes, int n_drafts, int vocab) {
    // Threads' runs short enough that a row has about four times as many as candidates are ever wanted, and not longer than 32 tokens (registers).
    VerifyPlan p;
    const int per_piece = type == 0 ? 4 : 8, most = 32 / per_piece;
    const int64_t pieces = ((int64_t)vocab + per_piece - 1 + per_piece - 1) / per_piece;   // with a first one that is shared with what is in front of the row
    while (p.vpt < most && pieces > (int64_t)p.vpt * 4096) p.vpt *= 2;
    p.runs = (int)((pieces + kScan * p.vpt - 1) / (kScan * p.vpt));
    const int64_t rows = (int64_t)lanes * (n_drafts + 1);
    p.results_at = (rows * p.runs * kScan * 4 + 255) / 256 * 256;
    p.rows_at = p.results_at + rows * p.runs * (int64_t)sizeof(Run);
    p.bytes = p.rows_at + rows * 8;
    return p;
}

void launch_verify_drafts(VerifyArgs a, const VerifyPlan& p, uint8_t* workspace, cudaStream_t s) {
    if (a.lanes <= 0) return;
    a.vpt = p.vpt;
    a.runs = p.runs;
    a.group_best = reinterpret_cast<float*>(workspace);
    a.run_results = workspace + p.results_at;
    a.rows = reinterpret_cast<int2*>(workspace + p.rows_at);
    const unsigned rows = (unsigned)(a.lanes * (a.n_drafts + 1));
    auto scan = [&](auto* kernel) {
        kernel<<<rows * (unsigned)p.runs, kScan, 0, s>>>(a);
        MK_LAUNCH_CHECK();
    };
    auto finish = [&](auto* kernel) {
        const int groups = p.runs * kScan;
        a.list_at = groups * 4;
        a.keys_at = (a.list_at + groups * 2 + 15) / 16 * 16;
        const size_t smem = (size_t)a.keys_at + kCandidates * 8 + kCounted * 8;
        ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
        // An SM holds two of these CTAs: with many lanes fewer to each (64 lanes with 4 drafts of 151936, whole vocabulary: 78 us with eight, 67 with four, 78 with two; 128 with 4 of
        // 128256: 131, 116, 114), but not where all but a few fit (40 with 6 drafts of 128256, top_k 64: 30 us with eight, 39 with four).
        int ctas = kMostCtas;
        while (ctas > 2 && (int64_t)a.lanes * ctas > 384) ctas /= 2;
        launch_pdl_cluster(kernel, ctas, dim3((unsigned)(a.lanes * ctas)), dim3(kThreads), smem, s, a);
    };
    if (a.type == 0) {
        switch (p.vpt) {
            case 1: scan(scan_rows_kernel<float, 1>); break;
            case 2: scan(scan_rows_kernel<float, 2>); break;
            case 4: scan(scan_rows_kernel<float, 4>); break;
            default: scan(scan_rows_kernel<float, 8>);
        }
        finish(finish_lanes_kernel<float>);
    } else if (a.type == 1) {
        switch (p.vpt) {
            case 1: scan(scan_rows_kernel<__half, 1>); break;
            case 2: scan(scan_rows_kernel<__half, 2>); break;
            default: scan(scan_rows_kernel<__half, 4>);
        }
        finish(finish_lanes_kernel<__half>);
    } else {
        switch (p.vpt) {
            case 1: scan(scan_rows_kernel<__nv_bfloat16, 1>); break;
            case 2: scan(scan_rows_kernel<__nv_bfloat16, 2>); break;
            default: scan(scan_rows_kernel<__nv_bfloat16, 4>);
        }
        finish(finish_lanes_kernel<__nv_bfloat16>);
    }
}

}  // namespace mk
