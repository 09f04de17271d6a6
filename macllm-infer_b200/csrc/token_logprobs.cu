// Log probabilities of given tokens, with the entropy of their distributions, their ranks and the likeliest tokens.
//
// For a row x of logits with maximum m and Z = sum e^(x_i - m):  log p_i = x_i - m - ln Z,  entropy = -sum p_i log p_i = ln Z - sum e^(x_i - m) (x_i - m) / Z.  The rank of
// a token is its place among all, by falling logit and, among equals, rising token; the likeliest tokens come in that order.
//
// One kernel, in which a row is read once from memory: by one CTA, or by a cluster of up to eight where rows are few, a run of the row to each.  A thread takes vectors of 16 bytes, eight of
// them at a time, and keeps its maximum, both sums under it, and how many values stand before the given token's; maxima and sums of threads, warps and CTAs join
// exactly but for roundings.  Differences x - m are taken before anything is scaled, so that they carry one rounding, and sums are 32-bit: a few hundred terms to a thread, then a tree.
// The likeliest `top` of a run: the top-th best of the threads' maxima is a bound that at least `top` values reach and few more do, only the vectors of threads that reach it are
// looked at again (in L2), and the candidates are ranked by counting.  Where too many reach it - thousands of equal logits, or most of them masked - a radix select over (value, token) finds the
// top-th key exactly, in up to seven more passes.  The leader of a cluster merges the sorted lists by binary search.
// What bounds it is HBM and, for 16-bit logits, instructions beside it (8 for a value): 2000 rows of 128256 bf16 logits 99.6 us, 5.2 TB/s (117 with sums of single numbers and bounds checked for each
// vector); 40 rows of 151936 f32 with 20 alternatives 17.1 us, 6 of them the alternatives; 5 rows of 32000 with 5 alternatives 9.1, of which 3.
#include "token_logprobs.h"
#include "attention_math.cuh"
#include <cuda_bf16.h>
#include <cooperative_groups.h>
#include <algorithm>

namespace mk {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBatch = 8;             // vectors of a thread on their way together
constexpr int kCandidates = 512;
constexpr int kMaxCluster = 8;

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

// Numbers as unsigned ones of the same order (no NaN; both zeros are one).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_ordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
// (value, token) of the same order as the likeliest come in: the larger key first.
__device__ __forceinline__ uint64_t key_of(float x, int token) { return (uint64_t)ordered(x) << 24 | (uint32_t)(0xffffff - token); }
__device__ __forceinline__ int token_of(uint64_t key) { return 0xffffff - (int)(key & 0xffffff); }
__device__ __forceinline__ float value_of(uint64_t key) { return of_ordered((uint32_t)(key >> 24)); }

// Vectors of 16 bytes: N values, taken two at a time with none below `least`; their maximum; and counts of those that reach a bound, in a form of the type's own that holds a batch's.
template <typename T>
struct Vec;
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
template <>
struct Vec<float> {
    static constexpr int N = 4;
    using Count = int;
    using Bound = float;
    static __device__ __forceinline__ float value(const uint4& v, int i) { return __uint_as_float(word_of(v, i)); }
    static constexpr float lowest = -3.4028234663852886e38f;
    static __device__ __forceinline__ Bound bound(float x) { return x; }
    static __device__ __forceinline__ FloatPair two(const uint4& v, int i, Bound least) { return FloatPair{fmaxf(value(v, 2 * i), least), fmaxf(value(v, 2 * i + 1), least)}; }
    static __device__ __forceinline__ float top(const uint4& v) { return max_nan(max_nan(value(v, 0), value(v, 1)), max_nan(value(v, 2), value(v, 3))); }
    static __device__ __forceinline__ void reach(const uint4& v, Bound b, Count& n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n += value(v, i) >= b ? 1 : 0;
    }
    static __device__ __forceinline__ int count(Count n) { return n; }
    static __device__ __forceinline__ float after(float x) {   // the next number up
        const uint32_t b = __float_as_uint(x + 0.f);
        return __uint_as_float(b & 0x80000000u ? b - 1 : b + 1);
    }
};
template <typename P>
__device__ __forceinline__ P as_pair(uint32_t w) { return *reinterpret_cast<const P*>(&w); }
template <typename P>
struct HalfVec {   // of two 16-bit types
    static constexpr int N = 8;
    using Count = P;   // up to 4 for each vector of a batch
    using Bound = P;
    static __device__ __forceinline__ float top(const uint4& v) {
        const P m = __hmax2_nan(__hmax2_nan(as_pair<P>(v.x), as_pair<P>(v.y)), __hmax2_nan(as_pair<P>(v.z), as_pair<P>(v.w)));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void reach(const uint4& v, Bound b, Count& n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n = __hadd2(n, __hge2(as_pair<P>(word_of(v, i)), b));
    }
    static __device__ __forceinline__ int count(Count n) { return (int)(__low2float(n) + __high2float(n)); }
};
template <>
struct Vec<__half> : HalfVec<__half2> {
    static __device__ __forceinline__ float value(const uint4& v, int i) {
        const float2 f = __half22float2(as_pair<__half2>(word_of(v, i >> 1)));
        return i & 1 ? f.y : f.x;
    }
    static constexpr float lowest = -65504.f;
    static __device__ __forceinline__ Bound bound(float x) { return __float2half2_rn(x); }
    static __device__ __forceinline__ FloatPair two(const uint4& v, int i, Bound least) {
        const float2 f = __half22float2(__hmax2(as_pair<__half2>(word_of(v, i)), least));
        return FloatPair{f.x, f.y};
    }
    static __device__ __forceinline__ float after(float x) {
        const unsigned short b = __half_as_ushort(__float2half_rn(x + 0.f));
        return __half2float(__ushort_as_half(b & 0x8000u ? b - 1 : b + 1));
    }
};
template <>
struct Vec<__nv_bfloat16> : HalfVec<__nv_bfloat162> {
    static __device__ __forceinline__ float value(const uint4& v, int i) {
        const uint32_t w = word_of(v, i >> 1);
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    static constexpr float lowest = -3.3895313892515355e38f;
    static __device__ __forceinline__ Bound bound(float x) { return __float2bfloat162_rn(x); }
    static __device__ __forceinline__ FloatPair two(const uint4& v, int i, Bound least) {
        const __nv_bfloat162 m = __hmax2(as_pair<__nv_bfloat162>(word_of(v, i)), least);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
        return FloatPair{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    }
    static __device__ __forceinline__ float after(float x) {
        const uint32_t b = __float_as_uint(x + 0.f) >> 16;
        return __uint_as_float((b & 0x8000u ? b - 1 : b + 1) << 16);
    }
};

// The values of a CTA's run of a row: `vectors` of 16 bytes from token `first` on, and, in single ones, those of the row in front of the first vector and behind the last.
template <typename T>
struct Run {
    const T* row;
    int first, vectors;
    int head, tail_at, tail;   // tokens [0, head) and [tail_at, tail_at + tail)
    __device__ __forceinline__ uint4 vector(int i) const { return __ldg(reinterpret_cast<const uint4*>(row + first) + i); }
    // f(value, token), `there` false where a thread of the warp has none; the warp's threads come together
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        constexpr int N = Vec<T>::N;
        for (int i0 = 0; i0 < vectors; i0 += kThreads) {
            const int i = i0 + (int)threadIdx.x;
            const bool there = i < vectors;
            const uint4 v = there ? vector(i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int j = 0; j < N; ++j) f(Vec<T>::value(v, j), first + i * N + j, there);
        }
        const int e = edge();
        f(e >= 0 ? (float)row[e] : 0.f, e, e >= 0);
    }
    __device__ __forceinline__ int edge() const {   // the thread's single token, or -1
        const int i = (int)threadIdx.x;
        return i < head ? i : (i < head + tail ? tail_at + i - head : -1);
    }
};

struct Sums {   // of a part of a row: maximum, sum of e^(x - m), sum of e^(x - m) (x - m), values in front of the given token's
    float m, z, zx;
    int before;
};
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    Sums r;
    r.m = max_nan(a.m, b.m);
    r.before = a.before + b.before;
    if (!(r.m > -INFINITY)) {   // nothing, or NaN
        r.z = a.z + b.z;
        r.zx = a.zx + b.zx;
        return r;
    }
    // a difference that overflows belongs to a sum that vanishes
    const float da = fmaxf(a.m - r.m, -3e38f), db = fmaxf(b.m - r.m, -3e38f), fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
    r.z = a.z * fa + b.z * fb;
    r.zx = (fa > 0.f ? fa * fmaf(a.z, da, a.zx) : 0.f) + (fb > 0.f ? fb * fmaf(b.z, db, b.zx) : 0.f);
    return r;
}

struct Shared {
    Sums warp_sums[kWarps], sums;
    uint32_t tops[kThreads];
    uint64_t candidates[kCandidates];
    uint64_t best[kLogprobMaxTop];          // of the run, in order
    uint64_t lists[kMaxCluster][kLogprobMaxTop];
    uint32_t histogram[256];
    uint64_t prefix;
    uint32_t bound;
    int n_candidates, n_best, left;
    int list_n[kMaxCluster];
};

// The `top` best keys of the run into s.best, in order; s.n_best of them.
template <typename T>
__device__ __forceinline__ void best_of_run(const Run<T>& run, float my_top, int top, Shared& s) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    s.tops[tid] = ordered(my_top);
    if (tid == 0) s.n_candidates = 0;
    __syncthreads();
    if (warp == 0) {   // a bound that `top` threads' maxima reach, and hardly twice as many
        uint32_t k[kThreads / 32], lo = UINT32_MAX, hi = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) {
            k[i] = s.tops[i * 32 + lane];
            lo = min(lo, k[i]);
            hi = max(hi, k[i]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);   // all reach it
        hi = __reduce_max_sync(0xffffffffu, hi);
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            int n = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) n += k[i] >= mid ? 1 : 0;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= top) lo = mid;
            else hi = mid - 1;
            if (n >= top && n <= top + top / 2) break;
        }
        if (lane == 0) s.bound = lo;
    }
    __syncthreads();
    const uint32_t bound = s.bound;
    if (ordered(my_top) >= bound) {
        constexpr int N = Vec<T>::N;
        auto offer = [&](float x, int token) {
            if (ordered(x) < bound) return;
            const int at = atomicAdd(&s.n_candidates, 1);
            if (at < kCandidates) s.candidates[at] = key_of(x, token);
        };
        const float least = of_ordered(bound);
        for (int i0 = tid; i0 < run.vectors; i0 += kThreads * 4) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = i0 + k * kThreads < run.vectors ? run.vector(i0 + k * kThreads) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * kThreads;
                if (i >= run.vectors || Vec<T>::top(v[k]) < least) continue;
#pragma unroll
                for (int j = 0; j < N; ++j) offer(Vec<T>::value(v[k], j), run.first + i * N + j);
            }
        }
        const int e = run.edge();
        if (e >= 0) offer((float)run.row[e], e);
    }
    __syncthreads();
    if (s.n_candidates > kCandidates) {   // digit by digit from the top: the key that `top` keys reach
        if (tid == 0) s.prefix = 0, s.left = top;   // more than kCandidates values are there
        for (int shift = 48; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kThreads) s.histogram[i] = 0;
            __syncthreads();
            const uint64_t prefix = s.prefix;
            run.each([&](float x, int token, bool there) {
                const uint64_t key = key_of(x, token);
                const bool in = there && key >> 8 >> shift == prefix;
                const int digit = (int)(key >> shift & 255);
                const uint32_t of = __ballot_sync(0xffffffffu, in);
                if (of == 0) return;
                // equal digits are counted at once: thousands of equal logits would queue at one counter
                const int first_digit = __shfl_sync(0xffffffffu, digit, __ffs(of) - 1);   // every thread of the warp comes here
                if (__all_sync(0xffffffffu, !in || digit == first_digit)) {
                    if (lane == __ffs(of) - 1) atomicAdd(&s.histogram[digit], __popc(of));
                } else if (in) {
                    atomicAdd(&s.histogram[digit], 1);
                }
            });
            __syncthreads();
            if (warp == 0) {   // the digit in which the top-th key lies: eight counters to a thread, from the top
                uint32_t mine = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) mine += s.histogram[255 - 8 * lane - i];
                uint32_t upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t before = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += before;
                }
                const uint32_t left = (uint32_t)s.left;
                __syncwarp();
                if (upto >= left && upto - mine < left) {
                    uint32_t rest = left - (upto - mine);
                    int d = 255 - 8 * lane;
                    while (s.histogram[d] < rest) rest -= s.histogram[d--];
                    s.prefix = prefix << 8 | (uint64_t)d;
                    s.left = (int)rest;
                    s.n_candidates = 0;
                }
            }
            __syncthreads();
        }
        const uint64_t least = s.prefix;
        run.each([&](float x, int token, bool there) {
            if (!there || key_of(x, token) < least) return;
            const int at = atomicAdd(&s.n_candidates, 1);
            if (at < kCandidates) s.candidates[at] = key_of(x, token);
        });
        __syncthreads();
    }
    const int n = min(s.n_candidates, kCandidates);
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t mine = s.candidates[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s.candidates[j] > mine ? 1 : 0;
        if (rank < top) s.best[rank] = mine;
    }
    if (tid == 0) s.n_best = min(n, top);
}

__device__ __forceinline__ void add_weights(FloatPair v, FloatPair minus_m, FloatPair& z, FloatPair& zx) {
    const FloatPair d = v + minus_m, y = d * FloatPair{kLog2e, kLog2e}, e{ex2(y.x), ex2(y.y)};
    z = z + e;
    zx = fma2(e, d, zx);
}
// A maximum at the end of the type's numbers has none that far below it, so that -inf counted like the lowest of them: the thread's values once more, one by one, -inf left out.  (Where a larger one
// came later, what was counted until then has vanished.)  Apart from the rest, which has 5 % more to do where these few lines are in line (2000 rows of bf16 logits 104.7 us, 99.6 so).
template <typename T>
__device__ __noinline__ float4 one_by_one(const T* row, int first, int vectors, int edge, float m) {
    FloatPair z{0.f, 0.f}, zx{0.f, 0.f};
    auto one = [&](float v) {
        if (v > -INFINITY) add_weights(FloatPair{v, -300.f}, FloatPair{-m, 0.f}, z, zx);   // and nothing
    };
    for (int i = threadIdx.x; i < vectors; i += kThreads)
        for (int j = 0; j < Vec<T>::N; ++j) one((float)row[first + i * Vec<T>::N + j]);
    if (edge >= 0) one((float)row[edge]);
    return make_float4(z.x, z.y, zx.x, zx.y);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const __grid_constant__ LogprobArgs a, int parts) {
    constexpr int N = Vec<T>::N;
    __shared__ Shared s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / parts;
    const int part = blockIdx.x - (int)row * parts;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int token = a.tokens[row];
    const bool given = token >= 0 && token < a.vocab;
    const float mine = given ? (float)x[token] : INFINITY;

    // the row's vectors, evenly shared out; its ends in single values go to the first CTA
    Run<T> run;
    {
        const int off = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), head = min(off, a.vocab), vectors = (a.vocab - head) / N;
        const int each = (vectors + parts - 1) / parts, from = min(part * each, vectors);
        run.row = x;
        run.first = head + from * N;
        run.vectors = min(each, vectors - from);
        run.head = part == 0 ? head : 0;
        run.tail_at = head + vectors * N;
        run.tail = part == 0 ? a.vocab - run.tail_at : 0;
    }
    // tokens in front of the given one count where they reach its logit, those behind it where they exceed it; its own vector's are looked at one by one
    const float above = given ? Vec<T>::after(mine) : INFINITY;
    const int own_vector = given && token >= run.first ? (token - run.first) / N : -1;
    const auto bound_mine = Vec<T>::bound(mine), bound_above = Vec<T>::bound(above), bound_none = Vec<T>::bound(INFINITY);

    FloatPair z{0.f, 0.f}, zx{0.f, 0.f};
    float m_run = -INFINITY;
    int before = 0;
    auto add = [&](FloatPair v, FloatPair minus_m) { add_weights(v, minus_m, z, zx); };
    auto raise = [&](float top) {   // the maximum to at least `top`; what to subtract
        const float m = max_nan(m_run, top);
        if (m > m_run) {
            const float d = fmaxf(m_run - m, -3e38f), f = ex2(d * kLog2e);
            zx = f > 0.f ? FloatPair{f, f} * fma2(z, FloatPair{d, d}, zx) : FloatPair{0.f, 0.f};
            z = z * FloatPair{f, f};
        }
        m_run = m;
        return m == -INFINITY ? 0.f : m;
    };
    // values whose weight is 0 anyway count as this far below the maximum: a weight of 0 times what is left of -inf would not be 0
    auto least_of = [](float m) { return fmaxf(m - 300.f - fabsf(m), Vec<T>::lowest); };
    auto batch = [&](int i0, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        uint4 v[kBatch];
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (kWhole || i0 + k * kThreads < run.vectors) v[k] = run.vector(i0 + k * kThreads);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (kWhole || i0 + k * kThreads < run.vectors) top = max_nan(top, Vec<T>::top(v[k]));
        const float m = raise(top);
        const auto least = Vec<T>::bound(least_of(m));
        typename Vec<T>::Count n{};
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * kThreads;
            if (!kWhole && i >= run.vectors) break;
#pragma unroll
            for (int j = 0; j < N / 2; ++j) add(Vec<T>::two(v[k], j, least), FloatPair{-m, -m});
            Vec<T>::reach(v[k], i < own_vector ? bound_mine : (i == own_vector ? bound_none : bound_above), n);
        }
        before += Vec<T>::count(n);
    };
    int i0 = tid;
    for (; i0 + (kBatch - 1) * kThreads < run.vectors; i0 += kThreads * kBatch) batch(i0, std::true_type{});
    if (i0 < run.vectors) batch(i0, std::false_type{});
    {
        const int e = run.edge();
        if (e >= 0) {
            const float v = (float)x[e], m = raise(v);
            add(FloatPair{fmaxf(v, least_of(m)), -300.f}, FloatPair{-m, 0.f});   // and nothing
            if (given) before += e < token ? v >= mine : v >= above;
        }
        if (own_vector >= 0 && own_vector < run.vectors && tid < N) {
            const int e = run.first + own_vector * N + tid;
            if (e != token) before += (float)x[e] >= (e < token ? mine : above) ? 1 : 0;
        }
    }
    if (m_run > -INFINITY && !(m_run - least_of(m_run) >= 150.f)) {
        const float4 sums = one_by_one(run.row, run.first, run.vectors, run.edge(), m_run);
        z = FloatPair{sums.x, sums.y}, zx = FloatPair{sums.z, sums.w};
    }
    const Sums my{m_run, z.x + z.y, zx.x + zx.y, before};
    const float my_top = my.m;
    Sums all = my;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums other;
        other.m = __shfl_xor_sync(0xffffffffu, all.m, o);
        other.z = __shfl_xor_sync(0xffffffffu, all.z, o);
        other.zx = __shfl_xor_sync(0xffffffffu, all.zx, o);
        other.before = __shfl_xor_sync(0xffffffffu, all.before, o);
        all = joined(all, other);
    }
    if (lane == 0) s.warp_sums[warp] = all;
    __syncthreads();
    if (tid == 0) {
        all = s.warp_sums[0];
        for (int w = 1; w < kWarps; ++w) all = joined(all, s.warp_sums[w]);
        s.sums = all;
        s.n_best = 0;
    }
    __syncthreads();
    const bool finite = s.sums.m < INFINITY;   // of this run: no NaN, no +inf
    if (a.top > 0 && finite) best_of_run(run, my_top, a.top, s);
    if (parts > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (part == 0) {
            if (tid < parts) s.list_n[tid] = cluster.map_shared_rank(&s, tid)->n_best;
            for (int i = tid; i < parts * a.top; i += kThreads) s.lists[i / a.top][i % a.top] = cluster.map_shared_rank(&s, i / a.top)->best[i % a.top];
            if (tid == 0) {
                all = s.sums;
                for (int c = 1; c < parts; ++c) all = joined(all, cluster.map_shared_rank(&s, c)->sums);
                s.warp_sums[0] = all;
            }
        }
        cluster.sync();
        if (part != 0) return;
        all = s.warp_sums[0];
    } else {
        __syncthreads();
        all = s.sums;
    }
    const bool bad = !(all.m < INFINITY) || all.m == -INFINITY;
    const float log_z = logf(all.z);
    if (tid == 0) {
        if (bad) tell(a.status, kDevBadRow);
        if (token >= a.vocab) tell(a.status, kDevBadRange);
        a.logprobs[row] = token < 0 ? 0.f : (given && !bad ? mine - all.m - log_z : NAN);
        a.entropy[row] = bad ? NAN : log_z - all.zx / all.z;
        a.ranks[row] = given && !bad ? all.before + 1 : 0;
    }
    if (a.top == 0) return;
    auto put = [&](int rank, uint64_t key) {
        a.top_tokens[row * a.top + rank] = token_of(key);
        a.top_logprobs[row * a.top + rank] = value_of(key) - all.m - log_z;
    };
    if (bad) {
        if (tid < a.top) {
            a.top_tokens[row * a.top + tid] = -1;
            a.top_logprobs[row * a.top + tid] = NAN;
        }
    } else if (parts == 1) {
        if (tid < s.n_best) put(tid, s.best[tid]);
    } else {
        for (int i = tid; i < parts * a.top; i += kThreads) {
            const int c = i / a.top, r = i - c * a.top;
            if (r >= s.list_n[c]) continue;
            const uint64_t key = s.lists[c][r];
            int rank = r;
            for (int o = 0; o < parts && rank < a.top; ++o) {
                if (o == c) continue;
                int lo = 0, hi = s.list_n[o];   // how many of the other's come first
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (s.lists[o][mid] > key) lo = mid + 1;
                    else hi = mid;
                }
                rank += lo;
            }
            if (rank < a.top) put(rank, key);
        }
    }
}

template <typename T>
void launch(const LogprobArgs& a, int parts, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    cuda_check(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a, parts), "kernel launch", __FILE__, __LINE__);
}

}  // namespace

void launch_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
    // as many CTAs to a row as give each SM one and each thread eight vectors (5 rows of 32000 logits: four 9.0 us, eight 10.2; 40 rows of 151936: four 16.9, eight 17.4; 12 of 256000: eight 15.5, four 18.6)
    const int64_t vectors = (int64_t)a.vocab * (a.kind == 0 ? 4 : 2) / 16;
    int parts = 1;
    while (parts < kMaxCluster && (int64_t)a.rows * parts < 148 && vectors > (int64_t)parts * kThreads * kBatch) parts *= 2;
    if (a.kind == 0) launch<float>(a, parts, s);
    else if (a.kind == 1) launch<__half>(a, parts, s);
    else launch<__nv_bfloat16>(a, parts, s);
}

}  // namespace mk
