// Rows of keys and values into pages of 4- or 8-bit codes, and back.
//
// Groups of 64 neighbouring values x_i of a head's row have a lowest value and a step of their own:
//   low = min x_i,  step = (max x_i - low) / L rounded to the rows' type (L = 15 or 255),  c_i = min(L, round((x_i - low) / step)), halves to even, 0 where step is 0;
// c_i stands for low + step c_i.  low is one of the values, so it needs no rounding; the step's is 2^-11 (f16) or 2^-8 (bf16) of it at most and moves no value by more than
// L times that, and since the codes are made with the rounded step they are the nearest ones under it.  A group with a value, or a range, that is not finite reads as NaN throughout.
#include "quantized_kv.h"
#include <algorithm>

namespace mk {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

template <typename T>
struct Two;
template <>
struct Two<__half> {
    static __device__ __forceinline__ float2 wide(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr float largest = 65504.f;
    using Pair = __half2;
    static constexpr int kCodeBits = 8;               // of a code in numbers kOne + c of this type, c exact
    static constexpr uint32_t kOne = 0x64006400u;     // 1024 + c
    static __device__ __forceinline__ Pair minus_one() { return __float2half2_rn(-1024.f); }
};
template <>
struct Two<__nv_bfloat16> {
    static __device__ __forceinline__ float2 wide(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr float largest = 3.3895313892515355e38f;
    using Pair = __nv_bfloat162;
    static constexpr int kCodeBits = 4;
    static constexpr uint32_t kOne = 0x43004300u;     // 128 + c
    static __device__ __forceinline__ Pair minus_one() { return __float2bfloat162_rn(-128.f); }
};
template <typename P>
__device__ __forceinline__ P as_pair(uint32_t w) { return *reinterpret_cast<const P*>(&w); }
template <typename P>
__device__ __forceinline__ uint32_t word_of(P v) { return *reinterpret_cast<const uint32_t*>(&v); }

// What eight codes stand for, as four words.  In numbers of the type themselves, a pair at a time, where they hold the codes (low + step c is rounded once either way), else in 32 bits.
template <typename T, int BITS>
__device__ __forceinline__ uint4 values_of(uint32_t pair, const uint32_t (&c)[BITS / 4]) {
    using W = Two<T>;
    uint32_t w[4];
    const float2 sl = W::wide(pair);
    if constexpr (BITS <= W::kCodeBits) {
        const auto step = as_pair<typename W::Pair>(__byte_perm(pair, 0, 0x1010)), low = as_pair<typename W::Pair>(__byte_perm(pair, 0, 0x3232));
        auto two = [&](uint32_t bits) { return word_of(__hfma2(__hadd2(as_pair<typename W::Pair>(bits), W::minus_one()), step, low)); };
        if constexpr (BITS == 4) {   // pairs (0, 4), (1, 5), (2, 6), (3, 7), then neighbours
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = two((c[0] >> 4 * j & 0x000f000fu) | W::kOne);
            w[0] = __byte_perm(u[0], u[1], 0x5410), w[1] = __byte_perm(u[2], u[3], 0x5410), w[2] = __byte_perm(u[0], u[1], 0x7632), w[3] = __byte_perm(u[2], u[3], 0x7632);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = two(__byte_perm(c[j >> 1], W::kOne, j & 1 ? 0x5352 : 0x5150));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)   // 2^23 + c by its bits
                v[h] = fmaf(sl.x, __uint_as_float((c[j * 2 * BITS / 32] >> (j * 2 + h) * BITS % 32 & ((1u << BITS) - 1)) | 0x4b000000u) - 8388608.f, sl.y);
            w[j] = W::pack(v[0], v[1]);
        }
    }
    // a rounded step may lead beyond the largest number
    if (fmaf(sl.x, (float)((1 << BITS) - 1), sl.y) > W::largest) {
        const auto most = as_pair<typename W::Pair>(W::pack(W::largest, W::largest));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = word_of(__hmin2_nan(as_pair<typename W::Pair>(w[j]), most));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The lane of row t, by a whole warp: the last one whose rows do not begin behind t, 32 of them looked at in each turn.  Whatever cu holds, the index is a lane's.
__device__ __forceinline__ int lane_of_row(const QuantLanes& a, int t) {
    int lo = 0;
    for (int n = a.lanes; n > 1;) {
        const int step = (n + 31) / 32, i = (int)(threadIdx.x & 31) * step;
        const uint32_t before = __ballot_sync(0xffffffffu, i < n && a.cu[lo + i] <= t);
        const int k = before != 0 ? 31 - __clz(before) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// Where a row's token is; page: -1 where it has none (in front of a lane's first token, or what the arrays should not hold), -2 where the row belongs to no lane.
struct Place {
    int page, in_page;
};
// Of row first + the thread's number in its warp, where that is below `rows`; the whole warp.
__device__ __forceinline__ Place place_of_row(const QuantLanes& a, const QuantPools& p, int first, int rows) {
    const int t = first + (threadIdx.x & 31);
    int lane = 0, begin, end;
    if (a.cu == nullptr) {
        lane = min(t, a.total - 1) / a.rows;
        begin = lane * a.rows;
        end = begin + a.rows;
    } else {
        lane = lane_of_row(a, first);
        for (int hi = a.lanes; rows > 1 && hi - lane > 1;) {   // the thread's own row, behind the first one's lane
            const int mid = (lane + hi) / 2;
            if (a.cu[mid] <= t) lane = mid;
            else hi = mid;
        }
        begin = a.cu[lane];
        end = a.cu[lane + 1];
    }
    Place r{-2, 0};
    if ((int)(threadIdx.x & 31) >= rows || t >= a.total || t < begin || t >= end) return r;   // a warp's last rows may lie behind the call's, wherever the list says that a lane ends
    r.page = -1;
    const int length = a.lengths[lane];
    if (begin < 0 || end > a.total || length < 0 || length > (int64_t)a.width << p.bt_shift) {
        tell(a.status, kDevBadRange);
        return r;
    }
    const int position = length - (end - t);
    if (position < 0) return r;
    const int page = a.tables[lane * a.ld_table + (position >> p.bt_shift)];
    if (page < 0 || page >= p.pages) {
        tell(a.status, kDevBadPage);
        return r;
    }
    r.page = page;
    r.in_page = position & (p.block_tokens - 1);
    return r;
}

// The code of x, which is c or next to it, where the difference d of x and low may have lost something: x - low = d + lost (see below).
__device__ __noinline__ uint32_t nearest(float x, float low, float step, uint32_t c, uint32_t most) {
    const float d = x - low, of_low = d - x, lost = (x - (d - of_low)) - (low + of_low), rest = fmaf(-(float)c, step, d), twice = 2.f * fabsf(rest), beyond = rest > 0.f ? lost : -lost;
    const bool other = twice > step || (twice == step && (beyond > 0.f || (beyond == 0.f && (c & 1u))));
    return other ? (rest > 0.f ? min(c + 1u, most) : c - 1u) : c;
}
// Codes of eight values x under (step, low); step is positive.  A reciprocal gives the quotient to 2^-22 of it, 2^-14 at most, which decides wherever it is not that near to a half; there, as bf16 values
// often are, the remainder does: d - c step is exact for the 32-bit difference d = x - low (c step has at most 19 bits), and twice that against the step says which code is nearer.  Where they are equal,
// what d lost in its rounding says it, and where it lost nothing the even code is meant; elsewhere the loss decides nothing, since twice the remainder is off the step by 2^-16 of it or more.  A difference
// of numbers of m bits loses nothing unless one of them is below 2^(m - 24) of it, and that is looked for first: with the loss of each value found anyway 16383 rows written and read took 47.8 us, so 46.0, without 44.7.
template <typename T, int BITS>
__device__ __forceinline__ void codes_of(const float (&x)[8], float low, float step, uint32_t (&word)[BITS / 4]) {
    constexpr uint32_t L = (1u << BITS) - 1;
    constexpr float kWhole = 12582912.f;   // 2^23 + 2^22: sums keep whole numbers, in their lowest bits
    const float inv = 1.0f / step;
    uint32_t c[8];
    float off = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = (x[j] - low) * inv, whole = fminf(q, (float)L) + kWhole;
        off = fmaxf(off, fabsf(q - (whole - kWhole)));
        c[j] = __float_as_uint(whole) & L;
    }
    if (!(inv < INFINITY)) {   // steps below 2^-128
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = min(L, (uint32_t)__float2int_rn(__fdiv_rn(x[j] - low, step)));
    } else if (off >= 0.4999f) {
        constexpr float kLoses = (float)(L + 1) / (std::is_same_v<T, __half> ? 8192.f : 65536.f);
        float least = low != 0.f ? fabsf(low) : INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j += 2) asm("{\n\t.reg .f32 a, b;\n\tabs.f32 a, %1;\n\tabs.f32 b, %2;\n\tmin.f32 %0, %0, a, b;\n\t}" : "+f"(least) : "f"(x[j]), "f"(x[j + 1]));
        if (least > step * kLoses) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float rest = fmaf(-(float)c[j], step, x[j] - low), twice = 2.f * fabsf(rest);
                const bool other = twice > step || (twice == step && (c[j] & 1u));
                c[j] = other ? (rest > 0.f ? min(c[j] + 1u, L) : c[j] - 1u) : c[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = nearest(x[j], low, step, c[j], L);
        }
    }
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
        constexpr int N = 32 / BITS;
        word[i] = c[i * N];
#pragma unroll
        for (int j = 1; j < N; ++j) word[i] |= c[i * N + j] << j * BITS;
    }
}

// A warp has ROWS rows of K or V, and their places in as many threads; eight values to a thread, a group to eight threads, four of a thread's pieces on their way together.
// What bounds it is instructions, about 16 for a value: 16383 rows of 8 heads of 128, K and V, bf16 into 4 bits (86 MB read and written): 32.3 us, 2.7 TB/s.  With a division for each value 38 us where it took 31.
constexpr int kAhead = 4;

template <typename T, int BITS, int ROWS>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ QuantRowsArgs a) {
    constexpr int L = (1 << BITS) - 1;
    const QuantPools& p = a.pools;
    const int lane = threadIdx.x & 31, first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * ROWS;
    if (first >= a.lanes.total) return;
    const Place place = place_of_row(a.lanes, p, first, ROWS);
    const bool keys = blockIdx.y == 0;
    const int64_t row_stride = keys ? a.k_row : a.v_row, head_stride = keys ? a.k_head : a.v_head;
    const int pieces_shift = p.d == 64 ? 3 : (p.d == 128 ? 4 : 5), n = p.kv_heads << pieces_shift;
#pragma unroll 1
    for (int r = 0; r < ROWS; ++r) {
        const int page = __shfl_sync(0xffffffffu, place.page, r), in_page = __shfl_sync(0xffffffffu, place.in_page, r);
        if (page < 0) continue;
        const T* row = static_cast<const T*>(keys ? a.k : a.v) + (first + r) * row_stride;
        uint8_t* codes = (keys ? p.k_codes : p.v_codes) + page * p.codes_stride;
        uint32_t* scales = (keys ? p.k_scales : p.v_scales) + page * p.scales_stride;
        for (int i0 = lane; i0 - lane < n; i0 += 32 * kAhead) {
            uint4 w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + 32 * k, head = i >> pieces_shift, piece = i & ((1 << pieces_shift) - 1);
                w[k] = i < n ? *reinterpret_cast<const uint4*>(row + head * head_stride + piece * 8) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + 32 * k, head = i >> pieces_shift, piece = i & ((1 << pieces_shift) - 1);
                if (i - lane >= n) break;
                using P = typename Two<T>::Pair;
                const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                // lowest and highest of the group, the latter as the lowest of what is turned round: one reduction for both
                P lows = __hmin2_nan(__hmin2_nan(as_pair<P>(u[0]), as_pair<P>(u[1])), __hmin2_nan(as_pair<P>(u[2]), as_pair<P>(u[3])));
                P highs = __hmax2_nan(__hmax2_nan(as_pair<P>(u[0]), as_pair<P>(u[1])), __hmax2_nan(as_pair<P>(u[2]), as_pair<P>(u[3])));
                highs = __hneg2(highs);
                P both = __hmin2_nan(as_pair<P>(__byte_perm(word_of(lows), word_of(highs), 0x5410)), as_pair<P>(__byte_perm(word_of(lows), word_of(highs), 0x7632)));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) both = __hmin2_nan(both, as_pair<P>(__shfl_xor_sync(0xffffffffu, word_of(both), o)));
                const float2 ends = Two<T>::wide(word_of(both));
                const float low = ends.x, high = -ends.y;
                const float range = high - low;
                uint32_t pair = Two<T>::pack(__fdiv_rn(range, (float)L), low);
                if (!isfinite(range)) pair = Two<T>::pack(NAN, NAN);
                const float step = Two<T>::wide(pair).x;
                uint32_t word[BITS / 4] = {};
                if (step > 0.f) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = Two<T>::wide(u[j]);
                        x[2 * j] = v.x;
                        x[2 * j + 1] = v.y;
                    }
                    codes_of<T, BITS>(x, low, step, word);
                }
                if (i >= n) break;
                const int64_t at = ((int64_t)head * p.block_tokens + in_page) << pieces_shift;   // in pieces
                uint8_t* to = codes + (at + piece) * BITS;
                if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(to) = word[0];
                else *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
                if ((lane & 7) == 0) scales[(at + piece) >> 3] = pair;
            }
        }
    }
}

// The same the other way; a row without a token becomes zeros, and a value beyond the type's largest that largest (a rounded step may lead there).  What bounds it is HBM, which takes four times what it gives:
// 95 thousand rows of 8 heads of 128 out of 4 bits (503 MB): 83 us, 6.1 TB/s; with conversions and sums in 32 bits 118 us.
template <typename T, int BITS, int ROWS>
__global__ void __launch_bounds__(kThreads) dequantize_rows_kernel(const __grid_constant__ QuantRowsArgs a) {
    const QuantPools& p = a.pools;
    const int lane = threadIdx.x & 31, first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * ROWS;
    if (first >= a.lanes.total) return;
    const Place place = place_of_row(a.lanes, p, first, ROWS);
    const bool keys = blockIdx.y == 0;
    const int64_t row_stride = keys ? a.k_row : a.v_row, head_stride = keys ? a.k_head : a.v_head;
    const int pieces_shift = p.d == 64 ? 3 : (p.d == 128 ? 4 : 5), n = p.kv_heads << pieces_shift;
#pragma unroll 1
    for (int r = 0; r < ROWS; ++r) {
        const int page = __shfl_sync(0xffffffffu, place.page, r), in_page = __shfl_sync(0xffffffffu, place.in_page, r);
        if (page < -1) continue;
        T* row = static_cast<T*>(keys ? a.k : a.v) + (first + r) * row_stride;
        const uint8_t* codes = (keys ? p.k_codes : p.v_codes) + page * p.codes_stride;
        const uint32_t* scales = (keys ? p.k_scales : p.v_scales) + page * p.scales_stride;
        for (int i0 = lane; i0 < n; i0 += 32 * kAhead) {
            uint32_t pair[kAhead], c[kAhead][BITS / 4];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + 32 * k, head = i >> pieces_shift, piece = i & ((1 << pieces_shift) - 1);
                pair[k] = c[k][0] = c[k][BITS / 4 - 1] = 0u;
                if (i >= n || page < 0) continue;
                const int64_t at = (((int64_t)head * p.block_tokens + in_page) << pieces_shift) + piece;
                pair[k] = scales[at >> 3];
                if constexpr (BITS == 4) {
                    c[k][0] = *reinterpret_cast<const uint32_t*>(codes + at * 4);
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(codes + at * 8);
                    c[k][0] = x.x;
                    c[k][1] = x.y;
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + 32 * k, head = i >> pieces_shift, piece = i & ((1 << pieces_shift) - 1);
                if (i < n) *reinterpret_cast<uint4*>(row + head * head_stride + piece * 8) = values_of<T, BITS>(pair[k], c[k]);
            }
        }
    }
}

// Rows of a warp: one where rows are few (a launch of 64 rows of 8 heads of 128 has 128 warps then), four where there are many, so that looking up their places hardly counts (eight leave fewer warps: 12 contexts
// of 8000 tokens 88 us where four take 83), two between (16383 rows written and read: 45 us, with four 48).
template <typename F>
void with_types(const QuantRowsArgs& a, F&& f) {
    auto with_rows = [&](auto type, auto bits) {
        auto run = [&](auto rows) {
            constexpr int kEach = decltype(rows)::value * (kThreads / 32);
            f(type, bits, rows, dim3((unsigned)((a.lanes.total + kEach - 1) / kEach), 2));
        };
        if (a.lanes.total < 4096) run(std::integral_constant<int, 1>{});
        else if (a.lanes.total < 40000) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 4>{});
    };
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    if (a.pools.bf16) a.pools.bits == 4 ? with_rows(__nv_bfloat16{}, Four{}) : with_rows(__nv_bfloat16{}, Eight{});
    else a.pools.bits == 4 ? with_rows(__half{}, Four{}) : with_rows(__half{}, Eight{});
}

}  // namespace

void launch_quantize_rows(const QuantRowsArgs& a, cudaStream_t s) {
    with_types(a, [&](auto type, auto bits, auto rows, dim3 grid) { quantize_rows_kernel<decltype(type), decltype(bits)::value, decltype(rows)::value><<<grid, kThreads, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

void launch_dequantize_rows(const QuantRowsArgs& a, cudaStream_t s) {
    with_types(a, [&](auto type, auto bits, auto rows, dim3 grid) { dequantize_rows_kernel<decltype(type), decltype(bits)::value, decltype(rows)::value><<<grid, kThreads, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

}  // namespace mk
