// Rows of keys and values into pages of 4- or 8-bit codes, and back.
//
// Groups of 64 neighbouring values x_i of a head's row have a lowest value and a step of their own:
//   low = min x_i,  step = (max x_i - low) / L rounded to the rows' type (L = 15 or 255),  c_i = min(L, round((x_i - low) / step)), halves to even, 0 where step is 0;
// c_i stands for low + step c_i.  low is one of the values, so it needs no rounding; the step's is 2^-11 (f16) or 2^-8 (bf16) of it at most and moves no value by more than
// L times that, and since the codes are made with the rounded step they are the nearest ones under it.  A group with a value, or a range, that is not finite reads as NaN throughout.
#include "quantized_kv.h"
#include "attention_math.cuh"
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
};
template <>
struct Two<__nv_bfloat16> {
    static __device__ __forceinline__ float2 wide(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr float largest = 3.3895313892515355e38f;
};

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

// Where a row's token is: its page, or -1 where it has none (rows of no lane, rows in front of a lane's first token, what the arrays should not hold).
struct Place {
    int page, in_page;
    bool mine;   // the row belongs to a lane
};
__device__ __forceinline__ Place place_of_row(const QuantLanes& a, const QuantPools& p, int t) {
    int lane, begin, end;
    if (a.cu == nullptr) {
        lane = t / a.rows;
        begin = lane * a.rows;
        end = begin + a.rows;
    } else {
        lane = lane_of_row(a, t);
        begin = a.cu[lane];
        end = a.cu[lane + 1];
    }
    Place r{-1, 0, t >= begin && t < end};
    if (!r.mine) return r;
    const int length = a.lengths[lane];
    const bool first = (threadIdx.x & 31) == 0;
    if (length < 0 || length > (int64_t)a.width << p.bt_shift) {
        if (first) tell(a.status, kDevBadRange);
        return r;
    }
    const int position = length - (end - t);
    if (position < 0) return r;
    const int page = a.tables[lane * a.ld_table + (position >> p.bt_shift)];
    if (page < 0 || page >= p.pages) {
        if (first) tell(a.status, kDevBadPage);
        return r;
    }
    r.page = page;
    r.in_page = position & (p.block_tokens - 1);
    return r;
}

// A warp has one row of K or V: eight values to a thread, a group to eight threads.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ QuantRowsArgs a) {
    constexpr int L = (1 << BITS) - 1;
    const QuantPools& p = a.pools;
    const int lane = threadIdx.x & 31, t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (t >= a.lanes.total) return;
    const Place at = place_of_row(a.lanes, p, t);
    if (at.page < 0) return;
    const bool keys = blockIdx.y == 0;
    const T* rows = static_cast<const T*>(keys ? a.k : a.v) + t * (keys ? a.k_row : a.v_row);
    const int64_t head_stride = keys ? a.k_head : a.v_head;
    uint8_t* codes = (keys ? p.k_codes : p.v_codes) + at.page * p.codes_stride;
    uint32_t* scales = (keys ? p.k_scales : p.v_scales) + at.page * p.scales_stride;
    const int pieces = p.d / 8, groups = p.d / kQuantGroup;
    for (int i0 = 0; i0 < p.kv_heads * pieces; i0 += 32) {
        const int i = i0 + lane, head = i / pieces, piece = i - head * pieces;
        if (i >= p.kv_heads * pieces) return;   // whole groups of eight threads
        const uint32_t group_mask = 0xffu << (lane & 24);
        const uint4 w = *reinterpret_cast<const uint4*>(rows + head * head_stride + piece * 8);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        float x[8], low = INFINITY, high = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = Two<T>::wide(u[j]);
            x[2 * j] = v.x;
            x[2 * j + 1] = v.y;
            low = min_nan(low, min_nan(v.x, v.y));
            high = max_nan(high, max_nan(v.x, v.y));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            low = min_nan(low, __shfl_xor_sync(group_mask, low, o));
            high = max_nan(high, __shfl_xor_sync(group_mask, high, o));
        }
        const float range = high - low;
        uint32_t pair = Two<T>::pack(__fdiv_rn(range, (float)L), low);
        if (!isfinite(range)) pair = Two<T>::pack(NAN, NAN);
        const float step = Two<T>::wide(pair).x;
        uint32_t word[BITS / 4] = {};
        if (step > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = min((uint32_t)L, (uint32_t)__float2int_rn(__fdiv_rn(x[j] - low, step)));
                word[j * BITS / 32] |= c << (j * BITS % 32);
            }
        }
        const int64_t row = (int64_t)head * p.block_tokens + at.in_page;
        uint8_t* to = codes + row * (p.d * BITS / 8) + piece * BITS;
        if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(to) = word[0];
        else *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
        if ((lane & 7) == 0) scales[row * groups + piece / 8] = pair;
    }
}

// The same the other way; a row without a token becomes zeros, and a value beyond the type's largest that largest (a rounded step may lead there).
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) dequantize_rows_kernel(const __grid_constant__ QuantRowsArgs a) {
    const QuantPools& p = a.pools;
    const int lane = threadIdx.x & 31, t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (t >= a.lanes.total) return;
    const Place at = place_of_row(a.lanes, p, t);
    if (!at.mine) return;
    const bool keys = blockIdx.y == 0;
    T* rows = static_cast<T*>(keys ? a.k : a.v) + t * (keys ? a.k_row : a.v_row);
    const int64_t head_stride = keys ? a.k_head : a.v_head;
    const int page = max(at.page, 0);
    const uint8_t* codes = (keys ? p.k_codes : p.v_codes) + page * p.codes_stride;
    const uint32_t* scales = (keys ? p.k_scales : p.v_scales) + page * p.scales_stride;
    const int pieces = p.d / 8, groups = p.d / kQuantGroup;
    for (int i = lane; i < p.kv_heads * pieces; i += 32) {
        const int head = i / pieces, piece = i - head * pieces;
        uint32_t w[4] = {};
        if (at.page >= 0) {
            const int64_t row = (int64_t)head * p.block_tokens + at.in_page;
            const float2 sl = Two<T>::wide(scales[row * groups + piece / 8]);
            const uint8_t* from = codes + row * (p.d * BITS / 8) + piece * BITS;
            uint32_t c[2];
            if constexpr (BITS == 4) c[0] = *reinterpret_cast<const uint32_t*>(from), c[1] = c[0] >> 16;
            else c[0] = reinterpret_cast<const uint2*>(from)->x, c[1] = reinterpret_cast<const uint2*>(from)->y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int b = (j & 1) * 2 + h;
                    const float y = fmaf(sl.x, (float)(c[j >> 1] >> (b * BITS) & ((1u << BITS) - 1)), sl.y);
                    v[h] = y > Two<T>::largest ? Two<T>::largest : y;   // NaN stays
                }
                w[j] = Two<T>::pack(v[0], v[1]);
            }
        }
        *reinterpret_cast<uint4*>(rows + head * head_stride + piece * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename F>
void with_types(const QuantPools& p, F&& f) {
    if (p.bf16) p.bits == 4 ? f(__nv_bfloat16{}, std::integral_constant<int, 4>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 8>{});
    else p.bits == 4 ? f(__half{}, std::integral_constant<int, 4>{}) : f(__half{}, std::integral_constant<int, 8>{});
}

dim3 row_grid(const QuantRowsArgs& a) { return dim3((unsigned)((a.lanes.total + kThreads / 32 - 1) / (kThreads / 32)), 2); }

}  // namespace

void launch_quantize_rows(const QuantRowsArgs& a, cudaStream_t s) {
    with_types(a.pools, [&](auto type, auto bits) { quantize_rows_kernel<decltype(type), decltype(bits)::value><<<row_grid(a), kThreads, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

void launch_dequantize_rows(const QuantRowsArgs& a, cudaStream_t s) {
    with_types(a.pools, [&](auto type, auto bits) { dequantize_rows_kernel<decltype(type), decltype(bits)::value><<<row_grid(a), kThreads, 0, s>>>(a); });
    MK_LAUNCH_CHECK();
}

}  // namespace mk
