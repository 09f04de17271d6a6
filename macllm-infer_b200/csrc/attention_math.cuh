// Small pieces that attention kernels over pages have in common.
#pragma once
#include "common.cuh"

namespace mk {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// cap * tanh(v / cap) as cap - 2 cap / (1 + exp(2 v / cap)), which rounds in parts of the cap: 2^-14 and less up to kCapOfDifference; NaN of NaN.
constexpr float kCapOfDifference = 256.f;
__device__ __forceinline__ float capped(float v, float cap, float two_over_cap) {
    return cap - __fdividef(2.0f * cap, 1.0f + __expf(min_nan(v * two_over_cap, 80.0f)));
}
// For caps above, by kernels of their own (beside the other in one kernel it cost calls without any cap 1.5 %): with x = v / cap below 1/4 as v (1 - x^2 / 3 + 2 x^4 / 15 - 17 x^6 / 315), whose next term is 3.4e-7 of v; from there on the roundings above are less than 2^-20 of v.
__device__ __forceinline__ float capped_wide(float v, float cap, float two_over_cap) {
    const float x = 0.5f * v * two_over_cap, y = x * x;
    return y < 0.0625f ? v * fmaf(y, fmaf(y, fmaf(y, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f) : capped(v, cap, two_over_cap);
}

// Two 32-bit numbers at once.
struct FloatPair {
    float x, y;
    __device__ __forceinline__ uint64_t bits() const {
        uint64_t b;
        asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(x), "f"(y));
        return b;
    }
    static __device__ __forceinline__ FloatPair of(uint64_t b) {
        FloatPair t;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(t.x), "=f"(t.y) : "l"(b));
        return t;
    }
};
__device__ __forceinline__ FloatPair operator+(FloatPair a, FloatPair b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits()), "l"(b.bits()));
    return FloatPair::of(r);
}
__device__ __forceinline__ FloatPair operator*(FloatPair a, FloatPair b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits()), "l"(b.bits()));
    return FloatPair::of(r);
}
__device__ __forceinline__ FloatPair fma2(FloatPair a, FloatPair b, FloatPair c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.bits()), "l"(b.bits()), "l"(c.bits()));
    return FloatPair::of(r);
}

// The 8 x 8 tile of 16-bit numbers that a warp holds as (row lane / 4, columns 2 (lane % 4), + 1), transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

}  // namespace mk
