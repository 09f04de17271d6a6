// Log probabilities of given tokens, with the entropy of their distributions, their ranks and the likeliest tokens.
//
// For a row x of logits with maximum m and Z = sum e^(x_i - m):  log p_i = x_i - m - ln Z,  entropy = -sum p_i log p_i = ln Z - sum e^(x_i - m) (x_i - m) / Z.  The rank of
// a token is its place among all, by falling logit and, among equals, rising token; the likeliest tokens come in that order.
#include "token_logprobs.h"
#include <cuda_bf16.h>

namespace mk {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float wide(T x) { return (float)x; }

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

// The best (value, token) of the block's threads, falling value first, then rising token.
__device__ __forceinline__ void block_best(float& v, int& i, float* red_v, int* red_i) {
    auto better = [](float v0, int i0, float v1, int i1) { return v0 > v1 || (v0 == v1 && i0 < i1); };
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (better(ov, oi, v, i)) v = ov, i = oi;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red_v[threadIdx.x >> 5] = v, red_i[threadIdx.x >> 5] = i;
    __syncthreads();
    v = red_v[0], i = red_i[0];
    for (int w = 1; w < kThreads / 32; ++w)
        if (better(red_v[w], red_i[w], v, i)) v = red_v[w], i = red_i[w];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    __shared__ float red[32];
    __shared__ int red_i[32];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int token = a.tokens[row];
    const bool given = token >= 0 && token < a.vocab;
    const float mine = given ? wide(x[token]) : 0.f;
    float top = -INFINITY, odd = 0.f;
    for (int i = tid; i < a.vocab; i += kThreads) {
        const float v = wide(x[i]);
        top = fmaxf(top, v);
        if (!(v < INFINITY)) odd = 1.f;
    }
    const float m = block_max(top, red);
    const bool bad = block_max(odd, red) != 0.f || m == -INFINITY;
    float z = 0.f, zx = 0.f, before = 0.f;
    if (!bad) {
        for (int i = tid; i < a.vocab; i += kThreads) {
            const float v = wide(x[i]), e = expf(v - m);
            z += e;
            if (v > -INFINITY) zx += e * (v - m);
            if (given && (v > mine || (v == mine && i < token))) before += 1.f;
        }
    }
    z = block_sum(z, red);
    zx = block_sum(zx, red);
    before = block_sum(before, red);
    const float log_z = logf(z);
    if (tid == 0) {
        if (bad) tell(a.status, kDevBadRow);
        if (token >= a.vocab) tell(a.status, kDevBadRange);
        a.logprobs[row] = token < 0 ? 0.f : (given && !bad ? mine - m - log_z : NAN);
        a.entropy[row] = bad ? NAN : log_z - zx / z;
        a.ranks[row] = given && !bad ? (int)before + 1 : 0;
    }
    float last_v = INFINITY;
    int last_i = -1;
    for (int k = 0; k < a.top; ++k) {
        float v = -INFINITY;
        int best = INT32_MAX;
        if (!bad) {
            for (int i = tid; i < a.vocab; i += kThreads) {
                const float y = wide(x[i]);
                if ((y < last_v || (y == last_v && i > last_i)) && (y > v || (y == v && i < best))) v = y, best = i;
            }
        }
        block_best(v, best, red, red_i);
        if (tid == 0) {
            a.top_tokens[row * a.top + k] = bad ? -1 : best;
            a.top_logprobs[row * a.top + k] = bad ? NAN : v - m - log_z;
        }
        last_v = v, last_i = best;
    }
}

}  // namespace

void launch_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
    if (a.kind == 0) token_logprobs_kernel<float><<<a.rows, kThreads, 0, s>>>(a);
    else if (a.kind == 1) token_logprobs_kernel<__half><<<a.rows, kThreads, 0, s>>>(a);
    else token_logprobs_kernel<__nv_bfloat16><<<a.rows, kThreads, 0, s>>>(a);
    MK_LAUNCH_CHECK();
}

}  // namespace mk
