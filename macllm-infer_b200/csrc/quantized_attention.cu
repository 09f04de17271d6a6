// Attention over paged keys and values in 4- or 8-bit codes.
//
// Row t of lane i has position p = length_i - n_i + t and sees the keys max(0, p - window + 1) .. p of the lane's pages:
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(cap(scale q . k_j) - m),
// with k_j and v_j what their codes stand for, low + step c, not rounded to 16 bits.  Scores, weights, maxima and sums are 32-bit.
#include "quantized_attention.h"
#include "kernels.h"

namespace mk {

namespace {

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

template <typename T>
__device__ __forceinline__ float2 wide_pair(uint32_t w) {
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// A warp to a (row, query head): D / 32 values to a thread, one key after the other.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(32) quantized_attention_kernel(const __grid_constant__ QuantAttnArgs a) {
    constexpr int V = D / 32, G = D / kQuantGroup;
    const QuantPools& p = a.pools;
    const int lane_id = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, kvh = head / (a.q_heads / p.kv_heads);
    int first = a.lanes.cu != nullptr ? a.lanes.cu[lane_id] : lane_id * a.lanes.rows, n = a.lanes.cu != nullptr ? a.lanes.cu[lane_id + 1] - first : a.lanes.rows;
    const int length = a.lanes.lengths[lane_id];
    const int keys = (int)min((int64_t)max(length, 0), (int64_t)a.lanes.width << p.bt_shift);
    if (first < 0 || first > a.lanes.total || n < 0 || n > a.lanes.rows || n > a.lanes.total - first || keys != length) {
        if (lane == 0) tell(a.lanes.status, kDevBadRange);
        if (first < 0 || first > a.lanes.total) first = 0, n = 0;
        n = min(max(n, 0), min(a.lanes.rows, a.lanes.total - first));
    }
    for (int r = blockIdx.z; r < n; r += gridDim.z) {
        const int position = keys - n + r;
        const T* q = static_cast<const T*>(a.q) + (int64_t)(first + r) * a.ldq + head * D + lane * V;
        float qv[V], o[V], m = -INFINITY, l = 0.f;
        for (int j = 0; j < V; ++j) qv[j] = (float)q[j], o[j] = 0.f;
        auto value = [&](const uint8_t* codes, const uint32_t* scales, int64_t row, float (&x)[V]) {
            const float2 sl = wide_pair<T>(scales[row * G + lane * V / kQuantGroup]);
            for (int j = 0; j < V; ++j) {
                const int i = lane * V + j;
                const uint32_t c = BITS == 8 ? codes[row * D + i] : codes[row * (D / 2) + i / 2] >> (i % 2 * 4) & 15;
                x[j] = fmaf(sl.x, (float)c, sl.y);
            }
        };
        for (int key = attention_first_key(max(position, 0), a.window, 0); key <= position; ++key) {
            int page = a.lanes.tables[lane_id * a.lanes.ld_table + (key >> p.bt_shift)];
            if (page < 0 || page >= p.pages) {
                if (lane == 0) tell(a.lanes.status, kDevBadPage);
                page = 0;
            }
            const int64_t row = (int64_t)kvh * p.block_tokens + (key & (p.block_tokens - 1));
            float x[V], s = 0.f;
            value(p.k_codes + page * p.codes_stride, p.k_scales + page * p.scales_stride, row, x);
            for (int j = 0; j < V; ++j) s = fmaf(qv[j], x[j], s);
            s = warp_sum(s) * a.scale;
            if (a.softcap != 0.f) s = a.softcap * tanhf(s / a.softcap);
            const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.f : m_new, alpha = expf(m - m_use), w = expf(s - m_use);
            m = m_new;
            l = fmaf(l, alpha, w);
            value(p.v_codes + page * p.codes_stride, p.v_scales + page * p.scales_stride, row, x);
            for (int j = 0; j < V; ++j) o[j] = fmaf(o[j], alpha, w * x[j]);
        }
        T* out = static_cast<T*>(a.out) + (int64_t)(first + r) * a.ldo + head * D + lane * V;
        for (int j = 0; j < V; ++j) out[j] = (T)(l == 0.f ? 0.f : o[j] / l);
    }
}

template <typename T, int BITS>
void launch(const QuantAttnArgs& a, cudaStream_t s) {
    const dim3 grid(a.lanes.lanes, a.q_heads, std::min(a.lanes.rows, 64));
    switch (a.pools.d) {
        case 64: quantized_attention_kernel<T, 64, BITS><<<grid, 32, 0, s>>>(a); break;
        case 128: quantized_attention_kernel<T, 128, BITS><<<grid, 32, 0, s>>>(a); break;
        default: quantized_attention_kernel<T, 256, BITS><<<grid, 32, 0, s>>>(a); break;
    }
    MK_LAUNCH_CHECK();
}

}  // namespace

QuantAttnPlan quantized_attention_plan(int, int, int, int, int, int, int, int, int, int) { return QuantAttnPlan{}; }

void launch_quantized_attention(const QuantAttnArgs& a, const QuantAttnPlan&, void*, cudaStream_t s) {
    if (a.pools.bf16) a.pools.bits == 4 ? launch<__nv_bfloat16, 4>(a, s) : launch<__nv_bfloat16, 8>(a, s);
    else a.pools.bits == 4 ? launch<__half, 4>(a, s) : launch<__half, 8>(a, s);
}

}  // namespace mk
