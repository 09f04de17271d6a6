// Attention of a batch whose lanes share their first pages.
//
// Row t of lane i has position p = length_i - n_i + t and sees the keys max(0, p - window + 1) .. p of the lane's pages:
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(cap(scale q . k_j) - m).
// Sums over disjoint parts of the keys join exactly: with (m_a, l_a, o_a) and (m_b, l_b, o_b) of two parts and m = max(m_a, m_b), l = l_a e^(m_a - m) +
// l_b e^(m_b - m), o likewise.  Maxima, sums and outputs of parts are 32-bit; weights are rounded to the pools' type for the product with V, as the
// result itself is at the end.
#include "shared_attention.h"
#include "attention_math.cuh"
#include "hgemm_tc.h"
#include "kernels.h"
#include "tile_phases.h"
#include "umma.cuh"
#include <cuda.h>
#include <cuda_bf16.h>
#include <algorithm>
#include <type_traits>

namespace mk {

namespace {

using namespace umma;

constexpr int kSms = 148;   // calls are cut without a device, for a B200

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {   // zeros where there is nothing
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Two warps at a named barrier, one of which waits for the other.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void pair_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

// Where a lane's rows and keys are; whatever the arrays hold, rows stay inside [0, total) and keys inside the table.
struct LaneRange {
    int first, n;       // rows
    int position;       // of its first row
    int keys;           // length, at most what the table holds
};
__device__ __forceinline__ LaneRange lane_range(const SharedAttnArgs& a, int lane) {
    LaneRange r;
    r.first = a.cu != nullptr ? a.cu[lane] : lane * a.rows;
    r.n = a.cu != nullptr ? a.cu[lane + 1] - r.first : a.rows;
    const int length = a.lengths[lane];
    r.keys = min(max(length, 0), a.width << a.bt_shift);
    if (r.first < 0 || r.first > a.total || r.n < 0 || r.n > a.rows || r.n > a.total - r.first || r.keys != length) {
        tell(a.status, kDevBadRange);
        if (r.first < 0 || r.first > a.total) r.first = 0, r.n = 0;
        r.n = min(max(r.n, 0), min(a.rows, a.total - r.first));
    }
    r.position = r.keys - r.n;
    return r;
}

// The parts [first, first + parts) of a row's results, added to a warp's (m, l, o), V values of o per thread.
template <int D, int AHEAD>
__device__ __forceinline__ void add_parts(const SharedAttnArgs& a, int64_t row, int parts, float& m, float& l, float (&o)[D / 32]) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t n_rows = (int64_t)a.total * a.q_heads;
    for (int s0 = 0; s0 < parts; s0 += 32) {
        const float2 ml = s0 + lane < parts ? __ldcg(a.part_ml + (s0 + lane) * n_rows + row) : make_float2(-INFINITY, 0.f);
        const float m_new = fmaxf(m, warp_max(ml.x)), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float old = ex2(m - m_use), f = ml.y == 0.f ? 0.f : ex2(ml.x - m_use);
        const uint32_t wrote = __ballot_sync(0xffffffffu, ml.y != 0.f);   // not by weights: one of 0 does not hide NaN
        l = l * old + warp_sum(ml.y * f);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] *= old;
        m = m_new;
        const int n = min(32, parts - s0);
        // AHEAD parts at a time, none of which waits for another's values where the compiler keeps their loads together (heads of 64 and 256: 100 registers; at heads of 128 it takes 48 and
        // the loads come one after the other); one without keys wrote no output
        for (int b = 0; b < n; b += AHEAD) {
            float x[AHEAD][V], w[AHEAD];
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
                w[s] = b + s < 32 ? __shfl_sync(0xffffffffu, f, b + s) : 0.f;
#pragma unroll
                for (int j = 0; j < V; ++j) x[s][j] = 0.f;
                if (b + s >= 32 || !(wrote >> (b + s) & 1u)) continue;
                const float* src = a.part_o + ((s0 + b + s) * n_rows + row) * D + lane * V;
                if constexpr (V == 2) {
                    const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
                    x[s][0] = y.x; x[s][1] = y.y;
                } else {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(src + j));
                        x[s][j] = y.x; x[s][j + 1] = y.y; x[s][j + 2] = y.z; x[s][j + 3] = y.w;
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < AHEAD; ++s)
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] += x[s][j] * w[s];
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* out, const float (&o)[V], float l) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;   // a row that sees nothing: zeros
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V; j += 2) w[j / 2] = Pair<T>::pack(o[j] * inv, o[j + 1] * inv);
    if constexpr (V == 2) *reinterpret_cast<uint32_t*>(out) = w[0];
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- a lane's keys -----------------------------------------------------------------------------------------------
//
// A CTA takes a share of one lane's keys for NT * 8 (row, head) items of one KV head.  Each of its warps walks tiles of 16 keys, which TMA brings into a ring of its own; the
// items are the short side of both products: S^T = K Q^T, O^T = V^T P^T.  What bounds it is HBM where lanes have much of their own, else the chain of dependent fetches at a
// CTA's two ends: so a warp asks for its first tiles before anything else, rings are short enough for three CTAs on an SM, and warps with one tile on its way each do better than
// half as many with two (heads of 256: 92 us where those take 104; heads of 64, 4 lanes of 1 to 60 keys: 8 warps 8.3 us, 4 warps 10.1, but 18 where 8 take 22 with two groups of items).
// 40 lanes of 16 heads of 256 over 8 with 300 to 4000 keys of their own: 79 us, 6.0 TB/s; 128 lanes of 32 heads of 128 over 8 with 20 to 700: 34 us, 3.0 TB/s.
constexpr int kTile = 16;

template <int D, int NT>
struct LaneSmem {
    static constexpr int WARPS = D == 64 && NT == 1 ? 8 : 4, THREADS = WARPS * 32;
    static constexpr int PANELS = D / 64, K_BYTES = kTile * D * 2, STAGE = 2 * K_BYTES;
    static constexpr int STAGES = 65536 / (WARPS * STAGE);   // at most
    static constexpr int QP = D + 8, OP = D + 4;
    __host__ __device__ static int ring(int stages) { return (max(stages * STAGE, NT * 8 * (OP + 2) * 4) + 1023) / 1024 * 1024; }
    static size_t bytes(int stages) { return 1024 + (size_t)WARPS * ring(stages) + (size_t)NT * 8 * QP * 2; }
};

template <typename T, int D, int NT, bool WIDE>
__global__ void __launch_bounds__(LaneSmem<D, NT>::THREADS) lane_keys_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ SharedAttnArgs a,
                                                                                   int chunk, int shares, int shared_parts, int join, int stage_bits) {
    using L = LaneSmem<D, NT>;
    using P = Pair<T>;
    constexpr int ITEMS = NT * 8, kWarps = L::WARPS;
    const int stages = 1 << stage_bits, ring_bytes = L::ring(stages);
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[kWarps * L::STAGES];
    uint8_t* rings = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    T* qs = reinterpret_cast<T*>(rings + kWarps * ring_bytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tq = lane & 3;
    const int lane_id = blockIdx.x / shares, share = blockIdx.x - lane_id * shares, kvh = blockIdx.y, g = a.q_heads / a.kv_heads;
    const LaneRange at = lane_range(a, lane_id);
    const int item0 = blockIdx.z * ITEMS, n_items = min(ITEMS, at.n * g - item0);
    if (n_items <= 0) {
        pdl_wait();   // also where no lane has rows, nobody behind this kernel overtakes the one before it
        return;
    }
    const int first_key = a.shared;
    const int p0 = at.position + item0 / g, p1 = at.position + (item0 + n_items - 1) / g;
    const int lo = max(first_key + share * chunk, attention_first_key(max(p0, 0), a.window, 0)), hi = min(min(p1 + 1, at.keys), shares > 1 ? first_key + (share + 1) * chunk : INT_MAX);
    const int begin = lo / kTile * kTile, n_tiles = hi > lo ? (hi - begin + kTile - 1) / kTile : 0;
    const int my_tiles = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;

    uint8_t* ring = rings + warp * ring_bytes;
    uint64_t* full = bars + warp * L::STAGES;
    const int32_t* table = a.tables + lane_id * a.ld_table;
    auto page_row = [&](int i) {
        const int pos = begin + (warp + kWarps * i) * kTile;
        int32_t page = table[pos >> a.bt_shift];
        if ((uint32_t)page >= (uint64_t)a.pool_pages) {
            tell(a.status, kDevBadPage);
            page = 0;
        }
        return (int)(page * a.page_rows) + kvh * a.block_tokens + (pos & (a.block_tokens - 1));
    };
    auto load_tile = [&](int i, int row) {   // one lane
        const int st = i & (stages - 1);
        const uint32_t dst = smem_u32(ring) + st * L::STAGE;
        bar_expect_tx(&full[st], L::STAGE);
#pragma unroll
        for (int p = 0; p < L::PANELS; ++p) {
            tma_load_2d(dst + p * (kTile * 128), &tm_k, p * 64, row, &full[st]);
            tma_load_2d(dst + L::K_BYTES + p * (kTile * 128), &tm_v, p * 64, row, &full[st]);
        }
    };
    int next_row = 0;   // of the tile that the ring takes next
    if (lane == 0 && my_tiles > 0) {
        const int ahead = min(stages, my_tiles);
        int rows[L::STAGES];
#pragma unroll
        for (int i = 0; i < L::STAGES; ++i) rows[i] = i < ahead ? page_row(i) : 0;
        next_row = stages < my_tiles ? page_row(stages) : 0;
        for (int i = 0; i < stages; ++i) bar_init(&full[i], 1);
        bar_init_fence();
#pragma unroll
        for (int i = 0; i < L::STAGES; ++i)
            if (i < ahead) load_tile(i, rows[i]);
    }
    for (int i = tid; i < ITEMS * (D / 8); i += L::THREADS) {
        const int item = i / (D / 8), c = (i - item * (D / 8)) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (item < n_items) {
            const int r = (item0 + item) / g, hq = (item0 + item) - r * g;
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(at.first + r) * a.ldq + (kvh * g + hq) * D + c);
        }
        *reinterpret_cast<uint4*>(qs + item * L::QP + c) = v;
    }
    __syncthreads();

    float o_acc[NT][D / 16][4], m_run[NT][2], l_run[NT][2];
    int see_lo[NT][2], see_hi[NT][2];   // keys that the lane's two items of a group of eight see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o_acc[n][j][0] = o_acc[n][j][1] = o_acc[n][j][2] = o_acc[n][j][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m_run[n][h] = -INFINITY;
            l_run[n][h] = 0.f;
            const int p = at.position + (item0 + n * 8 + 2 * tq + h) / g;
            see_lo[n][h] = max(lo, attention_first_key(max(p, 0), a.window, 0));
            see_hi[n][h] = min(hi, p + 1);
        }
    }
    const int all_lo = max(lo, attention_first_key(max(p1, 0), a.window, 0)), all_hi = min(hi, p0 + 1);   // keys that every item sees
    const float two_over_cap = a.softcap != 0.f ? 2.0f / a.softcap : 0.f, unit = a.softcap != 0.f ? a.scale : a.scale * kLog2e;
    const uint32_t q_at = smem_u32(qs) + (uint32_t)((lane & 7) * L::QP + (lane >> 3) * 8) * 2;
    bool ok = true;
    for (int i = 0; i < my_tiles; ++i) {
        const int st = i & (stages - 1);
        ok = __all_sync(0xffffffffu, bar_wait(&full[st], i >> stage_bits & 1));
        if (!ok) {
            if (lane == 0) tell(a.status, kDevWait);
            break;
        }
        const uint32_t kt = smem_u32(ring) + st * L::STAGE, vt = kt + L::K_BYTES;
        const int pos0 = begin + (warp + kWarps * i) * kTile;
        if (pos0 + kTile > hi) {   // rows behind the last key hold whatever the page held: weights of 0 need finite values there
            for (int j = lane; j < (kTile - (hi - pos0)) * 8 * L::PANELS; j += 32) {
                const int r = hi - pos0 + j / (8 * L::PANELS), c = j % (8 * L::PANELS);
                *reinterpret_cast<uint4*>(ring + st * L::STAGE + L::K_BYTES + (c >> 3) * (kTile * 128) + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            __syncwarp();
        }
        float sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
        const int kr = lane & 15;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
            uint32_t a0[4], a1[4];
            const uint32_t base = kt + (kk >> 1) * (kTile * 128) + kr * 128;
            const int cb = (kk & 1) * 64 + (lane >> 4) * 16;
            ldmatrix_x4(a0, base + (cb ^ ((kr & 7) << 4)));
            ldmatrix_x4(a1, base + ((cb + 32) ^ ((kr & 7) << 4)));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t b[4];
                ldmatrix_x4(b, q_at + (uint32_t)(n * 8 * L::QP + kk * 32) * 2);
                P::mma(sc[n], a0, b[0], b[1]);
                P::mma(sc[n], a1, b[2], b[3]);
            }
        }
        const bool whole = pos0 >= all_lo && pos0 + kTile <= all_hi;
        uint32_t b0[NT], b1[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int pos = pos0 + gid + 8 * (e >> 1);
                float v = sc[n][e] * unit;
                if (WIDE) v = capped_wide(v, a.softcap, two_over_cap) * kLog2e;
                else if (a.softcap != 0.f) v = capped(v, a.softcap, two_over_cap) * kLog2e;
                sc[n][e] = whole || (pos >= see_lo[n][e & 1] && pos < see_hi[n][e & 1]) ? v : -INFINITY;
            }
            float alpha[2], m_use[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float top = fmaxf(sc[n][h], sc[n][2 + h]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float m_new = fmaxf(m_run[n][h], top);
                m_use[h] = m_new == -INFINITY ? 0.f : m_new;
                alpha[h] = ex2(m_run[n][h] - m_use[h]);
                m_run[n][h] = m_new;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = ex2(sc[n][e] - m_use[e & 1]);
            l_run[n][0] = l_run[n][0] * alpha[0] + (sc[n][0] + sc[n][2]);
            l_run[n][1] = l_run[n][1] * alpha[1] + (sc[n][1] + sc[n][3]);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                o_acc[n][j][0] *= alpha[0];
                o_acc[n][j][1] *= alpha[1];
                o_acc[n][j][2] *= alpha[0];
                o_acc[n][j][3] *= alpha[1];
            }
            b0[n] = transpose_8x8(P::pack(sc[n][0], sc[n][1]));
            b1[n] = transpose_8x8(P::pack(sc[n][2], sc[n][3]));
        }
        const int vr = (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            uint32_t af[4];
            ldmatrix_x4_trans(af, vt + (j >> 2) * (kTile * 128) + vr * 128 + (((j & 3) * 32 + ((lane >> 3) & 1) * 16) ^ ((vr & 7) << 4)));
#pragma unroll
            for (int n = 0; n < NT; ++n) P::mma(o_acc[n][j], af, b0[n], b1[n]);
        }
        __syncwarp();
        if (lane == 0 && i + stages < my_tiles) {
            load_tile(i + stages, next_row);
            if (i + stages + 1 < my_tiles) next_row = page_row(i + stages + 1);
        }
    }
    if (!ok) {   // what this warp still has under way lands before the CTA ends; the result says so
        for (int i = 0; i < stages; ++i)
            if (i < my_tiles) bar_wait(&full[i], 0), bar_wait(&full[i], 1);
#pragma unroll
        for (int n = 0; n < NT; ++n) l_run[n][0] = l_run[n][1] = m_run[n][0] = m_run[n][1] = __int_as_float(0x7fffffff);
    }
    __syncwarp();
    // the warps' results meet in the rings
    float* w_o = reinterpret_cast<float*>(ring);
    float* w_ml = w_o + ITEMS * L::OP;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = l_run[n][h];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int item = n * 8 + 2 * tq + h;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                w_o[item * L::OP + j * 16 + gid] = o_acc[n][j][h];
                w_o[item * L::OP + j * 16 + gid + 8] = o_acc[n][j][2 + h];
            }
            if (gid == 0) {
                w_ml[item * 2] = m_run[n][h];
                w_ml[item * 2 + 1] = l;
            }
        }
    __syncthreads();
    constexpr int V = D / 32;
    const int step = ring_bytes / 4;
    const float* first = reinterpret_cast<const float*>(rings);
    pdl_wait();   // the shared keys' parts; and who comes after this kernel may rely on them too
    for (int item = warp; item < n_items; item += kWarps) {
        const int r = (item0 + item) / g, hq = item0 + item - r * g;
        float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = first[w * step + ITEMS * L::OP + item * 2];
            m = mw > m || mw != mw ? mw : m;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(first[w * step + ITEMS * L::OP + item * 2] - m_use);
            const float* x = first + w * step + item * L::OP + lane * V;
            l += first[w * step + ITEMS * L::OP + item * 2 + 1] * f;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] += x[j] * f;
        }
        const int64_t row = at.first + r, head = kvh * g + hq;
        if (join) {
            add_parts<D, 256 / D * 4>(a, row * a.q_heads + head, shared_parts, m, l, o);
            store_row<T, V>(static_cast<T*>(a.out) + row * a.ldo + head * D + lane * V, o, l);
        } else {
            const int64_t slot = ((int64_t)(shared_parts + share) * a.total + row) * a.q_heads + head;
            if (l != 0.f) {
#pragma unroll
                for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(a.part_o + slot * D + lane * V + j) = make_float2(o[j], o[j + 1]);
            }
            if (lane == 0) a.part_ml[slot] = make_float2(m, l);
        }
    }
}

// The parts of a row, joined: a warp per (row, head).
template <typename T, int D>
__global__ void __launch_bounds__(256) join_parts_kernel(const __grid_constant__ SharedAttnArgs a, int parts) {
    constexpr int V = D / 32;   // values of a thread
    pdl_wait();
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= (int64_t)a.total * a.q_heads) return;
    const int token = (int)(row / a.q_heads);
    if (a.cu != nullptr && (token < a.cu[0] || token >= a.cu[a.lanes])) return;
    float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = 0.f;
    add_parts<D, 32 / (D / 64)>(a, row, parts, m, l, o);
    store_row<T, V>(static_cast<T*>(a.out) + token * a.ldo + (row - (int64_t)token * a.q_heads) * D + lane * V, o, l);
}

// ---- the shared keys ---------------------------------------------------------------------------------------------
//
// All rows of the batch see the same keys, so they are the rows of one tall product: the (row, head) items of a KV head in tiles of 128, NQ tiles to a CTA, over a share of
// the keys in tiles of 64.  One warp brings keys and values by TMA (two with two tiles of items: a page of 16 tokens is 2 KB a box,
// and one warp's requests, sixteen a tile of keys, bounded the kernel at 2000 clocks for two tiles of items), one per tile of items issues the tcgen05 products, four do its softmax, a thread per item.  Scores of a tile
// of keys go to one of two areas of tensor memory that a tile of items has; its weights go back over its scores, as the A operand of O += P V; the scores of the next tile are
// made meanwhile.  With two tiles of items a key is fetched once for both; with one, two CTAs share an SM.  The running maximum follows only when a tile exceeds it by kSlack
// (weights stay below 2^kSlack).
//
// What bounds it, for two tiles of items and a tile of keys: the exponentials, 16 per clock and SM, take 1024 clocks; at heads of 128 the products take 1280 (measured alone: 48 clocks for
// 16 dimensions of 128 x 64 scores, whose operands shared memory delivers in that time, 65 for 16 keys of 128 x 128 outputs); at heads of 64 half of that.  Left alone, the warps that
// share a quarter of the SM fall into step and the exponential unit idles while both do the rest, so they take turns (a tile of keys, when that was built: heads of 64 1850 clocks, 1470 so; heads of 128 2000 and 1850).
// 128 lanes of 32 heads of 128 over 8 behind 32768 shared tokens: 73 us, 940 TFLOP/s, the tensor pipe 54 % and the exponential unit 55 % busy; 24 lanes of 16 heads over 4 with up to
// five rows behind 16384: 27 us.
constexpr float kSlack = 8.f;
constexpr int kItems = 128, kKeys = 64;

template <int D, int NQ>
struct SharedSmem {
    static constexpr int PANELS = D / 64, PANEL = kKeys * 128, QPANEL = kItems * 128, BYTES = PANELS * PANEL;
    static constexpr int STAGES = D == 256 || (D == 128 && NQ == 1) ? 2 : (D == 128 ? 4 : (NQ == 1 ? 5 : 6)), WARPS = NQ * 4, LOADERS = NQ, THREADS = (WARPS + LOADERS + NQ) * 32;   // WARPS: of the softmax
    static constexpr int CTAS = NQ == 1 && D <= 128 ? 2 : 1, TMEM = NQ * (D + 2 * kKeys) <= 256 ? 256 : 512;
    static constexpr size_t SMEM = 1024 + (size_t)NQ * PANELS * QPANEL + (size_t)STAGES * 2 * BYTES;
};

// OWN: the same for one lane's rows and its own keys, where a lane has so many (row, head) items that the small products of lane_keys_kernel would be made over and over.
template <typename T, int D, int NQ, bool OWN, bool WIDE>
__global__ void __launch_bounds__(SharedSmem<D, NQ>::THREADS, SharedSmem<D, NQ>::CTAS)
shared_keys_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ SharedAttnArgs a, int box, int splits, int chunk,
                   int lane_tiles, int first_part) {
    using L = SharedSmem<D, NQ>;
    constexpr int ST = L::STAGES, KEYS = kKeys, S_AT = NQ * D, AREAS = 2 * NQ;   // columns of tensor memory: outputs, then the areas
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[4 * ST + 3 * AREAS + 1 + NQ];
    __shared__ uint32_t tmem_slot;
    __shared__ int4 sees[L::WARPS];
    uint64_t *k_full = bars, *k_empty = bars + ST, *v_full = bars + 2 * ST, *v_empty = bars + 3 * ST, *s_full = bars + 4 * ST, *p_full = s_full + AREAS, *o_done = p_full + AREAS,
             *q_full = o_done + AREAS, *drained = q_full + 1;
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ks = qs + NQ * L::PANELS * L::QPANEL;
    uint8_t* vs = ks + ST * L::BYTES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = a.q_heads / a.kv_heads;
    const int split = blockIdx.x % splits, kvh = blockIdx.x / splits % a.kv_heads, block = blockIdx.x / splits / a.kv_heads, lane_id = OWN ? block / lane_tiles : 0,
              tile = OWN ? block - lane_id * lane_tiles : block;
    const LaneRange mine_range = OWN ? lane_range(a, lane_id) : LaneRange{0, a.total, 0, 0};
    if (OWN && tile * (NQ * kItems) >= mine_range.n * g) {
        pdl_wait();
        return;
    }
    const int base_key = OWN ? a.shared : 0, keys_end = OWN ? min(mine_range.keys, a.shared + (split + 1) * chunk) : a.shared;   // positions of tiles are counted from the first
    const int32_t* table = a.tables + lane_id * a.ld_table;
    constexpr bool kEarly = !OWN;
    const int all_tiles = (a.shared + KEYS - 1) / KEYS, first_tile = OWN ? split * chunk / KEYS : (int)((int64_t)all_tiles * split / splits),
              last_tile = OWN ? max(first_tile, (keys_end - base_key + KEYS - 1) / KEYS) : (int)((int64_t)all_tiles * (split + 1) / splits);
    // two loaders, one for keys and one for values, or one for both
    const bool loads = warp >= L::WARPS && warp < L::WARPS + L::LOADERS, loads_k = warp == L::WARPS, loads_v = warp == L::WARPS + L::LOADERS - 1;
    if (loads && lane == 0) {
        for (int i = 0; i < ST; ++i) {
            if (loads_k) {
                bar_init(&k_full[i], 1);
                bar_init(&k_empty[i], NQ);
            }
            if (loads_v) {
                bar_init(&v_full[i], 1);
                bar_init(&v_empty[i], NQ);
            }
        }
        bar_init_fence();
    }
    if (warp == L::WARPS + L::LOADERS) {
        if (lane == 0) {
            for (int i = 0; i < 2 * NQ; ++i) {
                bar_init(&s_full[i], 1);
                bar_init(&p_full[i], 4);
                bar_init(&o_done[i], 1);
            }
            bar_init(q_full, L::WARPS);
            for (int i = 0; i < NQ; ++i) bar_init(&drained[i], 1);
            bar_init_fence();
        }
        __syncwarp();
        tmem_alloc(&tmem_slot, L::TMEM);
        // Not before: a kernel behind this one (the own-keys form) holds tensor memory while it waits for this grid's end, which must not wait for that memory.
        pdl_trigger();
    }
    // The queries' pieces and the first tiles of keys and values are on their way before anything else is looked at (one after the other the queries took 0.6 us a piece, 10 us at
    // heads of 128).
    const int boxes = KEYS / box, of = lane % boxes, panel = lane / boxes;   // at most four boxes of each of the panels: 16
    const bool brings = loads && panel < L::PANELS;
    const int most_tiles = a.window != 0 && !OWN ? all_tiles : last_tile;
    auto page_row = [&](int t) {
        int pos = base_key + t * KEYS + of * box;
        if (pos >= keys_end) pos = (keys_end - 1) / box * box;   // keys behind the last one are not seen; they are read from where there is something
        int32_t page = brings && t < most_tiles ? table[pos >> a.bt_shift] : 0;
        if ((uint32_t)page >= (uint64_t)a.pool_pages) {
            tell(a.status, kDevBadPage);
            page = 0;
        }
        return (int)(page * a.page_rows) + kvh * a.block_tokens + (pos & (a.block_tokens - 1));
    };
    auto bring_k = [&](int st, int row) {
        if (lane == 0) bar_expect_tx(&k_full[st], L::BYTES);
        __syncwarp();
        if (brings) tma_load_2d(smem_u32(ks) + st * L::BYTES + panel * L::PANEL + of * box * 128, &tm_k, panel * 64, row, &k_full[st]);
    };
    auto bring_v = [&](int st, int row) {
        if (lane == 0) bar_expect_tx(&v_full[st], L::BYTES);
        __syncwarp();
        if (brings) tma_load_2d(smem_u32(vs) + st * L::BYTES + panel * L::PANEL + of * box * 128, &tm_v, panel * 64, row, &v_full[st]);
    };
    int early = 0;   // tiles asked for here; where there is a window, what is seen has to be known first
    if (kEarly && loads && a.window == 0) {
        __syncwarp();
        asm volatile("bar.arrive 15, %0;" ::"n"(L::THREADS) : "memory");
        early = min(ST, last_tile - first_tile);
        int rows[ST];
#pragma unroll
        for (int i = 0; i < ST; ++i) rows[i] = page_row(first_tile + i);
#pragma unroll
        for (int i = 0; i < ST; ++i)
            if (i < early) {
                if (loads_k) bring_k(i, rows[i]);
                if (loads_v) bring_v(i, rows[i]);
            }
    }
    const int q = warp >> 2, item = tile * (NQ * kItems) + tid, at_row = item / g, at_token = mine_range.first + at_row;   // total * q_heads is far below 2^31
    const bool exists = at_row < mine_range.n;   // of the batch, or of the lane
    if (warp < L::WARPS) {
        // eight threads to a piece of 128 bytes; where a row is comes from the thread whose item it is
        const int64_t mine = exists ? at_token * a.ldq + (kvh * g + item - at_row * g) * D : -1;
        const uint32_t to = smem_u32(qs) + q * L::PANELS * L::QPANEL + (warp & 3) * 32 * 128;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = k * 4 + lane / 8, c = lane % 8;
            const int64_t at = __shfl_sync(0xffffffffu, mine, r);
#pragma unroll
            for (int p = 0; p < L::PANELS; ++p)
                cp_async16(to + p * L::QPANEL + r * 128 + ((c ^ (r & 7)) << 4), static_cast<const T*>(a.q) + (at < 0 ? 0 : at + p * 64 + c * 8), at >= 0);
        }
    }
    // what this thread's item is, and what it sees
    int token = -1, head = 0, see_lo = 0, see_hi = 0;
    if (warp < L::WARPS) {
        if (exists) {
            LaneRange at = mine_range;
            if (!OWN) {
                int l = 0;
                if (a.cu == nullptr) {
                    l = at_token / a.rows;
                } else {   // the last lane that begins at or before this row
                    int hi = a.lanes;
                    while (hi - l > 1) {
                        const int mid = (l + hi) / 2;
                        if (a.cu[mid] <= at_token) l = mid;
                        else hi = mid;
                    }
                }
                at = lane_range(a, l);
            }
            if (at_token >= at.first && at_token < at.first + at.n) {
                token = at_token;
                head = kvh * g + item - at_row * g;
                const int p = at.position + token - at.first;
                see_lo = max(base_key, attention_first_key(max(p, 0), a.window, 0));
                see_hi = min(keys_end, p + 1);
            }
        }
        const bool live = token >= 0 && see_hi > see_lo;
        const int4 s = make_int4(__reduce_min_sync(0xffffffffu, live ? see_lo : INT_MAX), __reduce_max_sync(0xffffffffu, token >= 0 ? see_lo : 0),
                                 __reduce_min_sync(0xffffffffu, token >= 0 ? see_hi : INT_MAX), __reduce_max_sync(0xffffffffu, live ? see_hi : 0));
        if (lane == 0) sees[warp] = s;
    }
    fence_before();
    // nobody waits for the loader's first requests, and it needs nothing of the others where there is no window
    if (!kEarly || !loads || a.window != 0) asm volatile("bar.sync 15, %0;" ::"n"(L::THREADS) : "memory");
    fence_after();
    const uint32_t tmem = tmem_slot;
    int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = 0;
#pragma unroll
    for (int w = 0; w < L::WARPS; ++w) {
        lo_min = min(lo_min, sees[w].x);
        lo_max = max(lo_max, sees[w].y);
        hi_min = min(hi_min, sees[w].z);
        hi_max = max(hi_max, sees[w].w);
    }
    int t_begin = first_tile, t_end = last_tile;
    if (a.window != 0) {   // only what some item sees, shared out anew where all CTAs of the same items see it alike
        const int low = (min(lo_min, INT_MAX / 2) - base_key) / KEYS, high = (hi_max - base_key + KEYS - 1) / KEYS;
        t_begin = OWN ? max(first_tile, low) : low + (int)((int64_t)max(0, high - low) * split / splits);
        t_end = OWN ? min(last_tile, high) : low + (int)((int64_t)max(0, high - low) * (split + 1) / splits);
    }
    const int n_tiles = max(0, t_end - t_begin);

    if (loads) {
        // ---- loader
        bool ok = true;
        int t = early, row = page_row(t_begin + t);
        for (; t < n_tiles; ++t) {
            const int next = page_row(t_begin + t + 1), st = t % ST;
            const uint32_t ph = (uint32_t)(t / ST & 1) ^ 1;
            if (loads_k) {
                ok = __all_sync(0xffffffffu, bar_wait(&k_empty[st], ph));
                if (!ok) break;
                bring_k(st, row);
            }
            if (loads_v) {
                ok = __all_sync(0xffffffffu, bar_wait(&v_empty[st], ph));
                if (!ok) break;
                bring_v(st, row);
            }
            row = next;
        }
        if (!ok && lane == 0) tell(a.status, kDevWait);
        for (int u = max(0, t - ST); u <= t && u < n_tiles; ++u) {   // copies in flight land before the CTA ends, also where the others gave up
            if (loads_k && (u < t || loads_v)) bar_wait(&k_full[u % ST], u / ST & 1);
            if (loads_v && u < t) bar_wait(&v_full[u % ST], u / ST & 1);
        }
    } else if (warp >= L::WARPS + L::LOADERS) {
        // ---- products, a warp per tile of items: the one's waits pass under the other's products.  The whole warp walks along, so that descriptors and addresses are the same for
        // all of it, and one elected thread issues (a lane of its own: 2500 clocks a tile of keys, 100 a product)
        if (n_tiles > 0) {
            constexpr uint32_t kind = std::is_same<T, __nv_bfloat16>::value ? 1u << 7 | 1u << 10 : 0u;
            constexpr uint32_t i_scores = f16_idesc(kItems, KEYS, false) | kind, i_out = f16_idesc(kItems, D, true) | kind;
            const int q = NQ == 1 ? 0 : __shfl_sync(0xffffffffu, warp, 0) - L::WARPS - L::LOADERS;
            const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0), s_base = base + S_AT + q * 2 * KEYS, o_base = base + q * D;
            const uint64_t q_desc = sw128_desc(smem_u32(qs) + q * L::PANELS * L::QPANEL), k_desc = sw128_desc(smem_u32(ks)), v_desc = sw128_desc(smem_u32(vs), L::PANEL);
            const bool issues = elect_one();
            auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity)) != 0; };
            auto scores = [&](int t) {
                const int st = t % ST, at = tile_phase(t).at;
                if (!wait(&k_full[st], t / ST & 1)) return false;
                fence_after();
                if (issues) {
                    const uint64_t kd = k_desc + st * (L::BYTES / 16);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        mma(s_base + at * KEYS, q_desc + (i >> 2) * (L::QPANEL / 16) + (i & 3) * 2, kd + (i >> 2) * (L::PANEL / 16) + (i & 3) * 2, i_scores, i > 0);
                    commit(&k_empty[st]);
                    commit(&s_full[q * 2 + at]);
                }
                __syncwarp();
                return true;
            };
            bool ok = wait(q_full, 0);
            fence_after();
            ok = ok && scores(0);
            for (int t = 0; t < n_tiles && ok; ++t) {
                const int st = t % ST;
                const TilePhase ph = tile_phase(t);
                // the scores of tile t + 1 go where the weights of tile t - 1 were: their product was issued before, and products of one thread run in their order
                if (t + 1 < n_tiles) ok = scores(t + 1);
                ok = ok && wait(&v_full[st], t / ST & 1) && wait(&p_full[q * 2 + ph.at], ph.parity);
                if (!ok) break;
                fence_after();
                if (issues) {
                    const uint64_t vd = v_desc + st * (L::BYTES / 16);
#pragma unroll
                    for (int i = 0; i < KEYS / 16; ++i) mma_tmem_a(o_base, s_base + ph.at * KEYS + i * 8, vd + i * 128, i_out, t > 0 || i > 0);
                    commit(&v_empty[st]);
                    commit(&o_done[q * 2 + ph.at]);
                }
                __syncwarp();
            }
            if (!ok) {   // products under way end before their operands' memory is given back
                if (lane == 0) tell(a.status, kDevWait);
                if (issues) commit(&drained[q]);
                wait(&drained[q], 0);
            }
        }
    } else {
        // ---- softmax, an item per thread
        cp_async_wait_all();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) bar_arrive(q_full);

        const uint32_t my = tmem + ((uint32_t)((warp & 3) * 32) << 16), o_at = my + q * D;
        const float two_over_cap = a.softcap != 0.f ? 2.0f / a.softcap : 0.f, unit = a.softcap != 0.f ? kLog2e : a.scale * kLog2e;
        const int turn = 1 + (warp & 3) * 2;   // named barriers of the two warps, one for either's turn
        float m_run = -INFINITY, sum = 0.f;   // the maximum as a base-2 logarithm
        bool ok = true;   // once a wait gave up nothing is waited for any more, but every step is taken: the other warp counts on it
        if (NQ == 2 && q == 1 && n_tiles > 0) pair_arrive(turn);
        for (int t = 0; t < n_tiles; ++t) {
            const TilePhase ph = tile_phase(t);
            ok = ok && bar_wait(&s_full[q * 2 + ph.at], ph.parity);
            __syncwarp();
            fence_after();
            const uint32_t s_at = my + S_AT + (q * 2 + ph.at) * KEYS;
            float s[KEYS];
            tmem_ld32(s_at, reinterpret_cast<uint32_t*>(s));
            tmem_ld32(s_at + 32, reinterpret_cast<uint32_t*>(s) + 32);
            tmem_wait_ld();
            const int pos0 = base_key + (t_begin + t) * KEYS;
            if (WIDE) {
#pragma unroll
                for (int j = 0; j < KEYS; ++j) s[j] = capped_wide(s[j] * a.scale, a.softcap, two_over_cap);
            } else if (a.softcap != 0.f) {
#pragma unroll
                for (int j = 0; j < KEYS; ++j) s[j] = capped(s[j] * a.scale, a.softcap, two_over_cap);
            }
            if (pos0 + KEYS > hi_min || pos0 < lo_max) {   // uniform: some item does not see the whole tile
#pragma unroll
                for (int j = 0; j < KEYS; ++j) s[j] = pos0 + j >= see_lo && pos0 + j < see_hi ? s[j] : -INFINITY;
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int j = 4; j + 1 < KEYS; j += 2) top[j / 2 & 3] = max3(top[j / 2 & 3], s[j], s[j + 1]);
            const float m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * unit;
            const bool grow = m_tile > m_run + kSlack;   // also when there was none yet
            if (__any_sync(0xffffffffu, grow)) {
                const float m_new = grow ? m_tile : m_run;
                const float alpha = m_run == -INFINITY ? 1.0f : ex2(m_run - m_new);
                if (t > 0) {
                    const TilePhase before = tile_phase(t - 1);
                    ok = ok && bar_wait(&o_done[q * 2 + before.at], before.parity);
                    __syncwarp();
                    fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_at + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                        tmem_st32(o_at + c, o);
                    }
                }
                sum *= alpha;
                m_run = m_new;
            }
            const float m_use = m_run == -INFINITY ? 0.f : m_run;
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t w[KEYS / 2];
            if (NQ == 2) pair_sync(turn + q);
#pragma unroll
            for (int j = 0; j < KEYS; j += 2) {
                const float x = ex2(fmaf(s[j], unit, -m_use)), y = ex2(fmaf(s[j + 1], unit, -m_use));
                part[j & 3] += x;
                part[(j & 3) + 1] += y;
                w[j / 2] = Pair<T>::pack(x, y);
            }
            if (NQ == 2 && (q == 0 || t + 1 < n_tiles)) pair_arrive(turn + 1 - q);
            tmem_st32(s_at, w);
            sum += (part[0] + part[1]) + (part[2] + part[3]);
            if (OWN && pos0 + KEYS > keys_end) {
                // behind the lane's last key a page holds whatever it held: weights of 0 need finite values there
                ok = ok && bar_wait(&v_full[t % ST], t / ST & 1);
                const int first = max(0, keys_end - pos0), pieces = (KEYS - first) * 8;
                for (int i = tid & 127; i < pieces * L::PANELS; i += 128)
                    *reinterpret_cast<uint4*>(vs + (t % ST) * L::BYTES + i / pieces * L::PANEL + first * 128 + i % pieces * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_async_smem();
            }
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&p_full[q * 2 + ph.at]);
        }
        if (n_tiles > 0) {
            const TilePhase last = tile_phase(n_tiles - 1);
            ok = ok && bar_wait(&o_done[q * 2 + last.at], last.parity);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
            if (lane == 0) tell(a.status, kDevWait);
            sum = m_run = __int_as_float(0x7fffffff);   // the result says so
        }
        fence_after();
        const int64_t slot = ((int64_t)(first_part + split) * a.total + token) * a.q_heads + head;
        if (token >= 0) a.part_ml[slot] = sum == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m_run, sum);
        if (n_tiles > 0 && __any_sync(0xffffffffu, token >= 0)) {
            // Rows go out through where the queries were, half a row at a time, so that a warp writes whole rows (a thread a row: 2.6 us for heads of 128).
            constexpr int HALF = D / 2, PIECES = HALF / 4;   // values and 16-byte pieces of half a row
            float4* stage = reinterpret_cast<float4*>(qs + q * L::PANELS * L::QPANEL) + (warp & 3) * 32 * PIECES;
            const int64_t mine = token < 0 ? -1 : slot * D;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                __syncwarp();
#pragma unroll
                for (int c = 0; c < HALF; c += 32) {
                    float o[32];
                    tmem_ld32(o_at + half * HALF + c, reinterpret_cast<uint32_t*>(o));
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 8; ++j) stage[lane * PIECES + ((c / 4 + j) ^ (lane & 7))] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                }
                __syncwarp();
#pragma unroll 4
                for (int i = lane; i < 32 * PIECES; i += 32) {
                    const int r = i / PIECES, c = i % PIECES;
                    const int64_t at = __shfl_sync(0xffffffffu, mine, r);
                    if (at >= 0) *reinterpret_cast<float4*>(a.part_o + at + half * HALF + c * 4) = stage[r * PIECES + (c ^ (r & 7))];
                }
            }
        }
    }
    if (OWN) pdl_wait();   // who comes after this kernel relies on the one before it too
    fence_before();
    __syncthreads();
    if (warp == L::WARPS + L::LOADERS) {
        fence_after();
        tmem_dealloc(tmem, L::TMEM);
    }
}

// The pools as tensor maps with boxes of so many tokens; made anew only where a call's kernels differ in it (a map takes the host 0.6 us).
struct Maps {
    alignas(64) CUtensorMap k, v;
    int box = 0;
    void need(const SharedAttnArgs& a, int tokens) {
        if (box == tokens) return;
        const uint64_t rows = (uint64_t)(a.pool_pages - 1) * (uint64_t)a.page_rows + (uint64_t)a.kv_heads * (uint64_t)a.block_tokens;
        encode_tma_2d(&k, false, a.k_pool, (uint64_t)a.d, rows, (uint64_t)a.d * 2, 64, (uint32_t)tokens, true);
        encode_tma_2d(&v, false, a.v_pool, (uint64_t)a.d, rows, (uint64_t)a.d * 2, 64, (uint32_t)tokens, true);
        box = tokens;
    }
};

template <typename T, int D, int NQ, bool OWN>
void launch_tall(const SharedAttnArgs& a, const SharedAttnPlan& p, Maps& maps, cudaStream_t s) {
    using L = SharedSmem<D, NQ>;
    const int box = std::min(a.block_tokens, kKeys);
    maps.need(a, box);
    auto* kernel = a.softcap > kCapOfDifference ? shared_keys_kernel<T, D, NQ, OWN, true> : shared_keys_kernel<T, D, NQ, OWN, false>;
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::SMEM);
    if (!OWN) {
        kernel<<<(unsigned)(p.row_tiles * a.kv_heads * p.shared_parts), L::THREADS, L::SMEM, s>>>(maps.k, maps.v, a, box, p.shared_parts, 0, 0, 0);
        MK_LAUNCH_CHECK();
        return;
    }
    const unsigned grid = (unsigned)(a.lanes * p.item_tiles * a.kv_heads * p.shares);
    if (p.shared_parts > 0) launch_pdl(kernel, dim3(grid), dim3(L::THREADS), L::SMEM, s, maps.k, maps.v, a, box, p.shares, p.chunk, p.item_tiles, p.shared_parts);
    else kernel<<<grid, L::THREADS, L::SMEM, s>>>(maps.k, maps.v, a, box, p.shares, p.chunk, p.item_tiles, 0);
    MK_LAUNCH_CHECK();
}

template <typename T, int D, int NT>
void launch_lanes(const SharedAttnArgs& a, const SharedAttnPlan& p, Maps& maps, cudaStream_t s) {
    maps.need(a, kTile);
    using L = LaneSmem<D, NT>;
    auto* kernel = a.softcap > kCapOfDifference ? lane_keys_kernel<T, D, NT, true> : lane_keys_kernel<T, D, NT, false>;
    // Half the ring (32 KB) where there are more than two CTAs for each SM: more of them run at once, also beside a CTA of the shared keys, and what one waits for another uses (128
    // lanes of 8 heads with 1 to 60 keys 24.1 us and 20.3; 117 of 4 with one 16.6 and 12.7).  Fewer CTAs need more of their own on its way (32 lanes of 8 heads with 17 to 500 keys
    // 14.7 us with the whole ring, 15.9 with half; 8 with 3000 23.0 and 26.8).
    int stage_bits = 0;
    while ((2 << stage_bits) <= L::STAGES) ++stage_bits;
    if (stage_bits > 0 && (int64_t)a.lanes * p.shares * a.kv_heads > 2 * kSms) --stage_bits;
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::bytes(L::STAGES));
    const size_t smem = L::bytes(1 << stage_bits);
    const dim3 grid((unsigned)(a.lanes * p.shares), (unsigned)a.kv_heads, (unsigned)p.item_tiles);
    // behind the shared keys' kernel it starts early: what both read was there before that one
    if (p.shared_parts > 0) launch_pdl(kernel, grid, dim3(L::THREADS), smem, s, maps.k, maps.v, a, p.chunk, p.shares, p.shared_parts, p.joined ? 0 : 1, stage_bits);
    else kernel<<<grid, L::THREADS, smem, s>>>(maps.k, maps.v, a, p.chunk, p.shares, p.shared_parts, p.joined ? 0 : 1, stage_bits);
    MK_LAUNCH_CHECK();
}

template <typename T, int D>
void launch_typed(const SharedAttnArgs& a, const SharedAttnPlan& p, cudaStream_t s) {
    Maps maps;
    if (p.shared_parts > 0) {
        if constexpr (D <= 128) {
            if (p.item_rows == 2) launch_tall<T, D, 2, false>(a, p, maps, s);
            else launch_tall<T, D, 1, false>(a, p, maps, s);
        } else {
            launch_tall<T, D, 1, false>(a, p, maps, s);
        }
    }
    if (p.items >= kItems) {
        if constexpr (D <= 128) {
            if (p.items > kItems) launch_tall<T, D, 2, true>(a, p, maps, s);
            else launch_tall<T, D, 1, true>(a, p, maps, s);
        } else {
            launch_tall<T, D, 1, true>(a, p, maps, s);
        }
    } else {
        switch (p.items) {
            case 8: launch_lanes<T, D, 1>(a, p, maps, s); break;
            case 16: launch_lanes<T, D, 2>(a, p, maps, s); break;
            default:
                if constexpr (D <= 128) launch_lanes<T, D, 3>(a, p, maps, s);
        }
    }
    if (p.joined)
        launch_pdl(join_parts_kernel<T, D>, dim3((unsigned)(((int64_t)a.total * a.q_heads + 7) / 8)), dim3(256), 0, s, a, (int)p.parts);
}

}  // namespace

SharedAttnPlan shared_attention_plan(int q_heads, int kv_heads, int d, int block_tokens, int width, int lanes, int rows, int total, int shared, int window) {
    SharedAttnPlan p;
    const int g = q_heads / kv_heads;
    const int64_t items = (int64_t)rows * g;
    if (items <= 0 || lanes <= 0 || total <= 0) return p;
    const bool small = items <= 16 || (items <= 24 && d != 256 && lanes * (int64_t)kv_heads < kSms);
    // Few keys: every lane reads the shared ones too, in one launch without parts, as long as two CTAs an SM do for them.  Us so, and with the shared keys' kernel, by keys of a lane (48 of
    // them its own):
    //   4 lanes of 4 KV heads of 64    256: 4.9, 7.9   512: 6.8, 8.4    640: 7.7, 8.5    768: 8.5, 8.7    1024: 10.5, 9.0
    //   4 lanes of 8 KV heads of 128   256: 6.7, 8.8   384: 8.5, 8.9    448: 9.5, 9.0    512: 10.3, 9.0
    //   4 lanes of 8 KV heads of 256   256: 8.0, 11.2  384: 10.5, 12.0  448: 11.9, 12.2  512: 13.1, 12.2
    //   32 lanes of 8 KV heads         of 64 640: 8.8, 9.7   of 128 384: 9.8, 10.5   of 256 320: 11.7, 12.3, and 384: 13.2, 12.4
    const int64_t all_keys = std::min((int64_t)width * block_tokens, window > 0 ? (int64_t)window + rows : INT64_MAX);
    p.alone = shared > 0 && small && lanes * (int64_t)kv_heads <= 2 * kSms && all_keys <= (d == 64 ? 640 : 384);
    if (p.alone) shared = 0;
    const int64_t keys = (int64_t)width * block_tokens - shared;
    if (!small) {
        // Lanes of more items than the small products take at once (17 to 24: where lanes fill the device; 31 lanes of 20 items 39 us so, 47 with the others, 24 lanes 54 and 50): tiles of 128 or 256 of them, and their keys in shares until about two CTAs are there for each place on an SM
        p.items = d <= 128 && items > kItems ? 2 * kItems : kItems;
        p.item_tiles = (int)((items + p.items - 1) / p.items);
        const int64_t ctas = (int64_t)lanes * kv_heads * p.item_tiles, wanted = std::max<int64_t>(1, (2 * (p.items == kItems && d <= 128 ? 2 : 1) * kSms + ctas - 1) / ctas);
        p.chunk = (int)std::min<int64_t>(std::max<int64_t>(256, (keys + wanted - 1) / wanted + kKeys - 1), 4096) / kKeys * kKeys;
    } else {
        p.items = (int)((items + 7) / 8 * 8);
        p.item_tiles = 1;
        // A lane's own keys: whole where the lanes fill the device, else in shares of at least 256 keys; never more than 1024 (512 at heads of 256),
        // which take a CTA about 12 us: lanes differ in length.
        const int64_t ctas = (int64_t)lanes * kv_heads, wanted = std::max<int64_t>(1, (3 * kSms / 2 + ctas - 1) / ctas);
        p.chunk = (int)std::min<int64_t>(std::max<int64_t>(256, (keys + wanted - 1) / wanted + 15), d == 256 ? 512 : 1024) / 16 * 16;
    }
    if (p.alone) p.chunk = (int)((keys + 15) / 16 * 16);
    p.shares = (int)std::max<int64_t>(1, (keys + p.chunk - 1) / p.chunk);
    if (shared > 0) {
        // Tiles of items two at a time where there are more than one.  Shares of the shared keys: a CTA has an SM to itself; a tile of keys takes it about 0.7 us, or 1 us for two tiles of items, its start and end 4 us, and a share's results are written and read once (2.5 TB/s, and 0.1 us).
        const int64_t all = (int64_t)total * g;
        p.item_rows = d <= 128 && all > kItems ? 2 : 1;
        p.row_tiles = (int)((all + kItems * p.item_rows - 1) / (kItems * p.item_rows));
        const int tiles = (int)(std::min<int64_t>(shared, window > 0 ? (int64_t)window + rows : INT_MAX) + kKeys - 1) / kKeys;
        const double results_us = 0.1 + (double)total * q_heads * d * 8 / 2.5e6;
        double best = 0;
        for (int n = 1; n <= std::min(tiles, 148); ++n) {
            const int64_t slots = d <= 128 && p.item_rows == 1 ? 2 * kSms : kSms, waves = ((int64_t)p.row_tiles * kv_heads * n + slots - 1) / slots;
            const double us = waves * ((tiles + n - 1) / n * (p.item_rows == 2 ? 1.0 : 0.7) + 4.0) + n * results_us;
            if (n == 1 || us < best) best = us, p.shared_parts = n;
        }
    }
    // A lane's CTA joins the parts itself where its warps have at most two rows each to join, one after the other (1 lane, 5 rows of 2 heads of 256 each behind 768 shared tokens:
    // 20 us so, 15 with a kernel of its own).
    p.joined = p.shares > 1 || p.items >= kItems || (p.shared_parts > 0 && items > (d == 256 ? 4 : 8));
    p.parts = p.shared_parts + (p.joined ? p.shares : 0);
    return p;
}

void launch_shared_attention(SharedAttnArgs a, const SharedAttnPlan& p, cudaStream_t s) {
    if (a.lanes <= 0 || a.total <= 0 || a.rows <= 0) return;
    if (p.alone) a.shared = 0;
    for (a.bt_shift = 0; (1 << a.bt_shift) < a.block_tokens; ++a.bt_shift) {}
    a.part_ml = reinterpret_cast<float2*>(a.part_o + p.parts * a.total * a.q_heads * a.d);
    switch (a.d) {
        case 64: a.bf16 ? launch_typed<__nv_bfloat16, 64>(a, p, s) : launch_typed<__half, 64>(a, p, s); break;
        case 128: a.bf16 ? launch_typed<__nv_bfloat16, 128>(a, p, s) : launch_typed<__half, 128>(a, p, s); break;
        case 256: a.bf16 ? launch_typed<__nv_bfloat16, 256>(a, p, s) : launch_typed<__half, 256>(a, p, s); break;
        default: throw std::runtime_error("launch_shared_attention: unsupported head size");
    }
}

}  // namespace mk
