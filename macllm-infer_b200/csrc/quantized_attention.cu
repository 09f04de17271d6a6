// Attention over paged keys and values in 4- or 8-bit codes.
//
// Row t of lane i has position p = length_i - n_i + t and sees the keys max(0, p - window + 1) .. p of the lane's pages:
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(cap(scale q . k_j) - m),
// with k_j and v_j what their codes stand for, low + step c for each group of 64 values.
#include "quantized_attention.h"
#include "attention_math.cuh"
#include "kernels.h"
#include "umma.cuh"
#include <algorithm>

namespace mk {

namespace {

using namespace umma;

constexpr int kSms = 148;   // calls are cut without a device, for a B200

__device__ __forceinline__ void tell(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

template <typename T>
__device__ __forceinline__ float2 wide_pair(uint32_t w) {
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow_pair(float x, float y) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }   // of a positive number

// Where a lane's rows and keys are; whatever the arrays hold, rows stay inside [0, total) and keys inside the table.
struct LaneRange {
    int first, n;       // rows
    int position;       // of its first row
    int keys;           // length, at most what the table holds
};
__device__ __forceinline__ LaneRange lane_range(const QuantAttnArgs& a, int lane) {
    const QuantLanes& l = a.lanes;
    LaneRange r;
    r.first = l.cu != nullptr ? l.cu[lane] : lane * l.rows;
    r.n = l.cu != nullptr ? l.cu[lane + 1] - r.first : l.rows;
    const int length = l.lengths[lane];
    r.keys = min(max(length, 0), l.width << a.pools.bt_shift);
    if (r.first < 0 || r.first > l.total || r.n < 0 || r.n > l.rows || r.n > l.total - r.first || r.keys != length) {
        tell(l.status, kDevBadRange);
        if (r.first < 0 || r.first > l.total) r.first = 0, r.n = 0;
        r.n = min(max(r.n, 0), min(l.rows, l.total - r.first));
    }
    r.position = r.keys - r.n;
    return r;
}

// How the lanes' keys are shared out among CTAs.  With `want` CTAs for each KV head and block of items, a lane of n keys gets n / max(least, total / want) shares, rounded up: as many as its
// part of all keys asks for.  The lengths are the device's, so every CTA finds its lane and share by itself, from the number of its slot; a lane's slots follow one another.
struct Piece {
    int lane, share, shares, slot;   // the lane's first slot; lane < 0: none
};
// Of slot `slot`, or of the whole of lane `of_lane` where that is not negative; by a whole warp.
__device__ __forceinline__ Piece piece_of(const QuantAttnArgs& a, const QuantAttnCut& c, int slot, int of_lane) {
    const int n_lanes = a.lanes.lanes, lane = threadIdx.x & 31;
    if (!c.split) return Piece{of_lane >= 0 ? of_lane : slot, 0, 1, 0};
    auto keys_of = [&](int i) {
        if (i >= n_lanes) return 0;
        const int n = min(max(a.lanes.lengths[i], 0), a.lanes.width << a.pools.bt_shift);
        return a.window > 0 ? min(n, c.window_keys) : n;
    };
    const int mine = keys_of(lane);
    float total = (float)mine;
    for (int i = 32 + lane; i < n_lanes; i += 32) total += (float)keys_of(i);
    // The attention and the kernel that joins its shares count them each for itself: every rounding is spelled out, so that no compiler makes one of two in one kernel alone.
    const float per_share = __frcp_rn(fmaxf((float)c.least, __fdiv_rn(warp_sum(total), c.want)));
    // lanes with shares of more than half the largest size first: what is left at the end of a call is short
    int before = 0;
    for (int small = 0; small < 2; ++small)
        for (int i0 = 0; i0 < n_lanes; i0 += 32) {
            const float n = __fmul_rn((float)(i0 == 0 ? mine : keys_of(i0 + lane)), per_share);   // in largest shares
            const int shares = i0 + lane < n_lanes && (n < 0.5f) == (small != 0) ? max(1, (int)ceilf(__fsub_rn(n, 1e-3f))) : 0;   // roundings make no share
            int upto = shares;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            upto += before;
            const uint32_t hit = __ballot_sync(0xffffffffu, of_lane >= 0 ? shares > 0 && i0 + lane == of_lane : slot < upto);
            if (hit != 0) {
                const int at = __ffs(hit) - 1, its = __shfl_sync(0xffffffffu, shares, at), first = __shfl_sync(0xffffffffu, upto, at) - its;
                return Piece{i0 + at, of_lane >= 0 ? 0 : slot - first, its, first};
            }
            before = __shfl_sync(0xffffffffu, upto, 31);
        }
    return Piece{-1, 0, 1, 0};
}

// The keys of a block of items: `chunk` of them from `begin` on to each share, the last of which ends at `hi`.
struct Shares {
    int lo, hi, begin, chunk;
    __device__ __forceinline__ int used() const { return hi > lo ? (hi - begin + chunk - 1) / chunk : 0; }
};
__device__ __forceinline__ Shares shares_of(const QuantAttnArgs& a, const LaneRange& at, int item0, int n_items, int g, int shares) {
    const int p0 = at.position + item0 / g, p1 = at.position + (item0 + n_items - 1) / g;
    Shares s;
    s.lo = attention_first_key(max(p0, 0), a.window, 0);
    s.hi = min(p1 + 1, at.keys);
    s.begin = s.lo / 16 * 16;
    const int n = max(s.hi - s.begin, 0);
    s.chunk = shares == 1 ? (n + 15) / 16 * 16 : ((n + shares - 1) / shares + 15) / 16 * 16;
    s.chunk = max(s.chunk, 16);
    return s;
}

// ---- few items -----------------------------------------------------------------------------------------------------
//
// A CTA takes a share of one lane's keys for NT * 8 (row, query head) items of one KV head; each of its warps walks steps of 32 keys, whose codes and scales asynchronous
// copies of 16 bytes bring into a ring of its own (bulk copies take their operands from the warp's uniform registers: eight threads with one each cost 80 instructions for 16 keys).  Items are the short side of both products, S^T = K Q^T and O^T = V^T P^T, which run over the codes themselves: a code's bits alone
// are the f16 number c 2^-24 (a subnormal, which the tensor cores take in full), so that it costs a mask and half a shift.  With steps and lowest values of the groups
//   q . k = sum_g step_g (q_g . c_g) + low_g sum(q_g),   o = sum_j (w_j step_jg) c_j + sum_j w_j low_jg,
// steps multiply 32-bit partial scores, and weights before they are rounded: to two f16 numbers, 22 bits, since a weight's rounding counts for the whole range of a group.
// Queries are brought to f16 by a power of two per item, weights times steps by one per item and group; either is exact.  The running maximum follows only
// when a score exceeds it by more than 2^kSlack, which a vote of the warp tells, and the latter powers follow only when a step becomes too large for them, which the same vote tells: mostly they go by the
// largest step, where sizes are far apart by the largest weight times step that the item sees.  So what an item does not see, or sees with little weight, and other groups' sizes leave its results as exact as
// they are.  (One power of two for the largest step of all took ten bits off ordinary values' weights beside one of 6e4; it was faster by 2 % for single tokens at heads of 128, by 6 % for drafts at
// heads of 256.)
// The tensor cores cut a sum by its operands' exponent fields, which for subnormals are above the values: in 4 bits a score is off by 2^-22.0 of sum |q| |k| (root mean square, heads of 64).  With codes made normal
// numbers, an instruction more for each two, it is 2^-22.6, as in 8 bits either way; that takes 8 % longer for single tokens at heads of 128, 11 % for drafts at heads of 256.
// What bounds it is issue slots: about 370 instructions of a warp for 16 keys of heads of 128 (4096 values), half of the slots taken with twelve warps on an SM.  48 lanes of 200 to 6000 tokens, 32 heads of 128 over 8,
// 4 bits: 49.9 us, 1.9 TB/s; 3 contexts of up to 120001 tokens, 16 heads over 4: 42.4 us, 2.6 TB/s; 20 lanes of up to five rows, heads of 256, 8 bits: 152 us, 1.8 TB/s.  Before each item and group had a
// power of two of its own: 49, 42 and 144 us, with outputs of all tiles in one accumulator (but see there) 47, 40 and 123; codes by ordinary loads
// a tile ahead: 62, 124 and 149 us before the keys were shared out by lengths; 32 keys a step do 1.1 times as well as 16, four CTAs on an SM with 128 registers no better than three.
constexpr int kFewItems = 32;            // of a lane and KV head: more go to the tall kernel
constexpr int kTile = 16, kHalves = 2, kStep = kHalves * kTile;
constexpr int kWarps = 4;
constexpr float kSlack = 8.f;            // base-2 logarithm
constexpr int kMostBy = 118;             // of the exponents by which weights times steps are brought to f16: times 2^kSlack they are still numbers
constexpr float kStepLimit = 128.f;      // of steps brought to f16: times weights, 2^kSlack at most, they are below f16's largest

// CTAs on an SM: what registers allow.
__host__ __device__ constexpr int few_ctas(int d, int nt) { return d == 64 ? (nt == 1 ? 5 : 4) : (d == 128 ? (nt == 1 ? 3 : 2) : 2); }

template <int D, int BITS, int NT>
struct Few {
    static constexpr int G = D / kQuantGroup, ITEMS = NT * 8;
    static constexpr int ROW = D * BITS / 8, CODES = kTile * ROW, SCALES = kTile * G * 4, HALF = 2 * (CODES + SCALES), STAGE = kHalves * HALF;
    static constexpr int STAGES = STAGE <= 2400 ? 4 : 2;
    static constexpr int OP = D + 4;                                     // pitch of a warp's results, in floats
    static constexpr int RING = ((STAGES * STAGE > ITEMS * OP * 4 ? STAGES * STAGE : ITEMS * OP * 4) + 127) / 128 * 128;
    static constexpr int QP = D + 8;
    static constexpr size_t SMEM = 128 + (size_t)kWarps * RING + (size_t)ITEMS * QP * 2;
    static constexpr int CTAS = few_ctas(D, NT);
    static constexpr bool Q_IN_REGISTERS = NT * D <= 256;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }   // all but the last N groups are there
// N words of shared memory.
template <int N>
__device__ __forceinline__ void lds(uint32_t (&v)[N], uint32_t at) {
    if constexpr (N == 1) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(at));
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
    else asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}
// The key of a tile that row r of a product stands for.  A load of eight rows of K takes keys 0, 4, 1, 5 and 2, 6, 3, 7 at once, one of V keys 0 .. 3, or 4 .. 7, and so on.
__device__ __forceinline__ int key_of(int r) { return (r & 8) | (r & 7) >> 1 | (r & 1) << 2; }
// Where byte b of a key's codes lies in its tile: the 32 bytes that a load takes of each of four keys are on four different quarters of the banks (8-bit codes of heads of 64, whose loads of K
// take 64 bytes of two keys: on two of four).
template <int ROW>
__device__ __forceinline__ uint32_t place_in_tile(int key, int b) {
    const int turn = (key & 3) ^ (key >> 1 & 2);
    if constexpr (ROW == 32) return (key ^ (key >> 1 & 2)) * 32 + b;
    else if constexpr (ROW == 64) return key * 64 + (b ^ (turn & 2) << 4);
    else return key * ROW + (b ^ turn << 5);
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ float of_item(float top) {   // the largest of the threads that have the item
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    return fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
}
// The exponent by which weights times steps go into the second product where sizes are far apart: by the largest step that the item sees or, where its weight is small, by the largest weight times step.  The
// scores and steps of the thread's four keys, the maximum, what it has risen by (negative; 1: there was none), the exponent until now.  Apart from the kernel, whose loop it slowed by 1 to 2 % in line.
__device__ __noinline__ int careful_exponent(float4 score, float4 of_key, float maximum, float less, int now) {
    const float m = maximum == -INFINITY ? 0.f : maximum;
    float step = 0.f, x = 0.f;   // the largest that the item sees; the largest times its weight, 2^-10 of it
    auto key = [&](float score, float of_key) {
        if (!(score != -INFINITY && of_key < INFINITY)) return;
        step = fmaxf(step, of_key);
        x = fmaxf(x, ex2(score - m - 10.f) * of_key);
    };
    key(score.x, of_key.x);
    key(score.y, of_key.y);
    key(score.z, of_key.z);
    key(score.w, of_key.w);
    step = of_item(step), x = of_item(x);
    // what came so far has become less by 2^more, so that what comes may count for that much more
    const int more = less == 1.f ? 0 : min((int)fminf(-less, 240.f), kMostBy - now), e_step = exponent(step), e_x = exponent(x) + 10;
    return min(now + more, step > 0.f ? min(x > 0.f ? (e_x >= e_step - 8 ? 4 - e_step : 3 - e_x) : kMostBy, 120 - e_step) : kMostBy);
}

template <typename T, int D, int BITS, int NT, int CAP>
__global__ void __launch_bounds__(kWarps * 32, Few<D, BITS, NT>::CTAS) few_items_kernel(const __grid_constant__ QuantAttnArgs a, const __grid_constant__ QuantAttnCut cut, float* part_o, float2* part_ml) {
    using L = Few<D, BITS, NT>;
    constexpr int G = L::G;
    extern __shared__ uint8_t smem_raw[];
    __shared__ float item_factor[L::ITEMS], item_sums[L::ITEMS][G];
    __shared__ float2 warp_ml[kWarps][L::ITEMS];
    uint8_t* rings = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~(uintptr_t)127);   // a warp's results at the end
    __half* qs = reinterpret_cast<__half*>(rings + kWarps * L::RING);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tq = lane & 3;
    const QuantPools& p = a.pools;
    const int g = a.q_heads / p.kv_heads, slot = blockIdx.x, kvh = blockIdx.y;
    pdl_trigger();
    const Piece piece = piece_of(a, cut, slot, -1);
    if (piece.lane < 0) return;
    const int lane_id = piece.lane, share = piece.share, shares = piece.shares;
    const LaneRange at = lane_range(a, lane_id);
    const int item0 = blockIdx.z * L::ITEMS, n_items = min(L::ITEMS, at.n * g - item0);
    if (n_items <= 0) return;
    const Shares sh = shares_of(a, at, item0, n_items, g, shares);
    if (share > 0 && share >= sh.used()) return;
    const int lo = max(sh.lo, sh.begin + share * sh.chunk), hi = min(sh.hi, sh.begin + (share + 1) * sh.chunk);
    const int begin = sh.begin + share * sh.chunk, n_tiles = hi > lo ? (hi - begin + kTile - 1) / kTile : 0, n_steps = (n_tiles + kHalves - 1) / kHalves;
    const int my_steps = n_steps > warp ? (n_steps - warp + kWarps - 1) / kWarps : 0;

    const uint32_t ring = smem_u32(rings + warp * L::RING);
    const int32_t* table = a.lanes.tables + lane_id * a.lanes.ld_table;
    auto tile_of = [&](int i) { return ((i >> 1) * kWarps + warp) * kHalves + (i & 1); };   // of the warp's half i
    // the page numbers of 32 halves sit in the warp's threads, those of the next 32 on their way
    auto page_of = [&](int i) {
        const int tile = tile_of(i);
        if (tile >= n_tiles) return 0;
        const int32_t page = table[(begin + tile * kTile) >> p.bt_shift];
        if ((uint32_t)page < (uint64_t)p.pages) return page;
        tell(a.lanes.status, kDevBadPage);
        return 0;
    };
    int page_now = page_of(lane), page_next = my_steps > 16 ? page_of(32 + lane) : 0;
    // 16 bytes to a thread and copy: codes in runs of 512, the scales of 16 keys by neighbouring threads
    constexpr int RUNS = L::CODES / 512, SCALE_COPIES = L::SCALES / 16;   // 1 .. 8; 4, 8, 16
    static_assert(L::CODES % 512 == 0, "whole runs");
    uint32_t to[RUNS];
#pragma unroll
    for (int r = 0; r < RUNS; ++r) to[r] = ring + place_in_tile<L::ROW>((r * 512 + lane * 16) / L::ROW, (r * 512 + lane * 16) % L::ROW);
    const bool scale_of_keys = lane < SCALE_COPIES;
    const int scale_copy = scale_of_keys ? lane : lane - SCALE_COPIES;
    const uint32_t scale_to = ring + 2 * L::CODES + (scale_of_keys ? 0 : L::SCALES) + scale_copy * 16;
    const uint32_t* scales_from = (scale_of_keys ? p.k_scales : p.v_scales) + (int64_t)kvh * p.block_tokens * G + scale_copy * 4;
    const uint8_t *keys_from = p.k_codes + (int64_t)kvh * p.block_tokens * L::ROW + lane * 16, *values_from = p.v_codes + (int64_t)kvh * p.block_tokens * L::ROW + lane * 16;
    auto load_step = [&](int i) {   // the whole warp; a group of copies, an empty one behind the last step
        if (i < my_steps) {
            if ((i & 15) == 0 && i > 0) {
                page_now = page_next;
                page_next = page_of(2 * i + 32 + lane);
            }
            const uint32_t st = (i & (L::STAGES - 1)) * L::STAGE;
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const int64_t page = __shfl_sync(0xffffffffu, page_now, (2 * i + h) & 31);
                const int tile = tile_of(2 * i + h), row = (begin + tile * kTile) & (p.block_tokens - 1);
                if (tile >= n_tiles) break;
                const int64_t at = page * p.codes_stride + row * L::ROW;
#pragma unroll
                for (int r = 0; r < RUNS; ++r) {
                    copy16(to[r] + st + h * L::HALF, keys_from + at + r * 512);
                    copy16(to[r] + st + h * L::HALF + L::CODES, values_from + at + r * 512);
                }
                if (lane < 2 * SCALE_COPIES) copy16(scale_to + st + h * L::HALF, scales_from + page * p.scales_stride + row * G);
            }
        }
        copies_end();
    };
#pragma unroll 1
    for (int i = 0; i < L::STAGES; ++i) load_step(i);

    // queries: a warp has an item, V neighbouring values to a thread
    constexpr int V = D / 32;
    const float unit = CAP ? a.scale : a.scale * kLog2e;
    for (int item = warp; item < L::ITEMS; item += kWarps) {
        float x[V], sum = 0.f, top = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = 0.f;
        if (item < n_items) {
            const int r = (item0 + item) / g, hq = (item0 + item) - r * g;
            const T* q = static_cast<const T*>(a.q) + (int64_t)(at.first + r) * a.ldq + (kvh * g + hq) * D + lane * V;
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 y = wide_pair<T>(*reinterpret_cast<const uint32_t*>(q + j));
                x[j] = y.x;
                x[j + 1] = y.y;
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sum += x[j];
            top = fmaxf(top, fabsf(x[j]));
        }
        // the largest becomes 2^14 and a bit; powers of two that neither the factor here nor the one of the scores overflows
        top = warp_max(top);
        const int e = top > 0.f ? min(max(14 - (int)((__float_as_uint(top) >> 23) - 127), -86), 100) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<uint32_t*>(qs + item * L::QP + lane * V + j) = narrow_pair<__half>(x[j] * up, x[j + 1] * up);
        // sums of the groups, each of which 64 / V threads hold
#pragma unroll
        for (int o = 1; o < kQuantGroup / V; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane % (kQuantGroup / V) == 0) item_sums[item][lane * V / kQuantGroup] = sum * up * 0x1p-24f;
        if (lane == 0) item_factor[item] = unit * __uint_as_float((uint32_t)(127 + 24 - e) << 23);
    }
    __syncthreads();

    float o_acc[NT][G][4][4], low_acc[NT][G][2], m_run[NT][2], l_run[NT][2], factor[NT][2], sums[NT][G][2];
    int see_lo[NT][2], see_hi[NT][2];   // keys that the thread's two items of a group of eight see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < G; ++j) {
#pragma unroll
            for (int u = 0; u < 4; ++u) o_acc[n][j][u][0] = o_acc[n][j][u][1] = o_acc[n][j][u][2] = o_acc[n][j][u][3] = 0.f;
            low_acc[n][j][0] = low_acc[n][j][1] = 0.f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int item = n * 8 + 2 * tq + h, pos = at.position + (item0 + item) / g;
            m_run[n][h] = -INFINITY;
            l_run[n][h] = 0.f;
            factor[n][h] = item_factor[item];
#pragma unroll
            for (int j = 0; j < G; ++j) sums[n][j][h] = item_sums[item][j];
            see_lo[n][h] = max(lo, attention_first_key(max(pos, 0), a.window, 0));
            see_hi[n][h] = min(hi, pos + 1);
        }
    }
    const int p0 = at.position + item0 / g, p1 = at.position + (item0 + n_items - 1) / g;
    const int all_lo = max(lo, attention_first_key(max(p1, 0), a.window, 0)), all_hi = min(hi, p0 + 1);   // keys that every item sees
    const float two_over_cap = CAP ? 2.0f / a.softcap : 0.f;
    const bool wide_cap = CAP && a.softcap > kCapOfDifference;
    // queries as the B operand of step s of group j: the values that stand in the codes' order of the thread's words
    auto query = [&](int n, int j, int s, uint32_t& b0, uint32_t& b1) {
        const __half* q = qs + (n * 8 + gid) * L::QP + j * kQuantGroup + tq * 16;
        if constexpr (BITS == 4) {
            const __half* w = q + (s >> 1) * 8 + (s & 1) * 2;
            const __half2 x = __halves2half2(w[0], w[4]), y = __hmul2(__halves2half2(w[1], w[5]), __float2half2_rn(0.0625f));   // codes of the second pair are 16 times theirs
            b0 = *reinterpret_cast<const uint32_t*>(&x);
            b1 = *reinterpret_cast<const uint32_t*>(&y);
        } else {
            const __half* w = q + s * 4;
            const __half2 x = __halves2half2(w[0], w[2]), y = __halves2half2(w[1], w[3]);
            b0 = *reinterpret_cast<const uint32_t*>(&x);
            b1 = *reinterpret_cast<const uint32_t*>(&y);
        }
    };
    uint32_t q_reg[L::Q_IN_REGISTERS ? NT : 1][G][4][2];
    if constexpr (L::Q_IN_REGISTERS) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s) query(n, j, s, q_reg[n][j][s][0], q_reg[n][j][s][1]);
    }
    float by[NT][G][2];   // weights times steps of a group go into the second product by so much
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < G; ++j) by[n][j][0] = by[n][j][1] = power_of_two(kMostBy);
    const int key0 = key_of(gid), va = key_of(2 * tq), vb = key_of(2 * tq + 1);
#pragma unroll 1
    for (int i = 0; i < my_steps; ++i) {
        copies_wait<L::STAGES - 1>();
        __syncwarp();   // the other threads' too
        const uint32_t stage = ring + (i & (L::STAGES - 1)) * L::STAGE;
        const int pos0 = begin + tile_of(2 * i) * kTile;
        const bool whole = pos0 >= all_lo && pos0 + kStep <= all_hi;
        // ---- scores
        float sc[kHalves][NT][4];
        float2 v0[kHalves][G], v1[kHalves][G];   // (step, lowest) of the values of the thread's keys
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const uint32_t kt = stage + h * L::HALF, scales = kt + 2 * L::CODES + key0 * (G * 4);
            uint32_t kp[2][G], vp[2][G];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                lds(kp[r], scales + r * 8 * G * 4);
                lds(vp[r], scales + L::SCALES + r * 8 * G * 4);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[h][n][0] = sc[h][n][1] = sc[h][n][2] = sc[h][n][3] = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t w0[BITS / 2], w1[BITS / 2];   // words of the thread's two keys
                const uint32_t at_key = kt + place_in_tile<L::ROW>(key0, j * (kQuantGroup * BITS / 8) + tq * (BITS * 2));
                lds(w0, at_key);
                lds(w1, at_key + 8 * L::ROW);   // the same place of eight keys on
                float acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t a0, a1, a2, a3;
                    if constexpr (BITS == 4) {
                        const uint32_t x = s & 1 ? w0[s >> 1] >> 8 : w0[s >> 1], y = s & 1 ? w1[s >> 1] >> 8 : w1[s >> 1];
                        a0 = x & 0x000f000fu, a2 = x & 0x00f000f0u, a1 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
                    } else {
                        a0 = w0[s] & 0x00ff00ffu, a2 = w0[s] >> 8 & 0x00ff00ffu, a1 = w1[s] & 0x00ff00ffu, a3 = w1[s] >> 8 & 0x00ff00ffu;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t b0, b1;
                        if constexpr (L::Q_IN_REGISTERS) b0 = q_reg[n][j][s][0], b1 = q_reg[n][j][s][1];
                        else query(n, j, s, b0, b1);
                        mma_f16(acc[n], a0, a1, a2, a3, b0, b1);
                    }
                }
                const float2 sl0 = wide_pair<T>(kp[0][j]), sl1 = wide_pair<T>(kp[1][j]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    sc[h][n][0] = fmaf(sl0.x, acc[n][0], fmaf(sl0.y, sums[n][j][0], sc[h][n][0]));
                    sc[h][n][1] = fmaf(sl0.x, acc[n][1], fmaf(sl0.y, sums[n][j][1], sc[h][n][1]));
                    sc[h][n][2] = fmaf(sl1.x, acc[n][2], fmaf(sl1.y, sums[n][j][0], sc[h][n][2]));
                    sc[h][n][3] = fmaf(sl1.x, acc[n][3], fmaf(sl1.y, sums[n][j][1], sc[h][n][3]));
                }
                v0[h][j] = wide_pair<T>(vp[0][j]);
                v1[h][j] = wide_pair<T>(vp[1][j]);
            }
        }
        if (!whole) {   // keys that no item of the block sees may have any scales: those of values count as 0
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const int pos = pos0 + h * kTile + key0;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    if (pos < lo || pos >= hi) v0[h][j] = make_float2(0.f, 0.f);
                    if (pos + 8 < lo || pos + 8 >= hi) v1[h][j] = make_float2(0.f, 0.f);
                }
            }
        }
        bool up = false;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = sc[h][n][e] * factor[n][e & 1];
                    if (CAP) v = (wide_cap ? capped_wide(v, a.softcap, two_over_cap) : capped(v, a.softcap, two_over_cap)) * kLog2e;
                    if (!whole) {
                        const int pos = pos0 + h * kTile + key0 + (e >> 1) * 8;
                        v = pos >= see_lo[n][e & 1] && pos < see_hi[n][e & 1] ? v : -INFINITY;
                    }
                    sc[h][n][e] = v;
                    up |= v > m_run[n][e & 1] + kSlack;   // also when there was none yet
                }
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            float most = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) most = max3(most, by[n][j][0], by[n][j][1]);
            up |= max3(max3(v0[0][j].x, v1[0][j].x, v0[1][j].x), v1[1][j].x, 0.f) * most > kStepLimit;
        }
        if (__any_sync(0xffffffffu, up)) {
            float less[NT][2];   // what the maximum has risen by, negative; 1: there was none
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float m_new = fmaxf(m_run[n][c], of_item(fmaxf(fmaxf(sc[0][n][c], sc[0][n][2 + c]), fmaxf(sc[1][n][c], sc[1][n][2 + c]))));
                    less[n][c] = m_run[n][c] == -INFINITY ? 1.f : m_run[n][c] - m_new;
                    m_run[n][c] = m_new;
                    if (less[n][c] == 0.f || less[n][c] == 1.f) continue;
                    const float alpha = ex2(less[n][c]);
                    l_run[n][c] *= alpha;
#pragma unroll
                    for (int j = 0; j < G; ++j) {
                        low_acc[n][j][c] *= alpha;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            o_acc[n][j][u][c] *= alpha;
                            o_acc[n][j][u][2 + c] *= alpha;
                        }
                    }
                }
            // as nearly always: steps of like size, for items that have met none or ones of that size
            bool plain = true;
            float largest[G];
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float top = 0.f, least = INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float step = k & 1 ? v1[k >> 1][j].x : v0[k >> 1][j].x;
                    const int pos = pos0 + (k >> 1) * kTile + key0 + (k & 1) * 8;
                    top = max_nan(top, step);
                    if (whole || (pos >= lo && pos < hi)) least = fminf(least, step);
                }
                largest[j] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                const float smallest = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));   // the whole warp, whatever its threads have found so far
                plain = plain && largest[j] <= 256.f * smallest;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) plain = plain && (less[n][c] == 1.f || (largest[j] * by[n][j][c] <= kStepLimit && largest[j] * by[n][j][c] >= 0x1p-4f));
            }
            if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < G; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            if (less[n][c] == 1.f) by[n][j][c] = power_of_two(min(4 - exponent(largest[j]), kMostBy));
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < G; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int now = less[n][c] == 1.f ? kMostBy : exponent(by[n][j][c]);
                            const int then = careful_exponent(make_float4(sc[0][n][c], sc[0][n][2 + c], sc[1][n][c], sc[1][n][2 + c]), make_float4(v0[0][j].x, v1[0][j].x, v0[1][j].x, v1[1][j].x), m_run[n][c], less[n][c], now);
                            by[n][j][c] = power_of_two(then);
                            const float factor = power_of_two(max(then - now, -126));
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                o_acc[n][j][u][c] *= factor;
                                o_acc[n][j][u][2 + c] *= factor;
                            }
                        }
            }
        }
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            // ---- weights
            uint32_t hi_b[NT][G][2], lo_b[NT][G][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float m = m_run[n][e & 1];
                    w[e] = ex2(sc[h][n][e] - (m == -INFINITY ? 0.f : m));
                }
                l_run[n][0] += w[0] + w[2];
                l_run[n][1] += w[1] + w[3];
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    float x[4];
                    if (whole) {
                        low_acc[n][j][0] = fmaf(w[0], v0[h][j].y, fmaf(w[2], v1[h][j].y, low_acc[n][j][0]));
                        low_acc[n][j][1] = fmaf(w[1], v0[h][j].y, fmaf(w[3], v1[h][j].y, low_acc[n][j][1]));
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = w[e] * (by[n][j][e & 1] * (e < 2 ? v0[h][j].x : v1[h][j].x));
                    } else {   // what an item does not see does not count, also where it is not finite
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool seen = sc[h][n][e] != -INFINITY;
                            low_acc[n][j][e & 1] += seen ? w[e] * (e < 2 ? v0[h][j].y : v1[h][j].y) : 0.f;
                            x[e] = seen ? w[e] * (by[n][j][e & 1] * (e < 2 ? v0[h][j].x : v1[h][j].x)) : 0.f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t high = narrow_pair<__half>(x[2 * r], x[2 * r + 1]);
                        const float2 back = wide_pair<__half>(high);
                        hi_b[n][j][r] = transpose_8x8(high);
                        lo_b[n][j][r] = transpose_8x8(narrow_pair<__half>(x[2 * r] - back.x, x[2 * r + 1] - back.y));
                    }
                }
            }
            // ---- output; the thread's values are those of keys va, vb and the same eight further on
            const uint32_t vt = stage + h * L::HALF + L::CODES;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t w[4][BITS / 4];   // eight values of each of four keys
#pragma unroll
                for (int k = 0; k < 4; ++k) lds(w[k], vt + place_in_tile<L::ROW>(k & 1 ? vb : va, j * (kQuantGroup * BITS / 8) + gid * BITS) + (k >> 1) * 8 * L::ROW);
#pragma unroll
                for (int u = 0; u < 4; ++u) {   // values 2 u and 2 u + 1 of the eight
                    uint32_t a0, a1, a2, a3;
                    if constexpr (BITS == 4) {
                        uint32_t x = __byte_perm(w[0][0], w[1][0], u < 2 ? 0x5410 : 0x7632), y = __byte_perm(w[2][0], w[3][0], u < 2 ? 0x5410 : 0x7632);
                        if (u & 1) x >>= 8, y >>= 8;
                        a0 = x & 0x000f000fu, a1 = x & 0x00f000f0u, a2 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
                    } else {
                        const uint32_t x = __byte_perm(w[0][u >> 1], w[1][u >> 1], u & 1 ? 0x7632 : 0x5410), y = __byte_perm(w[2][u >> 1], w[3][u >> 1], u & 1 ? 0x7632 : 0x5410);
                        a0 = x & 0x00ff00ffu, a1 = x >> 8 & 0x00ff00ffu, a2 = y & 0x00ff00ffu, a3 = y >> 8 & 0x00ff00ffu;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        // Products align their sums by exponent fields, which for subnormal codes are up to 2^10 above the value: a sum is cut at 2^-14 of the largest weight's step at the most.  Over many
                        // tiles in one accumulator that would add up, so that each tile's is added in 32 bits: over 2048 keys results are off by 2^-20.8 of the mean of |v| in 4 bits, by 2^-22.4 in 8 (root mean squares).
                        float part[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_f16(part, a0, a1, a2, a3, hi_b[n][j][0], hi_b[n][j][1]);
                        mma_f16(part, a0, a1, a2, a3, lo_b[n][j][0], lo_b[n][j][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o_acc[n][j][u][e] += part[e];
                    }
                }
            }
        }
        __syncwarp();
        load_step(i + L::STAGES);
    }
    // ---- a warp's results, over its own sum: [item][D] and (maximum, sum)
    float* mine = reinterpret_cast<float*>(rings + warp * L::RING);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = l_run[n][h];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            const int item = n * 8 + 2 * tq + h;
            if (gid == 0) warp_ml[warp][item] = make_float2(m_run[n][h], l);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float low = low_acc[n][j][h];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) low += __shfl_xor_sync(0xffffffffu, low, o);
                low *= inv;
                const float back = power_of_two(-exponent(by[n][j][h]));
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // codes were c 2^-24, those of the second value 16 times that
                    const float x = o_acc[n][j][u][h] * inv * 0x1p24f, y = o_acc[n][j][u][2 + h] * inv * (BITS == 4 ? 0x1p20f : 0x1p24f);
                    *reinterpret_cast<float2*>(mine + item * L::OP + j * kQuantGroup + gid * 8 + 2 * u) = make_float2(fmaf(x, back, low), fmaf(y, back, low));
                }
            }
        }
    }
    __syncthreads();
    // ---- the warps' results together
    const bool last = shares == 1;
    for (int i = tid; i < n_items * (D / 4); i += kWarps * 32) {
        const int item = i / (D / 4), c = (i - item * (D / 4)) * 4;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_ml[w][item].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = warp_ml[w][item];
            if (ml.y == 0.f) continue;
            const float f = ml.y * ex2(ml.x - (m == -INFINITY ? 0.f : m));
            const float4 x = *reinterpret_cast<const float4*>(rings + w * L::RING + (item * L::OP + c) * 4);
            l += f;
            o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;   // a row that sees nothing: zeros
        o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
        const int r = (item0 + item) / g, hq = (item0 + item) - r * g;
        if (last) {
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(at.first + r) * a.ldo + (kvh * g + hq) * D + c) = make_uint2(narrow_pair<T>(o.x, o.y), narrow_pair<T>(o.z, o.w));
        } else {
            const int64_t row = ((int64_t)slot * a.lanes.rows + r) * a.q_heads + kvh * g + hq;
            *reinterpret_cast<float4*>(part_o + row * D + c) = o;
            if (c == 0) part_ml[row] = make_float2(m, l);
        }
    }
}

// ---- many items ----------------------------------------------------------------------------------------------------
//
// A CTA takes SUBS tiles of 128 (row, query head) items of a lane and KV head and walks the keys they see, or a share of them, in tiles of 64, on the fifth-generation tensor
// cores: scores Q K^T (128 x 64, f32) into one of two areas of tensor memory per tile of items, O += P V with P as the A operand in tensor memory, over its scores.  Four warps make
// numbers of keys out of their codes, 16 keys each, four of values: codes into registers two tiles ahead, f16 numbers into the swizzled rows that the products read.  A warp for each tile of items issues its
// products; four hold an item to a thread.  Two tiles of items share the numbers, and one's softmax runs under the other's products.
// What bounds it is the chain of a tile's softmax: 2700 clocks for 256 items by 64 keys of heads of 128, half of them exponentials (two warps of a scheduler come to them together), where products take 1024: tensor pipe
// 37 % busy.  4 portions of 1000 rows, 32 heads of 128 over 4, behind 2500 to 12000 tokens: 395 us, 729 TFLOP/s; 2048 rows of 32 heads over 8 behind 16384: 666 us, 774.  Where it took 400,
// one thread issuing all products took 498, codes through bulk copies and shared memory 441, turns at the exponentials 441, a fourth of the exponentials as polynomials on the other pipes 401.
// A code becomes 1024 + c by its bits, c by a subtraction, and low + step c by one fused multiply-add in f16: rounded once, to 11 bits, as a 16-bit cache would hold it; weights are
// rounded to 11 bits for the second product.  Scales come with a power of two of their own for every 16 keys (multiples of 2^8, so that neighbours share one): scores are multiplied by the
// keys', weights by the values' over the row's where they differ.  The row's goes by weights times sizes, so that values that it does not see, or sees with hardly any weight, take nothing off the others, whatever
// their size.  Where groups among the 16 keys are so far apart that f16 would cut off the smaller ones' steps, each key has an exponent of its own below the 16 keys', and its numbers are made in 32 bits: they have 11 bits
// down to 2^-21 of the key's largest.  (Exponents of 16 keys, and the largest of them for the weights, took all bits off a row's values beside an unseen one of 1e10.  Looking for such groups costs 4 % at heads of 256 in
// 4 bits and for drafts, nothing elsewhere.)  Values of a chunk of eight lie in the order in which the
// codes' masks give them; queries are laid out alike and results put back in order at the end.  Where a value's scales are not finite they count as zero, and the rows
// that see the key get NaN for that group at the end: a weight of 0 does not hide NaN from a product.
constexpr int kItemTile = 128, kKeyTile = 64, kCodeWarps = 8;   // four for keys, four for values
// Base-2 logarithm of the weight of a score at the maximum, in sums and products alike: with 2^kSlack above it is below f16's largest, down to 2^-21 of the largest weights have 11 bits, and what f16 loses
// of one is below 2^-32.  (With 0, thousands of weights of 2^-25 and less stayed in the sum alone; times are the same.)
constexpr float kWeightBits = 7.f;

template <int D, int BITS, int SUBS>
struct Many {
    static constexpr int G = D / kQuantGroup, PANELS = D / 64;
    static constexpr int Q_PANEL = kItemTile * 128, PANEL = kKeyTile * 128;
    static constexpr int Q_BYTES = PANELS * Q_PANEL, TILE_BYTES = PANELS * PANEL;
    static constexpr int K_STAGES = 2, V_STAGES = D == 256 ? 1 : 2;
    static constexpr size_t SMEM = 1024 + (size_t)SUBS * Q_BYTES + (size_t)(K_STAGES + V_STAGES) * TILE_BYTES;
    // a warp's codes of 16 keys in pieces of 16 bytes: PASSES to a thread, each CHUNKS times eight numbers
    static constexpr int ROW = D * BITS / 8, PIECES = ROW / 16, PASSES = ROW / 32, CHUNKS = 16 / BITS;
    static constexpr int ITEM_WARPS = 4 * SUBS, MMA_WARP = ITEM_WARPS + kCodeWarps, THREADS = (MMA_WARP + 4) * 32;
    // Twenty warps have 96 registers a thread at launch, 1920 of them a lane of all warps: eight warps of items then take 144, eight of codes keep 72, the last four 40 (1888).
    static constexpr bool SPLIT_REGISTERS = SUBS == 2;
    static constexpr int LAUNCH_REGISTERS = 96, ITEM_REGISTERS = 144, CODE_REGISTERS = 72, OTHER_REGISTERS = 40;
    static_assert(!SPLIT_REGISTERS || ITEM_WARPS * ITEM_REGISTERS + kCodeWarps * CODE_REGISTERS + 4 * OTHER_REGISTERS <= THREADS / 32 * LAUNCH_REGISTERS, "more registers than the launch has");
    static constexpr int S_AT = SUBS * D;   // columns of tensor memory: outputs, then scores
    static_assert(S_AT + SUBS * 2 * kKeyTile <= 512, "tensor memory");
};

// The exponent under which numbers up to `bound` are below 2^15, a multiple of eight; the one before stays while it leaves them above 2^-1, so that neighbours share one.
__device__ __forceinline__ int exponent_of(float bound, int before) {
    const int above = (int)(__float_as_uint(bound) >> 23) - 126;   // bound < 2^above
    const int e = bound > 0.f ? min(max(((above - 15 + 1024 + 7) / 8 - 128) * 8, -120), 120) : -120;
    return e <= before && (e >= before - 8 || bound == 0.f) ? before : e;
}
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
// The lane with the rank-th most tokens, the first of equals first, among up to kRanked lanes; more lanes keep their order.  All threads of the CTA.
constexpr int kRanked = 256;
__device__ __forceinline__ int lane_of_rank(const QuantLanes& l, int rank) {
    if (l.lanes == 1 || l.lanes > kRanked) return rank;
    __shared__ int lengths[kRanked], found;
    const int tid = threadIdx.x;
    if (tid < l.lanes) lengths[tid] = l.lengths[tid];
    if (tid == 0) found = rank;
    __syncthreads();
    if (tid < l.lanes) {
        const int mine = lengths[tid];
        int before = 0;
        for (int i = 0; i < l.lanes; ++i) before += lengths[i] > mine || (lengths[i] == mine && i < tid) ? 1 : 0;
        if (before == rank) found = tid;
    }
    __syncthreads();
    return found;
}

// The place of value i of eight in their chunk: as the masks give them.
template <int BITS>
__host__ __device__ constexpr int place_of(int i) { return BITS == 4 ? (i % 4) * 2 + i / 4 : i / 4 * 4 + (i % 2) * 2 + i % 4 / 2; }

template <typename T, int D, int BITS, int SUBS, int CAP>
__global__ void __launch_bounds__(Many<D, BITS, SUBS>::THREADS, 1) many_items_kernel(const __grid_constant__ QuantAttnArgs a, const __grid_constant__ QuantAttnCut cut, int blocks, float* part_o, float2* part_ml) {
    using L = Many<D, BITS, SUBS>;
    constexpr int G = L::G, KST = L::K_STAGES, VST = L::V_STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * KST + 2 * VST + 8 * SUBS];
    __shared__ uint32_t tmem_slot;
    __shared__ int4 k_info[4], v_info[4];               // exponents of each 16 keys and values of a tile, times 4; bit 0 tells of values' scales that are not finite, bit 1 of exponents for each key
    __shared__ int key_exponents[2][4][kKeyTile];       // of keys and of values, where the bit is set
    __shared__ uint32_t key_bounds[kCodeWarps][kTile];
    __shared__ uint32_t odd_groups[4][kKeyTile];        // groups of a key's values whose scales are not finite, where the bit is set
    uint64_t *k_full = bars, *k_empty = k_full + KST, *v_full = k_empty + KST, *v_empty = v_full + VST, *s_full = v_empty + VST, *p_full = s_full + 2 * SUBS,
             *o_done = p_full + 2 * SUBS, *q_full = o_done + 2 * SUBS, *drained = q_full + SUBS;
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ks = qs + SUBS * L::Q_BYTES;
    uint8_t* vs = ks + KST * L::TILE_BYTES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const QuantPools& p = a.pools;
    const int g = a.q_heads / p.kv_heads;
    // the longest lanes come first, and of each the last rows, which see the most keys: what is left at the end is short
    const int of_slot = p.kv_heads * blocks, slot = blockIdx.x / of_slot, rest = blockIdx.x - slot * of_slot, block = blocks - 1 - rest / p.kv_heads, kvh = rest % p.kv_heads;
    const Piece piece = piece_of(a, cut, slot, -1);
    if (piece.lane < 0) return;
    const int lane_id = cut.split ? piece.lane : lane_of_rank(a.lanes, slot), share = piece.share, shares = piece.shares;
    const LaneRange at = lane_range(a, lane_id);
    const int item0 = block * (SUBS * kItemTile), n_items = min(SUBS * kItemTile, at.n * g - item0);
    if (n_items <= 0) return;
    const Shares sh = shares_of(a, at, item0, n_items, g, shares);
    if (share > 0 && share >= sh.used()) return;
    const int begin = sh.begin + share * sh.chunk, lo = max(sh.lo, begin), hi = min(sh.hi, begin + sh.chunk);
    const int n_tiles = hi > lo ? (hi - begin + kKeyTile - 1) / kKeyTile : 0, subs = SUBS == 1 || n_items <= kItemTile ? 1 : 2;

    if (tid == 0) {
        for (int i = 0; i < KST; ++i) bar_init(&k_full[i], 4), bar_init(&k_empty[i], subs);
        for (int i = 0; i < VST; ++i) bar_init(&v_full[i], 4), bar_init(&v_empty[i], subs);
        for (int i = 0; i < 2 * SUBS; ++i) bar_init(&s_full[i], 1), bar_init(&p_full[i], kItemTile), bar_init(&o_done[i], 1);
        for (int i = 0; i < SUBS; ++i) bar_init(&q_full[i], kItemTile), bar_init(&drained[i], 1);
        bar_init_fence();
    }
    if (warp == L::MMA_WARP) tmem_alloc(&tmem_slot, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();   // with the tensor memory taken: the next kernel may wait for some

    if (warp >= L::ITEM_WARPS && warp < L::MMA_WARP) {
        // ---- codes to numbers: 16 keys, or their values, of each tile
        if constexpr (L::SPLIT_REGISTERS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::CODE_REGISTERS));
        const int w = warp & 3;
        const bool keys = warp - L::ITEM_WARPS < 4;
        const int32_t* table = a.lanes.tables + lane_id * a.lanes.ld_table;
        const uint8_t* codes_of = (keys ? p.k_codes : p.v_codes) + (int64_t)kvh * p.block_tokens * L::ROW;
        const uint32_t* scales_of = (keys ? p.k_scales : p.v_scales) + (int64_t)kvh * p.block_tokens * G;
        auto there = [&](int t) { return t < n_tiles && begin + t * kKeyTile + w * kTile < hi; };
        auto page_of = [&](int t) {   // the page of tile t's 16 keys
            if (!there(t)) return 0;
            const int32_t page = table[(begin + t * kKeyTile + w * kTile) >> p.bt_shift];
            if ((uint32_t)page < (uint64_t)p.pages) return page;
            tell(a.lanes.status, kDevBadPage);
            return 0;
        };
        int page_now = page_of(lane), page_next = n_tiles > 32 ? page_of(32 + lane) : 0;
        // A thread's pieces: eight threads that store at once have two pieces, 64 bytes of numbers apart, of four keys, whose chunks lie on eight different groups of banks.
        auto key_of_pass = [&](int i) { return (lane >> 1 & 3) + ((lane >> 3) + 4 * i) / (L::PIECES / 2) * 4; };
        auto piece_of_pass = [&](int i) {
            const int rest = ((lane >> 3) + 4 * i) % (L::PIECES / 2);
            return BITS == 4 ? (lane & 1) + 2 * rest : (lane & 1) * 2 + (rest & 1) + 4 * (rest >> 1);
        };
        struct Raw {
            uint4 codes[L::PASSES];
            uint32_t scales[L::PASSES];
        };
        auto load = [&](int t, Raw& r) {
            if ((t & 31) == 0 && t > 0) {
                page_now = page_next;
                page_next = page_of(t + 32 + lane);
            }
            const int64_t page = __shfl_sync(0xffffffffu, page_now, t & 31);
            if (!there(t)) {
                r = Raw{};
                return;
            }
            const int row = (begin + t * kKeyTile + w * kTile) & (p.block_tokens - 1);
            const uint8_t* codes = codes_of + page * p.codes_stride + row * L::ROW;
            const uint32_t* scales = scales_of + page * p.scales_stride + row * G;
#pragma unroll
            for (int i = 0; i < L::PASSES; ++i) {
                const int key = key_of_pass(i), piece = piece_of_pass(i);
                r.codes[i] = *reinterpret_cast<const uint4*>(codes + key * L::ROW + piece * 16);
                r.scales[i] = scales[key * G + piece * 8 * L::CHUNKS / kQuantGroup];
            }
        };
        uint64_t *mine_full = keys ? k_full : v_full, *mine_empty = keys ? k_empty : v_empty;
        const int stages = keys ? KST : VST;
        uint8_t* tiles = (keys ? ks : vs) + w * kTile * 128;
        int stage = 0, e = -120;
        uint32_t empty_parity = 1;
        float by = power_of_two(120);
        uint32_t most = 0, least = 1, fine = 1;   // bounds, as bits, for which the exponent stays; below which a group's numbers would have fewer than 11 bits
        auto make = [&](int t, const Raw& r) {
            const int pos0 = begin + t * kKeyTile + w * kTile;
            float2 sl[L::PASSES];
            uint32_t bound = 0, small = UINT32_MAX;   // of the numbers' absolute values, as bits: what is not finite is above all others; the smallest group's, less one, so that zeros are above too
            auto bound_of = [](float2 v) { return max_nan(fabsf(v.y), fabsf(fmaf(v.x, (float)((1 << BITS) - 1), v.y))); };
#pragma unroll
            for (int i = 0; i < L::PASSES; ++i) {
                const int pos = pos0 + key_of_pass(i);
                sl[i] = pos >= lo && pos < hi ? wide_pair<T>(r.scales[i]) : make_float2(0.f, 0.f);
                const uint32_t b = __float_as_uint(bound_of(sl[i]));
                bound = max(bound, b);
                small = min(small, b - 1u);
            }
            bound = __reduce_max_sync(0xffffffffu, bound);
            uint32_t odd = 0;   // passes
            auto follow = [&](int to) {
                e = to;
                by = power_of_two(-e);
                most = min((uint32_t)(127 + 15 + e) << 23, 0x7f7fffffu);
                least = (uint32_t)max(127 + 15 - 16 + e, 1) << 23;
                fine = (uint32_t)max(127 - 6 + e, 1) << 23;
            };
            if (bound > most || bound < least) {
                if (bound >= 0x7f800000u) {   // the largest of the finite ones; values whose scales are not count as 0
                    float fine_bound = 0.f;
#pragma unroll
                    for (int i = 0; i < L::PASSES; ++i) {
                        const float b = bound_of(sl[i]);
                        if (b < INFINITY) fine_bound = fmaxf(fine_bound, b);
                        else odd |= 1u << i;
                        if (!(b < INFINITY) && !keys) sl[i] = make_float2(0.f, 0.f);
                    }
                    bound = __reduce_max_sync(0xffffffffu, __float_as_uint(fine_bound));
                }
                follow(exponent_of(__uint_as_float(bound), e));
            }
            // a group whose step, and with it its numbers, f16 would cut off: exponents for each key, unless the 16 keys' had only stayed above
            bool apart = __any_sync(0xffffffffu, small < fine - 1u) != 0;
            if (apart && exponent_of(__uint_as_float(bound), -120) < e) {
                follow(exponent_of(__uint_as_float(bound), -120));
                apart = __any_sync(0xffffffffu, small < fine - 1u) != 0;
            }
            const bool any_odd = !keys && __any_sync(0xffffffffu, odd != 0);
            if (!__all_sync(0xffffffffu, bar_wait(&mine_empty[stage], empty_parity))) return false;
            if (any_odd) {
                if (lane < kTile) odd_groups[t & 3][w * kTile + lane] = 0;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < L::PASSES; ++i)
                    if (odd >> i & 1) atomicOr(&odd_groups[t & 3][w * kTile + key_of_pass(i)], 1u << (piece_of_pass(i) * 8 * L::CHUNKS / kQuantGroup));
            }
            if (lane == 0) reinterpret_cast<int*>(keys ? &k_info[t & 3] : &v_info[t & 3])[w] = e * 4 | (apart ? 2 : 0) | (any_odd ? 1 : 0);
            uint8_t* to = tiles + stage * L::TILE_BYTES;
            if (apart) {   // numbers from 32 bits; rare, so that codes and scales are read again, one pass after the other
                uint32_t* bounds = key_bounds[warp - L::ITEM_WARPS];
                if (lane < kTile) bounds[lane] = 0;
                __syncwarp();
                const int64_t page = page_of(t);
                const int row0 = pos0 & (p.block_tokens - 1);
                const uint32_t* scales = scales_of + page * p.scales_stride + row0 * G;
                auto scale_of = [&](int i) {
                    const int key = key_of_pass(i);
                    const float2 v = pos0 + key >= lo && pos0 + key < hi ? wide_pair<T>(scales[key * G + piece_of_pass(i) * 8 * L::CHUNKS / kQuantGroup]) : make_float2(0.f, 0.f);
                    return keys || bound_of(v) < INFINITY ? v : make_float2(0.f, 0.f);
                };
#pragma unroll 1
                for (int i = 0; i < L::PASSES; ++i) {
                    const uint32_t b = __float_as_uint(bound_of(scale_of(i)));
                    if (b < 0x7f800000u) atomicMax(&bounds[key_of_pass(i)], b);
                }
                __syncwarp();
                if (lane < kTile) key_exponents[keys ? 0 : 1][t & 3][w * kTile + lane] = exponent_of(__uint_as_float(bounds[lane]), -120);
#pragma unroll 1
                for (int i = 0; i < L::PASSES; ++i) {
                    const int key = key_of_pass(i), chunk0 = piece_of_pass(i) * L::CHUNKS;
                    const float2 v = scale_of(i);
                    const float by_key = power_of_two(-exponent_of(__uint_as_float(bounds[key]), -120)), step = v.x * by_key, low = v.y * by_key;
                    const uint4 codes = *reinterpret_cast<const uint4*>(codes_of + page * p.codes_stride + (row0 + key) * L::ROW + piece_of_pass(i) * 16);
                    const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
                    auto number = [&](uint32_t bits) { return narrow_pair<__half>(fmaf(step, (float)(bits & 0xffffu), low), fmaf(step, (float)(bits >> 16), low)); };
                    uint8_t* row = to + (chunk0 >> 3) * L::PANEL + key * 128;
#pragma unroll
                    for (int j = 0; j < L::CHUNKS; ++j) {
                        uint4 out;
                        if constexpr (BITS == 4) {
                            const uint32_t x = words[j];
                            out = make_uint4(number(x & 0x000f000fu), number(x >> 4 & 0x000f000fu), number(x >> 8 & 0x000f000fu), number(x >> 12 & 0x000f000fu));
                        } else {
                            const uint32_t x = words[2 * j], y = words[2 * j + 1];
                            out = make_uint4(number(x & 0x00ff00ffu), number(x >> 8 & 0x00ff00ffu), number(y & 0x00ff00ffu), number(y >> 8 & 0x00ff00ffu));
                        }
                        *reinterpret_cast<uint4*>(row + (((chunk0 + j & 7) ^ (key & 7)) << 4)) = out;
                    }
                }
            } else
#pragma unroll
            for (int i = 0; i < L::PASSES; ++i) {
                const __half2 step = __float2half2_rn(sl[i].x * by), part = __hmul2(step, __float2half2_rn(0.0625f)), low = __float2half2_rn(sl[i].y * by);   // codes in bits 4 .. 7 are 16 times theirs
                const uint32_t words[4] = {r.codes[i].x, r.codes[i].y, r.codes[i].z, r.codes[i].w};
                auto number = [&](uint32_t bits, __half2 by_step) {   // 1024 + c, c, low + step c
                    bits |= 0x64006400u;
                    const __half2 y = __hfma2(__hadd2(as_half2(bits), __float2half2_rn(-1024.f)), by_step, low);
                    return *reinterpret_cast<const uint32_t*>(&y);
                };
                const int key = key_of_pass(i), chunk0 = piece_of_pass(i) * L::CHUNKS;
                uint8_t* row = to + (chunk0 >> 3) * L::PANEL + key * 128;
#pragma unroll
                for (int j = 0; j < L::CHUNKS; ++j) {
                    uint4 out;
                    if constexpr (BITS == 4) {
                        const uint32_t x = words[j], y = x >> 8;
                        out = make_uint4(number(x & 0x000f000fu, step), number(x & 0x00f000f0u, part), number(y & 0x000f000fu, step), number(y & 0x00f000f0u, part));
                    } else {
                        const uint32_t x = words[2 * j], y = words[2 * j + 1];
                        out = make_uint4(number(x & 0x00ff00ffu, step), number(x >> 8 & 0x00ff00ffu, step), number(y & 0x00ff00ffu, step), number(y >> 8 & 0x00ff00ffu, step));
                    }
                    *reinterpret_cast<uint4*>(row + (((chunk0 + j & 7) ^ (key & 7)) << 4)) = out;
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(&mine_full[stage]);
            if (++stage == stages) stage = 0, empty_parity ^= 1;
            return true;
        };
        // two tiles on their way
        Raw even, uneven;
        load(0, even);
        load(1, uneven);
        bool ok = true;
#pragma unroll 1
        for (int t = 0; t < n_tiles; t += 2) {
            ok = make(t, even);
            if (!ok) break;
            load(t + 2, even);
            if (t + 1 == n_tiles) break;
            ok = make(t + 1, uneven);
            if (!ok) break;
            load(t + 3, uneven);
        }
        if (!ok && lane == 0) tell(a.lanes.status, kDevWait);
    } else if (warp >= L::MMA_WARP) {
        // ---- products
        if constexpr (L::SPLIT_REGISTERS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::OTHER_REGISTERS));
        const int sub = warp - L::MMA_WARP;   // a warp for each tile of items: the whole of it waits, one thread issues
        if (sub < subs && n_tiles > 0) {
            constexpr uint32_t i_scores = f16_idesc(kItemTile, kKeyTile, false), i_out = f16_idesc(kItemTile, D, true);
            const bool issues = elect_one();
            const uint64_t q = sw128_desc(smem_u32(qs) + sub * L::Q_BYTES), k0 = sw128_desc(smem_u32(ks)), v0 = sw128_desc(smem_u32(vs), L::PANEL);
            const uint32_t s_base = tmem + L::S_AT + sub * 2 * kKeyTile, o_base = tmem + sub * D;
            auto scores = [&](int t) {
                const int st = t % KST;
                if (!__all_sync(0xffffffffu, bar_wait(&k_full[st], t / KST & 1))) return false;
                fence_after();
                if (issues) {
                    const uint64_t k = k0 + st * (L::TILE_BYTES / 16);
                    const uint32_t to = s_base + (t & 1) * kKeyTile;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) mma(to, q + (i >> 2) * (L::Q_PANEL / 16) + (i & 3) * 2, k + (i >> 2) * (L::PANEL / 16) + (i & 3) * 2, i_scores, i > 0);
                    commit(&s_full[sub * 2 + (t & 1)]);
                    commit(&k_empty[st]);
                }
                __syncwarp();
                return true;
            };
            bool ok = __all_sync(0xffffffffu, bar_wait(&q_full[sub], 0));
            fence_after();
            ok = ok && scores(0);
            for (int t = 0; t < n_tiles && ok; ++t) {
                // scores of tile t + 1 go to the area that P of tile t - 1 occupied: its product was issued before, and products of one thread run in the order of their issue
                if (t + 1 < n_tiles && !scores(t + 1)) {
                    ok = false;
                    break;
                }
                const int st = t % VST;
                ok = __all_sync(0xffffffffu, bar_wait(&v_full[st], t / VST & 1) && bar_wait(&p_full[sub * 2 + (t & 1)], t >> 1 & 1));
                if (!ok) break;
                fence_after();
                if (issues) {
                    const uint64_t v = v0 + st * (L::TILE_BYTES / 16);
                    const uint32_t from = s_base + (t & 1) * kKeyTile;
#pragma unroll
                    for (int i = 0; i < kKeyTile / 16; ++i) mma_tmem_a(o_base, from + i * 8, v + i * 128, i_out, t > 0 || i > 0);
                    commit(&o_done[sub * 2 + (t & 1)]);
                    commit(&v_empty[st]);
                }
                __syncwarp();
            }
            if (!ok && lane == 0) tell(a.lanes.status, kDevWait);
            // products under way end before the memory of their operands and results is given back, whoever gave up a wait
            if (issues) commit(&drained[sub]);
            __all_sync(0xffffffffu, bar_wait(&drained[sub], 0));
        }
    } else if (warp < 4 * subs) {
        // ---- an item to a thread
        if constexpr (L::SPLIT_REGISTERS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::ITEM_REGISTERS));
        const int sub = warp >> 2, item = tid, row = item0 + item < at.n * g ? (item0 + item) / g : 0, head = item0 + item - row * g;
        const bool mine = item < n_items;
        const float unit = CAP ? a.scale : a.scale * kLog2e;
        float factor;   // of scores that come from scaled queries
        {
            const T* q = static_cast<const T*>(a.q) + (int64_t)(at.first + row) * a.ldq + (kvh * g + head) * D;
            float top = 0.f;
            if (mine) {
#pragma unroll 4
                for (int c = 0; c < D; c += 8) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + c);
                    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 y = wide_pair<T>(u[j]);
                        top = max3(top, fabsf(y.x), fabsf(y.y));
                    }
                }
            }
            // the largest becomes 2^14 and a bit, exactly
            const int e = top > 0.f ? min(max(14 - (int)((__float_as_uint(top) >> 23) - 127), -100), 100) : 0;
            const float up = power_of_two(e);
            factor = unit * power_of_two(-e);
            uint8_t* to = qs + sub * L::Q_BYTES + (item & 127) * 128;
#pragma unroll 4
            for (int c = 0; c < D; c += 8) {
                uint32_t out[4] = {0u, 0u, 0u, 0u};
                if (mine) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + c);
                    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 z = wide_pair<T>(u[j]);
                        y[place_of<BITS>(2 * j)] = z.x * up;
                        y[place_of<BITS>(2 * j + 1)] = z.y * up;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) out[j] = narrow_pair<__half>(y[2 * j], y[2 * j + 1]);
                }
                *reinterpret_cast<uint4*>(to + (c >> 6) * L::Q_PANEL + ((((c & 63) * 2) ^ ((item & 7) << 4)))) = make_uint4(out[0], out[1], out[2], out[3]);
            }
            fence_async_smem();
            bar_arrive(&q_full[sub]);
        }
        const int pos = at.position + row, see_lo = max(lo, attention_first_key(max(pos, 0), a.window, 0)), see_hi = mine ? min(hi, pos + 1) : 0;
        // keys that all rows of the tile of items see
        const int last = min(item0 + n_items, item0 + (sub + 1) * kItemTile) - 1, p0 = at.position + (item0 + sub * kItemTile) / g, p1 = at.position + last / g;
        const int all_lo = max(lo, attention_first_key(max(p1, 0), a.window, 0)), all_hi = min(hi, p0 + 1);
        const uint32_t my = tmem + ((uint32_t)((warp & 3) * 32) << 16), my_o = my + sub * D;
        const float two_over_cap = CAP ? 2.0f / a.softcap : 0.f;
        const bool wide_cap = CAP && a.softcap > kCapOfDifference;
        float m_run = -INFINITY, sum = 0.f;   // the score whose weight is 1: kWeightBits below a maximum
        int e_run = -120;
        uint32_t odd = 0;
        bool ok = true;
#pragma unroll 1
        for (int t = 0; t < n_tiles; ++t) {
            const int area = sub * 2 + (t & 1);
            ok = __all_sync(0xffffffffu, bar_wait(&s_full[area], t >> 1 & 1));
            if (!ok) break;
            fence_after();
            const uint32_t s_at = my + L::S_AT + area * kKeyTile;
            float s[kKeyTile];
            tmem_ld32(s_at, reinterpret_cast<uint32_t*>(s));
            tmem_ld32(s_at + 32, reinterpret_cast<uint32_t*>(s) + 32);
            const int4 ki = k_info[t & 3];
            const int pos0 = begin + t * kKeyTile;
            tmem_wait_ld();
            // neither 0 nor infinite: where it would be, scores are 0 or overflow whatever it is
            auto unit_of = [&](int e) { return fminf(fmaxf(factor * power_of_two(e), 1e-37f), 3e38f); };
            float u = unit_of(ki.x >> 2);
            if (CAP || ((ki.x ^ ki.y) | (ki.x ^ ki.z) | (ki.x ^ ki.w) | (ki.x & 2)) != 0) {   // scores one by one; then they are what is exponentiated
                const int info[4] = {ki.x, ki.y, ki.z, ki.w};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float ub = unit_of(info[b] >> 2);
                    if (info[b] & 2) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[b * 16 + j] *= unit_of(key_exponents[0][t & 3][b * 16 + j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[b * 16 + j] *= ub;
                    }
                    if (CAP) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float v = s[b * 16 + j];
                            s[b * 16 + j] = (wide_cap ? capped_wide(v, a.softcap, two_over_cap) : capped(v, a.softcap, two_over_cap)) * kLog2e;
                        }
                    }
                }
                u = 1.f;
            }
            if (pos0 < all_lo || pos0 + kKeyTile > all_hi) {   // uniform: some row does not see the whole tile
#pragma unroll
                for (int j = 0; j < kKeyTile; ++j) s[j] = pos0 + j >= see_lo && pos0 + j < see_hi ? s[j] : -INFINITY;
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int j = 4; j < kKeyTile; j += 8) {
#pragma unroll
                for (int k = 0; k < 4; ++k) top[k] = j + k + 4 < kKeyTile ? max3(top[k], s[j + k], s[j + k + 4]) : fmaxf(top[k], s[j + k]);
            }
            const float m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * u;
            const bool none = m_run == -INFINITY;
            float less = 0.f, alpha = 1.f;   // what the maximum has risen by, negative
            if (m_tile > m_run + (kSlack + kWeightBits)) {   // also when there was none yet
                less = none ? 0.f : m_run - (m_tile - kWeightBits);
                alpha = ex2(less);
                sum *= alpha;
                m_run = m_tile - kWeightBits;
            }
            const float m_use = m_run == -INFINITY ? 0.f : m_run;
            FloatPair part[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
            for (int j = 0; j < kKeyTile; j += 2) {
                const FloatPair y = fma2(FloatPair{s[j], s[j + 1]}, FloatPair{u, u}, FloatPair{-m_use, -m_use}), e{ex2(y.x), ex2(y.y)};
                s[j] = e.x;
                s[j + 1] = e.y;
                part[j >> 1 & 1] = part[j >> 1 & 1] + e;
            }
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
            ok = __all_sync(0xffffffffu, bar_wait(&v_full[t % VST], t / VST & 1));
            if (!ok) break;
            const int4 vi = v_info[t & 3];
            // Exponents of the values: one for all, by which weights are scaled where a tile's differ.  It follows what the row's weights make of them, so that large values that it does not see, or
            // sees with little weight, take nothing off the others.
            if (none && ((vi.x ^ vi.y) | (vi.x ^ vi.z) | (vi.x ^ vi.w) | (vi.x & 3)) == 0) {
                if (m_run != -INFINITY) e_run = vi.x >> 2;   // its largest weight is 2^kWeightBits
            } else if (((vi.x ^ e_run * 4) | (vi.y ^ e_run * 4) | (vi.z ^ e_run * 4) | (vi.w ^ e_run * 4)) != 0) {
                const int info[4] = {vi.x, vi.y, vi.z, vi.w}, ev[4] = {vi.x >> 2, vi.y >> 2, vi.z >> 2, vi.w >> 2};
                const int* of_keys = key_exponents[1][t & 3];
                int top = -1000;   // weights times 2^e are below 2^top
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (info[b] & 2) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (s[b * 16 + j] > 0.f) top = max(top, of_keys[b * 16 + j] + exponent(fminf(s[b * 16 + j], 32767.f)) + 1);
                    } else {
                        float most = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) most = fmaxf(most, s[b * 16 + j]);
                        if (most > 0.f) top = max(top, ev[b] + exponent(fminf(most, 32767.f)) + 1);
                    }
                }
                const int low = max(e_run - (int)fminf(-less, 240.f), -120);   // what came so far has become less
                const bool alike = ev[0] == ev[1] && ev[0] == ev[2] && ev[0] == ev[3] && ((vi.x | vi.y | vi.z | vi.w) & 2) == 0;
                const int e = alike && top >= ev[0] + 4 && top <= ev[0] + 15 && low <= ev[0] + 8 ? ev[0] : (top > low + 15 ? top - 8 : low);
                alpha = ex2(less + (float)(e_run - e));
                e_run = e;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    auto to = [&](int from) { return from - e < -126 ? 0.f : power_of_two(min(from - e, 126)); };
                    const float all = to(ev[b]);
                    if (info[b] & 2) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[b * 16 + j] *= to(of_keys[b * 16 + j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[b * 16 + j] *= all;
                    }
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (!(info[b] & 1)) continue;
                    for (int j = b * 16; j < b * 16 + 16; ++j)
                        if (pos0 + j >= see_lo && pos0 + j < see_hi) odd |= odd_groups[t & 3][j];
                }
            }
            if (t > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                ok = __all_sync(0xffffffffu, bar_wait(&o_done[sub * 2 + (t - 1 & 1)], t - 1 >> 1 & 1));
                if (!ok) break;
                fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(my_o + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                    tmem_st32(my_o + c, o);
                }
            }
            uint32_t w[kKeyTile / 2];
#pragma unroll
            for (int j = 0; j < kKeyTile / 2; ++j) w[j] = narrow_pair<__half>(s[2 * j], s[2 * j + 1]);
            tmem_st32(s_at, w);
            tmem_wait_st();
            fence_before();
            bar_arrive(&p_full[area]);
        }
        if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, bar_wait(&o_done[sub * 2 + (n_tiles - 1 & 1)], n_tiles - 1 >> 1 & 1));
        if (!ok && lane == 0) tell(a.lanes.status, kDevWait);
        fence_after();
        const float inv = !ok ? NAN : (sum == 0.f ? 0.f : 1.0f / sum), back = power_of_two(e_run);
        const int64_t out_row = (int64_t)(at.first + row), part_row = ((int64_t)slot * a.lanes.rows + row) * a.q_heads + kvh * g + head;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (n_tiles > 0 && ok) {
                tmem_ld32(my_o + c, o);
                tmem_wait_ld();
            }
            if (!mine) continue;
            float x[32];
            const bool none = sum == 0.f && ok, not_a_number = odd >> (c / kQuantGroup) & 1;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float v = __uint_as_float(o[j / 8 * 8 + place_of<BITS>(j % 8)]);
                x[j] = none ? 0.f : (not_a_number ? NAN : v * inv * back);
            }
            if (shares == 1) {
                T* to = static_cast<T*>(a.out) + out_row * a.ldo + (kvh * g + head) * D + c;
#pragma unroll
                for (int j = 0; j < 32; j += 8)
                    *reinterpret_cast<uint4*>(to + j) = make_uint4(narrow_pair<T>(x[j], x[j + 1]), narrow_pair<T>(x[j + 2], x[j + 3]), narrow_pair<T>(x[j + 4], x[j + 5]), narrow_pair<T>(x[j + 6], x[j + 7]));
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(part_o + part_row * D + c + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            }
        }
        if (mine && shares > 1) part_ml[part_row] = make_float2(m_run, ok ? sum : NAN);
    }
    fence_before();
    __syncthreads();
    if (warp == L::MMA_WARP) {
        fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- shares joined ---------------------------------------------------------------------------------------------------
//
// WARPS warps to a (row, query head), a part to each in turn, eight of them on their way; where parts are many and rows few, the chain of loads is what it takes (48 rows of 100 parts: 18 us with a warp each).
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ QuantAttnArgs a, const __grid_constant__ QuantAttnCut cut, int items_of_block, const float* part_o, const float2* part_ml) {
    constexpr int V = D / 32, ROWS = 4 / WARPS, AHEAD = 8;
    __shared__ float sums[WARPS > 1 ? WARPS : 1][D];
    __shared__ float2 warp_ml[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = a.q_heads / a.pools.kv_heads, mine = warp % WARPS;
    const int lane_id = blockIdx.x;
    const Piece piece = piece_of(a, cut, 0, lane_id);
    const LaneRange at = lane_range(a, lane_id);
    pdl_wait();
    if (piece.shares == 1) return;   // written as it is
    const int64_t n_rows = (int64_t)a.lanes.rows * a.q_heads, n = (int64_t)at.n * a.q_heads;
    for (int64_t row0 = (int64_t)blockIdx.y * ROWS; row0 < n; row0 += (int64_t)gridDim.y * ROWS) {
        const int64_t at_row = row0 + warp / WARPS;
        const bool there = at_row < n;
        const int r = there ? (int)(at_row / a.q_heads) : 0, head = there ? (int)(at_row - (int64_t)r * a.q_heads) : 0, item = r * g + head % g, item0 = item / items_of_block * items_of_block;
        const int used = there ? max(1, shares_of(a, at, item0, min(items_of_block, at.n * g - item0), g, piece.shares).used()) : 0;
        const int64_t row = piece.slot * n_rows + at_row;
        float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
        for (int s0 = mine * 32; s0 < used; s0 += WARPS * 32) {
            const float2 ml = s0 + lane < used ? __ldcg(part_ml + (s0 + lane) * n_rows + row) : make_float2(-INFINITY, 0.f);
            const float m_new = fmaxf(m, warp_max(ml.x)), m_use = m_new == -INFINITY ? 0.f : m_new;
            const float old = ex2(m - m_use), f = ml.y == 0.f ? 0.f : ml.y * ex2(ml.x - m_use);
            l = l * old + warp_sum(f);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] *= old;
            m = m_new;
            const int parts = min(32, used - s0);
            for (int b = 0; b < parts; b += AHEAD) {
                float x[AHEAD][V], w[AHEAD];
#pragma unroll
                for (int s = 0; s < AHEAD; ++s) {
                    w[s] = b + s < 32 ? __shfl_sync(0xffffffffu, f, b + s) : 0.f;
#pragma unroll
                    for (int j = 0; j < V; ++j) x[s][j] = 0.f;
                    if (b + s >= parts) continue;   // not by its weight: one of 0 does not hide NaN
                    const float* src = part_o + ((s0 + b + s) * n_rows + row) * D + lane * V;
#pragma unroll
                    for (int j = 0; j < V; j += 2) {
                        const float2 y = __ldcg(reinterpret_cast<const float2*>(src + j));
                        x[s][j] = y.x;
                        x[s][j + 1] = y.y;
                    }
                }
#pragma unroll
                for (int s = 0; s < AHEAD; ++s)
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = fmaf(w[s], x[s][j], o[j]);
            }
        }
        if constexpr (WARPS > 1) {
            if (lane == 0) warp_ml[warp] = make_float2(m, l);
#pragma unroll
            for (int j = 0; j < V; ++j) sums[mine][lane * V + j] = o[j];
            __syncthreads();
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, warp_ml[w].x);
            l = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 ml = warp_ml[w];
                if (ml.y == 0.f) continue;
                const float f = ex2(ml.x - (top == -INFINITY ? 0.f : top));
                l = fmaf(ml.y, f, l);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = fmaf(f, sums[w][lane * V + j], o[j]);
            }
            __syncthreads();
        }
        if (!there || mine != 0) continue;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* out = static_cast<T*>(a.out) + (int64_t)(at.first + r) * a.ldo + head * D + lane * V;
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<uint32_t*>(out + j) = narrow_pair<T>(o[j] * inv, o[j + 1] * inv);
    }
}

template <typename T, int D, int BITS, int NT, int CAP>
void launch_few(const QuantAttnArgs& a, const QuantAttnPlan& p, float* part_o, float2* part_ml, cudaStream_t s) {
    auto* kernel = few_items_kernel<T, D, BITS, NT, CAP>;
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), Few<D, BITS, NT>::SMEM);
    kernel<<<dim3((unsigned)p.slots, (unsigned)a.pools.kv_heads, (unsigned)p.blocks), kWarps * 32, Few<D, BITS, NT>::SMEM, s>>>(a, p.cut, part_o, part_ml);
    MK_LAUNCH_CHECK();
}

template <typename T, int D, int BITS, int CAP>
void launch_many(const QuantAttnArgs& a, const QuantAttnPlan& p, float* part_o, float2* part_ml, cudaStream_t s) {
    constexpr int SUBS = D == 256 ? 1 : 2;
    using L = Many<D, BITS, SUBS>;
    auto* kernel = many_items_kernel<T, D, BITS, SUBS, CAP>;
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::SMEM);
    if constexpr (L::SPLIT_REGISTERS) {   // warps that ask for more registers than the launch has would wait for good
        static const int registers = [&] {
            cudaFuncAttributes at{};
            cuda_check(cudaFuncGetAttributes(&at, kernel), "function attributes", __FILE__, __LINE__);
            return at.numRegs;
        }();
        if (registers < L::LAUNCH_REGISTERS) throw std::runtime_error("quantized attention: the kernel was built with fewer registers than its warps share out");
    }
    kernel<<<(unsigned)(p.slots * a.pools.kv_heads * p.blocks), L::THREADS, L::SMEM, s>>>(a, p.cut, p.blocks, part_o, part_ml);
    MK_LAUNCH_CHECK();
}

template <typename T, int D>
void launch(const QuantAttnArgs& a, const QuantAttnPlan& p, void* workspace, cudaStream_t s) {
    float* part_o = static_cast<float*>(workspace);
    float2* part_ml = reinterpret_cast<float2*>(part_o + (p.cut.split ? p.slots * (int64_t)a.lanes.rows * a.q_heads * D : 0));
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    auto few = [&](auto bits, auto nt) {
        constexpr int B = decltype(bits)::value, N = decltype(nt)::value;
        a.softcap != 0.f ? launch_few<T, D, B, N, 1>(a, p, part_o, part_ml, s) : launch_few<T, D, B, N, 0>(a, p, part_o, part_ml, s);
    };
    auto many = [&](auto bits) {
        constexpr int B = decltype(bits)::value;
        a.softcap != 0.f ? launch_many<T, D, B, 1>(a, p, part_o, part_ml, s) : launch_many<T, D, B, 0>(a, p, part_o, part_ml, s);
    };
    if (p.items > 16) {
        a.pools.bits == 4 ? many(Four{}) : many(Eight{});
    } else if (p.items == 8) {
        a.pools.bits == 4 ? few(Four{}, One{}) : few(Eight{}, One{});
    } else {
        if constexpr (D != 256) a.pools.bits == 4 ? few(Four{}, Two{}) : few(Eight{}, Two{});   // heads of 256: 255 registers and more, so they take two blocks instead
    }
    if (p.cut.split) {
        const int64_t rows = (int64_t)a.lanes.rows * a.q_heads;
        // rows that do not fill the SMs with a warp each get four
        const bool few_rows = rows * a.lanes.lanes <= 4 * 16 * kSms;
        launch_pdl(few_rows ? join_kernel<T, D, 4> : join_kernel<T, D, 1>, dim3((unsigned)a.lanes.lanes, (unsigned)std::min<int64_t>(few_rows ? rows : (rows + 3) / 4, 4096)), dim3(128), 0, s, a, p.cut,
                   p.items, (const float*)part_o, (const float2*)part_ml);
        MK_LAUNCH_CHECK();
    }
}

}  // namespace

QuantAttnPlan quantized_attention_plan(int q_heads, int kv_heads, int d, int bits, int block_tokens, int width, int lanes, int rows, int total, int window) {
    QuantAttnPlan p;
    const int64_t items = (int64_t)rows * (q_heads / kv_heads);
    // Up to 32 items go by blocks of 16 (heads of 256: of 8), each of which walks the keys, out of L2 but for the first: 24 lanes of 20 items, heads of 128, 137 us where the tall kernel takes 145; 8 lanes of 32 60 and 59;
    // heads of 256, 12 lanes of 24, 111 and 125.  With 48 items it is the other way round: 88 and 61, 196 and 146, heads of 64 47 and 36.
    p.items = items <= 8 || (items <= kFewItems && d == 256) ? 8 : (items <= kFewItems ? 16 : (d == 256 ? kItemTile : 2 * kItemTile));
    p.blocks = (int)std::max<int64_t>(1, (items + p.items - 1) / p.items);
    // one wave of CTAs
    const int ctas = p.items > 16 ? 1 : few_ctas(d, p.items / 8);
    const double want = (double)kSms * ctas / ((double)kv_heads * p.blocks);
    const int64_t table = (int64_t)width * block_tokens, window_keys = (int64_t)window + rows + 16;
    p.cut.window_keys = (int)std::min<int64_t>(window_keys, INT32_MAX);
    p.cut.least = p.items > 16 ? 256 : 512;
    // Lanes that fill the SMs by themselves, or four times over where they have few items, are not shared out: 4 portions of 375 to 875 rows take 395 us so and 469 shared out, 24 lanes of 12 rows 149 and 163.  The
    // bound does not look at the lengths, which are the device's, and one lane far longer than the others pays for that: 19 lanes of 64 items, one of 12000 tokens among ones of 300, take 207 us and would take 45
    // (18 lanes, which are shared out, 55); 222 single tokens, one of 40000 among ones of 300, 433 and would take 111.
    p.cut.split = (window > 0 ? std::min(table, window_keys) : table) > p.cut.least && lanes < (p.items > 16 ? 1 : 4) * want;
    // A lane's last share is a part of one, so `want` less the lanes is one wave: CTAs of many items are alone on an SM, and few lanes' CTAs all last as long (3 contexts of up to 120001 tokens: 42.3 us,
    // with half as many more shares 52.5).  Many lanes' differ, and a second wave of smaller ones evens them out (48 lanes of 200 to 6000 tokens: 49.9 us; shares of the largest size for one
    // wave 54.9, 2.5 times as many 54.2; 20 lanes of up to five rows, heads of 256: 152, 158 and 149).
    const double shares = p.items > 16 || lanes <= want / 4 ? std::max(want / 2, want - lanes) : 1.5 * want;
    p.cut.want = (float)shares;
    p.slots = p.cut.split ? lanes + (int)std::min(shares, (double)lanes * (double)table / p.cut.least) + 1 : lanes;
    if (p.cut.split) p.bytes = (int64_t)p.slots * rows * q_heads * ((int64_t)d * 4 + 8);
    return p;
}

void launch_quantized_attention(const QuantAttnArgs& a, const QuantAttnPlan& p, void* workspace, cudaStream_t s) {
    auto with_type = [&](auto type) {
        using T = decltype(type);
        switch (a.pools.d) {
            case 64: launch<T, 64>(a, p, workspace, s); break;
            case 128: launch<T, 128>(a, p, workspace, s); break;
            default: launch<T, 256>(a, p, workspace, s); break;
        }
    };
    a.pools.bf16 ? with_type(__nv_bfloat16{}) : with_type(__half{});
}

}  // namespace mk
