// kv8_prefill.cuh — attention of many query rows per request over the paged 8-bit cache (prompts, chunks)
// on the 5th-generation tensor cores.
//
//   s = (Q . Kcode^T) * k_scale * scale * log2 e,  p = 2^(s - m),  O = sum over keys of p * v_scale * Vcode,  out = O / sum p
//
// Bound: the matrix unit (4 head_dim operations per visible pair) and, as large here, the exponentials:
// 128 x 128 of them per tile at 16 a clock take as long as the tile's products. 2048 rows of 32 heads of 128 at 30000
// keys: 1.29 ms, 804 TFLOP/s (half of the measured matrix rate); what is left is the softmax's chain of latencies per tile.
//
//  * Work is the list of 128-key tiles of every (request, KV head, group of query rows), cut into runs of
//    equal cost, one per CTA, as in the decode kernel: causal groups of any length fill all SMs alike. Units
//    that span CTAs are joined through the workspace in key order.
//  * Rows of a group are (token, query head of the KV head): grouped heads share every K and V tile.
//    Two streams of 128 rows per CTA take turns on the matrix unit: while one stream's softmax warps
//    work, the other's products run. fp32 activations (SPLIT): one group of 128 rows, q and the weights as
//    pairs of fp16, and the two streams take the even and the odd tiles. head_dim 256: both take every tile of
//    64 keys, and half the output channels (the scores are made twice: the sums of 256 channels fill two streams' space).
//  * Codes become fp16 exactly, once per tile for both streams, by four converter warps, from stages that
//    TMA fills a tile ahead, and stored as they lie, keys by channels, in 128-byte swizzled shared
//    memory: a K-major operand for S, an MN-major one for O. Scales never touch the codes: k_scale is
//    part of a score's factor and log2 v_scale of the exponent, both constant over 16 keys; the references of a
//    row are its own, as in the decode kernel.
//  * S, then P in its place as fp16 (the weights are the A operand straight from tensor memory), and O
//    stay in tensor memory: 2 x (128 + head_dim) of its 512 columns.
//  * O is rescaled only when one of a row's references grows by more than 2^8 (fp16 weights have that room).
#pragma once

#include "kv8_decode.cuh"

namespace fence {

constexpr int KP_SMS = 148;
constexpr int KP_W_CONV = 8, KP_W_PREP = 12, KP_W_MMA = 13, KP_W_LOAD = 14, KP_THREADS = 480;
constexpr int KP_MIN_TILES = 2, KP_SLOTS = 4;
constexpr int KP_UNIT = 4;  // a unit's start and end cost about as much as four tiles: counted so when the runs are cut
// The matrix unit's additions cut the sum's last bit off, half of it on average and always towards zero: 128 of them (8
// tiles) cost 2e-6, 30000 keys 1.2e-4, and 131000 keys in one go 7e-4, more than fp16's rounding (2^-12 at least). So the sums are
// added, rounded, to the stream's record from time to time: every 4 tiles of a stream for fp32 activations, every
// KP_TURN_KEYS keys for 16 bits (every 8192 keys took 1382 us where this takes 1280, 2048 rows at 30000 keys).
constexpr int KP_TURN_SPLIT = 4, KP_TURN_KEYS = 32768;

template <int HD, bool SPLIT>
struct KPShape {
    static_assert(HD <= 128 || !SPLIT, "two parts of 256 channels of q leave no room for the keys");
    static constexpr bool HALVES = HD == 256;       // the streams share rows and tiles and take 128 output channels each
    static constexpr int KT = HALVES ? 64 : 128;    // keys per tile
    static constexpr int HDO = HALVES ? 128 : HD;   // channels of a stream's sums
    static constexpr int ROWS = SPLIT || HALVES ? 128 : 256;  // per group
    static constexpr int Q_TILE = 128 * HD * 2;     // 128 rows as fp16
    static constexpr int OP = KT * HD * 2;          // a K or V operand tile
    static constexpr int O_Q = 0;  // two tiles: the streams' rows, or the high and low parts; one where the rows are shared
    static constexpr int O_K = (HALVES ? 1 : 2) * Q_TILE;
    static constexpr int O_V = O_K + 2 * OP;
    static constexpr int RAW = KT * HD;             // staged codes of a K or V tile
    static constexpr int O_RAW = O_V + 2 * OP;
    static constexpr int O_BAR = O_RAW + 2 * RAW;
    static constexpr int O_MISC = O_BAR + 256;
    static constexpr int O_PREP = O_MISC + 64;  // [KP_SLOTS][24]: k_scale, log2 v_scale, 1 / v_scale of 8 x 16 keys; [KP_SLOTS][8]: the pool's row of their first
    static constexpr int SMEM = O_PREP + KP_SLOTS * 128 + 1024;
    // tiles between two times; the first of a stream after one is among the next STEP
    static constexpr int STEP = SPLIT ? 2 : 1, TURN = SPLIT ? 2 * KP_TURN_SPLIT : KP_TURN_KEYS / KT;
    static constexpr int REC = 128 * (HDO + 2);  // floats of one stream's partial result
};

// The rows of q as the prefill kernel multiplies them, in its order (KV head, token, query head of the KV head): by a power of
// two into [256, 512), so that fp16 holds them whatever their range is, and what fp16 leaves of them (SPLIT). A pass of
// its own over q: done by the softmax warps at each unit's start it took them 9 us every time (short of independent
// work, with code that the tiles' loops had pushed out of the instruction cache), and TMA can fetch the finished rows while
// the unit before ends. A warp per row.
constexpr int KQ_WARPS = 8;
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(32 * KQ_WARPS) kv8_q_rows_kernel(const KAttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int EPL = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long i = (long long)blockIdx.x * KQ_WARPS + (threadIdx.x >> 5), per_head = (long long)a.n_tokens * a.G;
    if (i >= per_head * a.c.n_kv_heads) return;
    const int tok = (int)(i / a.n_q_heads), head = (int)(i % a.n_q_heads);  // in q's order
    const long long src = tok * a.q_stride + (long long)head * HD + lane * EPL;
    float x[EPL];
    if (SPLIT) {
        const float* p = static_cast<const float*>(a.q) + src;
        if (a.q_wide && EPL == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            x[0] = v.x, x[1] = v.y, x[EPL - 2] = v.z, x[EPL - 1] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e] = p[e];
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(a.q) + src;
        uint32_t w[EPL / 2];
        if (a.q_wide && EPL == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[EPL / 2 - 1] = v.y;
        } else if (a.q_wide && EPL == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1 % (EPL / 2)] = v.y, w[2 % (EPL / 2)] = v.z, w[3 % (EPL / 2)] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < EPL / 2; ++e) w[e] = (uint32_t)p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
        }
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e) {
            if (a.type == FENCE_F16) {
                x[2 * e] = half_bits_to_float(w[e]), x[2 * e + 1] = half_bits_to_float(w[e] >> 16);
            } else {
                x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    }
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
    big = __reduce_max_sync(0xffffffffu, big);
    const int ex = (int)(big >> 23);
    const bool plain = ex == 255;  // infinity or NaN in the row
    const int sh = plain ? 0 : max(ex, 1) - 127 - 8;
    const float f1 = __uint_as_float((uint32_t)(127 - max(min(sh, 126), -126)) << 23);
    const float f2 = sh < -126 ? __uint_as_float((uint32_t)(1 - sh) << 23) : 1.f;
    const int h = head / a.G;
    const long long row = h * per_head + (long long)tok * a.G + (head - h * a.G);
    if (lane == 0) a.q_scale[row] = (plain ? 1.f : ldexpf(1.f, sh)) * a.scale_log2;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.q_rows + row * HD) + lane * (EPL / 2);
    uint32_t* low = dst + per_head * a.c.n_kv_heads * HD / 2;
#pragma unroll
    for (int e = 0; e < EPL; e += 2) {
        const float u = x[e] * f1 * f2, v = x[e + 1] * f1 * f2;
        const uint32_t hi = kd_pack(u, v);
        dst[e / 2] = hi;
        if (SPLIT) low[e / 2] = kd_pack_rest(u, v, hi);
    }
}

// What every role derives for itself from the run's position.
struct KPSeg {
    KReq q;
    int h, row0, nrows, tile0, cnt, first, tiles;  // this CTA's tiles of the unit, its place in the unit, the unit's tiles
    int unit0, next;                               // where the unit's place in the list begins, where this CTA's next one is
    int lo[2], hi[2];                              // the tiles that rows of each stream see
};

template <int KT>
__device__ __forceinline__ void kp_group(const KAttnArgs& a, const KReq& q, int rows_per_group, int gi, int* lo_tile, int* tiles) {
    const int nrows = q.n * a.G, r_lo = gi * rows_per_group, r_hi = min(r_lo + rows_per_group, nrows) - 1;
    const int first = q.kv - q.n + r_lo / a.G, last = q.kv - q.n + r_hi / a.G;
    const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
    *lo_tile = last < 0 ? 0 : lo / KT;
    *tiles = last < 0 ? 1 : last / KT - *lo_tile + 1;
}

// Walks a CTA's run of tiles; every warp does so for itself, all lanes together.
template <int ROWS, int KT>
struct KPWalk {
    int r, base, per_head;  // request, tiles before it, tiles of one of its heads
    KReq q;
    int lane;
    __device__ __forceinline__ int count(const KAttnArgs& a, const KReq& x) const {  // tiles of one head of request x
        int sum = 0;
        for (int g0 = 0; g0 < x.groups; g0 += 32) {
            int lo, t = 0;
            if (g0 + lane < x.groups) {
                kp_group<KT>(a, x, ROWS, g0 + lane, &lo, &t);
                t += KP_UNIT;
            }
            sum += __reduce_add_sync(0xffffffffu, (unsigned)t);
        }
        return sum;
    }
    __device__ __forceinline__ bool mine(const KAttnArgs& a, const KReq& x) const {
        return x.n > 0 && (long long)x.n * a.G > a.min_rows;
    }
    __device__ __forceinline__ void enter(const KAttnArgs& a, int request, int before) {
        r = request, base = before;
        q = kd_request(a, r, ROWS, KT, false);
        per_head = mine(a, q) ? count(a, q) : 0;
    }
    // to the tile `cur` of the list, cur < total
    __device__ __forceinline__ KPSeg seek(const KAttnArgs& a, int cur, int end) {
        while (per_head == 0 || cur >= base + per_head * a.c.n_kv_heads) {
            const int before = base + per_head * a.c.n_kv_heads;
            int next = r + 1;
            for (;;) {  // the next request of this kernel, 32 at a time
                bool m = false;
                if (next + lane < a.n_req) m = mine(a, kd_request(a, next + lane, ROWS, KT, false));
                const unsigned b = __ballot_sync(0xffffffffu, m);
                if (b || next >= a.n_req) {
                    next += b ? __ffs(b) - 1 : 0;
                    break;
                }
                next += 32;
            }
            enter(a, min(next, a.n_req - 1), before);
            if (next >= a.n_req) break;
        }
        KPSeg s;
        s.q = q;
        s.h = (cur - base) / per_head;
        int rest = (cur - base) - s.h * per_head, gi = 0, lo = 0, t = 0;
        for (int g0 = 0; g0 < q.groups; g0 += 32) {
            t = 0;
            if (g0 + lane < q.groups) {
                kp_group<KT>(a, q, ROWS, g0 + lane, &lo, &t);
                t += KP_UNIT;
            }
            int v = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            const int all = __shfl_sync(0xffffffffu, v, 31);
            if (rest < all) {
                const int at = __ffs(__ballot_sync(0xffffffffu, v > rest)) - 1;
                rest -= __shfl_sync(0xffffffffu, v - t, at);
                lo = __shfl_sync(0xffffffffu, lo, at);
                t = __shfl_sync(0xffffffffu, t, at);
                gi = g0 + at;
                break;
            }
            rest -= all;
        }
        s.row0 = gi * ROWS;
        s.nrows = min(ROWS, q.n * a.G - s.row0);
        s.unit0 = cur - rest;
        s.tiles = t - KP_UNIT;
        s.first = max(0, rest - KP_UNIT);
        s.tile0 = lo + s.first;
        s.cnt = min(s.tiles, end - s.unit0 - KP_UNIT) - s.first;  // none: the run ends in this unit's start, its tiles are the next CTA's
        s.next = s.cnt > 0 ? s.unit0 + KP_UNIT + s.first + s.cnt : INT_MAX;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r_lo = s.row0 + (ROWS == 256 ? 128 * x : 0), r_hi = min(r_lo + 128, s.row0 + s.nrows) - 1;
            const int first = q.kv - q.n + r_lo / a.G, last = q.kv - q.n + r_hi / a.G;
            s.lo[x] = a.window > 0 ? max(0, first - a.window + 1) / KT : 0;
            s.hi[x] = r_hi < r_lo || last < 0 ? -1 : last / KT;
        }
        return s;
    }
};

// Whether stream s has rows that see the tile of keys kt.
template <bool SPLIT>
__device__ __forceinline__ bool kp_active(int lo, int hi, int s, int kt) {
    return kt >= lo && kt <= hi && (!SPLIT || (kt & 1) == s);
}
template <bool SPLIT>
__device__ __forceinline__ bool kp_active(const KPSeg& g, int s, int kt) {
    return kp_active<SPLIT>(g.lo[s], g.hi[s], s, kt);
}

#define KP_LD32(r, addr)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"             \
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                                                   \
        : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]),    \
          "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]),             \
          "=r"((r)[15]), "=r"((r)[16]), "=r"((r)[17]), "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]),           \
          "=r"((r)[22]), "=r"((r)[23]), "=r"((r)[24]), "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]),           \
          "=r"((r)[29]), "=r"((r)[30]), "=r"((r)[31])                                                                        \
        : "r"(addr)                                                                                                          \
        : "memory")
#define KP_LD16(r, addr)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"             \
        : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]),    \
          "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]),             \
          "=r"((r)[15])                                                                                                      \
        : "r"(addr)                                                                                                          \
        : "memory")
#define KP_ST16(addr, r)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), \
        "r"((r)[0]), "r"((r)[1]), "r"((r)[2]), "r"((r)[3]), "r"((r)[4]), "r"((r)[5]), "r"((r)[6]), "r"((r)[7]), "r"((r)[8]),        \
        "r"((r)[9]), "r"((r)[10]), "r"((r)[11]), "r"((r)[12]), "r"((r)[13]), "r"((r)[14]), "r"((r)[15])                       \
        : "memory")

__device__ __forceinline__ void kp_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kp_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// what this thread wrote to shared memory is visible to the matrix unit's reads
__device__ __forceinline__ void kp_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// One lane of the warp, always the same: the matrix unit's calls are made by it.
__device__ __forceinline__ bool kp_elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void kp_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D (tensor memory) (+)= A (shared memory) . B^T, and the same with A in tensor memory
__device__ __forceinline__ void kp_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void kp_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(ta), "l"(db), "r"(idesc), "r"(add)
        : "memory");
}
// two fp32 at once
__device__ __forceinline__ uint64_t kp_two(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 kp_both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t kp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t kp_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// shared-memory descriptor of an MN-major operand, 128-byte swizzle: 8 keys of 128 bytes after 8 keys
// (stride offset 1024), 64 channels after 64 channels (leading offset)
__device__ __forceinline__ uint64_t kp_desc_mn(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
__device__ __forceinline__ void kp_sts128(uint32_t sa, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sa), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <int FMT, int HD, bool SPLIT>
__global__ void __launch_bounds__(KP_THREADS, 1)
    kv8_prefill_kernel(const KAttnArgs a, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
    using S = KPShape<HD, SPLIT>;
    constexpr int ROWS = S::ROWS, KT = S::KT, HDO = S::HDO, LINE = HD == 64 ? 64 : 128;
    constexpr bool HALVES = S::HALVES, SHARED = SPLIT || HALVES;  // SHARED: both streams have the same rows
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + S::O_BAR);
    uint64_t *q_full = bar, *k_full = bar + 2, *k_empty = bar + 4, *v_full = bar + 6, *v_empty = bar + 8, *s_full = bar + 10,
             *p_full = bar + 12, *o_full = bar + 14, *seg_done = bar + 15, *prep_full = bar + 16, *prep_empty = prep_full + KP_SLOTS,
             *raw_full = bar + 24, *raw_empty = bar + 26, *q_empty = bar + 28;
    int* s_misc = reinterpret_cast<int*>(smem + S::O_MISC);
    float* s_prep = reinterpret_cast<float*>(smem + S::O_PREP);
    int* s_row = reinterpret_cast<int*>(smem + S::O_PREP + KP_SLOTS * 96);

    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&k_full[s], 4);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 4);
            mbar_init(&v_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 4);
            mbar_init(&raw_full[s], 1);
            mbar_init(&raw_empty[s], 4);
        }
        mbar_init(o_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(seg_done, 8);
        for (int s = 0; s < KP_SLOTS; ++s) {
            mbar_init(&prep_full[s], 1);
            mbar_init(&prep_empty[s], 9);
        }
        fence_barrier_init();
    }
    if (warp == KP_W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_misc)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The q rows' kernel lets this one start while it waits itself for what came before: all of that has to be done here too.
    pdl_wait();
    pdl_launch_dependents();
    // ---- where this CTA's run begins: prefix sums over the requests, in the space of the operands
    KPWalk<ROWS, KT> walk;
    walk.lane = lane;
    {
        int* s_cnt = reinterpret_cast<int*>(smem);  // [n_req] tiles of each
        long long* s_w = reinterpret_cast<long long*>(smem + 4 * FENCE_PAGED_MAX_REQ);
        for (int r0 = warp * 32; r0 < a.n_req; r0 += KP_THREADS) {
            KReq q{};
            if (r0 + lane < a.n_req) q = kd_request(a, r0 + lane, ROWS, KT, blockIdx.x == 0);
            unsigned todo = __ballot_sync(0xffffffffu, walk.mine(a, q));
            int own = 0;
            while (todo) {  // few: requests with many rows
                const int l = __ffs(todo) - 1;
                todo &= todo - 1;
                KReq x;
                x.start = 0;
                x.n = __shfl_sync(0xffffffffu, q.n, l);
                x.kv = __shfl_sync(0xffffffffu, q.kv, l);
                x.groups = __shfl_sync(0xffffffffu, q.groups, l);
                const long long w = (long long)walk.count(a, x) * a.c.n_kv_heads;
                if (lane == l) own = (int)min(w, (long long)INT_MAX);
            }
            if (r0 + lane < a.n_req) s_cnt[r0 + lane] = own;
        }
        __syncthreads();
        const int per_t = (a.n_req + KP_THREADS - 1) / KP_THREADS;
        const int r0 = min(a.n_req, tid * per_t), r1 = min(a.n_req, r0 + per_t);
        long long sum = 0;
        for (int r = r0; r < r1; ++r) sum += s_cnt[r];
        long long v = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) s_w[warp] = v;
        __syncthreads();
        long long all = 0;
        for (int w = 0; w < KP_THREADS / 32; ++w) {
            if (w < warp) v += s_w[w];
            all += s_w[w];
        }
        if (all > INT_MAX / 2) {
            if (tid == 0) set_device_error(KV8_BAD);
            all = 0;  // no such list fits a pool
        }
        const int per = max(KP_MIN_TILES + KP_UNIT, (int)((all + gridDim.x - 1) / gridDim.x));
        const long long begin = (long long)blockIdx.x * per;
        if (tid == 0) s_misc[1] = (int)all;
        long long at = v - sum;
        for (int r = r0; r < r1; ++r) {
            if (begin >= at && begin < at + s_cnt[r]) {
                s_misc[2] = r;
                s_misc[3] = (int)at;
            }
            at += s_cnt[r];
        }
        __syncthreads();
    }
    const int total = s_misc[1];
    const int per = max(KP_MIN_TILES + KP_UNIT, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int begin = (int)min((long long)total, (long long)blockIdx.x * per), end = min(total, begin + min(per, total - begin));
    if (begin < end) walk.enter(a, s_misc[2], s_misc[3]);
    kp_fence_before();
    __syncthreads();
    kp_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(s_misc);
    // S of stream s at column 128 s, O of it at 256 + 128 s
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t n) {  // the n-th completion (from 0)
        if (ok) ok = mbar_wait(b, n & 1u);
    };

    if (warp >= KP_W_CONV && warp < KP_W_PREP) {
        // ---------------------------------------------------------------- codes -> fp16 operands
        // 8 keys x 64 channels a warp and step; rows r and r ^ 5 side by side: neither the loads nor the stores of a
        // quarter-warp meet on a bank (the staged codes are swizzled too)
        constexpr int HALF = HD / 64, STEPS = KT / 8 * HALF / 4, STEP_ROWS = 32 / HALF;
        const int cw = warp - KP_W_CONV, r8 = (lane >> 3) ^ ((lane >> 2 & 1) * 5);
        // this thread's row in the first step, its place in the operand and in the stage
        const int row0 = (cw / HALF) * 8 + r8, half = cw % HALF, c16 = (half & 1) * 4 + (lane & 3);
        const uint32_t dst0 = (uint32_t)(half * (KT * 128) + row0 * 128 + (((2 * (lane & 3)) ^ r8) << 4));
        const uint32_t raw0 = sbase + S::O_RAW + (HD == 64 ? (uint32_t)(row0 * 64 + ((c16 ^ ((row0 >> 1) & 3)) << 4))
                                                           : (uint32_t)((half >> 1) * (KT * 128) + row0 * 128 + ((c16 ^ r8) << 4)));
        uint32_t it = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            if (g.cnt <= 0) break;
            const int any_lo = a.window > 0 ? max(0, g.q.kv - g.q.n + g.row0 / a.G - a.window + 1) : 0;
            // the tiles that some row sees follow one another
            const int t0 = max(g.tile0, min(g.hi[0] < 0 ? INT_MAX : g.lo[0], g.hi[1] < 0 ? INT_MAX : g.lo[1]));
            const int t1 = min(g.tile0 + g.cnt - 1, max(g.hi[0], g.hi[1]));
            for (int kt = t0; kt <= t1; ++kt, ++it) {
                const uint32_t b = it & 1u;
                const int lo = any_lo - kt * KT - row0, hi = g.q.kv - kt * KT - row0;
                const bool edge = hi + row0 < KT || lo + row0 > 0;  // keys there may hold anything: they count as zero
#pragma unroll 1
                for (int v = 0; v < 2; ++v) {
                    wait(&raw_full[v], it);
                    if (it >= 2) wait((v ? v_empty : k_empty) + b, (it >> 1) - 1);
                    __syncwarp();
                    const uint32_t op = sbase + (v ? S::O_V : S::O_K) + b * S::OP + dst0, raw = raw0 + v * S::RAW;
#pragma unroll 1
                    for (int i0 = 0; i0 < STEPS; i0 += 4) {
                        uint4 x[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = lds128(raw + (i0 + i) * (STEP_ROWS * LINE));
                        if (edge) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if ((i0 + i) * STEP_ROWS >= hi || (i0 + i) * STEP_ROWS < lo) x[i] = make_uint4(0, 0, 0, 0);
                        }
                        const uint32_t dst = op + i0 * (STEP_ROWS * 128);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t y[4] = {kd_bias<FMT>(x[i].x), kd_bias<FMT>(x[i].y), kd_bias<FMT>(x[i].z), kd_bias<FMT>(x[i].w)};
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                kp_sts128((dst + i * (STEP_ROWS * 128)) ^ (k << 4), kd_half2<FMT>(y[2 * k], false),
                                          kd_half2<FMT>(y[2 * k], true), kd_half2<FMT>(y[2 * k + 1], false),
                                          kd_half2<FMT>(y[2 * k + 1], true));
                        }
                    }
                    kp_fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&raw_empty[v]);
                        mbar_arrive((v ? v_full : k_full) + b);
                    }
                }
            }
            cur = g.next;
        }
    } else if (warp == KP_W_LOAD) {
        // ---------------------------------------------------------------- codes into the stages
        const int box = min(a.c.page_tokens, 64), boxes = KT / box;
        // fetched: units whose q rows were fetched. Units with no tile that a row sees (a prompt that was not placed) have none, and
        // no phase of q_empty: both sides count the same units, or a wait by parity would pass a unit too early.
        uint32_t it = 0, fetched = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            if (g.cnt <= 0) break;
            bool q_due = true;
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j;
                if (!kp_active<SPLIT>(g, 0, kt) && !kp_active<SPLIT>(g, 1, kt)) continue;
                const uint32_t slot = it % KP_SLOTS;
                wait(&prep_full[slot], it / KP_SLOTS);
                const bool load = lane < boxes && kt * KT + lane * box < g.q.kv;
                const int y = load ? s_row[slot * 8 + lane * (box / 16)] : 0, n = __popc(__ballot_sync(0xffffffffu, load));
                if (lane == 0) mbar_arrive(&prep_empty[slot]);
#pragma unroll 1
                for (int v = 0; v < 2; ++v) {
                    if (it > 0) wait(&raw_empty[v], it - 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&raw_full[v], (uint32_t)(n * box * HD));
                    __syncwarp();
                    if (load) {
#pragma unroll
                        for (int x = 0; x < (HALVES ? 2 : 1); ++x)
                            kd_tma(sbase + S::O_RAW + v * S::RAW + x * KT * 128 + lane * box * LINE, v ? &tm_v : &tm_k, x * 128, y,
                                   &raw_full[v]);
                    }
                }
                ++it;
                if (q_due && ok) {  // the unit's q rows, behind its first tile; once the last unit's scores are done
                    q_due = false;
                    if (fetched > 0) wait(q_empty, fetched - 1);
                    ++fetched;
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok && lane == 0) {
                        const int per_head = a.n_tokens * a.G, y = g.h * per_head + g.q.start * a.G + g.row0;
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            if (HALVES && s == 1) continue;
                            if (!SPLIT && max(g.lo[s], g.tile0) > min(g.hi[s], g.tile0 + g.cnt - 1)) continue;  // no rows here
                            uint64_t* full = &q_full[SHARED ? 0 : s];
                            if (!SPLIT || s == 0) mbar_arrive_expect_tx(full, (SPLIT ? 2 : 1) * S::Q_TILE);
#pragma unroll
                            for (int x = 0; x < HD / 64; ++x)
                                kd_tma(sbase + S::O_Q + s * S::Q_TILE + x * 128 * 128, &tm_q, x * 64,
                                       SPLIT ? y + s * per_head * a.c.n_kv_heads : y + 128 * s, full);
                        }
                    }
                    __syncwarp();
                }
            }
            cur = g.next;
        }
    } else if (warp == KP_W_PREP) {
        // ---------------------------------------------------------------- pages and scales of 8 x 16 keys, some tiles ahead
        uint32_t it = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            if (g.cnt <= 0) break;
            const int* table = a.block_table + (size_t)walk.r * a.max_pages;
            // the first key that some row of the unit sees: pages before it may be anyone's by now
            const int any_lo = a.window > 0 ? max(0, g.q.kv - g.q.n + g.row0 / a.G - a.window + 1) : 0;
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j, key = kt * KT + lane * 16;
                if (!kp_active<SPLIT>(g, 0, kt) && !kp_active<SPLIT>(g, 1, kt)) continue;
                int unit = 0;
                float ks = 0.f, vs = 0.f;
                if (lane < KT / 16 && key < g.q.kv && (key | (a.c.page_tokens - 1)) >= any_lo) {
                    int p = table[key >> a.shift];
                    if (p < 0 || p >= a.c.n_pages) {
                        set_device_error(KV8_BAD);
                        p = 0;
                    }
                    unit = p * a.c.n_kv_heads + g.h;
                    ks = a.c.k_scale[unit];
                    vs = a.c.v_scale[unit];
                }
                const uint32_t slot = it % KP_SLOTS;
                if (it >= KP_SLOTS) wait(&prep_empty[slot], it / KP_SLOTS - 1);
                __syncwarp();
                if (lane < KT / 16) {
                    float lv = -INFINITY, rv = 1.f;
                    if (vs >= 1.17549435e-38f && vs < INFINITY) {
                        lv = log2f(vs);
                        rv = 1.f / vs;
                    } else if (!(vs < INFINITY)) {
                        ks = __uint_as_float(0x7fffffffu);  // NaN for whoever sees these keys
                    }
                    float* d = s_prep + slot * 24;
                    d[lane] = ks;
                    d[8 + lane] = lv;
                    d[16 + lane] = rv;
                    s_row[slot * 8 + lane] = unit * a.c.page_tokens + (key & (a.c.page_tokens - 1));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&prep_full[slot]);
                ++it;
            }
            cur = g.next;
        }
    } else if (warp == KP_W_MMA) {
        // ---------------------------------------------------------------- products
        // one copy of the code for both streams: it runs four times a tile and should find itself in the instruction cache
        constexpr uint32_t id_s = tg_idesc(128, KT), id_o = tg_idesc(128, HDO) | (1u << 16);  // V: MN-major
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        uint32_t it = 0, nq = 0, np = 0, segs = 0;  // nq, np: 16 bits per stream, of which the lowest counts
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            if (g.cnt <= 0) break;
            int pend0 = -1, pend1 = -1;      // the tile (count) whose weights a stream is making
            uint32_t have = 0, left = 0;  // have: q (bits 0, 1) and o (2, 3) of the streams; left: streams that still need V, 8 bits per buffer
            const int last = g.tile0 + g.cnt;
            // one more round than tiles, two where the streams take turns, to finish the last weights
            for (int kt = g.tile0; kt < last + (SPLIT ? 2 : 1); ++kt) {
                const uint32_t b = it & 1u;
                bool used = false;
#pragma unroll 1
                for (int s = 0; s < 2; ++s) {
                    const bool act = kt < last && kp_active<SPLIT>(s ? g.lo[1] : g.lo[0], s ? g.hi[1] : g.hi[0], s, kt);
                    const int p = s ? pend1 : pend0;
                    if (p >= 0 && (!SPLIT || (kt & 1) == s)) {  // O_s += P_s . V of the pending tile
                        const uint32_t pb = (uint32_t)p & 1u;
                        wait(&v_full[pb], (uint32_t)p >> 1);
                        wait(&p_full[s], np >> (16 * s));
                        np ^= 1u << (16 * s);
                        left -= 1u << (8 * pb);
                        const uint32_t add = (have >> (2 + s)) & (uint32_t)((kt - S::STEP - g.tile0) % S::TURN >= S::STEP);
                        have |= 4u << s;
                        kp_fence_after();
                        const uint32_t d = __shfl_sync(0xffffffffu, tm + 256 + 128 * s, 0), ta = __shfl_sync(0xffffffffu, tm + 128 * s, 0);
                        const uint64_t db = kp_desc_mn(__shfl_sync(0xffffffffu, sbase + S::O_V + pb * S::OP + (HALVES ? s * 2 * KT * 128 : 0), 0), KT * 128);
                        if (kp_elect() && ok) {
#pragma unroll
                            for (int x = 0; x < (SPLIT ? 2 : 1); ++x)
#pragma unroll
                                for (int k = 0; k < KT / 16; ++k)  // 16 keys: 2048 bytes further
                                    kp_mma_ts(d, ta + (k >> 1) * 32 + x * 16 + (k & 1) * 8, db + k * 128, id_o, x > 0 || k > 0 ? 1u : add);
                            if (((left >> (8 * pb)) & 255u) == 0) kp_commit(&v_empty[pb]);
                        }
                        if (s) pend1 = -1;
                        else pend0 = -1;
                    }
                    if (act) {  // S_s = Q_s . K^T
                        const int qi = SHARED ? 0 : s;
                        if (!((have >> qi) & 1u)) {
                            have |= 1u << qi;
                            wait(&q_full[qi], nq >> (16 * qi));
                            nq ^= 1u << (16 * qi);
                        }
                        wait(&k_full[b], it >> 1);
                        kp_fence_after();
                        const uint32_t d = __shfl_sync(0xffffffffu, tm + 128 * s, 0);
                        const uint64_t db = tg_desc(__shfl_sync(0xffffffffu, sbase + S::O_K + b * S::OP, 0));
                        const uint64_t da = tg_desc(__shfl_sync(0xffffffffu, sbase + S::O_Q + qi * S::Q_TILE, 0));
                        if (kp_elect() && ok) {
                            // 16 channels: 32 bytes further, 64 channels: the next slab; the low parts of q first
#pragma unroll
                            for (int x = SPLIT ? 1 : 0; x >= 0; --x)
#pragma unroll
                                for (int k = 0; k < HD / 16; ++k)
                                    kp_mma_ss(d, da + (x * S::Q_TILE + (k >> 2) * 128 * 128 + (k & 3) * 32) / 16,
                                              db + ((k >> 2) * KT * 128 + (k & 3) * 32) / 16, id_s, (SPLIT && x == 0) || k > 0);
                            kp_commit(&s_full[s]);
                        }
                        if (s) pend1 = (int)it;
                        else pend0 = (int)it;
                        left += 1u << (8 * b);
                        used = true;
                    }
                }
                if (used) {
                    if (kp_elect() && ok) kp_commit(&k_empty[b]);
                    ++it;
                }
            }
            if ((have & 3u) && kp_elect() && ok) kp_commit(q_empty);  // only where scores were made: the loader's count
            __syncwarp();
            // a stream without tiles here may still be at the last unit's end: o_full must not run two ahead of it
            if (segs > 0) wait(seg_done, segs - 1);
            ++segs;
            if (kp_elect() && ok) kp_commit(o_full);
            __syncwarp();
            cur = g.next;
        }
    } else if (warp < KP_W_CONV) {
        // ---------------------------------------------------------------- softmax, a thread per row
        const int s = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_s = t_lane + 128 * s, t_o = t_lane + 256 + 128 * s;
        uint32_t n_s = 0, n_o = 0, it = 0;
        // rows that belong to no request
        if (a.min_rows == 0) {
            const int used = max(0, min(a.new_start[a.n_req], a.n_tokens));
            const long long w = (long long)a.n_q_heads * HD, n = (a.n_tokens - used) * w;
            for (long long i = blockIdx.x * 256 + tid; i < n; i += gridDim.x * 256)
                kv8_st1(a.out, (used + i / w) * a.out_stride + i % w, a.type, 0.f);
            if (a.lse)
                for (long long i = blockIdx.x * 256 + tid; i < (long long)(a.n_tokens - used) * a.n_q_heads; i += gridDim.x * 256)
                    a.lse[(long long)used * a.n_q_heads + i] = -INFINITY;
        }
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            if (g.cnt <= 0) break;
            const int i_row = (SHARED ? 0 : 128 * s) + row;  // in the group
            const bool valid = i_row < g.nrows;
            const int tok_i = (g.row0 + (valid ? i_row : 0)) / a.G;
            const int head = g.h * a.G + (g.row0 + (valid ? i_row : 0)) % a.G;
            const long long tok = g.q.start + tok_i;
            const int ch0 = HALVES ? s * HDO : 0;  // this stream's channels
            const int lim = valid ? g.q.kv - g.q.n + tok_i : -1;
            const int lim_lo = a.window > 0 ? lim - a.window + 1 : 0;
            // tiles that all of this stream's rows see whole need no mask
            const int r_lo = g.row0 + (SHARED ? 0 : 128 * s), r_hi = min(r_lo + 128, g.row0 + g.nrows) - 1;
            const int lim_first = g.q.kv - g.q.n + r_lo / a.G, lim_last = g.q.kv - g.q.n + r_hi / a.G;
            const float qs = valid ? a.q_scale[(long long)g.h * a.n_tokens * a.G + tok * a.G + (g.row0 + i_row) % a.G] : 1.f;
            // m, u: the row's references, as in the decode kernel; up = KD_UP + m - u, down = 2^-up
            float m = -INFINITY, u = -INFINITY, l = 0.f, up = 0.f, down = 1.f;
            bool have_o = false;
            // the record of (CTA, slot, stream): m and l of each row, then the sums, four channels of all rows after one another
            auto record = [&]() { return a.part + ((long long)blockIdx.x * 4 + (g.first > 0 ? 0 : 2) + s) * S::REC; };
            const bool whole = g.cnt == g.tiles, direct = whole && !SPLIT && g.cnt <= S::TURN;  // the same for both streams
            bool again = false;  // the record holds sums already
            for (int j = 0;;) {
                for (const int stop = min(g.cnt, j + S::TURN); j < stop; ++j) {
                    const int kt = g.tile0 + j, key0 = kt * KT;
                    const bool act = kp_active<SPLIT>(g, s, kt);
                    if (!act && !kp_active<SPLIT>(g, 1 - s, kt)) continue;
                    const uint32_t slot = it % KP_SLOTS, use = it / KP_SLOTS;
                    ++it;
                    wait(&prep_full[slot], use);  // also where this stream has no rows: it must not give back a slot before its time
                    __syncwarp();
                    if (!act) {
                        if (lane == 0) mbar_arrive(&prep_empty[slot]);
                        continue;
                    }
                    wait(&s_full[s], n_s++);
                    __syncwarp();
                    kp_fence_after();
                    const float* pr = s_prep + slot * 24;  // k_scale, log2 and reciprocal of v_scale of 8 x 16 keys
                    // Loops of 32 columns, not unrolled: the roles' code has to share the instruction cache.
                    const bool edge = key0 + KT - 1 > lim_first || (a.window > 0 && key0 < lim_last - a.window + 1);
                    uint32_t bad = 0;  // of an edge tile: blocks of 16 keys with a scale that is no number, of which this row sees some
                    if (edge) {        // -infinity in the columns that this row does not see
#pragma unroll 1
                        for (int c = 0; c < KT / 32; ++c) {
                            uint32_t x[32];
                            KP_LD32(x, t_s + 32 * c);
                            kp_wait_ld();
                            const int h = lim - key0 - 32 * c, l0 = lim_lo - key0 - 32 * c;  // sees the columns l0 .. h
                            uint32_t see = h < 0 ? 0u : h >= 31 ? ~0u : (2u << h) - 1u;
                            if (l0 > 0) see &= l0 >= 32 ? 0u : ~0u << l0;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!((see >> e) & 1u)) x[e] = 0xff800000u;
                            KP_ST16(t_s + 32 * c, x);
                            KP_ST16(t_s + 32 * c + 16, (x + 16));
                            if (!(pr[2 * c] * qs < INFINITY) && (see & 0xffffu)) bad |= 1u << (2 * c);
                            if (!(pr[2 * c + 1] * qs < INFINITY) && (see >> 16)) bad |= 2u << (2 * c);
                        }
                        kp_wait_st();
                    }
                    // factor of a block's scores; -infinity has to stay so in an edge tile: none of 0 or NaN there
                    auto factor = [&](int b) {
                        float f = pr[b] * qs;
                        if (edge) f = f < INFINITY ? fmaxf(f, 1e-30f) : 1e-30f;
                        return f;
                    };
                    constexpr int CH = 32, NB = CH / 16;
                    float mt = -INFINITY, ut = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < KT; c += CH) {
                        uint32_t x[CH];
#pragma unroll
                        for (int k = 0; k < CH; k += 32) KP_LD32((x + k), t_s + c + k);
                        float f[NB];
#pragma unroll
                        for (int k = 0; k < NB; ++k) f[k] = factor(c / 16 + k);
                        kp_wait_ld();
#pragma unroll
                        for (int k = 0; k < NB; ++k) {
                            float y = __uint_as_float(x[16 * k]);
#pragma unroll
                            for (int e = 1; e < 16; ++e) y = fmaxf(y, __uint_as_float(x[16 * k + e]));
                            y *= f[k];
                            mt = fmaxf(mt, y);
                            ut = fmaxf(ut, y + pr[8 + c / 16 + k]);
                        }
                    }
                    if (__any_sync(0xffffffffu, mt > m + KD_LAZY || ut > u + KD_LAZY)) {
                        // each row by itself: what another row sees has no say
                        const float mn = mt > m + KD_LAZY ? ceilf(mt) : m;
                        const float un = fmaxf(ut > u + KD_LAZY ? ceilf(ut) : u, mn - KD_FLOOR);
                        l *= mn == -INFINITY ? 1.f : kd_exp2(m - mn);
                        const float al = un == -INFINITY ? 1.f : kd_exp2(u - un);
                        m = mn, u = un;
                        up = m == -INFINITY ? 0.f : KD_UP + m - u;
                        down = kd_exp2(-up);
                        if (have_o) {  // the products of the tiles before have ended: S came after them
#pragma unroll 1
                            for (int c = 0; c < HDO; c += 16) {
                                uint32_t r[16];
                                KP_LD16(r, t_o + c);
                                kp_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * al);
                                KP_ST16(t_o + c, r);
                            }
                        }
                    }
                    have_o = true;
                    const float mm = m == -INFINITY ? 0.f : m;
                    // ---- weights, in place of the scores
#pragma unroll 1
                    for (int c = 0; c < KT; c += CH) {
                        uint32_t x[CH];
#pragma unroll
                        for (int k = 0; k < CH; k += 32) KP_LD32((x + k), t_s + c + k);
                        float cf[NB], add[NB], fb[NB], fl[NB];
#pragma unroll
                        for (int k = 0; k < NB; ++k) {
                            const int b = c / 16 + k;
                            const float d = pr[8 + b] + up;
                            const bool tiny = !(d >= -40.f);  // a page of zeros, or next to it for this row
                            cf[k] = factor(b);
                            add[k] = SPLIT ? -mm : (tiny ? -40.f : d) - mm;
                            if ((bad >> b) & 1u) add[k] = __uint_as_float(0x7fffffffu);
                            fb[k] = SPLIT ? (tiny ? 0.f : kd_exp2(fminf(d, 127.f))) : 0.f;
                            fl[k] = SPLIT ? 1.f : tiny ? 1.0995116e12f : pr[16 + b] * down;
                        }
                        kp_wait_ld();
#pragma unroll
                        for (int h = 0; h < CH / 32; ++h) {
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int kb = 2 * h + k;
                                const uint64_t cf2 = kp_two(cf[kb], cf[kb]), add2 = kp_two(add[kb], add[kb]);
                                uint64_t sum2 = 0;
#pragma unroll
                                for (int e = 0; e < 16; e += 2) {
                                    const float2 y = kp_both(kp_fma2(
                                        kp_two(__uint_as_float(x[16 * kb + e]), __uint_as_float(x[16 * kb + e + 1])), cf2, add2));
                                    float p0 = kd_exp2(y.x), p1 = kd_exp2(y.y);
                                    sum2 = kp_add2(sum2, kp_two(p0, p1));
                                    if (SPLIT) p0 *= fb[kb], p1 *= fb[kb];
                                    const int at = k * 8 + (e >> 1);
                                    hi[at] = kd_pack(p0, p1);
                                    if (SPLIT) lo[at] = kd_pack_rest(p0, p1, hi[at]);
                                }
                                const float2 sum = kp_both(sum2);
                                l += (sum.x + sum.y) * fl[kb];
                            }
                            KP_ST16(t_s + c + h * 32, hi);
                            if (SPLIT) KP_ST16(t_s + c + h * 32 + 16, lo);
                        }
                    }
                    kp_wait_st();
                    kp_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&p_full[s]);
                        mbar_arrive(&prep_empty[slot]);
                    }
                }
                // ---- the end of the unit (or of this part), or of a turn
                const bool end_of = j >= g.cnt;
                if (end_of) {
                    wait(o_full, n_o++);
                } else {
                    // the scores of this stream's next tile come after the products before them; without one the sums wait for the end
                    const bool next = kp_active<SPLIT>(g, s, g.tile0 + j) || (SPLIT && j + 1 < g.cnt && kp_active<SPLIT>(g, s, g.tile0 + j + 1));
                    if (!next || !have_o) continue;
                    wait(&s_full[s], n_s);
                }
                __syncwarp();
                kp_fence_after();
                float mul = direct ? (l == 0.f ? 0.f : 1.f / l) : 1.f, f = 0.f;
                float2* ml = reinterpret_cast<float2*>(record()) + row;
                float4* rec = reinterpret_cast<float4*>(record() + 256) + row;
                if (again) {
                    const float2 v = __ldcg(ml);
                    const float mn = fmaxf(m, v.x), mz = mn == -INFINITY ? 0.f : mn;
                    mul = kd_exp2(m - mz), f = kd_exp2(v.x - mz);
                    l = l * mul + v.y * f;
                    m = mn;
                }
#pragma unroll 1
                for (int c = 0; c < HDO; c += 16) {
                    uint32_t r[16];
                    float x[16];
                    if (have_o) {
                        KP_LD16(r, t_o + c);
                        kp_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = have_o && mul != 0.f ? __uint_as_float(r[e]) * mul * down : 0.f;
                    if (direct) {
                        const long long at = tok * a.out_stride + (long long)head * HD + ch0 + c;
                        if (valid) {
                            kv8_st8(a.out, at, a.type, a.out_wide, *reinterpret_cast<const float(*)[8]>(x));
                            kv8_st8(a.out, at + 8, a.type, a.out_wide, *reinterpret_cast<const float(*)[8]>(x + 8));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            float4* at = rec + ((c + e) >> 2) * 128;
                            if (again) {
                                const float4 v = __ldcg(at);
                                x[e] = fmaf(v.x, f, x[e]), x[e + 1] = fmaf(v.y, f, x[e + 1]);
                                x[e + 2] = fmaf(v.z, f, x[e + 2]), x[e + 3] = fmaf(v.w, f, x[e + 3]);
                            }
                            __stcg(at, make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]));
                        }
                    }
                }
                if (!direct) __stcg(ml, make_float2(m, l));
                if (end_of) break;
                again = true, have_o = false;
                m = u = -INFINITY, l = 0.f, up = 0.f, down = 1.f;
                kp_fence_before();
            }
            const int c_first = (g.unit0 + KP_UNIT) / per, c_last = (g.unit0 + KP_UNIT + g.tiles - 1) / per;
            if (direct) {
                if (valid && a.lse && (!HALVES || s == 0)) a.lse[tok * a.n_q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
            } else {
                __threadfence();
                named_bar_sync(1, 256);
                if (tid == 0) {
                    const int n = whole ? 0 : atomicAdd(a.arrived + c_first, 1);
                    const bool last = whole || n == c_last - c_first;
                    if (last && !whole) a.arrived[c_first] = 0;  // ready for the next call
                    __threadfence();
                    s_misc[4] = last;
                }
                named_bar_sync(1, 256);
                if (s_misc[4]) {
                    // join the parts in the order of the keys; SPLIT: both streams' parts of the same rows, half the channels each
                    constexpr int STREAMS = SPLIT ? 2 : 1;
                    const int c0 = SPLIT ? s * (HD / 2) : 0, c1 = SPLIT ? c0 + HD / 2 : HDO;
                    float M = -INFINITY, L = 0.f;
#pragma unroll 1
                    for (int k = c_first; k <= c_last; ++k)
#pragma unroll
                        for (int x = 0; x < STREAMS; ++x) {
                            const float* pr = a.part + ((long long)k * 4 + (k == c_first ? 2 : 0) + (SPLIT ? x : s)) * S::REC;
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr) + row);
                            const float mn = fmaxf(M, ml.x), mz = mn == -INFINITY ? 0.f : mn;
                            L = L * kd_exp2(M - mz) + ml.y * kd_exp2(ml.x - mz);
                            M = mn;
                        }
                    const float mz = M == -INFINITY ? 0.f : M, inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
                    for (int c = c0; c < c1; c += 32) {
                        float acc[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[e] = 0.f;
#pragma unroll 1
                        for (int k = c_first; k <= c_last; ++k)
#pragma unroll
                            for (int x = 0; x < STREAMS; ++x) {
                                const float* pr = a.part + ((long long)k * 4 + (k == c_first ? 2 : 0) + (SPLIT ? x : s)) * S::REC;
                                const float w = kd_exp2(__ldcg(reinterpret_cast<const float2*>(pr) + row).x - mz);
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    const float4 v = __ldcg(reinterpret_cast<const float4*>(pr + 256) + ((c + e) >> 2) * 128 + row);
                                    acc[e] += v.x * w;
                                    acc[e + 1] += v.y * w;
                                    acc[e + 2] += v.z * w;
                                    acc[e + 3] += v.w * w;
                                }
                            }
                        if (valid) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                float x[8];
#pragma unroll
                                for (int y = 0; y < 8; ++y) x[y] = acc[e + y] * inv;
                                kv8_st8(a.out, tok * a.out_stride + (long long)head * HD + ch0 + c + e, a.type, a.out_wide, x);
                            }
                        }
                    }
                    if (valid && a.lse && (!SHARED || s == 0))
                        a.lse[tok * a.n_q_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945f;
                }
            }
            kp_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_done);
            cur = g.next;
        }
    }
    kp_fence_before();
    __syncthreads();
    if (warp == KP_W_MMA)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace fence
