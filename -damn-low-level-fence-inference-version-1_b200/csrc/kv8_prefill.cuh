// kv8_prefill.cuh — attention of many query rows per request over the paged 8-bit cache (prompts, chunks)
// on the 5th-generation tensor cores.
//
//   S = Q . Kcode^T,  p = 2^(S * k_scale * scale * log2 e - m),  O = sum over keys of p * v_scale * Vcode,  out = O / sum p
//
// Bound: the matrix unit (4 head_dim operations per visible pair) and, as large here, the exponentials:
// 128 x 128 of them per tile at 16 a clock take as long as the tile's products.
//
//  * Work is the list of 128-key tiles of every (request, KV head, group of query rows), cut into equal
//    runs, one per CTA, as in the decode kernel: causal groups of any length fill all SMs alike. Units
//    that span CTAs are joined through the workspace in key order.
//  * Rows of a group are (token, query head of the KV head): grouped heads share every K and V tile.
//    Two streams of 128 rows per CTA take turns on the matrix unit: while one stream's softmax warps
//    work, the other's products run. fp32 activations (SPLIT): one group of 128 rows, q and the weights as
//    pairs of fp16, and the two streams take the even and the odd tiles.
//  * Codes become fp16 exactly, once per tile for both streams, by four converter warps: K rows as they
//    are, V transposed, so that both are K-major operands in 128-byte swizzled shared memory. Scales never
//    touch the codes: k_scale is part of a score's factor and v_scale / (a running reference) of the
//    exponent, both constant over 16 keys.
//  * S, then P in its place as fp16 (the weights are the A operand straight from tensor memory), and O
//    stay in tensor memory: 2 x (128 + head_dim) of its 512 columns.
//  * O is rescaled only when a row's maximum grows by more than 2^8 (fp16 weights have that room).
#pragma once

#include "kv8_decode.cuh"

namespace fence {

constexpr int KP_KT = 128, KP_SMS = 148;
constexpr int KP_W_CONV = 8, KP_W_LOAD = 12, KP_W_MMA = 13, KP_THREADS = 14 * 32;
constexpr int KP_MIN_TILES = 2;

template <int HD, bool SPLIT>
struct KPShape {
    static constexpr int ROWS = SPLIT ? 128 : 256;  // per group
    static constexpr int Q_TILE = 128 * HD * 2;     // 128 rows as fp16
    static constexpr int OP = KP_KT * HD * 2;       // a K or V operand tile
    static constexpr int RAW = KP_KT * HD;
    static constexpr int O_Q = 0;  // two tiles: the streams' rows, or the high and low parts
    static constexpr int O_K = 2 * Q_TILE;
    static constexpr int O_V = O_K + 2 * OP;
    static constexpr int O_RK = O_V + 2 * OP;
    static constexpr int O_RV = O_RK + RAW;
    static constexpr int O_BAR = O_RV + RAW;
    static constexpr int O_MISC = O_BAR + 256;
    static constexpr int O_RSC = O_MISC + 64;    // raw scales K 8, V 8
    static constexpr int O_PREP = O_RSC + 64;    // [4][24]: k_scale, log2 v_scale, 1 / v_scale of 8 x 16 keys
    static constexpr int SMEM = O_PREP + 4 * 96 + 1024;
    static constexpr int REC = 128 * (HD + 2);   // floats of one stream's partial result
};

// What every role derives for itself from the run's position.
struct KPSeg {
    KReq q;
    int h, row0, nrows, tile0, cnt, first, tiles;  // this CTA's tiles of the unit, its place in the unit, the unit's tiles
};

__device__ __forceinline__ void kp_group(const KAttnArgs& a, const KReq& q, int rows_per_group, int gi, int* lo_tile, int* tiles) {
    const int nrows = q.n * a.G, r_lo = gi * rows_per_group, r_hi = min(r_lo + rows_per_group, nrows) - 1;
    const int first = q.kv - q.n + r_lo / a.G, last = q.kv - q.n + r_hi / a.G;
    const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
    *lo_tile = last < 0 ? 0 : lo / KP_KT;
    *tiles = last < 0 ? 1 : last / KP_KT - *lo_tile + 1;
}

// Walks a CTA's run of tiles; every warp does so for itself, all lanes together.
template <int ROWS>
struct KPWalk {
    int r, base, per_head;  // request, tiles before it, tiles of one of its heads
    KReq q;
    int lane;
    __device__ __forceinline__ int count(const KAttnArgs& a, const KReq& x) const {  // tiles of one head of request x
        int sum = 0;
        for (int g0 = 0; g0 < x.groups; g0 += 32) {
            int lo, t = 0;
            if (g0 + lane < x.groups) kp_group(a, x, ROWS, g0 + lane, &lo, &t);
            sum += __reduce_add_sync(0xffffffffu, (unsigned)t);
        }
        return sum;
    }
    __device__ __forceinline__ bool mine(const KAttnArgs& a, const KReq& x) const {
        return x.n > 0 && (long long)x.n * a.G > a.min_rows;
    }
    __device__ __forceinline__ void enter(const KAttnArgs& a, int request, int before) {
        r = request, base = before;
        q = kd_request(a, r, ROWS, KP_KT, false);
        per_head = mine(a, q) ? count(a, q) : 0;
    }
    // to the tile `cur` of the list, cur < total
    __device__ __forceinline__ KPSeg seek(const KAttnArgs& a, int cur, int end) {
        while (per_head == 0 || cur >= base + per_head * a.c.n_kv_heads) {
            const int before = base + per_head * a.c.n_kv_heads;
            int next = r + 1;
            for (;;) {  // the next request of this kernel, 32 at a time
                bool m = false;
                if (next + lane < a.n_req) m = mine(a, kd_request(a, next + lane, ROWS, KP_KT, false));
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
            if (g0 + lane < q.groups) kp_group(a, q, ROWS, g0 + lane, &lo, &t);
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
        s.first = rest;
        s.tiles = t;
        s.tile0 = lo + rest;
        s.cnt = min(t - rest, end - cur);
        return s;
    }
};

// Whether stream s has rows that see the tile of keys kt.
template <bool SPLIT>
__device__ __forceinline__ bool kp_active(const KAttnArgs& a, const KPSeg& g, int s, int kt) {
    if (SPLIT && (kt & 1) != s) return false;
    const int r_lo = g.row0 + (SPLIT ? 0 : 128 * s), r_hi = min(r_lo + 128, g.row0 + g.nrows) - 1;
    if (r_hi < r_lo) return false;
    const int first = g.q.kv - g.q.n + r_lo / a.G, last = g.q.kv - g.q.n + r_hi / a.G;
    const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
    return last >= 0 && kt * KP_KT <= last && (kt + 1) * KP_KT > lo;
}

#define KP_LD32(r, addr)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"             \
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                                                   \
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),        \
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),             \
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),            \
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])                          \
        : "r"(addr)                                                                                                          \
        : "memory")
#define KP_ST32(addr, r)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"          \
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),                                         \
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),        \
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),          \
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),          \
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])                                                                       \
        : "memory")
#define KP_ST16(addr, r)                                                                                                     \
    asm volatile(                                                                                                            \
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), \
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),        \
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])                                               \
        : "memory")

__device__ __forceinline__ void kp_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kp_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// what this thread wrote to shared memory is visible to the matrix unit's reads
__device__ __forceinline__ void kp_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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
__device__ __forceinline__ void kp_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(ta), "l"(db), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void kp_sts32(uint32_t sa, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(sa), "r"(v) : "memory");
}
__device__ __forceinline__ void kp_sts128(uint32_t sa, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sa), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <int FMT, int HD, bool SPLIT>
__global__ void __launch_bounds__(KP_THREADS, 1)
    kv8_prefill_kernel(const KAttnArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using S = KPShape<HD, SPLIT>;
    constexpr int ROWS = S::ROWS, LINE = HD == 64 ? 64 : 128;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + S::O_BAR);
    uint64_t *q_full = bar, *rk_full = bar + 2, *rk_empty = bar + 3, *rv_full = bar + 4, *rv_empty = bar + 5, *k_full = bar + 6,
             *k_empty = bar + 8, *v_full = bar + 10, *v_empty = bar + 12, *s_full = bar + 14, *p_full = bar + 16, *o_full = bar + 18,
             *prep_full = bar + 19, *seg_done = bar + 23;
    int* s_misc = reinterpret_cast<int*>(smem + S::O_MISC);
    float* s_rsc = reinterpret_cast<float*>(smem + S::O_RSC);
    float* s_prep = reinterpret_cast<float*>(smem + S::O_PREP);

    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 4);
            mbar_init(&k_full[s], 4);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 4);
            mbar_init(&v_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 4);
        }
        mbar_init(rk_full, 33);
        mbar_init(rk_empty, 4);
        mbar_init(rv_full, 1);
        mbar_init(rv_empty, 4);
        mbar_init(o_full, 1);
        mbar_init(seg_done, 8);
        for (int s = 0; s < 4; ++s) mbar_init(&prep_full[s], 1);
        fence_barrier_init();
    }
    if (warp == KP_W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_misc)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- where this CTA's run begins: prefix sums over the requests, in the space of the operands
    KPWalk<ROWS> walk;
    walk.lane = lane;
    {
        int* s_cnt = reinterpret_cast<int*>(smem);  // [n_req] tiles of each
        long long* s_w = reinterpret_cast<long long*>(smem + 4 * FENCE_PAGED_MAX_REQ);
        for (int r0 = warp * 32; r0 < a.n_req; r0 += KP_THREADS) {
            KReq q{};
            if (r0 + lane < a.n_req) q = kd_request(a, r0 + lane, ROWS, KP_KT, blockIdx.x == 0);
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
        const int per = max(KP_MIN_TILES, (int)((all + gridDim.x - 1) / gridDim.x));
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
    const int per = max(KP_MIN_TILES, (total + (int)gridDim.x - 1) / (int)gridDim.x);
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

    if (warp == KP_W_LOAD) {
        // ---------------------------------------------------------------- raw tiles and scales
        const int P = a.c.page_tokens, box = min(P, 64), boxes = KP_KT / box;
        uint32_t it = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            const int* table = a.block_table + (size_t)walk.r * a.max_pages;
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j, key0 = kt * KP_KT;
                if (!kp_active<SPLIT>(a, g, 0, kt) && !kp_active<SPLIT>(a, g, 1, kt)) continue;
                // page of the 16 keys of lanes 0..7 (scales) and of this lane's box
                auto page_at = [&](int key) {
                    int p = table[key >> a.shift];
                    if (p < 0 || p >= a.c.n_pages) {
                        set_device_error(KV8_BAD);
                        p = 0;
                    }
                    return p * a.c.n_kv_heads + g.h;
                };
                const int k_box = key0 + lane * box, k_sc = key0 + lane * 16;
                const bool load = lane < boxes && k_box < g.q.kv, scale = lane < 8 && k_sc < g.q.kv;
                const int u_box = load ? page_at(k_box) : 0, u_sc = scale ? page_at(k_sc) : 0;
                const int n = __popc(__ballot_sync(0xffffffffu, load));
                if (it > 0) wait(rk_empty, it - 1);
                if (!__all_sync(0xffffffffu, ok)) ok = false;
                if (ok) {
                    if (lane == 0) mbar_arrive_expect_tx(rk_full, (uint32_t)(n * box * HD));
                    __syncwarp();
                    if (load) kd_tma(sbase + S::O_RK + lane * box * LINE, &tm_k, 0, u_box * P + (k_box & (P - 1)), rk_full);
                    if (scale) {
                        cp_async4(s_rsc + lane, a.c.k_scale + u_sc);
                        cp_async4(s_rsc + 8 + lane, a.c.v_scale + u_sc);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(rk_full)) : "memory");
                }
                if (it > 0) wait(rv_empty, it - 1);
                if (!__all_sync(0xffffffffu, ok)) ok = false;
                if (ok) {
                    if (lane == 0) mbar_arrive_expect_tx(rv_full, (uint32_t)(n * box * HD));
                    __syncwarp();
                    if (load) kd_tma(sbase + S::O_RV + lane * box * LINE, &tm_v, 0, u_box * P + (k_box & (P - 1)), rv_full);
                }
                ++it;
            }
            cur += g.cnt;
        }
        cp_async_wait_all();
    } else if (warp >= KP_W_CONV && warp < KP_W_LOAD) {
        // ---------------------------------------------------------------- codes -> fp16 operands
        const int cw = warp - KP_W_CONV;
        uint32_t it = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            const int any_lo = a.window > 0 ? max(0, g.q.kv - g.q.n + g.row0 / a.G - a.window + 1) : 0;
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j, key0 = kt * KP_KT;
                if (!kp_active<SPLIT>(a, g, 0, kt) && !kp_active<SPLIT>(a, g, 1, kt)) continue;
                const uint32_t b = it & 1u;
                // ---- K: rows as they are; a thread turns 16 codes into two 16-byte chunks
                wait(rk_full, it);
                if (it >= 2) wait(&k_empty[b], (it >> 1) - 1);
                __syncwarp();
                if (cw == 0) {
                    if (lane < 8) {
                        const bool in = key0 + lane * 16 < g.q.kv;
                        float ks = in ? s_rsc[lane] : 0.f;
                        const float vs = in ? s_rsc[8 + lane] : 0.f;
                        float lv = -INFINITY, rv = 1.f;
                        if (vs > 0.f && vs < INFINITY) {
                            lv = log2f(vs);
                            rv = 1.f / vs;
                        } else if (vs != 0.f) {
                            ks = __uint_as_float(0x7fffffffu);  // NaN for whoever sees these keys
                        }
                        float* d = s_prep + (it & 3u) * 24;
                        d[lane] = ks;
                        d[8 + lane] = lv;
                        d[16 + lane] = rv;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&prep_full[it & 3u]);
                }
                constexpr int CPR = HD / 16;  // 16-code chunks per row
                const uint32_t kop = sbase + S::O_K + b * S::OP;
#pragma unroll 4
                for (int i = cw * 32 + lane; i < KP_KT * CPR; i += 128) {
                    const int row = i / CPR, c = i % CPR;
                    const uint32_t src = HD == 64 ? (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4))
                                                  : (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4));
                    const uint4 w = lds128(sbase + S::O_RK + src);
                    const uint32_t x[4] = {kd_bias<FMT>(w.x), kd_bias<FMT>(w.y), kd_bias<FMT>(w.z), kd_bias<FMT>(w.w)};
                    uint32_t y[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        y[2 * k] = kd_half2<FMT>(x[k], false);
                        y[2 * k + 1] = kd_half2<FMT>(x[k], true);
                    }
                    const uint32_t dst = kop + (uint32_t)((c >> 2) * (KP_KT * 128) + row * 128);
                    const uint32_t c0 = (uint32_t)((2 * c) & 7), f = (uint32_t)(row & 7);
                    // the second slab's lanes store their chunks the other way round: no two on one bank
                    const bool sw = HD == 128 && (c >> 2);
                    const uint32_t ca = (c0 + (sw ? 1u : 0u)) ^ f, cb = (c0 + (sw ? 0u : 1u)) ^ f;
                    kp_sts128(dst + (ca << 4), sw ? y[4] : y[0], sw ? y[5] : y[1], sw ? y[6] : y[2], sw ? y[7] : y[3]);
                    kp_sts128(dst + (cb << 4), sw ? y[0] : y[4], sw ? y[1] : y[5], sw ? y[2] : y[6], sw ? y[3] : y[7]);
                }
                kp_fence_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(rk_empty);
                    mbar_arrive(&k_full[b]);
                }
                // ---- V transposed: lanes are 32 pairs of keys, a thread turns 2 keys x 16 channels into 16 rows' words
                wait(rv_full, it);
                if (it >= 2) wait(&v_empty[b], (it >> 1) - 1);
                __syncwarp();
                const uint32_t vop = sbase + S::O_V + b * S::OP;
                const bool edge = key0 + KP_KT > g.q.kv || key0 < any_lo;  // keys there may hold anything: they count as zero
                const bool odd = (lane >> 2) & 1;  // these lanes read the odd key first: no two on one bank
#pragma unroll 2
                for (int i = cw; i < 2 * CPR; i += 4) {
                    const int slab = i / CPR, c = i % CPR, row = slab * 64 + 2 * lane + (odd ? 1 : 0), row2 = row ^ 1;
                    const uint32_t s1 = HD == 64 ? (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4))
                                                 : (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4));
                    const uint32_t s2 = HD == 64 ? (uint32_t)(row2 * 64 + ((c ^ ((row2 >> 1) & 3)) << 4))
                                                 : (uint32_t)(row2 * 128 + ((c ^ (row2 & 7)) << 4));
                    uint4 u = lds128(sbase + S::O_RV + s1), v = lds128(sbase + S::O_RV + s2);
                    if (edge) {
                        const int k1 = key0 + row, k2 = key0 + row2;
                        if (k1 >= g.q.kv || k1 < any_lo) u = make_uint4(0, 0, 0, 0);
                        if (k2 >= g.q.kv || k2 < any_lo) v = make_uint4(0, 0, 0, 0);
                    }
                    const uint32_t lo = odd ? 0x1504 : 0x5140, hi = odd ? 0x3726 : 0x7362;
                    const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
                    const uint32_t dst = vop + (uint32_t)(slab * HD * 128 + c * 16 * 128 + (lane & 3) * 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = kd_bias<FMT>(__byte_perm(uu[k], vv[k], lo)), y = kd_bias<FMT>(__byte_perm(uu[k], vv[k], hi));
                        const uint32_t w[4] = {kd_half2<FMT>(x, false), kd_half2<FMT>(x, true), kd_half2<FMT>(y, false),
                                               kd_half2<FMT>(y, true)};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t d = 4 * k + e;  // channel 16 c + d: row of the operand, d & 7 its place in the swizzle
                            kp_sts32(dst + d * 128 + ((((uint32_t)lane >> 2) ^ (d & 7u)) << 4), w[e]);
                        }
                    }
                }
                kp_fence_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(rv_empty);
                    mbar_arrive(&v_full[b]);
                }
                ++it;
            }
            cur += g.cnt;
        }
    } else if (warp == KP_W_MMA) {
        // ---------------------------------------------------------------- products
        constexpr uint32_t id_s = tg_idesc(128, KP_KT), id_o = tg_idesc(128, HD);
        uint32_t it = 0, nq[2] = {0, 0}, np[2] = {0, 0}, segs = 0;
        for (int cur = begin; cur < end;) {
            const KPSeg g = walk.seek(a, cur, end);
            int pend[2] = {-1, -1};          // the tile (count) whose weights stream s is making
            bool have_q[2] = {false, false}, have_o[2] = {false, false};
            int left[2] = {0, 0};            // streams that still need the V operand
            auto weigh = [&](int s) {        // O_s += P_s . V of its pending tile
                const uint32_t t = (uint32_t)pend[s], b = t & 1u;
                wait(&v_full[b], t >> 1);
                wait(&p_full[s], np[s]++);
                __syncwarp();
                kp_fence_after();
                if (lane == 0 && ok) {
                    const uint32_t vop = sbase + S::O_V + b * S::OP;
#pragma unroll
                    for (int x = 0; x < (SPLIT ? 2 : 1); ++x) {
#pragma unroll
                        for (int k = 0; k < KP_KT / 16; ++k)
                            kp_mma_ts(tmem + 256 + 128 * s, tmem + 128 * s + (k >> 1) * 32 + x * 16 + (k & 1) * 8,
                                      tg_desc(vop + (k >> 2) * HD * 128 + (k & 3) * 32), id_o, have_o[s] || x > 0 || k > 0);
                    }
                }
                have_o[s] = true;
                if (--left[b] == 0 && lane == 0 && ok) kp_commit(&v_empty[b]);
                pend[s] = -1;
            };
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j;
                const bool act[2] = {kp_active<SPLIT>(a, g, 0, kt), kp_active<SPLIT>(a, g, 1, kt)};
                if (!act[0] && !act[1]) continue;
                const uint32_t b = it & 1u;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (pend[s] >= 0 && (!SPLIT || act[s])) weigh(s);
                    if (!act[s]) continue;
                    if (!have_q[SPLIT ? 0 : s]) {
                        have_q[SPLIT ? 0 : s] = true;
                        wait(&q_full[SPLIT ? 0 : s], nq[SPLIT ? 0 : s]++);
                    }
                    wait(&k_full[b], it >> 1);
                    __syncwarp();
                    kp_fence_after();
                    if (lane == 0 && ok) {
                        const uint32_t kop = sbase + S::O_K + b * S::OP;
#pragma unroll
                        for (int x = SPLIT ? 1 : 0; x >= 0; --x) {  // the low parts first
                            const uint32_t qop = sbase + S::O_Q + (SPLIT ? x : s) * S::Q_TILE;
#pragma unroll
                            for (int k = 0; k < HD / 16; ++k)
                                kp_mma_ss(tmem + 128 * s, tg_desc(qop + (k >> 2) * 128 * 128 + (k & 3) * 32),
                                          tg_desc(kop + (k >> 2) * KP_KT * 128 + (k & 3) * 32), id_s, (SPLIT && x == 0) || k > 0);
                        }
                        kp_commit(&s_full[s]);
                    }
                    pend[s] = (int)it;
                }
                left[b] = (act[0] ? 1 : 0) + (act[1] ? 1 : 0);
                if (lane == 0 && ok) kp_commit(&k_empty[b]);
                ++it;
            }
            // the last tiles' weights, in the order of the tiles
            const int s0 = pend[0] >= 0 && (pend[1] < 0 || pend[0] <= pend[1]) ? 0 : 1;
            if (pend[s0] >= 0) weigh(s0);
            if (pend[1 - s0] >= 0) weigh(1 - s0);
            // a stream without tiles here may still be at the last unit's end: o_full must not run two ahead of it
            if (segs > 0) wait(seg_done, segs - 1);
            ++segs;
            if (lane == 0 && ok) kp_commit(o_full);
            __syncwarp();
            cur += g.cnt;
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
            const int i_row = (SPLIT ? 0 : 128 * s) + row;  // in the group
            const bool valid = i_row < g.nrows;
            const int tok_i = (g.row0 + (valid ? i_row : 0)) / a.G;
            const int head = g.h * a.G + (g.row0 + (valid ? i_row : 0)) % a.G;
            const long long tok = g.q.start + tok_i;
            const int lim = valid ? g.q.kv - g.q.n + tok_i : -1;
            const int lim_lo = a.window > 0 ? lim - a.window + 1 : 0;
            // tiles that all of this stream's rows see whole need no mask
            const int r_lo = g.row0 + (SPLIT ? 0 : 128 * s), r_hi = min(r_lo + 128, g.row0 + g.nrows) - 1;
            const bool rows_full = r_hi - r_lo == 127;
            const int lim_first = g.q.kv - g.q.n + r_lo / a.G, lim_last = g.q.kv - g.q.n + r_hi / a.G;
            bool any = false;
            for (int j = 0; j < g.cnt && !any; ++j) any = kp_active<SPLIT>(a, g, s, g.tile0 + j);
            bool any_q = any;
            if (SPLIT && s == 0)
                for (int j = 0; j < g.cnt && !any_q; ++j) any_q = kp_active<SPLIT>(a, g, 1, g.tile0 + j);
            float qs = 1.f;
            if (any_q) {
                // ---- this row of q: by a power of two into [256, 512), fp16 (and what fp16 leaves)
                const long long at = tok * a.q_stride + (long long)head * HD;
                uint32_t big = 0;
#pragma unroll 4
                for (int c = 0; c < HD; c += 8) {
                    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (valid) kv8_ld8(a.q, at + c, a.type, a.q_wide, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                const int ex = (int)(big >> 23);
                const bool plain = ex == 255;
                const int sh = plain ? 0 : max(ex, 1) - 127 - 8;
                const float f1 = __uint_as_float((uint32_t)(127 - max(min(sh, 126), -126)) << 23);
                const float f2 = sh < -126 ? __uint_as_float((uint32_t)(1 - sh) << 23) : 1.f;
                qs = (plain ? 1.f : ldexpf(1.f, sh)) * a.scale_log2;
                if (!SPLIT || s == 0) {
                    const uint32_t dst = sbase + S::O_Q + (SPLIT ? 0 : s * S::Q_TILE) + row * 128;
#pragma unroll 4
                    for (int c = 0; c < HD; c += 8) {
                        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                        if (valid) kv8_ld8(a.q, at + c, a.type, a.q_wide, x);
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float u = x[2 * e] * f1 * f2, v = x[2 * e + 1] * f1 * f2;
                            hi[e] = kd_pack(u, v);
                            if (SPLIT) lo[e] = kd_pack_rest(u, v, hi[e]);
                        }
                        const uint32_t o = dst + (c >> 6) * (128 * 128) + ((((c >> 3) & 7) ^ (row & 7)) << 4);
                        kp_sts128(o, hi[0], hi[1], hi[2], hi[3]);
                        if (SPLIT) kp_sts128(o + S::Q_TILE, lo[0], lo[1], lo[2], lo[3]);
                    }
                    kp_fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[SPLIT ? 0 : s]);
                }
            }
            float m = -INFINITY, l = 0.f, lvref = -INFINITY, vref = 0.f;
            bool have_o = false;
            for (int j = 0; j < g.cnt; ++j) {
                const int kt = g.tile0 + j, key0 = kt * KP_KT;
                const bool act = kp_active<SPLIT>(a, g, s, kt);
                if (!act && !kp_active<SPLIT>(a, g, 1 - s, kt)) continue;
                const uint32_t slot = it & 3u, use = it >> 2;
                ++it;
                if (!act) continue;
                wait(&prep_full[slot], use);
                wait(&s_full[s], n_s++);
                __syncwarp();
                kp_fence_after();
                const float* pr = s_prep + slot * 24;
                const bool masked = !rows_full || key0 + KP_KT - 1 > lim_first || (a.window > 0 && key0 < lim_last - a.window + 1);
                const int c_hi = lim - key0, c_lo = lim_lo - key0;  // this row sees the columns c_lo .. c_hi
                // ---- the row's largest
                float mt = -INFINITY, lvmax = -INFINITY;
#pragma unroll
                for (int b = 0; b < 8; ++b) lvmax = fmaxf(lvmax, pr[8 + b]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    KP_LD32(r, t_s + c * 32);
                    kp_wait_ld();
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        float x = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int col = c * 32 + b * 16 + e;
                            float y = __uint_as_float(r[b * 16 + e]);
                            if (masked && (col > c_hi || col < c_lo)) y = -INFINITY;
                            x = fmaxf(x, y);
                        }
                        mt = fmaxf(mt, x * (pr[c * 2 + b] * qs));
                    }
                }
                const bool move_v = lvmax > lvref + 4.f;
                if (__any_sync(0xffffffffu, move_v || mt > m + KD_LAZY)) {
                    const float mn = fmaxf(m, mt), lvn = move_v ? lvmax : lvref;
                    float al = mn == -INFINITY ? 1.f : kd_exp2(m - mn);
                    l *= al;
                    if (move_v) {
                        al *= lvref == -INFINITY ? 0.f : kd_exp2(lvref - lvn);
                        lvref = lvn;
                        vref = exp2f(lvn);
                    }
                    m = mn;
                    if (have_o) {  // the products of the tiles before have ended: S came after them
#pragma unroll
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t r[32];
                            KP_LD32(r, t_o + c);
                            kp_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * al);
                            KP_ST32(t_o + c, r);
                        }
                    }
                }
                have_o = true;
                const float mm = m == -INFINITY ? 0.f : m, lv0 = lvref == -INFINITY ? 0.f : lvref;
                // ---- weights, in place of the scores
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32], hi[16], lo[16];
                    KP_LD32(r, t_s + c * 32);
                    kp_wait_ld();
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const float cf = pr[c * 2 + b] * qs, d = pr[8 + c * 2 + b] - lv0;
                        const bool tiny = !(d >= -40.f);  // a page of zeros, or next to it
                        const float add = SPLIT ? -mm : (tiny ? -40.f : d) - mm;
                        const float fb = SPLIT ? (tiny ? 0.f : kd_exp2(d)) : 0.f;
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float p[2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int col = c * 32 + b * 16 + e + y;
                                p[y] = kd_exp2(fmaf(__uint_as_float(r[b * 16 + e + y]), cf, add));
                                if (masked && (col > c_hi || col < c_lo)) p[y] = 0.f;
                                sum += p[y];
                                if (SPLIT) p[y] *= fb;
                            }
                            const int at = b * 8 + (e >> 1);
                            hi[at] = kd_pack(p[0], p[1]);
                            if (SPLIT) lo[at] = kd_pack_rest(p[0], p[1], hi[at]);
                        }
                        l += SPLIT ? sum : sum * (tiny ? 1.0995116e12f : pr[16 + c * 2 + b] * (lvref == -INFINITY ? 1.f : vref));
                    }
                    KP_ST16(t_s + c * 32, hi);
                    if (SPLIT) KP_ST16(t_s + c * 32 + 16, lo);
                }
                kp_wait_st();
                kp_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[s]);
            }
            // ---- the unit's (or this part's) end
            wait(o_full, n_o++);
            __syncwarp();
            kp_fence_after();
            const bool whole = g.cnt == g.tiles, direct = whole && !SPLIT;
            const int unit0 = cur - g.first;
            const int c_first = unit0 / per, c_last = (unit0 + g.tiles - 1) / per;
            if (direct) {
                const float inv = l == 0.f ? 0.f : vref / l;
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t r[32];
                    if (have_o) {
                        KP_LD32(r, t_o + c);
                        kp_wait_ld();
                    }
                    if (valid) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            float x[8];
#pragma unroll
                            for (int y = 0; y < 8; ++y) x[y] = have_o && l != 0.f ? __uint_as_float(r[e + y]) * inv : 0.f;
                            kv8_st8(a.out, tok * a.out_stride + (long long)head * HD + c + e, a.type, a.out_wide, x);
                        }
                    }
                }
                if (valid && a.lse) a.lse[tok * a.n_q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
            } else {
                // record of (CTA, slot, stream): m and l of each row, then the sums, four channels of all rows after one another
                float* rec = a.part + ((long long)blockIdx.x * 4 + (g.first > 0 ? 0 : 2) + s) * S::REC;
                __stcg(reinterpret_cast<float2*>(rec) + row, make_float2(m, l));
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t r[32];
                    if (have_o) {
                        KP_LD32(r, t_o + c);
                        kp_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (have_o)
                            v = make_float4(__uint_as_float(r[e]) * vref, __uint_as_float(r[e + 1]) * vref,
                                            __uint_as_float(r[e + 2]) * vref, __uint_as_float(r[e + 3]) * vref);
                        __stcg(reinterpret_cast<float4*>(rec + 256) + ((c + e) >> 2) * 128 + row, v);
                    }
                }
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
                    const int c0 = SPLIT ? s * (HD / 2) : 0, c1 = SPLIT ? c0 + HD / 2 : HD;
                    float M = -INFINITY, L = 0.f;
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
                    for (int c = c0; c < c1; c += 32) {
                        float acc[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[e] = 0.f;
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
                                kv8_st8(a.out, tok * a.out_stride + (long long)head * HD + c + e, a.type, a.out_wide, x);
                            }
                        }
                    }
                    if (valid && a.lse && (!SPLIT || s == 0))
                        a.lse[tok * a.n_q_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945f;
                }
            }
            kp_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_done);
            cur += g.cnt;
        }
    }
    kp_fence_before();
    __syncthreads();
    if (warp == KP_W_MMA)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace fence
