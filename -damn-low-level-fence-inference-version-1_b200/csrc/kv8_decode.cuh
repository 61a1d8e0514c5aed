// kv8_decode.cuh — attention of up to 48 query rows per request and KV head over the paged 8-bit cache (decode, drafts).
//
//   s[j][h] = (K code row j . q row h) * k_scale[page] * scale,  p = softmax(s),  out = p . (V code rows * v_scale[page])
//
// Bound: HBM, two bytes per key, head and channel; the kernel has to keep the codes coming and turn them
// into matrix operands fast enough. 3 requests of 90k to 131k keys, 8 heads of 128, e4m3: 639 MB in 120 us (82 % of the
// measured copy bandwidth); 64 requests of 60 to 8000 keys: 199 MB in 50 us, a third of it starts and ends of units.
//
//  * Work is the list of 32-key tiles of every (request, KV head, group of 8 NT query rows), cut into
//    runs of equal cost, one per CTA, whatever the lengths are: a CTA's run may begin and end inside a unit. Such a
//    unit's partial results go to the workspace and the last of its CTAs to arrive joins them in the
//    order of the keys, so the result does not depend on timing.
//  * One producer warp per CTA copies each tile's pages (TMA, 16 or more rows at a time, swizzled so
//    that all operand loads are free of bank conflicts) and their scales into a ring of stages.
//  * Four consumer warps take the tiles in turn, each with a softmax state of its own: keys are the
//    rows of the matrix products (S^T = K Q^T: 16 keys x 8 rows, O^T = V^T P^T: 16 channels x 8 rows),
//    so 8 query rows fill the instruction and nothing is padded for grouped heads. A page holds 16 or
//    more keys: 16 keys share their scales. (A tile shared by the warps, 16 keys each, spent a third
//    more instructions on the softmax state per key.)
//  * Codes become fp16 exactly. Scales never touch them: k_scale multiplies the scores, v_scale the
//    weights. q rows are brought to [256, 512) by a power of two, so that fp16 holds them whatever their
//    range. SPLIT (fp32 activations): q and the weights as a pair of fp16 (22 bits), and the products of
//    16 keys are added to the sums in fp32 outside the matrix unit. 16-bit rows add up inside it, where additions truncate:
//    mean relative error -1.4e-4 where one CTA takes all of 131000 keys (fp16 rounds by 2^-12 at least), less where units are cut.
//  * Two references per row, both of keys that the row sees: m for the sum of the weights, near the largest
//    score s, and u for the sums of values, near the largest s + log2 v_scale. What is rounded to fp16 is
//    2^(s - u + KD_UP) * v_scale: large where the row's own output comes from, whatever the scale of a page that it gives
//    little weight (with the largest v_scale for a reference, pages 2^25 below it counted as zero). References are
//    whole numbers: bringing sums to a new one is exact.
#pragma once

#include <cuda.h>

#include "kv8.cuh"

namespace fence {

struct KAttnArgs {
    fence_kv8_cache c;
    const int* block_table;
    const int* kv_len;
    const int* new_start;
    int n_req, n_tokens, max_pages, shift, G, n_q_heads, window, type;
    const void* q;
    void* out;
    float* lse;
    long long q_stride, out_stride;
    float scale_log2;  // scale * log2(e): scores are kept as exponents of 2
    int max_rows;      // decode kernel: requests of more query rows per KV head are left to the prefill kernel
    int behind_prefill;    // decode kernel: the kernel before is this call's prefill kernel, with other rows: no need to wait for it
    int min_rows;      // prefill kernel: requests of at most this many are the decode kernel's
    int q_wide, out_wide;  // rows are 16-byte aligned
    __half* q_rows;        // prefill kernel: [2][n_kv_heads][n_tokens * G][head_dim], rows of q as it multiplies them (high, low)
    float* q_scale;        // [n_kv_heads][n_tokens * G]: times this gives scores
    int* arrived;      // [CTAs] partial results of the unit that starts in this CTA and goes on in the next
    float* part;       // [CTAs][2][rows * (head_dim + 2)]
};

constexpr int KD_TILE = 32, KD_WARPS = 4, KD_THREADS = 32 * (KD_WARPS + 1);
constexpr int KD_MIN_TILES = 4;  // tiles per CTA below which more CTAs only add joins
constexpr int KD_UNIT = 8;       // a unit's start and end cost about as much as eight tiles: counted so when the runs are cut
constexpr float KD_LAZY = 8.f;   // the references may lag by 2^8
constexpr float KD_UP = 6.f;     // weights enter fp16 times 2^6: below 2^(8 + 6 + 1), so small ones keep more of their bits
constexpr float KD_FLOOR = 120.f;  // u >= m - 120, so that 2^(u - m) and its reciprocal are normal numbers (for v_scale near 2^-126)

template <int HD, bool SPLIT, int NT>
struct KDShape {
    // CTAs per SM, by the registers that the sums take (256 channels of fp32: 103 us with one, 109 with the registers of two, 4
    // requests of 30000 to 60000 keys)
    static constexpr int CTAS = HD == 256 ? (NT == 2 || SPLIT ? 1 : 2) : (HD == 128 && NT == 2 ? 2 : 3);
    // twice as many stages as warps: with one each, every tile's load began when the tile before it was done with
    // (SPLIT's second part of q takes the place of one: with 12 a single CTA fitted, 47 us against 37 for drafts of 4)
    static constexpr int STAGES = HD == 64 ? 12 : HD == 128 ? (CTAS == 3 ? 8 : SPLIT ? 11 : 12) : CTAS == 1 ? 10 : 6;
    static constexpr int KV_BYTES = KD_TILE * HD;
    static constexpr int STAGE = 2 * KV_BYTES;
    static constexpr int ROWS = 8 * NT;
    static constexpr int SLAB = HD + 4;
    // after the ring: scales, barriers, q fragments (high and low), rows' scales, the warps' (m, l), the slab
    static constexpr int O_SCALE = STAGES * STAGE;
    static constexpr int O_BAR = O_SCALE + STAGES * 32;
    static constexpr int O_Q = O_BAR + 2 * STAGES * 8;
    static constexpr int O_QS = O_Q + NT * (SPLIT ? 2 : 1) * (HD / 16) * 256;
    static constexpr int O_ML = O_QS + ROWS * 4;
    static constexpr int O_SLAB = O_ML + KD_WARPS * ROWS * 8;
    static constexpr int O_SCAN = O_SLAB + ROWS * SLAB * 4;
    static constexpr int SMEM = O_SCAN + 64 + 1024;  // + the prefix sums [n_req + 1], + alignment
    static_assert(CTAS * (SMEM + 4 * 257 + 1024) <= 228 * 1024, "CTAS of them fit an SM, for up to 256 requests");
};

__device__ __forceinline__ void kd_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t kd_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float kd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t kd_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// what fp16 leaves of a and b
__device__ __forceinline__ uint32_t kd_pack_rest(float a, float b, uint32_t hi) {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return kd_pack(a - h.x, b - h.y);
}
__device__ __forceinline__ uint2 kd_lds64(uint32_t sa) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(sa));
    return v;
}
__device__ __forceinline__ void kd_tma(uint32_t dst, const CUtensorMap* tm, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// What one request contributes: its rows in the token buffers and the keys that they can see.
struct KReq {
    int start, n, kv, tile0, tiles, groups;
};
__device__ __forceinline__ KReq kd_request(const KAttnArgs& a, int r, int rows_per_group, int tile_keys, bool report) {
    KReq q{};
    q.start = a.new_start[r];
    int end = a.new_start[r + 1], kv = a.kv_len[r];
    const int most = a.max_pages << a.shift;
    if (q.start < 0 || end < q.start || end > a.n_tokens || kv < 0 || kv > most) {
        if (report) set_device_error(KV8_BAD);
        q.start = max(0, min(q.start, a.n_tokens));
        end = max(q.start, min(end, a.n_tokens));
        kv = max(0, min(kv, most));
    }
    q.n = end - q.start;
    q.kv = kv;
    if (q.n == 0) return q;
    const int lo = a.window > 0 ? max(0, kv - q.n - a.window + 1) : 0;  // the first row's first key
    q.tile0 = lo / tile_keys;
    q.tiles = kv > 0 ? (kv - 1) / tile_keys - q.tile0 + 1 : 1;  // a request that sees nothing still has its rows written
    q.groups = (int)(((long long)q.n * a.G + rows_per_group - 1) / rows_per_group);
    return q;
}

template <int FMT, int HD, bool SPLIT, int NT>
__global__ void __launch_bounds__(KD_THREADS, KDShape<HD, SPLIT, NT>::CTAS)
    kv8_decode_kernel(const KAttnArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using S = KDShape<HD, SPLIT, NT>;
    constexpr int ROWS = S::ROWS, KS = HD / 16, MT = HD / 16, HALVES = HD == 256 ? 2 : 1, LINE = HD == 64 ? 64 : 128;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    float* s_scale = reinterpret_cast<float*>(smem + S::O_SCALE);  // [stage][K 4, V 4]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::O_BAR);
    uint64_t* empty = full + S::STAGES;
    uint2* s_q = reinterpret_cast<uint2*>(smem + S::O_Q);  // [NT][high, SPLIT: low][KS][32]
    float* s_qs = reinterpret_cast<float*>(smem + S::O_QS);
    float2* s_ml = reinterpret_cast<float2*>(smem + S::O_ML);  // [warp][ROWS]
    float* s_slab = reinterpret_cast<float*>(smem + S::O_SLAB);
    int* s_misc = reinterpret_cast<int*>(smem + S::O_SCAN);
    int* s_pre = s_misc + 16;  // [n_req + 1] tiles before each request

    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&full[s], 33);
            mbar_init(&empty[s], 1);
        }
        fence_barrier_init();
    }
    // The prefill kernel of the same call lets this one start once it has itself waited for all before it.
    if (!a.behind_prefill) {
        pdl_launch_dependents();
        pdl_wait();
    }
    // ---- prefix sums of the requests' tiles
    {
        const int per = (a.n_req + KD_THREADS - 1) / KD_THREADS;
        const int r0 = min(a.n_req, tid * per), r1 = min(a.n_req, r0 + per);
        long long sum = 0;
        for (int r = r0; r < r1; ++r) {
            const KReq q = kd_request(a, r, ROWS, KD_TILE, blockIdx.x == 0);
            const long long w = (long long)q.n * a.G > a.max_rows ? 0 : (long long)(q.tiles + KD_UNIT) * q.groups * a.c.n_kv_heads;
            s_pre[r] = (int)min(w, (long long)INT_MAX);
            sum += w;
        }
        long long v = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        long long* s_w = reinterpret_cast<long long*>(s_ml);
        if (lane == 31) s_w[warp] = v;
        __syncthreads();
        for (int w = 0; w < warp; ++w) v += s_w[w];
        v -= sum;
        for (int r = r0; r < r1; ++r) {
            const int w = s_pre[r];
            s_pre[r] = (int)min(v, (long long)INT_MAX);
            v += w;
        }
        if (tid == KD_THREADS - 1) {
            if (v > INT_MAX) set_device_error(KV8_BAD);
            s_pre[a.n_req] = (int)min(v, (long long)INT_MAX);
        }
        __syncthreads();
    }
    const int total = s_pre[a.n_req];
    const int per = max(KD_MIN_TILES + KD_UNIT, (int)(((long long)total + gridDim.x - 1) / gridDim.x));
    const int begin = (int)min((long long)total, (long long)blockIdx.x * per), end = min(total, begin + min(per, total - begin));
    // the request of the run's first tile
    int r = 0;
    {
        int hi = a.n_req;
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if (s_pre[mid] <= begin) r = mid;
            else hi = mid;
        }
    }
    bool ok = true;
    const int P = a.c.page_tokens, box = min(P, KD_TILE), boxes = KD_TILE / box;

    if (warp == KD_WARPS) {
        // ---------------------------------------------------------------- producer
        int it = 0;
        for (int cur = begin; cur < end;) {
            while (s_pre[r + 1] <= cur) ++r;
            const KReq q = kd_request(a, r, ROWS, KD_TILE, false);
            const int span = q.tiles + KD_UNIT, unit = (cur - s_pre[r]) / span, unit0 = s_pre[r] + unit * span;
            const int first = max(0, cur - unit0 - KD_UNIT), cnt = min(q.tiles, end - unit0 - KD_UNIT) - first, h = unit / q.groups;
            if (cnt <= 0) break;  // the run ends in this unit's start: its tiles are the next CTA's
            const int lo = a.window > 0 ? max(0, q.kv - q.n - a.window + 1) : 0;
            const int* table = a.block_table + (size_t)r * a.max_pages;
            int ids = 0, ids_at = -1;  // this lane's page id of a run of 32 pages
            for (int i = 0; i < cnt; ++i, ++it) {
                const int s = it % S::STAGES, key0 = (q.tile0 + first + i) * KD_TILE;
                const int p0 = key0 >> a.shift;
                if (ids_at < 0 || p0 >= ids_at + 32 || p0 < ids_at) {
                    ids_at = p0 & ~(boxes - 1);
                    const int j = ids_at + lane;
                    ids = (j << a.shift) < q.kv ? table[j] : 0;
                }
                if (ok && it >= S::STAGES) ok = mbar_wait(&empty[s], (uint32_t)(it / S::STAGES - 1) & 1u);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                int page = __shfl_sync(0xffffffffu, ids, (p0 - ids_at + lane) & 31);
                const int k_lo = key0 + lane * box;
                bool mine = lane < boxes && k_lo < q.kv && k_lo + box > lo;
                if (mine && (page < 0 || page >= a.c.n_pages)) {
                    set_device_error(KV8_BAD);
                    page = 0;
                }
                const int loads = __popc(__ballot_sync(0xffffffffu, mine));
                if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(loads * box * HD * 2));
                __syncwarp();
                if (mine) {
                    const int unit_row = page * a.c.n_kv_heads + h;
                    const int y = unit_row * P + (k_lo & (P - 1));
                    const uint32_t dst = sbase + (uint32_t)(s * S::STAGE + lane * box * LINE);
#pragma unroll
                    for (int x = 0; x < HALVES; ++x) {
                        kd_tma(dst + x * KD_TILE * LINE, &tm_k, x * 128, y, &full[s]);
                        kd_tma(dst + S::KV_BYTES + x * KD_TILE * LINE, &tm_v, x * 128, y, &full[s]);
                    }
                    cp_async4(s_scale + s * 8 + lane, a.c.k_scale + unit_row);
                    cp_async4(s_scale + s * 8 + 4 + lane, a.c.v_scale + unit_row);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
            }
            if (!ok) break;
            cur = unit0 + KD_UNIT + first + cnt;
        }
        cp_async_wait_all();
        if (a.behind_prefill) pdl_wait();  // so that what comes next waits for both
        return;
    }
    // -------------------------------------------------------------------- consumers
    // rows that belong to no request
    {
        const int used = max(0, min(a.new_start[a.n_req], a.n_tokens));
        const long long row = (long long)a.n_q_heads * HD, n = (a.n_tokens - used) * row;
        const int ct = blockIdx.x * 128 + tid, cs = gridDim.x * 128;
        for (long long i = ct; i < n; i += cs) kv8_st1(a.out, (used + i / row) * a.out_stride + i % row, a.type, 0.f);
        if (a.lse)
            for (long long i = ct; i < (long long)(a.n_tokens - used) * a.n_q_heads; i += cs)
                a.lse[(long long)used * a.n_q_heads + i] = -INFINITY;
    }
    int it = 0;
    for (int cur = begin; cur < end;) {
        while (s_pre[r + 1] <= cur) ++r;
        const KReq q = kd_request(a, r, ROWS, KD_TILE, false);
        const int span = q.tiles + KD_UNIT, unit = (cur - s_pre[r]) / span, unit0 = s_pre[r] + unit * span;
        const int first = max(0, cur - unit0 - KD_UNIT), cnt = min(q.tiles, end - unit0 - KD_UNIT) - first;
        if (cnt <= 0) break;
        const int h = unit / q.groups, row0 = (unit - h * q.groups) * ROWS;
        const int rows = min(ROWS, q.n * a.G - row0);  // row = token * G + head in the group
        // ---- q rows: scaled by a power of two into [256, 512), as B fragments
        for (int i = warp; i < ROWS; i += KD_WARPS) {
            constexpr int EPL = HD / 32;  // elements per lane: 2, 4 or 8
            float x[EPL];
            uint32_t big = 0;
            const int tok = q.start + (row0 + i) / a.G, head = h * a.G + (row0 + i) % a.G;
            const long long at = tok * a.q_stride + (long long)head * HD + lane * EPL;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                x[e] = i >= rows ? 0.f
                       : a.type == FENCE_F32 ? static_cast<const float*>(a.q)[at + e]
                       : a.type == FENCE_F16 ? __half2float(static_cast<const __half*>(a.q)[at + e])
                                             : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at + e]);
                big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
            }
            big = __reduce_max_sync(0xffffffffu, big);
            const int ex = (int)(big >> 23);  // biased exponent
            const bool plain = ex == 255;     // infinity or NaN in the row
            const int sh = plain ? 0 : max(ex, 1) - 127 - 8;  // times 2^-sh
            const float f1 = __uint_as_float((uint32_t)(127 - max(min(sh, 126), -126)) << 23);
            const float f2 = sh > 126 ? 0.5f : sh < -126 ? __uint_as_float((uint32_t)(127 - sh - 126) << 23) : 1.f;
            if (lane == 0) s_qs[i] = plain ? 1.f : ldexpf(1.f, sh);
#pragma unroll
            for (int e = 0; e < EPL; e += 2) {
                const float u = x[e] * f1 * f2, v = x[e + 1] * f1 * f2;
                const uint32_t hi = kd_pack(u, v);
                const int c = lane * EPL + e;  // channel: k step j, thread ct of the quad, pair
                const int half = c / 128, cc = c % 128;
                const int ct = HD == 64 ? cc / 16 : cc / 32, j = HD == 64 ? (cc % 16) / 4 : half * 8 + (cc % 32) / 4;
                uint32_t* dst = reinterpret_cast<uint32_t*>(s_q) +
                                ((((i >> 3) * (SPLIT ? 2 : 1)) * KS + j) * 32 + (i & 7) * 4 + ct) * 2 + ((c >> 1) & 1);
                dst[0] = hi;
                if (SPLIT) dst[KS * 64] = kd_pack_rest(u, v, hi);
            }
        }
        named_bar_sync(1, 32 * KD_WARPS);
        // ---- this thread's rows 8 nt + 2 t + e: scale and last visible position
        float qs[NT][2], m[NT][2], u[NT][2], l[NT][2];
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = nt * 8 + 2 * t + e;
                qs[nt][e] = s_qs[i] * a.scale_log2;
                lim[nt][e] = i < rows ? q.kv - q.n + (row0 + i) / a.G : -1;
                m[nt][e] = u[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
            }
        // keys that every row sees, and keys that some row sees
        const int lim_first = q.kv - q.n + row0 / a.G, lim_last = q.kv - q.n + (row0 + rows - 1) / a.G;
        const int all_lo = a.window > 0 ? lim_last - a.window + 1 : 0, any_lo = a.window > 0 ? lim_first - a.window + 1 : 0;
        float o[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;

        for (int i = warp; i < cnt; i += KD_WARPS) {
            const uint32_t n = (uint32_t)(it + i);
            const int s = n % S::STAGES, key0 = (q.tile0 + first + i) * KD_TILE;
            if (ok) ok = mbar_wait(&full[s], (n / S::STAGES) & 1u);
            __syncwarp();
            if (key0 <= lim_last && key0 + KD_TILE - 1 >= any_lo && lim_last >= 0) {
                constexpr int MK = KD_TILE / 16;  // blocks of 16 keys: one page each, or a part of one
                const uint32_t kb = sbase + (uint32_t)(s * S::STAGE), vb = kb + S::KV_BYTES;
                float sk[MK], sv[MK];
#pragma unroll
                for (int y = 0; y < MK; ++y) {
                    sk[y] = s_scale[s * 8 + (box == 16 ? y : 0)];  // a box of 32 keys holds the tile
                    sv[y] = s_scale[s * 8 + 4 + (box == 16 ? y : 0)];
                }
                // ---- scores of 32 keys: two products side by side
                float acc[MK][NT][4], low[SPLIT ? MK : 1][NT][4];
#pragma unroll
                for (int y = 0; y < MK; ++y)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            acc[y][nt][e] = 0.f;
                            if (SPLIT) low[y][nt][e] = 0.f;
                        }
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {  // 16 bytes of each of the rows g and g + 8 of every block
                    const uint32_t off = HD == 64 ? (uint32_t)(g * 64 + ((t ^ ((g >> 1) & 3)) << 4))
                                                  : (uint32_t)((c >> 1) * KD_TILE * 128 + g * 128 + (((2 * t + (c & 1)) ^ g) << 4));
                    uint4 ka[MK], kc[MK];
#pragma unroll
                    for (int y = 0; y < MK; ++y) {
                        ka[y] = lds128(kb + off + y * 16 * LINE);
                        kc[y] = lds128(kb + off + (y * 16 + 8) * LINE);
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int j = HD == 64 ? w : (c >> 1) * 8 + (c & 1) * 4 + w;
                        uint2 bq[NT], bl[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            bq[nt] = s_q[((nt * (SPLIT ? 2 : 1)) * KS + j) * 32 + lane];
                            if (SPLIT) bl[nt] = s_q[((nt * 2 + 1) * KS + j) * 32 + lane];
                        }
#pragma unroll
                        for (int y = 0; y < MK; ++y) {
                            const uint32_t xa = kd_bias<FMT>(w == 0 ? ka[y].x : w == 1 ? ka[y].y : w == 2 ? ka[y].z : ka[y].w);
                            const uint32_t xb = kd_bias<FMT>(w == 0 ? kc[y].x : w == 1 ? kc[y].y : w == 2 ? kc[y].z : kc[y].w);
                            const uint32_t a0 = kd_half2<FMT>(xa, false), a1 = kd_half2<FMT>(xb, false);
                            const uint32_t a2 = kd_half2<FMT>(xa, true), a3 = kd_half2<FMT>(xb, true);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                kd_mma(acc[y][nt], a0, a1, a2, a3, bq[nt].x, bq[nt].y);
                                if (SPLIT) kd_mma(low[y][nt], a0, a1, a2, a3, bl[nt].x, bl[nt].y);
                            }
                        }
                    }
                }
                // ---- scale, mask, the largest of each row
                const bool masked = key0 + KD_TILE - 1 > lim_first || (a.window > 0 && key0 < all_lo);
                float lv[MK];  // whole part of log2 v_scale
#pragma unroll
                for (int y = 0; y < MK; ++y) {
                    // out of every row's sight the page was not fetched, nor its scales
                    if (masked && (key0 + y * 16 > lim_last || key0 + y * 16 + 15 < any_lo)) sv[y] = 0.f;
                    lv[y] = sv[y] > 0.f && sv[y] < INFINITY ? (float)((int)(__float_as_uint(sv[y]) >> 23) - 127) : -INFINITY;
                }
                bool move = false;
                float mt[NT][2], ut[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int y = 0; y < MK; ++y)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float x = acc[y][nt][e];
                            if (SPLIT) x += low[y][nt][e];
                            acc[y][nt][e] = x * (qs[nt][e & 1] * sk[y]);
                        }
                    if (masked) {
#pragma unroll
                        for (int y = 0; y < MK; ++y)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = key0 + y * 16 + g + (e >> 1) * 8, li = lim[nt][e & 1];
                                if (key > li || (a.window > 0 && key <= li - a.window)) acc[y][nt][e] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {  // this thread's keys; the whole row's only if a reference has to move
                        float x = -INFINITY, w = -INFINITY;
#pragma unroll
                        for (int y = 0; y < MK; ++y) {
                            const float z = fmaxf(acc[y][nt][e], acc[y][nt][e + 2]);
                            x = fmaxf(x, z);
                            w = fmaxf(w, z + lv[y]);
                        }
                        mt[nt][e] = x;
                        ut[nt][e] = w;
                        move |= x > m[nt][e] + KD_LAZY || w > u[nt][e] + KD_LAZY;  // also the first: -inf
                    }
                }
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = mt[nt][e], w = ut[nt][e];
#pragma unroll
                            for (int z = 4; z < 32; z *= 2) {
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, z));
                                w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, z));
                            }
                            // each row by itself: what another row sees has no say
                            const float mn = x > m[nt][e] + KD_LAZY ? ceilf(x) : m[nt][e];
                            const float un = fmaxf(w > u[nt][e] + KD_LAZY ? ceilf(w) : u[nt][e], mn - KD_FLOOR);
                            l[nt][e] *= mn == -INFINITY ? 1.f : kd_exp2(m[nt][e] - mn);
                            const float al = un == -INFINITY ? 1.f : kd_exp2(u[nt][e] - un);
                            m[nt][e] = mn;
                            u[nt][e] = un;
#pragma unroll
                            for (int i2 = 0; i2 < MT; ++i2) {
                                o[i2][nt][e] *= al;
                                o[i2][nt][e + 2] *= al;
                            }
                        }
                }
                // ---- the weights as B fragments, with the V scale
                float mm[NT][2], fu[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        mm[nt][e] = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
                        fu[nt][e] = m[nt][e] == -INFINITY ? 1.f : kd_exp2(KD_UP + m[nt][e] - u[nt][e]);
                    }
                uint32_t b0[MK][NT], b1[MK][NT], c0[SPLIT ? MK : 1][NT], c1[SPLIT ? MK : 1][NT];
#pragma unroll
                for (int y = 0; y < MK; ++y) {
                    // a NaN or infinite scale gives NaN to whoever sees the key
                    if (!(sv[y] < INFINITY)) sv[y] = __uint_as_float(0x7fffffffu);
                    const bool apart = masked && !(sv[y] < INFINITY);  // to nobody else
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float p[4], fv[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            fv[e] = sv[y] * fu[nt][e];
                            if (fv[e] > 3e38f) fv[e] = 3e38f;  // a weight of 0 stays so; a NaN scale too
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = kd_exp2(acc[y][nt][e] - mm[nt][e & 1]);
                            l[nt][e & 1] += x;
                            p[e] = x * fv[e & 1];
                        }
                        if (apart) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (acc[y][nt][e] == -INFINITY) p[e] = 0.f;
                        }
                        const uint32_t h0 = kd_pack(p[0], p[1]), h1 = kd_pack(p[2], p[3]);
                        b0[y][nt] = kd_transpose(h0);
                        b1[y][nt] = kd_transpose(h1);
                        if (SPLIT) {
                            c0[y][nt] = kd_transpose(kd_pack_rest(p[0], p[1], h0));
                            c1[y][nt] = kd_transpose(kd_pack_rest(p[2], p[3], h1));
                        }
                    }
                }
                // ---- O^T += V^T P^T; keys that no row sees count as zero, whatever their codes are
#pragma unroll
                for (int y = 0; y < MK; ++y) {
                    const int rv = y * 16 + 2 * t;
#pragma unroll
                    for (int x = 0; x < HALVES; ++x) {
                        constexpr int WORDS = HD == 64 ? 2 : 4;
                        uint32_t w[4][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int row = rv + (e & 1) + (e >> 1) * 8;
                            if (HD == 64) {
                                const uint2 v = kd_lds64(vb + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + ((g & 1) << 3));
                                w[e][0] = v.x, w[e][1] = v.y;
                            } else {
                                const uint4 v = lds128(vb + x * KD_TILE * 128 + row * 128 + ((g ^ (row & 7)) << 4));
                                w[e][0] = v.x, w[e][1] = v.y, w[e][2] = v.z, w[e][3] = v.w;
                            }
                        }
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = key0 + rv + (e & 1) + (e >> 1) * 8;
                                if (key > lim_last || key < any_lo) {
#pragma unroll
                                    for (int k = 0; k < WORDS; ++k) w[e][k] = 0;
                                }
                            }
                        }
#pragma unroll
                        for (int k = 0; k < WORDS; ++k) {
#pragma unroll
                            for (int z = 0; z < 2; ++z) {  // bytes 0, 1 or 2, 3 of the word: two channels
                                const uint32_t sel = z ? 0x7362 : 0x5140;
                                const uint32_t u = kd_bias<FMT>(__byte_perm(w[0][k], w[1][k], sel));
                                const uint32_t v = kd_bias<FMT>(__byte_perm(w[2][k], w[3][k], sel));
                                const uint32_t a0 = kd_half2<FMT>(u, false), a1 = kd_half2<FMT>(u, true);
                                const uint32_t a2 = kd_half2<FMT>(v, false), a3 = kd_half2<FMT>(v, true);
                                const int i2 = x * 8 + 2 * k + z;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    if (SPLIT) {
                                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                                        kd_mma(d, a0, a1, a2, a3, c0[y][nt], c1[y][nt]);
                                        kd_mma(d, a0, a1, a2, a3, b0[y][nt], b1[y][nt]);
#pragma unroll
                                        for (int e = 0; e < 4; ++e) o[i2][nt][e] += d[e];
                                    } else {
                                        kd_mma(o[i2][nt], a0, a1, a2, a3, b0[y][nt], b1[y][nt]);
                                    }
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        it += cnt;
        // ---- the four warps' results into one: largest m, then sum of o * 2^(u - KD_UP - M)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) s_ml[warp * ROWS + nt * 8 + 2 * t + e] = make_float2(m[nt][e], x);
            }
        named_bar_sync(1, 32 * KD_WARPS);
        float w_row[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, s_ml[w * ROWS + nt * 8 + 2 * t + e].x);
                w_row[nt][e] = exp2f(u[nt][e] - KD_UP - (M == -INFINITY ? 0.f : M));  // a power of 2, maybe a subnormal one
            }
        for (int w = 0; w < KD_WARPS; ++w) {
            if (w == warp) {
#pragma unroll
                for (int i2 = 0; i2 < MT; ++i2)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            // columns in the order (channel tile, g, 2 channels)
                            float2* d = reinterpret_cast<float2*>(s_slab + (nt * 8 + 2 * t + e) * S::SLAB + i2 * 16 + 2 * g);
                            float2 v = make_float2(o[i2][nt][e] * w_row[nt][e], o[i2][nt][e + 2] * w_row[nt][e]);
                            if (w > 0) {
                                const float2 u = *d;
                                v.x += u.x;
                                v.y += u.y;
                            }
                            *d = v;
                        }
            }
            named_bar_sync(1, 32 * KD_WARPS);
        }
        // channel of slab column c
        auto channel = [](int c) {
            const int i2 = c >> 4, gg = (c >> 1) & 7, e = c & 1;
            return HD == 64 ? gg * 8 + 2 * i2 + e : (i2 >> 3) * 128 + gg * 16 + 2 * (i2 & 7) + e;
        };
        const bool whole = cnt == q.tiles;
        const int c_first = (unit0 + KD_UNIT) / per, c_last = (unit0 + KD_UNIT + q.tiles - 1) / per;
        const int stride = ROWS * (HD + 2);
        bool write = whole;
        if (!whole) {
            float* rec = a.part + ((long long)blockIdx.x * 2 + (first > 0 ? 0 : 1)) * stride;
            for (int i = tid; i < ROWS * (HD / 4); i += 128) {
                const int row = i / (HD / 4), c = (i % (HD / 4)) * 4;
                const float* s4 = s_slab + row * S::SLAB + c;
                __stcg(reinterpret_cast<float4*>(rec + row * HD + c), make_float4(s4[0], s4[1], s4[2], s4[3]));
            }
            if (tid < ROWS) {
                float M = -INFINITY, L = 0.f;
                for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, s_ml[w * ROWS + tid].x);
                for (int w = 0; w < KD_WARPS; ++w) {
                    const float2 v = s_ml[w * ROWS + tid];
                    L += v.y * kd_exp2(v.x - (M == -INFINITY ? 0.f : M));
                }
                __stcg(reinterpret_cast<float2*>(rec + ROWS * HD) + tid, make_float2(M, L));
            }
            __threadfence();
            named_bar_sync(1, 32 * KD_WARPS);
            if (tid == 0) {
                const int n = atomicAdd(a.arrived + c_first, 1);
                const bool last = n == c_last - c_first;
                if (last) a.arrived[c_first] = 0;  // ready for the next call
                __threadfence();
                s_misc[0] = last;
            }
            named_bar_sync(1, 32 * KD_WARPS);
            write = s_misc[0] != 0;
            if (write) {
                // join the parts in the order of the keys
                for (int i = tid; i < ROWS * (HD / 4); i += 128) {
                    const int row = i / (HD / 4), c = (i % (HD / 4)) * 4;
                    float M = -INFINITY, L = 0.f;
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int k = c_first; k <= c_last; ++k) {
                        const float* pr = a.part + ((long long)k * 2 + (k == c_first ? 1 : 0)) * stride;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + ROWS * HD) + row);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(pr + row * HD + c));
                        const float mn = fmaxf(M, ml.x), mm = mn == -INFINITY ? 0.f : mn;
                        const float al = kd_exp2(M - mm), be = kd_exp2(ml.x - mm);
                        M = mn;
                        L = L * al + ml.y * be;
                        sum.x = sum.x * al + v.x * be;
                        sum.y = sum.y * al + v.y * be;
                        sum.z = sum.z * al + v.z * be;
                        sum.w = sum.w * al + v.w * be;
                    }
                    float* s4 = s_slab + row * S::SLAB + c;
                    s4[0] = sum.x, s4[1] = sum.y, s4[2] = sum.z, s4[3] = sum.w;
                    if (c == 0) {
                        s_ml[row] = make_float2(M, L);
#pragma unroll
                        for (int w = 1; w < KD_WARPS; ++w) s_ml[w * ROWS + row] = make_float2(-INFINITY, 0.f);
                    }
                }
                named_bar_sync(1, 32 * KD_WARPS);
            }
        }
        if (write) {
            for (int i = warp; i < rows; i += KD_WARPS) {
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, s_ml[w * ROWS + i].x);
#pragma unroll
                for (int w = 0; w < KD_WARPS; ++w) {
                    const float2 v = s_ml[w * ROWS + i];
                    L += v.y * kd_exp2(v.x - (M == -INFINITY ? 0.f : M));
                }
                const int tok = q.start + (row0 + i) / a.G, head = h * a.G + (row0 + i) % a.G;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                for (int c = lane; c < HD; c += 32)
                    kv8_st1(a.out, tok * a.out_stride + (long long)head * HD + channel(c), a.type, s_slab[i * S::SLAB + c] * inv);
                if (a.lse && lane == 0)
                    a.lse[(long long)tok * a.n_q_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945f;
            }
        }
        named_bar_sync(1, 32 * KD_WARPS);
        cur = unit0 + KD_UNIT + first + cnt;
    }
    if (a.behind_prefill) pdl_wait();
}

}  // namespace fence
