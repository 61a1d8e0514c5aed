// paged_plan.cu — fence_paged_plan: one step's block tables, slot map, positions and page list from the
// requests' lengths, in one launch and without the host.
//
// The plan is three prefix sums over the requests (new tokens, pages needed, pages given back) and a
// fourth over the placed ones (pages that get tokens); everything else is a function of them:
//   page j that the call hands out = stack[avail - 1 - j], stack = free pages, then the ended requests' pages
//   token t belongs to the last request whose start is <= t; its page is its table's entry, or if the
//   call has just handed it out, page N_r + (pos / P - held) of the call.
// What bounds it is latency: the launch, the lengths' load, the scans, one dependent load of a page id
// (6.5 us alone for 48 requests, 13.5 us for 2000 requests with 46 thousand tokens, cold caches).
// So every CTA repeats the scans for itself in shared memory (at most 4096 requests: 16 KB of lengths
// from L2) and then writes its share of the outputs; nothing waits on another CTA, and no CTA reads what
// another one writes: table entries below `held`, free pages below n_free and the ended requests' rows
// are only read, new entries and pages above n_free only written.
#include "kv8.cuh"

namespace fence {

struct PlanArgs {
    fence_paged_batch b;
    int shift;  // log2(page_tokens)
};

// Inclusive scan of one value per thread over the CTA (at most 1024 threads); total in *sum.
__device__ __forceinline__ long long plan_scan(long long v, long long* s_warp, long long* sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();  // s_warp may still be read from the scan before
    if (lane == 31) s_warp[w] = v;
    __syncthreads();
    if (w == 0) {
        long long x = lane < nw ? s_warp[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += u;
        }
        s_warp[lane] = x;
    }
    __syncthreads();
    *sum = s_warp[31];
    return v + (w ? s_warp[w - 1] : 0);
}
__device__ __forceinline__ int plan_clip(long long v) { return (int)min(v, (long long)INT_MAX); }
// The last i in [0, n) with a[i] <= v, for a[0] = 0 <= v and a ascending.
__device__ __forceinline__ int plan_find(const int* a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void paged_plan_kernel(const PlanArgs p) {
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ int s_mem[];
    __shared__ long long s_warp[32];
    __shared__ int s_used;
    const fence_paged_batch& b = p.b;
    const int n = b.n_req, sh = p.shift, P = b.page_tokens, MP = b.max_pages;
    int* s_start = s_mem;             // [n + 1] first token
    int* s_need = s_start + n + 1;    // [n + 1] pages handed out before this request
    int* s_back = s_need + n + 1;     // [n + 1] pages given back before it
    int* s_touch = s_back + n + 1;    // [n + 1] pages with new tokens before it
    int* s_ctx = s_touch + n + 1;     // [n] tokens in the cache before the step
    int* s_kv = s_ctx + n;            // [n] with the step's; 0 not placed
    const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
    const int r0 = min(n, (int)threadIdx.x * per), r1 = min(n, r0 + per);

    int n_free = *b.n_free;
    if (n_free < 0 || n_free > b.n_pages) {
        if (threadIdx.x == 0) set_device_error(KV8_BAD);
        n_free = max(0, min(n_free, b.n_pages));
    }
    if (threadIdx.x == 0) s_used = 0;
    long long t_new = 0, t_need = 0, t_back = 0;
    for (int r = r0; r < r1; ++r) {
        const int ctx = max(0, b.ctx_len[r]), raw = b.new_len[r], nw = max(0, raw);
        const long long both = (long long)ctx + nw;
        const bool fits = both <= (long long)MP << sh;
        const int held = (int)(((long long)ctx + P - 1) >> sh);
        const int need = raw >= 0 && fits ? (int)((both + P - 1) >> sh) - held : 0;
        const int back = raw < 0 ? min(held, MP) : 0;
        if (blockIdx.x == 0 && (b.ctx_len[r] < 0 || held > MP)) set_device_error(KV8_BAD);  // taken as 0; not placed
        s_ctx[r] = ctx;
        s_start[r] = nw;
        s_need[r] = need;
        s_back[r] = back;
        s_kv[r] = raw >= 0 && fits ? (int)both : -1;
        t_new += nw;
        t_need += need;
        t_back += back;
    }
    long long all_new, all_need, all_back;
    long long e_new = plan_scan(t_new, s_warp, &all_new) - t_new;
    long long e_need = plan_scan(t_need, s_warp, &all_need) - t_need;
    long long e_back = plan_scan(t_back, s_warp, &all_back) - t_back;
    if (threadIdx.x == 0 && blockIdx.x == 0 && (all_new > b.n_tokens || n_free + all_back > b.n_pages))
        set_device_error(KV8_BAD);
    const int n_back = (int)min(all_back, (long long)(b.n_pages - n_free));
    const int avail = n_free + n_back;
    long long t_touch = 0;
    int used = 0;
    for (int r = r0; r < r1; ++r) {
        const int nw = s_start[r], need = s_need[r], back = s_back[r];
        s_start[r] = plan_clip(e_new);
        s_need[r] = plan_clip(e_need);
        s_back[r] = plan_clip(e_back);
        const bool placed = s_kv[r] >= 0 && (need == 0 || e_need + need <= avail);
        const int ctx = s_ctx[r], kv = placed ? s_kv[r] : 0;
        s_kv[r] = kv;
        if (placed && need > 0) used = (int)(e_need + need);
        const int touched = placed && nw > 0 ? ((kv - 1) >> sh) - (ctx >> sh) + 1 : 0;
        s_touch[r] = touched;
        t_touch += touched;
        e_new += nw;
        e_need += need;
        e_back += back;
        if (blockIdx.x == 0) {
            const int raw = b.new_len[r];
            b.ctx_out[r] = raw < 0 ? 0 : placed ? kv : ctx;
            b.kv_len[r] = kv;
            b.new_start[r] = s_start[r];
        }
    }
    if (used) atomicMax(&s_used, used);
    long long all_touch;
    long long e_touch = plan_scan(t_touch, s_warp, &all_touch) - t_touch;
    for (int r = r0; r < r1; ++r) {
        const int c = s_touch[r];
        s_touch[r] = plan_clip(e_touch);
        e_touch += c;
    }
    if (threadIdx.x == 0) {
        s_start[n] = plan_clip(all_new);
        s_need[n] = plan_clip(all_need);
        s_back[n] = plan_clip(all_back);
        s_touch[n] = plan_clip(all_touch);
    }
    __syncthreads();
    used = s_used;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        b.new_start[n] = s_start[n];
        *b.n_free_out = avail - used;
    }

    auto stack_at = [&](int i) -> int {  // i < avail
        if (i < n_free) return b.free_pages[i];
        const int k = i - n_free, r = plan_find(s_back, n, k);
        return b.block_table[(size_t)r * MP + (k - s_back[r])];
    };
    // page id of position pos of the placed request r
    auto page_of = [&](int r, int pos) -> int {
        const int j = pos >> sh, held = (s_ctx[r] + P - 1) >> sh;
        return j < held ? b.block_table[(size_t)r * MP + j] : stack_at(avail - 1 - (s_need[r] + j - held));
    };
    const int g0 = blockIdx.x * blockDim.x + threadIdx.x, gs = gridDim.x * blockDim.x;
    const int total = s_start[n];
    for (int t = g0; t < b.n_tokens; t += gs) {
        int pos = -1, slot = -1;
        if (t < total) {
            const int r = plan_find(s_start, n, t);
            if (s_kv[r] > 0) {
                pos = s_ctx[r] + t - s_start[r];
                slot = (page_of(r, pos) << sh) + (pos & (P - 1));
            }
        }
        b.slot[t] = slot;
        b.pos[t] = pos;
    }
    const int n_touch = s_touch[n];
    for (int u = g0; u < b.n_touch; u += gs) {
        int4 e = make_int4(-1, 0, 0, 0);
        if (u < n_touch) {
            const int r = plan_find(s_touch, n, u);
            const int ctx = s_ctx[r], j = (ctx >> sh) + u - s_touch[r];
            const int lo = max(ctx, j << sh), hi = min(s_kv[r], (j + 1) << sh);
            e = make_int4(page_of(r, lo), lo & (P - 1), s_start[r] + lo - ctx, hi - lo);
        }
        reinterpret_cast<int4*>(b.touch)[u] = e;
    }
    for (int j = g0; j < used; j += gs) {  // the pages handed out, into their tables
        const int r = plan_find(s_need, n, j);
        b.block_table[(size_t)r * MP + ((s_ctx[r] + P - 1) >> sh) + (j - s_need[r])] = stack_at(avail - 1 - j);
    }
    for (int i = g0; i < n_back - used; i += gs)  // the ended requests' pages that stay free
        b.free_pages[n_free + i] = stack_at(n_free + i);
}

static int ilog2(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

int kv8_check_cache(const fence_kv8_cache* c, const char* who) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale)
        return set_error(FENCE_E_ARG, "%s: null cache or cache pointer", who);
    if (c->n_pages <= 0 || c->n_kv_heads <= 0)
        return set_error(FENCE_E_ARG, "%s: n_pages %d, n_kv_heads %d", who, c->n_pages, c->n_kv_heads);
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        return set_error(FENCE_E_UNSUPPORTED, "%s: page_tokens %d not in {16,32,64,128}", who, c->page_tokens);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(FENCE_E_UNSUPPORTED, "%s: head_dim %d not in {64,128,256}", who, c->head_dim);
    if (c->format != KV8_INT8 && c->format != KV8_E4M3)
        return set_error(FENCE_E_UNSUPPORTED, "%s: code format %d", who, c->format);
    if ((long long)c->n_pages * c->page_tokens * c->n_kv_heads > INT_MAX)
        return set_error(FENCE_E_UNSUPPORTED, "%s: more than 2^31 - 1 rows in the pool", who);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return set_error(FENCE_E_ALIGN, "%s: codes must be 16-byte aligned", who);
    return FENCE_OK;
}

int kv8_check_batch(const fence_paged_batch* b, const fence_kv8_cache* c, const char* who) {
    if (!b) return set_error(FENCE_E_ARG, "%s: null batch", who);
    if (b->n_req <= 0 || b->n_tokens < 0 || b->max_pages <= 0 || b->n_pages <= 0)
        return set_error(FENCE_E_ARG, "%s: n_req %d, n_tokens %d, max_pages %d, n_pages %d", who, b->n_req, b->n_tokens,
                         b->max_pages, b->n_pages);
    if (b->n_req > FENCE_PAGED_MAX_REQ)
        return set_error(FENCE_E_UNSUPPORTED, "%s: %d requests, at most %d", who, b->n_req, FENCE_PAGED_MAX_REQ);
    if (b->page_tokens != 16 && b->page_tokens != 32 && b->page_tokens != 64 && b->page_tokens != 128)
        return set_error(FENCE_E_UNSUPPORTED, "%s: page_tokens %d not in {16,32,64,128}", who, b->page_tokens);
    if ((long long)b->max_pages * b->page_tokens > INT_MAX / 2 || (long long)b->n_pages * b->page_tokens > INT_MAX)
        return set_error(FENCE_E_UNSUPPORTED, "%s: positions or slots past 31 bits", who);
    if (c && (b->page_tokens != c->page_tokens || b->n_pages != c->n_pages))
        return set_error(FENCE_E_ARG, "%s: batch and cache differ: page_tokens %d / %d, n_pages %d / %d", who,
                         b->page_tokens, c->page_tokens, b->n_pages, c->n_pages);
    return FENCE_OK;
}

}  // namespace fence

extern "C" int fence_paged_plan(const fence_paged_batch* b, fence_stream_t stream) {
    using namespace fence;
    if (int e = kv8_check_batch(b, nullptr, "paged_plan")) return e;
    if (!b->ctx_len || !b->new_len || !b->block_table || !b->free_pages || !b->n_free || !b->n_free_out || !b->ctx_out ||
        !b->kv_len || !b->new_start || (b->n_tokens > 0 && (!b->slot || !b->pos || !b->touch)))
        return set_error(FENCE_E_ARG, "paged_plan: null pointer");
    if (b->ctx_out == b->ctx_len || b->kv_len == b->ctx_len || b->n_free_out == b->n_free || b->ctx_out == b->new_len ||
        b->kv_len == b->new_len)
        return set_error(FENCE_E_ARG, "paged_plan: an output is also an input");
    const long long want = b->n_tokens < 2LL * b->n_req + b->n_tokens / b->page_tokens
                               ? b->n_tokens : 2LL * b->n_req + b->n_tokens / b->page_tokens;
    if (b->n_touch < want) return set_error(FENCE_E_ARG, "paged_plan: n_touch %d, needs %lld", b->n_touch, want);
    if (reinterpret_cast<uintptr_t>(b->touch) & 15)
        return set_error(FENCE_E_ALIGN, "paged_plan: touch must be 16-byte aligned");
    PlanArgs p{*b, ilog2(b->page_tokens)};
    const int threads = b->n_req <= 512 ? 256 : 1024;
    long long work = b->n_tokens > b->n_pages ? b->n_tokens : b->n_pages;
    const int cap = threads == 256 ? 296 : 148;
    int grid = (int)((work + threads - 1) / threads);
    grid = grid < 1 ? 1 : grid > cap ? cap : grid;
    const int smem = (6 * b->n_req + 4) * (int)sizeof(int);
    // a launch may use 48 KB without asking, the kernel's own arrays among them (48880 bytes were refused): ask well before
    if (smem > 32 * 1024)
        FENCE_CUDA_TRY(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (6 * FENCE_PAGED_MAX_REQ + 4) * (int)sizeof(int)));
    return cuda_status(kv8_launch(paged_plan_kernel, dim3((unsigned)grid), threads, smem, (cudaStream_t)stream, p), "paged_plan");
}
