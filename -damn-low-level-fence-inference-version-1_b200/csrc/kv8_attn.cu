// kv8_attn.cu — fence_kv8_attention: causal grouped-query attention of a ragged batch over the paged
// 8-bit cache.
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
};

constexpr int KS_THREADS = 128, KS_G = 8;

// One CTA per (token, KV head): 128 keys at a time, a thread per key for the scores of up to 8 query
// heads, then a thread per output channel for the sum over the keys.
template <int FMT, int HD>
__global__ void __launch_bounds__(KS_THREADS) kv8_attn_simple_kernel(const KAttnArgs a) {
    __shared__ float s_q[KS_G][HD], s_p[KS_G][KS_THREADS], s_red[KS_G][4];
    __shared__ int s_r;
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, P = a.c.page_tokens;
    if (tid == 0) {
        int lo = 0, hi = a.n_req;  // the last request that starts at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.new_start[mid] <= t) lo = mid;
            else hi = mid;
        }
        s_r = lo;
    }
    __syncthreads();
    const int r = s_r, start = a.new_start[r], end = a.new_start[r + 1];
    int kv = a.kv_len[r];
    if (kv < 0 || kv > a.max_pages * P || end > a.n_tokens) {
        if (tid == 0) set_device_error(KV8_BAD);
        kv = max(0, min(kv, a.max_pages * P));
    }
    const int pos = t < end ? kv - (end - start) + (t - start) : -1;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const uint8_t* K = static_cast<const uint8_t*>(a.c.k);
    const uint8_t* V = static_cast<const uint8_t*>(a.c.v);
    for (int g0 = 0; g0 < a.G; g0 += KS_G) {
        const int ng = min(KS_G, a.G - g0);
        __syncthreads();
        for (int i = tid; i < ng * HD; i += KS_THREADS) {
            const long long at = t * a.q_stride + ((long long)h * a.G + g0) * HD + i;
            s_q[i / HD][i % HD] = a.type == FENCE_F32 ? static_cast<const float*>(a.q)[at]
                                  : a.type == FENCE_F16 ? __half2float(static_cast<const __half*>(a.q)[at])
                                                        : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
        }
        __syncthreads();
        float m[KS_G], l[KS_G], o[KS_G][(HD + 127) / 128];
#pragma unroll
        for (int g = 0; g < KS_G; ++g) {
            m[g] = -INFINITY, l[g] = 0.f;
            for (int d = 0; d < (HD + 127) / 128; ++d) o[g][d] = 0.f;
        }
        for (int k0 = first & ~(KS_THREADS - 1); k0 <= pos; k0 += KS_THREADS) {
            const int key = k0 + tid;
            float s[KS_G];
#pragma unroll
            for (int g = 0; g < KS_G; ++g) s[g] = -INFINITY;
            if (key <= pos && key >= first) {
                int page = a.block_table[(size_t)r * a.max_pages + (key >> a.shift)];
                if (page < 0 || page >= a.c.n_pages) {
                    set_device_error(KV8_BAD);
                    page = 0;
                }
                const long long unit = (long long)page * a.c.n_kv_heads + h;
                const uint8_t* row = K + (unit * P + (key & (P - 1))) * HD;
                float acc[KS_G] = {};
                for (int i = 0; i < HD; i += 4) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + i);
                    for (int j = 0; j < 4; ++j) {
                        const float x = kv8_value<FMT>((w >> (8 * j)) & 0xff);
#pragma unroll
                        for (int g = 0; g < KS_G; ++g) acc[g] += x * s_q[g][i + j];
                    }
                }
                const float sc = a.c.k_scale[unit] * a.scale_log2;
#pragma unroll
                for (int g = 0; g < KS_G; ++g) s[g] = acc[g] * sc;
            }
            __syncthreads();
#pragma unroll
            for (int g = 0; g < KS_G; ++g) {
                const float x = warp_max(s[g]);
                if ((tid & 31) == 0) s_red[g][tid >> 5] = x;
            }
            __syncthreads();
#pragma unroll
            for (int g = 0; g < KS_G; ++g) {
                float mn = m[g];
                for (int w = 0; w < 4; ++w) mn = fmaxf(mn, s_red[g][w]);
                const float c = mn == -INFINITY ? 1.f : exp2f(m[g] - mn);
                m[g] = mn;
                l[g] *= c;
                for (int d = 0; d < (HD + 127) / 128; ++d) o[g][d] *= c;
                const bool seen = key <= pos && key >= first;
                s_p[g][tid] = !seen ? 0.f : mn == -INFINITY ? s[g] - s[g] : exp2f(s[g] - mn);
            }
            __syncthreads();
            const int nk = min(KS_THREADS, pos - k0 + 1);
            for (int kk = max(0, first - k0); kk < nk; ++kk) {
                int page = a.block_table[(size_t)r * a.max_pages + ((k0 + kk) >> a.shift)];
                if (page < 0 || page >= a.c.n_pages) page = 0;
                const long long unit = (long long)page * a.c.n_kv_heads + h;
                const float sv = a.c.v_scale[unit];
                for (int d = 0; d < (HD + 127) / 128; ++d) {
                    const int col = tid + d * 128;
                    const float x = col < HD ? kv8_value<FMT>(V[(unit * P + ((k0 + kk) & (P - 1))) * HD + col]) * sv : 0.f;
#pragma unroll
                    for (int g = 0; g < KS_G; ++g) {
                        const float p = s_p[g][kk];
                        if (d == 0) l[g] += p;
                        o[g][d] += p * x;
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int g = 0; g < KS_G; ++g) {
            if (g >= ng) break;
            const int head = h * a.G + g0 + g;
            for (int d = 0; d < (HD + 127) / 128; ++d)
                if (tid + d * 128 < HD)
                    kv8_st1(a.out, t * a.out_stride + (long long)head * HD + tid + d * 128, a.type, pos < 0 ? 0.f : o[g][d] / l[g]);
            if (tid == 0 && a.lse)
                a.lse[(long long)t * a.n_q_heads + head] = pos < 0 ? -INFINITY : (m[g] + log2f(l[g])) * 0.69314718056f;
        }
    }
}

static int kv8_attn_check(const fence_kv8_cache* c, const fence_paged_batch* b, const fence_kv8_attn* a, const char* who) {
    if (int e = kv8_check_cache(c, who)) return e;
    if (int e = kv8_check_batch(b, c, who)) return e;
    if (!a) return set_error(FENCE_E_ARG, "%s: null operands", who);
    if (a->n_q_heads <= 0 || a->n_q_heads % c->n_kv_heads)
        return set_error(FENCE_E_ARG, "%s: %d query heads over %d kv heads", who, a->n_q_heads, c->n_kv_heads);
    if (!kv8_type_ok(a->type)) return set_error(FENCE_E_UNSUPPORTED, "%s: element type %d", who, a->type);
    if (a->max_new <= 0) return set_error(FENCE_E_ARG, "%s: max_new %d", who, a->max_new);
    return FENCE_OK;
}

template <int FMT, int HD>
static int kv8_launch_attn(const KAttnArgs& p, cudaStream_t st) {
    kv8_attn_simple_kernel<FMT, HD><<<dim3((unsigned)p.n_tokens, (unsigned)p.c.n_kv_heads), KS_THREADS, 0, st>>>(p);
    return cuda_status(cudaGetLastError(), "kv8_attention");
}

}  // namespace fence

extern "C" size_t fence_kv8_attention_workspace_bytes(const fence_kv8_cache* c, const fence_paged_batch* b,
                                                      const fence_kv8_attn* a) {
    using namespace fence;
    if (kv8_attn_check(c, b, a, "kv8_attention_workspace_bytes")) return 0;
    return 256;
}

extern "C" int fence_kv8_attention(const fence_kv8_cache* c, const fence_paged_batch* b, const fence_kv8_attn* a,
                                   fence_stream_t stream) {
    using namespace fence;
    if (int e = kv8_attn_check(c, b, a, "kv8_attention")) return e;
    if (b->n_tokens == 0) return FENCE_OK;
    if (!a->q || !a->out || !a->workspace || !b->block_table || !b->kv_len || !b->new_start)
        return set_error(FENCE_E_ARG, "kv8_attention: null pointer");
    const long long row = (long long)a->n_q_heads * c->head_dim;
    if (a->q_stride < row || a->out_stride < row)
        return set_error(FENCE_E_ARG, "kv8_attention: strides %lld, %lld below a row of %lld", a->q_stride, a->out_stride, row);
    const uintptr_t es = (uintptr_t)kv8_elem_size(a->type);
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % es)
        return set_error(FENCE_E_ALIGN, "kv8_attention: q and out must be aligned to their elements");
    if (reinterpret_cast<uintptr_t>(a->workspace) & 255)
        return set_error(FENCE_E_ALIGN, "kv8_attention: workspace must be 256-byte aligned");
    const size_t need = fence_kv8_attention_workspace_bytes(c, b, a);
    if (a->workspace_bytes < need)
        return set_error(FENCE_E_SCRATCH, "kv8_attention: workspace of %zu bytes, needs %zu", a->workspace_bytes, need);
    KAttnArgs p{*c, b->block_table, b->kv_len, b->new_start, b->n_req, b->n_tokens, b->max_pages, ilog2(c->page_tokens),
                a->n_q_heads / c->n_kv_heads, a->n_q_heads, a->window > 0 ? a->window : 0, a->type, a->q, a->out, a->lse,
                a->q_stride, a->out_stride, a->scale * 1.4426950408889634f};
    const cudaStream_t st = (cudaStream_t)stream;
    const int kind = (c->format == KV8_E4M3 ? 3 : 0) + (c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2);
    switch (kind) {
        case 0: return kv8_launch_attn<KV8_INT8, 64>(p, st);
        case 1: return kv8_launch_attn<KV8_INT8, 128>(p, st);
        case 2: return kv8_launch_attn<KV8_INT8, 256>(p, st);
        case 3: return kv8_launch_attn<KV8_E4M3, 64>(p, st);
        case 4: return kv8_launch_attn<KV8_E4M3, 128>(p, st);
        default: return kv8_launch_attn<KV8_E4M3, 256>(p, st);
    }
}
