// kv8_store.cu — fence_kv8_store and fence_kv8_load: rows into and out of the paged 8-bit cache.
#include "kv8.cuh"

namespace fence {

struct StoreArgs {
    fence_kv8_cache c;
    const int4* touch;
    int n_tokens;
    const void* x[2];  // k, v
    long long stride[2];
    int type, wide[2];
};

constexpr int KV8_ST_THREADS = 128;

// One CTA per touched page, KV head and K or V. Pass 1: the largest |x| of the new rows, as the largest
// bit pattern of |x| (so that NaN wins over everything). Then the page's scale, the older rows if it
// grew, and the new rows' codes.
template <int FMT>
__global__ void __launch_bounds__(KV8_ST_THREADS) kv8_store_kernel(const StoreArgs a) {
    const int4 e = a.touch[blockIdx.x];  // page, first row, first token, rows
    if (e.x < 0) return;
    const int P = a.c.page_tokens, hd = a.c.head_dim, h = blockIdx.y, kv = blockIdx.z, cpr = hd / 8;
    if (e.x >= a.c.n_pages || e.y < 0 || e.w < 0 || e.y + e.w > P || e.z < 0 || e.z > a.n_tokens - e.w) {
        if (threadIdx.x == 0) set_device_error(KV8_BAD);
        return;
    }
    const void* x = a.x[kv];
    const bool wide = a.wide[kv];
    const long long unit = (long long)e.x * a.c.n_kv_heads + h;
    uint8_t* codes = static_cast<uint8_t*>(kv ? a.c.v : a.c.k) + unit * P * hd;
    float* scale = (kv ? a.c.v_scale : a.c.k_scale) + unit;
    const float s0 = e.y > 0 ? *scale : 0.f;

    uint32_t m = 0;
    for (int i = threadIdx.x; i < e.w * cpr; i += KV8_ST_THREADS) {
        float v[8];
        kv8_ld8(x, (e.z + i / cpr) * a.stride[kv] + h * hd + (i % cpr) * 8, a.type, wide, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    __shared__ uint32_t s_m[KV8_ST_THREADS / 32];
    if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KV8_ST_THREADS / 32; ++w) m = max(m, s_m[w]);
    float s1 = __uint_as_float(m) * kv8_limit_inv<FMT>();
    if (s1 < 1.17549435e-38f) s1 = 0.f;
    // the bit patterns' order: NaN is the largest, and stays
    const bool grown = (__float_as_uint(s1) & 0x7fffffffu) > (__float_as_uint(s0) & 0x7fffffffu);
    if (!grown) s1 = s0;
    const float inv = s1 > 0.f ? __frcp_rn(s1) : 0.f;
    if (grown) {
        for (int i = threadIdx.x; i < e.y * cpr; i += KV8_ST_THREADS) {
            uint2 w = reinterpret_cast<uint2*>(codes)[i];
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = ((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 0xffu;
                o[j >> 2] |= kv8_code<FMT>(kv8_value<FMT>(c) * s0 * inv) << (8 * (j & 3));
            }
            reinterpret_cast<uint2*>(codes)[i] = make_uint2(o[0], o[1]);
        }
    }
    for (int i = threadIdx.x; i < e.w * cpr; i += KV8_ST_THREADS) {
        float v[8];
        kv8_ld8(x, (e.z + i / cpr) * a.stride[kv] + h * hd + (i % cpr) * 8, a.type, wide, v);
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j >> 2] |= kv8_code<FMT>(v[j] * inv) << (8 * (j & 3));
        reinterpret_cast<uint2*>(codes)[e.y * cpr + i] = make_uint2(o[0], o[1]);
    }
    if (threadIdx.x == 0 && (grown || e.y == 0)) *scale = s1;
}

struct LoadArgs {
    fence_kv8_cache c;
    const int* slot;
    int n, shift;
    void* x[2];
    long long stride[2];
    int type, wide[2];
};

// A thread per 8 codes.
template <int FMT>
__global__ void __launch_bounds__(256) kv8_load_kernel(const LoadArgs a) {
    const int hd = a.c.head_dim, cpr = hd / 8, row = a.c.n_kv_heads * cpr, kv = blockIdx.y;
    if (!a.x[kv]) return;
    const uint8_t* codes = static_cast<const uint8_t*>(kv ? a.c.v : a.c.k);
    const float* scale = kv ? a.c.v_scale : a.c.k_scale;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)a.n * row; i += (long long)gridDim.x * 256) {
        const int t = (int)(i / row), c = (int)(i % row), h = c / cpr, col = (c % cpr) * 8;
        const int slot = a.slot[t], page = slot >> a.shift;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (slot >= 0 && page < a.c.n_pages) {
            const long long unit = (long long)page * a.c.n_kv_heads + h;
            const uint2 w = *reinterpret_cast<const uint2*>(codes + (unit * a.c.page_tokens + (slot & (a.c.page_tokens - 1))) * hd + col);
            const float s = scale[unit];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = kv8_value<FMT>(((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 0xffu) * s;
        } else if (slot != -1) {
            set_device_error(KV8_BAD);
        }
        kv8_st8(a.x[kv], (long long)t * a.stride[kv] + h * hd + col, a.type, a.wide[kv], v);
    }
}

}  // namespace fence

extern "C" int fence_kv8_store(const fence_kv8_cache* c, const fence_paged_batch* b, const void* k, const void* v, int type,
                               long long k_stride, long long v_stride, fence_stream_t stream) {
    using namespace fence;
    if (int e = kv8_check_cache(c, "kv8_store")) return e;
    if (int e = kv8_check_batch(b, c, "kv8_store")) return e;
    if (b->n_tokens == 0 || b->n_touch == 0) return FENCE_OK;
    if (!k || !v || !b->touch || b->n_touch < 0) return set_error(FENCE_E_ARG, "kv8_store: null pointer");
    if (!kv8_type_ok(type)) return set_error(FENCE_E_UNSUPPORTED, "kv8_store: element type %d", type);
    const long long row = (long long)c->n_kv_heads * c->head_dim;
    if (k_stride < row || v_stride < row)
        return set_error(FENCE_E_ARG, "kv8_store: strides %lld, %lld below a row of %lld", k_stride, v_stride, row);
    const uintptr_t es = (uintptr_t)kv8_elem_size(type);
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % es)
        return set_error(FENCE_E_ALIGN, "kv8_store: k and v must be aligned to their elements");
    if (reinterpret_cast<uintptr_t>(b->touch) & 15)
        return set_error(FENCE_E_ALIGN, "kv8_store: touch must be 16-byte aligned");
    if (c->n_kv_heads > 65535) return set_error(FENCE_E_UNSUPPORTED, "kv8_store: %d heads", c->n_kv_heads);
    StoreArgs a{*c, reinterpret_cast<const int4*>(b->touch), b->n_tokens, {k, v}, {k_stride, v_stride}, type,
                {kv8_wide(k, k_stride, type), kv8_wide(v, v_stride, type)}};
    const dim3 grid((unsigned)b->n_touch, (unsigned)c->n_kv_heads, 2);
    if (c->format == KV8_INT8) kv8_store_kernel<KV8_INT8><<<grid, KV8_ST_THREADS, 0, (cudaStream_t)stream>>>(a);
    else kv8_store_kernel<KV8_E4M3><<<grid, KV8_ST_THREADS, 0, (cudaStream_t)stream>>>(a);
    return cuda_status(cudaGetLastError(), "kv8_store");
}

extern "C" int fence_kv8_load(const fence_kv8_cache* c, const int* slot, int n, void* k, void* v, int type, long long k_stride,
                              long long v_stride, fence_stream_t stream) {
    using namespace fence;
    if (int e = kv8_check_cache(c, "kv8_load")) return e;
    if (n < 0 || (n > 0 && (!slot || (!k && !v)))) return set_error(FENCE_E_ARG, "kv8_load: bad arguments (n=%d)", n);
    if (!kv8_type_ok(type)) return set_error(FENCE_E_UNSUPPORTED, "kv8_load: element type %d", type);
    if (n == 0) return FENCE_OK;
    const long long row = (long long)c->n_kv_heads * c->head_dim;
    if ((k && k_stride < row) || (v && v_stride < row))
        return set_error(FENCE_E_ARG, "kv8_load: strides %lld, %lld below a row of %lld", k_stride, v_stride, row);
    const uintptr_t es = (uintptr_t)kv8_elem_size(type);
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % es)
        return set_error(FENCE_E_ALIGN, "kv8_load: k and v must be aligned to their elements");
    LoadArgs a{*c, slot, n, ilog2(c->page_tokens), {k, v}, {k_stride, v_stride}, type,
               {kv8_wide(k, k_stride, type), kv8_wide(v, v_stride, type)}};
    const long long items = (long long)n * c->n_kv_heads * (c->head_dim / 8);
    const long long want = (items + 255) / 256;
    const dim3 grid((unsigned)(want > 148 * 16 ? 148 * 16 : want), 2);
    if (c->format == KV8_INT8) kv8_load_kernel<KV8_INT8><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
    else kv8_load_kernel<KV8_E4M3><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
    return cuda_status(cudaGetLastError(), "kv8_load");
}
