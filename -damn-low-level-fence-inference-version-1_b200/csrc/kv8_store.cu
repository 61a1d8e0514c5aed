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

constexpr int KV8_ST_CHUNKS = 8;  // of 8 elements, at most, per thread: a page of one head stays in the CTA's registers

// One CTA per touched page, KV head and K or V: the largest |x| of the new rows, as the largest bit
// pattern of |x| (so that NaN wins over everything), then the page's scale, the older rows if it grew, and
// the new rows' codes. Bound: HBM, each element read once and its code written once; all of a thread's
// loads are in flight together and the rows stay in registers between the two steps (read twice, in
// loops, 8000 rows of 8 x 128 bf16 took 23 us; so 12.4, against 7.6 us of traffic). Threads: the page's elements / 64, 128 to 512.
template <int FMT, int TYPE, bool WIDE>
__global__ void __launch_bounds__(512) kv8_store_kernel(const StoreArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int4 e = a.touch[blockIdx.x];  // page, first row, first token, rows
    if (e.x < 0) return;
    const int P = a.c.page_tokens, hd = a.c.head_dim, h = blockIdx.y, kv = blockIdx.z, cpr = hd / 8, shift = 31 - __clz(cpr);
    if (e.x >= a.c.n_pages || e.y < 0 || e.w < 0 || e.y + e.w > P || e.z < 0 || e.z > a.n_tokens - e.w) {
        if (threadIdx.x == 0) set_device_error(KV8_BAD);
        return;
    }
    const void* x = a.x[kv];
    const long long unit = (long long)e.x * a.c.n_kv_heads + h, stride = a.stride[kv];
    uint8_t* codes = static_cast<uint8_t*>(kv ? a.c.v : a.c.k) + unit * P * hd;
    float* scale = (kv ? a.c.v_scale : a.c.k_scale) + unit;
    const float s0 = e.y > 0 ? *scale : 0.f;
    const int n = e.w << shift, nt = (int)blockDim.x;

    uint32_t w[KV8_ST_CHUNKS][TYPE == FENCE_F32 ? 8 : 4];
#pragma unroll
    for (int j = 0; j < KV8_ST_CHUNKS; ++j) {
        const int i = (int)threadIdx.x + j * nt;
#pragma unroll
        for (int k = 0; k < (TYPE == FENCE_F32 ? 8 : 4); ++k) w[j][k] = 0;
        if (j * nt < n && i < n) kv8_raw8<TYPE, WIDE>(x, (e.z + (i >> shift)) * stride + h * hd + (i & (cpr - 1)) * 8, w[j]);
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < KV8_ST_CHUNKS; ++j)
        if (j * nt < n) {  // the same for all threads: one row costs one round
#pragma unroll
            for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(kv8_elem<TYPE>(w[j], k)) & 0x7fffffffu);
        }
    m = __reduce_max_sync(0xffffffffu, m);
    __shared__ uint32_t s_m[16];
    if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int k = 0; k < nt >> 5; ++k) m = max(m, s_m[k]);
    float s1 = __uint_as_float(m) * kv8_limit_inv<FMT>();
    if (s1 < 1.17549435e-38f) s1 = 0.f;
    // the bit patterns' order: NaN is the largest, and stays
    const bool grown = (__float_as_uint(s1) & 0x7fffffffu) > (__float_as_uint(s0) & 0x7fffffffu);
    if (!grown) s1 = s0;
    const float inv = s1 > 0.f ? __frcp_rn(s1) : 0.f;
    if (grown) {
        for (int i = threadIdx.x; i < e.y << shift; i += nt) {
            const uint2 c = reinterpret_cast<uint2*>(codes)[i];
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j >> 2] |= kv8_code<FMT>(kv8_value<FMT>(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xffu) * s0 * inv) << (8 * (j & 3));
            reinterpret_cast<uint2*>(codes)[i] = make_uint2(o[0], o[1]);
        }
    }
#pragma unroll
    for (int j = 0; j < KV8_ST_CHUNKS; ++j) {
        const int i = (int)threadIdx.x + j * nt;
        if (j * nt < n && i < n) {
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                o[k >> 2] |= kv8_code2<FMT>(kv8_elem<TYPE>(w[j], k) * inv, kv8_elem<TYPE>(w[j], k + 1) * inv) << (8 * (k & 3));
            reinterpret_cast<uint2*>(codes)[(e.y << shift) + i] = make_uint2(o[0], o[1]);
        }
    }
    if (threadIdx.x == 0 && (grown || e.y == 0)) *scale = s1;
}

struct LoadArgs {
    fence_kv8_cache c;
    const int* slot;
    int n, shift, rows;  // rows: per block
    void* x[2];
    long long stride[2];
    int type, wide[2];
};

// A block takes whole rows, about 256 x KV8_LD_ITEMS pieces of 8 codes; a thread's loads are in flight together and a warp's
// stores fill whole lines. Bound: HBM (one byte in, one element out): 8000 rows of 8 x 128 to bf16 16.1 us against 7.6 us of
// traffic, the rest the chain slot, page, codes.
constexpr int KV8_LD_ITEMS = 4;
template <int FMT>
__global__ void __launch_bounds__(256) kv8_load_kernel(const LoadArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int hd = a.c.head_dim, cpr = hd / 8, row = a.c.n_kv_heads * cpr, kv = blockIdx.y, shift = 31 - __clz(cpr);
    if (!a.x[kv]) return;
    const uint8_t* codes = static_cast<const uint8_t*>(kv ? a.c.v : a.c.k);
    const float* scale = kv ? a.c.v_scale : a.c.k_scale;
    const int t0 = blockIdx.x * a.rows, n = min(a.rows, a.n - t0) * row;
    for (int base = (int)threadIdx.x; base < n; base += 256 * KV8_LD_ITEMS) {
        uint2 w[KV8_LD_ITEMS];
        float s[KV8_LD_ITEMS];
        int t[KV8_LD_ITEMS], c[KV8_LD_ITEMS];
#pragma unroll
        for (int j = 0; j < KV8_LD_ITEMS; ++j) {
            const int i = base + j * 256, q = i / row;
            t[j] = q;
            c[j] = i - q * row;
            w[j] = make_uint2(0, 0);
            s[j] = 0.f;
            if (i < n) {
                const int slot = a.slot[t0 + q], page = slot >> a.shift, h = c[j] >> shift;
                if (slot >= 0 && page < a.c.n_pages) {
                    const long long unit = (long long)page * a.c.n_kv_heads + h;
                    w[j] = *reinterpret_cast<const uint2*>(codes + (unit * a.c.page_tokens + (slot & (a.c.page_tokens - 1))) * hd +
                                                           (c[j] & (cpr - 1)) * 8);
                    s[j] = scale[unit];
                } else if (slot != -1) {
                    set_device_error(KV8_BAD);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < KV8_LD_ITEMS; ++j) {
            if (base + j * 256 >= n) continue;
            float v[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t b = kd_bias<FMT>(k ? w[j].y : w[j].x), lo = kd_half2<FMT>(b, false), hi = kd_half2<FMT>(b, true);
                v[4 * k] = half_bits_to_float(lo) * s[j];
                v[4 * k + 1] = half_bits_to_float(lo >> 16) * s[j];
                v[4 * k + 2] = half_bits_to_float(hi) * s[j];
                v[4 * k + 3] = half_bits_to_float(hi >> 16) * s[j];
            }
            kv8_st8(a.x[kv], (long long)(t0 + t[j]) * a.stride[kv] + c[j] * 8, a.type, a.wide[kv], v);
        }
    }
}

template <int FMT, int TYPE>
static cudaError_t kv8_launch_store(const StoreArgs& a, dim3 grid, int threads, cudaStream_t st) {
    if (a.wide[0] && a.wide[1]) return kv8_launch(kv8_store_kernel<FMT, TYPE, true>, grid, threads, 0, st, a);
    return kv8_launch(kv8_store_kernel<FMT, TYPE, false>, grid, threads, 0, st, a);
}
template <int FMT>
static cudaError_t kv8_launch_store(const StoreArgs& a, dim3 grid, int threads, cudaStream_t st) {
    if (a.type == FENCE_F32) return kv8_launch_store<FMT, FENCE_F32>(a, grid, threads, st);
    if (a.type == FENCE_F16) return kv8_launch_store<FMT, FENCE_F16>(a, grid, threads, st);
    return kv8_launch_store<FMT, FENCE_BF16>(a, grid, threads, st);
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
    int threads = c->page_tokens * c->head_dim / (8 * KV8_ST_CHUNKS);
    threads = threads < 128 ? 128 : threads;  // at most 128 * 256 / 64 = 512
    const cudaStream_t st = (cudaStream_t)stream;
    return cuda_status(c->format == KV8_INT8 ? kv8_launch_store<KV8_INT8>(a, grid, threads, st)
                                             : kv8_launch_store<KV8_E4M3>(a, grid, threads, st),
                       "kv8_store");
}

extern "C" int fence_kv8_load(const fence_kv8_cache* c, const int* slot, int n, void* k, void* v, int type, long long k_stride,
                              long long v_stride, fence_stream_t stream) {
    using namespace fence;
    if (int e = kv8_check_cache(c, "kv8_load")) return e;
    if (c->n_kv_heads > 65535) return set_error(FENCE_E_UNSUPPORTED, "kv8_load: %d heads", c->n_kv_heads);
    if (n < 0 || (n > 0 && (!slot || (!k && !v)))) return set_error(FENCE_E_ARG, "kv8_load: bad arguments (n=%d)", n);
    if (!kv8_type_ok(type)) return set_error(FENCE_E_UNSUPPORTED, "kv8_load: element type %d", type);
    if (n == 0) return FENCE_OK;
    const long long row = (long long)c->n_kv_heads * c->head_dim;
    if ((k && k_stride < row) || (v && v_stride < row))
        return set_error(FENCE_E_ARG, "kv8_load: strides %lld, %lld below a row of %lld", k_stride, v_stride, row);
    const uintptr_t es = (uintptr_t)kv8_elem_size(type);
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % es)
        return set_error(FENCE_E_ALIGN, "kv8_load: k and v must be aligned to their elements");
    const int pieces = 256 * KV8_LD_ITEMS, per_row = (int)(row / 8), rows = per_row < pieces ? pieces / per_row : 1;
    LoadArgs a{*c, slot, n, ilog2(c->page_tokens), rows, {k, v}, {k_stride, v_stride}, type,
               {kv8_wide(k, k_stride, type), kv8_wide(v, v_stride, type)}};
    const dim3 grid((unsigned)((n + (long long)rows - 1) / rows), 2);
    return cuda_status(kv8_launch(c->format == KV8_INT8 ? kv8_load_kernel<KV8_INT8> : kv8_load_kernel<KV8_E4M3>, grid, 256, 0,
                                  (cudaStream_t)stream, a),
                       "kv8_load");
}
