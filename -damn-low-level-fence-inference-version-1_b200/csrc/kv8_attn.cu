// kv8_attn.cu — fence_kv8_attention: causal grouped-query attention of a ragged batch over the paged
// 8-bit cache.
#include "kv8_prefill.cuh"

namespace fence {

// 2-D codes [n_pages * n_kv_heads * page_tokens][head_dim], box of at most 128 bytes x box_rows, swizzled
static bool kv8_tensor_map(CUtensorMap* tm, const fence_kv8_cache* c, void* base, int box_rows) {
    PFN_cuTensorMapEncodeTiled enc = tg_encode_fn();
    if (!enc) return false;
    const cuuint32_t line = c->head_dim < 128 ? 64 : 128;
    const cuuint64_t dims[2] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->n_pages * c->n_kv_heads * c->page_tokens};
    const cuuint64_t strides[1] = {(cuuint64_t)c->head_dim};
    const cuuint32_t box[2] = {line, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               line == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Sets a kernel's dynamic shared memory limit once per device.
template <typename F>
static cudaError_t kv8_opt_in(F kern, int bytes, int (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        done[dev] = 1;
    }
    return cudaSuccess;
}

constexpr int KV8_SMS = 148;

template <int FMT, int HD, bool SPLIT, int NT>
static int kv8_launch_decode(const KAttnArgs& p, cudaStream_t st) {
    using S = KDShape<HD, SPLIT, NT>;
    static int done[64] = {};
    CUtensorMap tm_k, tm_v;
    const int box = p.c.page_tokens < KD_TILE ? p.c.page_tokens : KD_TILE;
    if (!kv8_tensor_map(&tm_k, &p.c, p.c.k, box) || !kv8_tensor_map(&tm_v, &p.c, p.c.v, box))
        return set_error(FENCE_E_UNSUPPORTED, "kv8_attention: no tensor map for the cache");
    auto kern = kv8_decode_kernel<FMT, HD, SPLIT, NT>;
    FENCE_CUDA_TRY(kv8_opt_in(kern, S::SMEM + 4 * (FENCE_PAGED_MAX_REQ + 1), done));
    const int smem = S::SMEM + 4 * (p.n_req + 1), fit = 228 * 1024 / (smem + 1024);  // many requests' prefix sums can cost a CTA
    const dim3 grid((unsigned)(KV8_SMS * (fit < S::CTAS ? fit : S::CTAS)));
    return cuda_status(kv8_launch(kern, grid, KD_THREADS, smem, st, p, tm_k, tm_v), "kv8_attention");
}

template <int FMT, int HD, bool SPLIT>
static int kv8_launch_prefill(const KAttnArgs& p, cudaStream_t st) {
    using S = KPShape<HD, SPLIT>;
    static int done[64] = {};
    CUtensorMap tm_q, tm_k, tm_v;
    const int box = p.c.page_tokens < 64 ? p.c.page_tokens : 64;
    if (!kv8_tensor_map(&tm_k, &p.c, p.c.k, box) || !kv8_tensor_map(&tm_v, &p.c, p.c.v, box))
        return set_error(FENCE_E_UNSUPPORTED, "kv8_attention: no tensor map for the cache");
    const long long rows = (long long)p.n_tokens * p.n_q_heads;
    if (!tg_tensor_map(&tm_q, p.q_rows, (int)(rows * (SPLIT ? 2 : 1)), HD, 128))
        return set_error(FENCE_E_UNSUPPORTED, "kv8_attention: no tensor map for the query rows");
    FENCE_CUDA_TRY(kv8_launch(kv8_q_rows_kernel<HD, SPLIT>, dim3((unsigned)((rows + KQ_WARPS - 1) / KQ_WARPS)), 32 * KQ_WARPS, 0, st, p));
    auto kern = kv8_prefill_kernel<FMT, HD, SPLIT>;
    FENCE_CUDA_TRY(kv8_opt_in(kern, S::SMEM, done));
    return cuda_status(kv8_launch(kern, dim3(KP_SMS), KP_THREADS, S::SMEM, st, p, tm_q, tm_k, tm_v), "kv8_attention");
}

constexpr size_t KV8_ARRIVED_BYTES = 4096;  // counters, at the workspace's start: 2048 for each kernel
// The most query rows per KV head of a request that the decode kernel takes (16 in one pass over the keys, more in several).
// Both kernels measured, heads 32/8 of 128, int8, bf16, us (decode / prefill kernel): 16 requests at 8000 keys 137 / 196 with
// 32 rows, 257 / 197 with 64; at 30000 keys 449 / 587 and 881 / 585; one request at 1000 keys 19 / 37 and 20 / 38. The rule
// goes by rows alone, so that the workspace and the launches follow from the shapes on the host: with few keys the prefill
// kernel loses up to those 18 us. Heads of 64 and 256 and fp32 use the same border, unmeasured.
constexpr int KV8_DECODE_ROWS = 48;

// Whether the batch needs the prefill kernel.
static bool kv8_has_prefill(const fence_kv8_cache* c, const fence_kv8_attn* a) {
    // 256 channels of fp32 queries, as pairs, leave no room for the keys there
    return (c->head_dim <= 128 || a->type != FENCE_F32) && (long long)a->max_new * (a->n_q_heads / c->n_kv_heads) > KV8_DECODE_ROWS;
}
// The workspace: counters, the decode kernel's partial results, the prefill kernel's, its query rows and their scales.
static size_t kv8_prefill_part_bytes(const fence_kv8_cache* c) {
    return (size_t)KP_SMS * 4 * 128 * ((c->head_dim < 128 ? c->head_dim : 128) + 2) * sizeof(float);
}
static size_t kv8_q_rows_bytes(const fence_kv8_cache* c, const fence_paged_batch* b, const fence_kv8_attn* a) {
    return ((size_t)b->n_tokens * a->n_q_heads * c->head_dim * 2 * (a->type == FENCE_F32 ? 2 : 1) + 255) & ~(size_t)255;
}
static size_t kv8_decode_part_bytes(const fence_kv8_cache* c) {
    return (size_t)KV8_SMS * 3 * 2 * 16 * (c->head_dim + 2) * sizeof(float);
}

template <int FMT, int HD>
static int kv8_launch_attn(const KAttnArgs& pd, bool split, int nt, bool prefill, char* ws, size_t q_bytes,
                           cudaStream_t st) {
    KAttnArgs p = pd;
    if (prefill) {
        // one request: the prefill kernel takes it whatever its length is
        p.min_rows = p.n_req == 1 ? 0 : KV8_DECODE_ROWS;
        p.arrived = reinterpret_cast<int*>(ws + 2048);
        char* at = ws + KV8_ARRIVED_BYTES + kv8_decode_part_bytes(&p.c);
        p.part = reinterpret_cast<float*>(at);
        at += kv8_prefill_part_bytes(&p.c);
        p.q_rows = reinterpret_cast<__half*>(at);
        p.q_scale = reinterpret_cast<float*>(at + q_bytes);
        int e;
        if constexpr (HD <= 128) e = split ? kv8_launch_prefill<FMT, HD, true>(p, st) : kv8_launch_prefill<FMT, HD, false>(p, st);
        else e = kv8_launch_prefill<FMT, HD, false>(p, st);
        if (e || p.n_req == 1) return e;
        p.max_rows = KV8_DECODE_ROWS;
        p.behind_prefill = 1;
        p.arrived = pd.arrived;
        p.part = pd.part;
    }
    if (split) return nt == 1 ? kv8_launch_decode<FMT, HD, true, 1>(p, st) : kv8_launch_decode<FMT, HD, true, 2>(p, st);
    return nt == 1 ? kv8_launch_decode<FMT, HD, false, 1>(p, st) : kv8_launch_decode<FMT, HD, false, 2>(p, st);
}

static int kv8_attn_check(const fence_kv8_cache* c, const fence_paged_batch* b, const fence_kv8_attn* a, const char* who) {
    if (int e = kv8_check_cache(c, who)) return e;
    if (int e = kv8_check_batch(b, c, who)) return e;
    if (!a) return set_error(FENCE_E_ARG, "%s: null operands", who);
    if (a->n_q_heads <= 0 || a->n_q_heads % c->n_kv_heads)
        return set_error(FENCE_E_ARG, "%s: %d query heads over %d kv heads", who, a->n_q_heads, c->n_kv_heads);
    if (!kv8_type_ok(a->type)) return set_error(FENCE_E_UNSUPPORTED, "%s: element type %d", who, a->type);
    if (!(a->scale >= 0.f && a->scale < INFINITY)) return set_error(FENCE_E_ARG, "%s: scale %g", who, (double)a->scale);
    if ((long long)b->n_tokens * a->n_q_heads > INT_MAX / 2)
        return set_error(FENCE_E_UNSUPPORTED, "%s: more than 2^30 query rows", who);
    if (a->max_new <= 0) return set_error(FENCE_E_ARG, "%s: max_new %d", who, a->max_new);
    return FENCE_OK;
}

}  // namespace fence

extern "C" size_t fence_kv8_attention_workspace_bytes(const fence_kv8_cache* c, const fence_paged_batch* b,
                                                      const fence_kv8_attn* a) {
    using namespace fence;
    if (kv8_attn_check(c, b, a, "kv8_attention_workspace_bytes")) return 0;
    size_t n = KV8_ARRIVED_BYTES + kv8_decode_part_bytes(c);
    if (kv8_has_prefill(c, a))
        n += kv8_prefill_part_bytes(c) + kv8_q_rows_bytes(c, b, a) + (size_t)b->n_tokens * a->n_q_heads * sizeof(float);
    return n;
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
    // a window as long as any request is none; positions less a window (at most 2^30 each) stay within 32 bits
    const int window = a->window > 0 && a->window < (long long)b->max_pages * b->page_tokens ? a->window : 0;
    KAttnArgs p{*c, b->block_table, b->kv_len, b->new_start, b->n_req, b->n_tokens, b->max_pages, ilog2(c->page_tokens),
                a->n_q_heads / c->n_kv_heads, a->n_q_heads, window, a->type, a->q, a->out, a->lse,
                a->q_stride, a->out_stride, (float)(a->scale * 1.4426950408889634), INT_MAX, 0, 0, kv8_wide(a->q, a->q_stride, a->type),
                kv8_wide(a->out, a->out_stride, a->type), nullptr, nullptr, static_cast<int*>(a->workspace),
                reinterpret_cast<float*>(static_cast<char*>(a->workspace) + KV8_ARRIVED_BYTES)};
    const bool split = a->type == FENCE_F32, prefill = kv8_has_prefill(c, a);
    const int nt = (long long)a->max_new * p.G <= 8 ? 1 : 2;
    const cudaStream_t st = (cudaStream_t)stream;
    char* ws = static_cast<char*>(a->workspace);
    const size_t q_bytes = kv8_q_rows_bytes(c, b, a);
    const int kind = (c->format == KV8_E4M3 ? 3 : 0) + (c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2);
    switch (kind) {
        case 0: return kv8_launch_attn<KV8_INT8, 64>(p, split, nt, prefill, ws, q_bytes, st);
        case 1: return kv8_launch_attn<KV8_INT8, 128>(p, split, nt, prefill, ws, q_bytes, st);
        case 2: return kv8_launch_attn<KV8_INT8, 256>(p, split, nt, prefill, ws, q_bytes, st);
        case 3: return kv8_launch_attn<KV8_E4M3, 64>(p, split, nt, prefill, ws, q_bytes, st);
        case 4: return kv8_launch_attn<KV8_E4M3, 128>(p, split, nt, prefill, ws, q_bytes, st);
        default: return kv8_launch_attn<KV8_E4M3, 256>(p, split, nt, prefill, ws, q_bytes, st);
    }
}

