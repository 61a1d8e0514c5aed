// kv8.cuh — the paged 8-bit KV cache: what its kernels share. Pages of page_tokens positions, codes
// [n_pages][n_kv_heads][page_tokens][head_dim] one byte each, a float scale per page and head.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "host.h"

namespace fence {

constexpr int KV8_INT8 = FENCE_KV8_INT8, KV8_E4M3 = FENCE_KV8_E4M3;
constexpr int KV8_BAD = FENCE_E_ARG;  // the device error word for lengths, pages or slots out of range

// The largest code, and its reciprocal: a page's scale is its largest |x| times the reciprocal.
template <int FMT>
__host__ __device__ constexpr float kv8_limit_inv() {
    return FMT == KV8_INT8 ? (float)(1.0 / 127.0) : (float)(1.0 / 448.0);
}

// Code of y = x / scale, to nearest, ties to even; NaN gives 0.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_code(float y) {
    if (FMT == KV8_INT8) {
        const int c = __float2int_rn(y);  // NaN: 0
        return (uint32_t)max(-127, min(127, c)) & 0xffu;
    }
    return y != y ? 0u : (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
// Codes of two values, the first in the low byte.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_code2(float a, float b) {
    if (FMT == KV8_INT8) return kv8_code<FMT>(a) | (kv8_code<FMT>(b) << 8);
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a != a ? 0.f : a, b != b ? 0.f : b), __NV_SATFINITE, __NV_E4M3);
}
template <int FMT>
__device__ __forceinline__ float kv8_value(uint32_t code) {
    if (FMT == KV8_INT8) return (float)(int8_t)code;
    // sign, exponent (bias 7) and mantissa moved to fp16's places (bias 15): 2^8 too small, subnormals too
    const uint32_t h = ((code & 0x80u) << 8) | ((code & 0x7fu) << 7);
    return half_bits_to_float(h) * 256.f;
}

// two codes (bytes lo and lo + 1 of w) -> two fp16, exactly
template <int FMT>
__device__ __forceinline__ uint32_t kd_half2(uint32_t w, bool high) {
    if (FMT == KV8_INT8) {
        // w holds code + 128: bytes beside 0x64 are the fp16 numbers 1024 + byte; less 1152
        const uint32_t x = __byte_perm(w, 0x64646464u, high ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    uint32_t h;
    if (high) asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, u;\n\t}" : "=r"(h) : "r"(w));
    else asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(h) : "r"(w));
    return h;
}
template <int FMT>
__device__ __forceinline__ uint32_t kd_bias(uint32_t w) { return FMT == KV8_INT8 ? w ^ 0x80808080u : w; }

// 8 consecutive elements of a row of activations, raw: 16 bytes of 16-bit types, 32 of floats (WIDE: the row is 16-byte aligned),
// and their values.
template <int TYPE, bool WIDE>
__device__ __forceinline__ void kv8_raw8(const void* base, long long i, uint32_t (&w)[TYPE == FENCE_F32 ? 8 : 4]) {
    if (TYPE == FENCE_F32) {
        const uint32_t* p = static_cast<const uint32_t*>(base) + i;
        if (WIDE) {
            const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4);
            constexpr int O = TYPE == FENCE_F32 ? 4 : 0;
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[O] = b.x, w[O + 1] = b.y, w[O + 2] = b.z, w[O + 3] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < (TYPE == FENCE_F32 ? 8 : 4); ++j) w[j] = p[j];
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + i;
        if (WIDE) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (uint32_t)p[2 * j] | ((uint32_t)p[2 * j + 1] << 16);
        }
    }
}
template <int TYPE>
__device__ __forceinline__ float kv8_elem(const uint32_t (&w)[TYPE == FENCE_F32 ? 8 : 4], int j) {  // j a constant
    if (TYPE == FENCE_F32) return __uint_as_float(w[TYPE == FENCE_F32 ? j : 0]);
    const uint32_t x = w[TYPE == FENCE_F32 ? 0 : j >> 1];
    if (TYPE == FENCE_F16) return half_bits_to_float(j & 1 ? x >> 16 : x);
    return __uint_as_float(j & 1 ? x & 0xffff0000u : x << 16);
}
__device__ __forceinline__ uint32_t kv8_pack2(float a, float b, int type) {
    if (type == FENCE_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void kv8_st8(void* base, long long i, int type, bool wide, const float (&x)[8]) {
    if (type == FENCE_F32) {
        float* p = static_cast<float*>(base) + i;
        if (wide) {
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = x[j];
        }
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = kv8_pack2(x[2 * j], x[2 * j + 1], type);
    uint16_t* p = static_cast<uint16_t*>(base) + i;
    if (wide) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[2 * j] = (uint16_t)w[j];
            p[2 * j + 1] = (uint16_t)(w[j] >> 16);
        }
    }
}
__device__ __forceinline__ void kv8_st1(void* base, long long i, int type, float x) {
    if (type == FENCE_F32) static_cast<float*>(base)[i] = x;
    else if (type == FENCE_F16) static_cast<__half*>(base)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// Launches with programmatic stream serialization: the kernel's launch and set-up overlap the end of the kernel before it.
// Every kernel launched so waits for that one (pdl_wait) before it touches global memory, so the order is the stream's.
template <typename... P, typename... A>
inline cudaError_t kv8_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

inline int kv8_elem_size(int type) { return type == FENCE_F32 ? 4 : 2; }
// whether every row of a [rows][stride] buffer that starts at a multiple of 8 elements is 16-byte aligned
inline bool kv8_wide(const void* p, long long stride, int type) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * kv8_elem_size(type)) % 16 == 0;
}
inline bool kv8_type_ok(int type) { return type == FENCE_F32 || type == FENCE_F16 || type == FENCE_BF16; }

// Checks what every call needs of a cache. Returns 0 or a status with the message set.
int kv8_check_cache(const fence_kv8_cache* c, const char* who);
// Checks a batch against the cache (null: the plan's own call).
int kv8_check_batch(const fence_paged_batch* b, const fence_kv8_cache* c, const char* who);

}  // namespace fence
