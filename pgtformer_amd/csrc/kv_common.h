// Shared by the cached-attention kernels (qk_rope.hip, kv_cache.hip, kv_attention.hip).
#pragma once
#include "common.h"

// fp32 -> half, saturating at +-65504 as every half store of this library, but NaN stays NaN (v_med3_f32 would give -65504)
__device__ __forceinline__ float clamp_half(float v) { return v > 65504.f ? 65504.f : (v < -65504.f ? -65504.f : v); }
__device__ __forceinline__ uint32_t half2_of(float a, float b) { return f2h2_nosat(clamp_half(a), clamp_half(b)); }
// {a, b} in the 16-bit type T
template <typename T> __device__ __forceinline__ uint32_t pair_of(float a, float b) {
    if constexpr (__is_same(T, bf16_t)) return f2bf2(a, b);
    else return half2_of(a, b);
}
template <typename T> __device__ __forceinline__ void store2(T* p, float a, float b) {
    if constexpr (__is_same(T, float)) *reinterpret_cast<float2*>(p) = make_float2(a, b);
    else *reinterpret_cast<uint32_t*>(p) = pair_of<T>(a, b);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float* f) {
    if constexpr (__is_same(T, float)) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pair_of<T>(f[0], f[1]), pair_of<T>(f[2], f[3]));
}

template <typename T> __device__ __forceinline__ void store_nan(T* p) {      // T: bf16_t, half_t
    *reinterpret_cast<uint16_t*>(p) = 0x7fff;                                 // a NaN in both
}

// log2 of a page's number of tokens, -1 if it is none of 16, 32, 64, 128
static inline int kv_page_shift(int page) {
    for (int s = 4; s <= 7; ++s)
        if (page == 1 << s) return s;
    return -1;
}
