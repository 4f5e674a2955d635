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

// Loads that write LDS: 64 lanes x 16 (4) bytes from a pointer per lane to dst + lane * 16 (4), dst uniform.  One opaque statement: the compiler
// neither models nor drains the transfer; completion is a counted s_waitcnt vmcnt of the caller's.  ONCE: streaming policy (7.1 instead of
// 6.3 TB/s on a plain read of 2 GiB), for data that no other workgroup of the launch reads (with it, 1024 query rows over the same pages
// took 1.5 times as long).
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
template <bool ONCE = false> __device__ __forceinline__ void lds_load16(const void* src, uint32_t dst) {
    uint32_t m0;
    if constexpr (ONCE)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0) : "v"(src), "s"(dst) : "memory");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0) : "v"(src), "s"(dst) : "memory");
}
__device__ __forceinline__ void lds_load4(const void* src, uint32_t dst) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(src), "s"(dst) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }      // all but the last N
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// log2 of a page's number of tokens, -1 if it is none of 16, 32, 64, 128
static inline int kv_page_shift(int page) {
    for (int s = 4; s <= 7; ++s)
        if (page == 1 << s) return s;
    return -1;
}
