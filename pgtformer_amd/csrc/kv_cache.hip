// Key / value cache in 8 bits: quantise tokens as they are written, read them back.
//
// A page holds `page` tokens of every kv head.  Per (page, head) K and V each have one scale 2^e, e the least exponent in [-32, 32] with
// max |x| <= 448 * 2^e over the finite x, and codes e4m3(x * 2^-e): with a power of two the product is exact, so the code is the one rounding there is
// (half a step, 2^-4 of the value above 2^-6 * 2^e), and a page that later receives a larger token is re-expressed exactly but for what
// falls under the new scale's smallest normal number.  A mantissa in the scale would gain nothing: the step of a floating-point
// code is relative.  Infinities and NaN do not count for the scale (one infinity would take e to 32 and its page's other tokens to zero): infinities, as
// values beyond 448 * 2^32, become +-448 * 2^e, NaN stays NaN.
//
// Layouts are the operand order of the attention that reads them (16 bytes = what one lane feeds to two matrix instructions):
//   K (pages, kv, hd / 16, page, 16): 16 dims of one token          V (pages, kv, page / 16, hd, 16): 16 tokens of one dim
//
// One workgroup per (page, head, K | V), 32 elements per thread: a maximum over the new tokens, then the codes.  K: two runs of 16 dims
// of a token; V: 16 tokens x 2 dims, transposed in registers.
// Much at once - 16396 tokens of 8 heads of 64 in half, 50 MB each way - is bound by the start and end of 7392 short workgroups: append 18 us (2.8
// TB/s; they live some 6 us each, with K and V in one workgroup the same), read 14 (3.5; a copy: 5.1).  A token for each of 48 sequences: 5.8 and
// 4.6 us, the chain of index, scale and data loads.
#include <cfloat>

#include "kv_common.h"
#include "pgt_internal.h"

namespace {

constexpr int E_MIN = -32, E_MAX = 32;

// least e in [E_MIN, E_MAX] with amax <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, E_MIN), E_MAX);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= FLT_MAX ? a : 0.f;
}
__device__ __forceinline__ float clamp_to(float v, float top) { return v > top ? top : (v < -top ? -top : v); }      // NaN passes
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void value4(uint32_t w, float* f) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
__device__ __forceinline__ void value16(const uint4& w, float* f) {
    value4(w.x, f); value4(w.y, f + 4); value4(w.z, f + 8); value4(w.w, f + 12);
}
__device__ __forceinline__ uint4 code16(const float* f, float inv) {
    return make_uint4(code4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), code4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv),
                      code4(f[8] * inv, f[9] * inv, f[10] * inv, f[11] * inv), code4(f[12] * inv, f[13] * inv, f[14] * inv, f[15] * inv));
}
template <typename T> __device__ __forceinline__ void ld16(const T* p, float* f) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) Vec16<T>::unpack(reinterpret_cast<const uint4*>(p)[i], f + i * N);
}
template <typename T> __device__ __forceinline__ void st16(T* p, const float* f) {
    if constexpr (__is_same(T, float)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store4(p + 4 * i, f + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<uint4*>(p)[i] = make_uint4(pair_of<T>(f[8 * i], f[8 * i + 1]), pair_of<T>(f[8 * i + 2], f[8 * i + 3]),
                                                        pair_of<T>(f[8 * i + 4], f[8 * i + 5]), pair_of<T>(f[8 * i + 6], f[8 * i + 7]));
    }
}
template <typename T> __device__ __forceinline__ void ld2(const T* p, float& a, float& b) {
    if constexpr (__is_same(T, float)) {
        const float2 w = *reinterpret_cast<const float2*>(p);
        a = w.x; b = w.y;
    } else if constexpr (__is_same(T, bf16_t)) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u);
    } else {
        const halfx2 w = __builtin_bit_cast(halfx2, *reinterpret_cast<const uint32_t*>(p));
        a = (float)w.x; b = (float)w.y;
    }
}

struct KvP {
    const void *k, *v;              // append: new rows; read: unused
    void *ko, *vo;                  // read: output rows
    uint8_t *kp, *vp;
    float *ks, *vs;
    const int32_t *table, *lens, *cu;
    int64_t ldk, ldv;               // row strides (read: of the outputs)
    int pages, kv, hd, pshift, ldt, width, B, rows, per_seq, npg;
};

// what the workgroup works on: sequence b, its packed rows, page `idx` of the sequence, or nothing
struct Spot {
    bool any;
    int row0, t_lo, t_hi, half, head;      // token t of the page is packed row row0 + (t - t_off)
    int t_off;
    size_t id;
};
__device__ __forceinline__ Spot find(const KvP& p) {
    Spot s;
    // pages first, then sequences, then heads: 16396 tokens 19 us, with the heads first 23
    const int pages = p.npg * p.B, hh = blockIdx.x / pages, w = blockIdx.x - hh * pages;
    s.half = hh & 1; s.head = hh >> 1;
    const int b = w / p.npg, pi = w - b * p.npg;
    const int page = 1 << p.pshift;
    int r0, n;
    if (p.cu) {
        r0 = min(max(p.cu[b], 0), p.rows);
        n = min(max(p.cu[b + 1], r0), p.rows) - r0;
        n = min(n, p.per_seq);
    } else {
        r0 = b * p.per_seq;
        n = p.per_seq;
    }
    const int64_t len = max(p.lens[b], 0);
    const int64_t cap = (int64_t)p.width << p.pshift;
    const int64_t idx = (len >> p.pshift) + pi, base = idx << p.pshift;
    const int64_t lo = max(len, base), hi = min(min(len + n, cap), base + page);
    s.any = false;
    if (lo >= hi) return s;
    const int id = p.table[(size_t)b * p.ldt + idx];
    if (id < 0 || id >= p.pages) return s;
    s.any = true;
    s.id = id;
    s.row0 = r0;
    s.t_lo = (int)(lo - base);
    s.t_hi = (int)(hi - base);
    s.t_off = (int)(len - base);      // may be negative: the sequence's first row lies in an earlier page
    return s;
}

template <typename T> __global__ __launch_bounds__(512) void kv_append_kernel(const KvP p) {
    __shared__ uint32_t wmax[8];
    const Spot s = find(p);
    if (!s.any) return;
    const int tid = threadIdx.x, page = 1 << p.pshift, hd = p.hd, nch = hd >> 4, nthr = page * hd >> 5;
    const bool active = tid < nthr;
    const size_t base = (s.id * p.kv + s.head) * (size_t)(page * hd);
    float* scale = (s.half ? p.vs : p.ks) + s.id * p.kv + s.head;
    const bool fresh = s.t_lo == 0;      // no earlier token in the page
    uint8_t* dst = (s.half ? p.vp : p.kp) + base;
    const T* src = (const T*)(s.half ? p.v : p.k) + s.head * hd;
    const int64_t ld = s.half ? p.ldv : p.ldk;
    float f[32];
    uint32_t top = 0;      // bits of the largest |x|: not below infinity's if there is one, or a NaN
    // K: units tid, tid + nthr of (token, 16 dims); V: one unit of (16 tokens, 2 dims)
    const int blk = tid / (hd >> 1), d0 = 2 * (tid % (hd >> 1));
#pragma unroll
    for (int e = 0; e < 32; ++e) f[e] = 0.f;
    if (active && s.half == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = tid + i * nthr, t = u / nch, c = u % nch;
            if (t >= s.t_lo && t < s.t_hi) ld16(src + (s.row0 + t - s.t_off) * ld + c * 16, f + 16 * i);
        }
    } else if (active) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int t = blk * 16 + e;
            if (t >= s.t_lo && t < s.t_hi) ld2(src + (s.row0 + t - s.t_off) * ld + d0, f[e], f[16 + e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
    const float was = *scale;      // read before the barrier, written behind it
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((tid & 63) == 0) wmax[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < ((int)blockDim.x + 63) >> 6; ++w) top = max(top, wmax[w]);
    const bool rare = top > __float_as_uint(448.f * 0x1p32f);      // something saturates, is infinite or NaN
    if (rare) {
        float am = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) am = fmaxf(am, finite_abs(f[e]));
        am = wave_max(am);
        __syncthreads();
        if ((tid & 63) == 0) wmax[tid >> 6] = __float_as_uint(am);
        __syncthreads();
        top = 0;
        for (int w = 0; w < ((int)blockDim.x + 63) >> 6; ++w) top = max(top, wmax[w]);
    }
    int e = scale_exponent(__uint_as_float(top));
    const int e_old = min(max((int)((__float_as_uint(was) >> 23) & 255) - 127, E_MIN), E_MAX);
    if (!fresh) e = max(e, e_old);
    const bool grew = !fresh && e > e_old;
    const float inv = pow2(-e), back = pow2(e_old - e);
    if (rare) {
#pragma unroll
        for (int k = 0; k < 32; ++k) f[k] = clamp_to(f[k], 448.f * pow2(e));
    }
    if (tid == 0 && (fresh || grew)) *scale = pow2(e);
    if (!active) return;
    if (s.half == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = tid + i * nthr, t = u / nch, c = u % nch;
            uint4* o = reinterpret_cast<uint4*>(dst) + c * page + t;
            if (t >= s.t_lo && t < s.t_hi) *o = code16(f + 16 * i, inv);
            else if (t < s.t_lo) {
                if (grew) {
                    float g[16];
                    value16(*o, g);
                    *o = code16(g, back);
                }
            } else if (fresh) *o = make_uint4(0, 0, 0, 0);
        }
    } else {
        const int t0 = blk * 16;
        if (t0 >= s.t_hi && !fresh) return;
        if (t0 + 16 <= s.t_lo && !grew) return;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint4* o = reinterpret_cast<uint4*>(dst) + blk * hd + d0 + j;
            uint4 w = code16(f + 16 * j, inv);
            if (!fresh && (t0 < s.t_lo || t0 + 16 > s.t_hi)) {      // tokens of the block that stay
                const uint4 was4 = *o;
                uint4 old = was4;
                if (grew) {
                    float g[16];
                    value16(was4, g);
                    old = code16(g, back);
                }
                uint32_t ow[4] = {old.x, old.y, old.z, old.w}, aw[4] = {was4.x, was4.y, was4.z, was4.w}, nw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t r = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int t = t0 + 4 * q + b;
                        const uint32_t from = t < s.t_lo ? ow[q] : (t < s.t_hi ? nw[q] : aw[q]);
                        r |= from & (0xffu << (8 * b));
                    }
                    nw[q] = r;
                }
                w = make_uint4(nw[0], nw[1], nw[2], nw[3]);
            }
            *o = w;
        }
    }
}

template <typename T> __global__ __launch_bounds__(512) void kv_read_kernel(const KvP p) {
    int w = blockIdx.x;
    const int half = w & 1; w >>= 1;
    const int head = w % p.kv; w /= p.kv;
    const int pi = w % p.npg, b = w / p.npg;
    const int tid = threadIdx.x, page = 1 << p.pshift, hd = p.hd, nch = hd >> 4, nthr = page * hd >> 5;
    if (tid >= nthr) return;
    int r0, n;
    if (p.cu) {
        r0 = min(max(p.cu[b], 0), p.rows);
        n = min(max(p.cu[b + 1], r0), p.rows) - r0;
        n = min(n, p.per_seq);
    } else {
        r0 = b * p.per_seq;
        n = p.per_seq;
    }
    const int64_t len = max(p.lens[b], 0);
    const int64_t idx = (len >> p.pshift) + pi, off = len - (idx << p.pshift);
    const int t_lo = (int)max(off, (int64_t)0), t_hi = (int)min(off + n, (int64_t)page);
    if (t_lo >= t_hi) return;
    const int id = idx < p.width ? p.table[(size_t)b * p.ldt + idx] : -1;
    const bool have = id >= 0 && id < p.pages;      // tokens that the cache does not hold read as zeros
    const size_t base = have ? ((size_t)id * p.kv + head) * (size_t)(page * hd) : 0;
    const float sc = have ? (half ? p.vs : p.ks)[(size_t)id * p.kv + head] : 0.f;
    const uint4* src = reinterpret_cast<const uint4*>((half ? p.vp : p.kp) + base);
    T* dst = (T*)(half ? p.vo : p.ko) + head * hd;
    const int64_t ld = half ? p.ldv : p.ldk;
    if (half == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = tid + i * nthr, t = u / nch, c = u % nch;
            if (t < t_lo || t >= t_hi) continue;
            float f[16];
            value16(have ? src[c * page + t] : make_uint4(0, 0, 0, 0), f);
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] *= sc;
            st16(dst + (r0 + t - off) * ld + c * 16, f);
        }
    } else {
        const int blk = tid / (hd >> 1), d0 = 2 * (tid % (hd >> 1)), t0 = blk * 16;
        if (t0 >= t_hi || t0 + 16 <= t_lo) return;
        float f[32];
        value16(have ? src[blk * hd + d0] : make_uint4(0, 0, 0, 0), f);
        value16(have ? src[blk * hd + d0 + 1] : make_uint4(0, 0, 0, 0), f + 16);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int t = t0 + e;
            if (t >= t_lo && t < t_hi) store2(dst + (r0 + t - off) * ld + d0, f[e] * sc, f[16 + e] * sc);
        }
    }
}

int check(const char* what, int dtype, const KvP& p, int page, const void* a, const void* b, int lda, int ldb) {
    PGT_CHECK(dtype == PGT_F32 || dtype == PGT_BF16 || dtype == PGT_F16, "%s: bad dtype %d", what, dtype);
    PGT_CHECK(p.pshift > 0, "%s: page=%d unsupported (16, 32, 64, 128)", what, page);
    PGT_CHECK(p.hd == 64 || p.hd == 128, "%s: head_dim=%d unsupported (64, 128)", what, p.hd);
    PGT_CHECK(p.kv > 0 && p.kv <= 65536 && p.pages > 0 && p.B >= 0 && p.rows >= 0 && p.per_seq >= 0 && p.width >= 0 && p.ldt >= p.width,
              "%s: kv_heads=%d pages=%d B=%d rows=%d tokens per sequence=%d table width=%d", what, p.kv, p.pages, p.B, p.rows, p.per_seq, p.width);
    PGT_CHECK(p.kp && p.vp && p.ks && p.vs, "%s: null cache", what);
    PGT_CHECK((((uintptr_t)p.kp | (uintptr_t)p.vp) & 15) == 0, "%s: misaligned cache", what);
    if (p.B == 0 || p.rows == 0 || p.per_seq == 0) return 0;
    PGT_CHECK(a && b && p.lens && (p.width == 0 || p.table), "%s: null argument", what);
    PGT_CHECK(p.cu || (int64_t)p.B * p.per_seq <= p.rows, "%s: %d sequences of %d tokens in %d rows", what, p.B, p.per_seq, p.rows);
    const int al = dtype == PGT_F32 ? 4 : 8;
    PGT_CHECK(lda >= p.kv * p.hd && ldb >= p.kv * p.hd && lda % al == 0 && ldb % al == 0,
              "%s: row strides must cover kv_heads * head_dim and be multiples of 16 bytes", what);
    PGT_CHECK((((uintptr_t)a | (uintptr_t)b) & 15) == 0, "%s: misaligned pointer", what);
    return 0;
}
// workgroups of a launch: every page that `per_seq` tokens can touch, each kv head, K and V; 0 = does not fit a grid, whose threads are counted in 32 bits
unsigned threads(const KvP& p) { return max((p.hd << p.pshift) / 32, 64); }
unsigned groups(KvP& p) {
    const int64_t page = 1 << p.pshift;
    p.npg = (int)((p.per_seq + 2 * page - 2) / page);
    const int64_t g = (int64_t)p.B * p.npg * p.kv * 2;
    return g < (1LL << 31) && g * threads(p) < (1LL << 32) ? (unsigned)g : 0;
}

}  // namespace

extern "C" int pgt_kv_append(int32_t dtype, const void* k, int32_t ldk, const void* v, int32_t ldv, void* k_pages, void* v_pages,
                             float* k_scale, float* v_scale, int32_t pages, int32_t page, int32_t kv_heads, int32_t hd,
                             const int32_t* table, int32_t ld_table, int32_t width, const int32_t* lens, const int32_t* cu, int32_t B,
                             int32_t rows, int32_t max_new, pgt_stream_t stream) {
    KvP p = {};
    p.k = k; p.v = v; p.kp = (uint8_t*)k_pages; p.vp = (uint8_t*)v_pages; p.ks = k_scale; p.vs = v_scale;
    p.table = table; p.lens = lens; p.cu = cu; p.ldk = ldk; p.ldv = ldv; p.pages = pages; p.kv = kv_heads; p.hd = hd;
    p.pshift = kv_page_shift(page); p.ldt = ld_table; p.width = width; p.B = B; p.rows = rows; p.per_seq = max_new;
    if (const int rc = check("kv_append", dtype, p, page, k, v, ldk, ldv)) return rc;
    if (B == 0 || rows == 0 || max_new == 0 || width == 0) return 0;
    const unsigned g = groups(p);
    PGT_CHECK(g, "kv_append: %d sequences of up to %d tokens each exceed one launch", B, max_new);
    const dim3 blk(threads(p));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PGT_F32) hipLaunchKernelGGL(kv_append_kernel<float>, dim3(g), blk, 0, st, p);
    else if (dtype == PGT_BF16) hipLaunchKernelGGL(kv_append_kernel<bf16_t>, dim3(g), blk, 0, st, p);
    else hipLaunchKernelGGL(kv_append_kernel<half_t>, dim3(g), blk, 0, st, p);
    PGT_LAUNCH_CHECK();
    return 0;
}

extern "C" int pgt_kv_read(int32_t dtype, void* k_out, int32_t ldk, void* v_out, int32_t ldv, const void* k_pages, const void* v_pages,
                           const float* k_scale, const float* v_scale, int32_t pages, int32_t page, int32_t kv_heads, int32_t hd,
                           const int32_t* table, int32_t ld_table, int32_t width, const int32_t* start, const int32_t* cu, int32_t B,
                           int32_t rows, int32_t max_rows, pgt_stream_t stream) {
    KvP p = {};
    p.ko = k_out; p.vo = v_out; p.kp = (uint8_t*)k_pages; p.vp = (uint8_t*)v_pages; p.ks = (float*)k_scale; p.vs = (float*)v_scale;
    p.table = table; p.lens = start; p.cu = cu; p.ldk = ldk; p.ldv = ldv; p.pages = pages; p.kv = kv_heads; p.hd = hd;
    p.pshift = kv_page_shift(page); p.ldt = ld_table; p.width = width; p.B = B; p.rows = rows; p.per_seq = max_rows;
    if (const int rc = check("kv_read", dtype, p, page, k_out, v_out, ldk, ldv)) return rc;
    if (B == 0 || rows == 0 || max_rows == 0) return 0;
    const unsigned g = groups(p);
    PGT_CHECK(g, "kv_read: %d sequences of up to %d tokens each exceed one launch", B, max_rows);
    const dim3 blk(threads(p));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PGT_F32) hipLaunchKernelGGL(kv_read_kernel<float>, dim3(g), blk, 0, st, p);
    else if (dtype == PGT_BF16) hipLaunchKernelGGL(kv_read_kernel<bf16_t>, dim3(g), blk, 0, st, p);
    else hipLaunchKernelGGL(kv_read_kernel<half_t>, dim3(g), blk, 0, st, p);
    PGT_LAUNCH_CHECK();
    return 0;
}
