// Shared by the two kernels of the attention over the 8-bit cache: kv_attention.hip (few query rows) and kv_attention_rows.hip (many).
#pragma once
#include "kv_common.h"

namespace {

// 8 e4m3 codes -> 8 halves / bf16, exact
__device__ __forceinline__ uint4 half8(uint32_t a, uint32_t b) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true)));
}
__device__ __forceinline__ uint4 bfloat8(uint32_t a, uint32_t b) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true)));
}
__device__ __forceinline__ f32x4 mma_h(const uint4& a, const uint4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_b(const uint4& a, const uint4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// 16 bytes of the cache.  ONCE: with the streaming policy (7.1 instead of 6.3 TB/s on a plain read of 2 GiB), for launches in which no other
// workgroup reads them (with it, 1024 query rows over the same pages took 1.5 times as long)
template <bool ONCE> __device__ __forceinline__ uint4 load16(const uint8_t* p) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4* q = reinterpret_cast<const u32x4*>(p);
    if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(q));
    else return __builtin_bit_cast(uint4, *q);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// does any of the four codes stand for NaN (0x7f, 0xff)?
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

struct AttnP {
    const void* q;
    void* out;
    const uint8_t *kp, *vp;
    const float *ks, *vs;
    const int32_t *table, *lens, *cu;
    float *po, *pml;                  // partial results: (slot, columns, hd), (slot, columns, {m, l})
    int64_t ldq, ldo;
    int pages, pshift, ldt, width, B, rows, max_new, heads, kv, group, cshift, nct, wgs, causal, window;      // column tiles of 2^cshift; wgs: workgroups that share the work, 0 = one per column tile
    float c;                          // scale * log2 e
};

// sequence b: its packed rows and its tokens in the cache (which end with the rows' own)
struct Seq {
    int r0, n, len;
};
__device__ __forceinline__ Seq seq_of(const AttnP& p, int b) {
    Seq s;
    if (p.cu) {
        s.r0 = min(max(p.cu[b], 0), p.rows);
        s.n = min(min(max(p.cu[b + 1], s.r0), p.rows) - s.r0, p.max_new);
    } else {
        s.r0 = b * p.max_new;
        s.n = p.max_new;
    }
    const int64_t cap = min((int64_t)p.width << p.pshift, (int64_t)0x7fffff00);
    s.len = (int)min((int64_t)max(p.lens[b], 0), cap);
    return s;
}
// tokens [lo, hi) that the query at position pos (of a sequence of len tokens) sees
__device__ __forceinline__ void sees(const AttnP& p, int len, int pos, int& lo, int& hi) {
    lo = 0;
    hi = len;
    if (p.causal) {
        const uint32_t end = ((uint32_t)max(pos, 0) / (uint32_t)p.causal + 1) * (uint32_t)p.causal;      // < 2^32: pos + causal at most
        hi = (int)min(end, (uint32_t)len);
        if (p.window) lo = (int)min(end > (uint32_t)p.window ? end - (uint32_t)p.window : 0u, (uint32_t)len);
    }
    if (pos < 0) hi = 0;      // more rows than tokens: nothing to see
    lo = min(lo, hi);
}

constexpr int MIN_SHARE = 4;      // tiles of a piece: one per wave of a workgroup with few rows

// Work sharing (wgs > 0).  The tiles of 64 tokens of all (sequence, kv head, column tile) in this order are one line that is cut into wgs equal
// pieces, whatever the lengths: every workgroup streams the same number of bytes, and as many run as fit the chip at once.  A column tile
// that is cut leaves a partial result per piece - workgroup w and column tile i meet in slot w + i, which no other pair has - and the join
// adds them.  Lengths are only known on the device: each workgroup sums them up.
struct Line {
    int total, share;
};
// tiles of each column tile of sequence b (the range that its first to last query see), and its column tiles
__device__ __forceinline__ int seq_tiles(const AttnP& p, const Seq& s, int& first, int& nct) {
    int lo, hi, dummy;
    sees(p, s.len, s.len - s.n, lo, dummy);
    sees(p, s.len, s.len - 1, dummy, hi);
    first = lo >> 6;
    nct = (s.n * p.group + (1 << p.cshift) - 1) >> p.cshift;
    return s.n > 0 ? max(((hi + 63) >> 6) - first, 0) : 0;
}
__device__ __forceinline__ int seq_units(const AttnP& p, int b) {
    int first, nct;
    const int t = seq_tiles(p, seq_of(p, b), first, nct);
    return t * nct * p.kv;
}
__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// the whole line, and the part of it before sequence b (all 64 * W threads; red: 2 * W ints)
template <int W> __device__ __forceinline__ Line line_of(const AttnP& p, int b, int& before, int* red) {
    int all = 0, pre = 0;
    for (int i = threadIdx.x; i < p.B; i += 64 * W) {
        const int u = seq_units(p, i);
        all += u;
        if (i < b) pre += u;
    }
    all = wave_sum_i(all);
    pre = wave_sum_i(pre);
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = all;
        red[W + (threadIdx.x >> 6)] = pre;
    }
    __syncthreads();
    Line l;
    l.total = before = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        l.total += red[w];
        before += red[W + w];
    }
    l.share = max((l.total + p.wgs - 1) / p.wgs, MIN_SHARE);
    return l;
}
// the sequence that place `pos` of the line lies in, and the line before it
template <int W> __device__ __forceinline__ void locate(const AttnP& p, int pos, int& b, int& before, int* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int run = 0;
    for (int c = 0; c < p.B; c += 64 * W) {
        const int u = c + tid < p.B ? seq_units(p, c + tid) : 0;
        int v = u;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int w = __shfl_up(v, o, 64);
            if (lane >= o) v += w;
        }
        __syncthreads();
        if (lane == 63) red[wave] = v;
        __syncthreads();
        int e = run + v - u;
        for (int w = 0; w < wave; ++w) e += red[w];
        if (pos >= e && pos < e + u) {
            red[W] = c + tid;
            red[W + 1] = e;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) run += red[w];
        if (run > pos) break;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(red[W]);
    before = __builtin_amdgcn_readfirstlane(red[W + 1]);
    __syncthreads();
}

}  // namespace

// kv_attention_rows.hip: bf16 / half, column tiles of 256; p is an AttnP
int pgt_kv_attention_rows_launch(const void* p, int bf16, int hd, unsigned groups, hipStream_t st);
