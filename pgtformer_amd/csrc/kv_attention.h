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
    int2* ends;                       // per segment: the workgroups that hold its first and its last piece
    int64_t ldq, ldo;
    int pages, pshift, ldt, width, B, rows, max_new, heads, kv, group, cshift, nct, wgs, jrows, causal, window;      // column tiles of 2^cshift; wgs: workgroups that share the work, 0 = one per
                                      // column tile; jrows: rows of a column tile that the join looks at
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
        const uint32_t at = (uint32_t)max(pos, 0), c = (uint32_t)p.causal;
        const uint32_t end = c == 1 ? at + 1 : (at / c + 1) * c;      // < 2^32: pos + causal at most
        hi = (int)min(end, (uint32_t)len);
        if (p.window) lo = (int)min(end > (uint32_t)p.window ? end - (uint32_t)p.window : 0u, (uint32_t)len);
    }
    if (pos < 0) hi = 0;      // more rows than tokens: nothing to see
    lo = min(lo, hi);
}

// values that every lane of a wave holds alike but that came from memory, into scalar registers
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Seq uni(const Seq& s) { return {uni(s.r0), uni(s.n), uni(s.len)}; }
__device__ __forceinline__ void sees_uni(const AttnP& p, int len, int pos, int& lo, int& hi) {
    sees(p, len, pos, lo, hi);
    lo = uni(lo);
    hi = uni(hi);
}

constexpr float NEVER = -1e30f;      // reference of a query that has seen nothing (finite: differences and products stay numbers)
constexpr int MIN_SHARE = 4;         // tiles of a piece: one per wave of a workgroup with few rows

// Work sharing (wgs > 0).  The tiles of 64 tokens of all segments - (sequence, kv head, column tile), in this order - are one line that is cut
// into wgs equal pieces, whatever the lengths: every workgroup does the same work, and as many run as fit the chip at once.  A segment that
// is cut leaves a partial result per piece - workgroup w and segment e meet in slot w + e, which no other pair has - and the join adds
// them; one that is not is finished where it was computed.  Lengths are only known on the device: each workgroup sums them up.
struct Segment {
    int b, hk, ct, first, tiles;      // first tile, tiles
};
__device__ __forceinline__ Segment segment_of(const AttnP& p, int e) {
    Segment g;
    g.ct = e % p.nct;
    e /= p.nct;
    g.hk = e % p.kv;
    g.b = e / p.kv;
    const Seq s = seq_of(p, g.b);
    const int cols = s.n * p.group, c0 = g.ct << p.cshift, cz = min(c0 + (1 << p.cshift), cols) - 1;
    g.first = g.tiles = 0;
    if (c0 < cols) {
        int lo, hi, dummy;
        sees(p, s.len, s.len - s.n + c0 / p.group, lo, dummy);
        sees(p, s.len, s.len - s.n + cz / p.group, dummy, hi);
        g.first = lo >> 6;
        g.tiles = max(((hi + 63) >> 6) - g.first, 0);
    }
    return g;
}
__device__ __forceinline__ Segment uni(const Segment& g) { return {uni(g.b), uni(g.hk), uni(g.ct), uni(g.first), uni(g.tiles)}; }
__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
struct Line {
    int total, share;
};
// the whole line (all 64 * W threads; red: 2 * W ints)
template <int W> __device__ __forceinline__ Line line_of(const AttnP& p, int* red) {
    const int segs = p.B * p.kv * p.nct;
    int all = 0;
    for (int i = threadIdx.x; i < segs; i += 64 * W) all += segment_of(p, i).tiles;
    all = wave_sum_i(all);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = all;
    __syncthreads();
    Line l;
    l.total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) l.total += red[w];
    l.total = uni(l.total);
    l.share = uni(max((l.total + p.wgs - 1) / p.wgs, MIN_SHARE));
    return l;
}
// the segment that place `pos` of the line lies in, and the line before it
template <int W> __device__ __forceinline__ void locate(const AttnP& p, int pos, int& e, int& before, int* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, segs = p.B * p.kv * p.nct;
    int run = 0;
    for (int c = 0; c < segs; c += 64 * W) {
        const int u = c + tid < segs ? segment_of(p, c + tid).tiles : 0;
        int v = u;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int w = __shfl_up(v, o, 64);
            if (lane >= o) v += w;
        }
        __syncthreads();
        if (lane == 63) red[wave] = v;
        __syncthreads();
        int at = run + v - u;
        for (int w = 0; w < wave; ++w) at += red[w];
        if (pos >= at && pos < at + u) {
            red[W] = c + tid;
            red[W + 1] = at;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) run += red[w];
        if (run > pos) break;
    }
    __syncthreads();
    e = uni(red[W]);
    before = uni(red[W + 1]);
    __syncthreads();
}

}  // namespace

// kv_attention_rows.hip: bf16 / half, column tiles of 256; p is an AttnP
int pgt_kv_attention_rows_launch(const void* p, int bf16, int hd, unsigned groups, hipStream_t st);
