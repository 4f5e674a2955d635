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
// 8 floats as three bf16 planes: hi + mid + lo is the float but for 2^-25 of it
__device__ __forceinline__ void split3(const float* p, uint4& hi, uint4& mid, uint4& lo) {
    float f[8];
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(p + 4);
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = f2bf2(f[2 * e], f[2 * e + 1]);
            x3_opaque(w[e]);
            f[2 * e] -= __uint_as_float(w[e] << 16);
            f[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
        }
        (pl == 0 ? hi : pl == 1 ? mid : lo) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// log2 of a page's scale, a power of two from 2^-32 on (0 - memory that was only cleared - as that: its tokens count as the zeros they are)
__device__ __forceinline__ float log2_scale(float s) { return (float)max((int)((__float_as_uint(s) >> 23) & 255) - 127, -32); }
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
    int pages, pshift, ldt, width, B, rows, max_new, heads, kv, group, causal, window;
    int cshift, nct, wgs, jrows;      // column tiles of 2^cshift, nct per sequence and kv head; workgroups that share the work, 0 = one per
                                      // column tile; rows of a column tile that the join looks at
    float c;                          // scale * log2 e
};

// sequence b: its packed rows (those that are processed: max_new at most), its tokens in the cache (which end with ALL its rows' own) and the position of
// its first row
struct Seq {
    int r0, n, len, p0;
};
__device__ __forceinline__ Seq seq_of(const AttnP& p, int b) {
    Seq s;
    int n = p.max_new;
    if (p.cu) {
        s.r0 = min(max(p.cu[b], 0), p.rows);
        n = min(max(p.cu[b + 1], s.r0), p.rows) - s.r0;
    } else {
        s.r0 = b * p.max_new;
    }
    s.n = min(n, p.max_new);
    s.len = min(max(p.lens[b], 0), p.width << p.pshift);
    s.p0 = s.len - n;
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
__device__ __forceinline__ Seq uni(const Seq& s) { return {uni(s.r0), uni(s.n), uni(s.len), uni(s.p0)}; }
__device__ __forceinline__ void sees_uni(const AttnP& p, int len, int pos, int& lo, int& hi) {
    sees(p, len, pos, lo, hi);
    lo = uni(lo);
    hi = uni(hi);
}

constexpr float NEVER = -3.402823466e38f;      // reference of a query that has seen nothing: below every score, finite (so that NEVER - NEVER is 0)
constexpr int MIN_SHARE = 4;         // tiles of a piece

// Work sharing (wgs > 0).  The tiles of 64 tokens of all segments - (sequence, column tile, kv head), in an order of the kernel's - are one line
// that is cut into wgs equal pieces, whatever the lengths: every workgroup does the same work, and as many run as fit the chip at once.  A
// segment that is cut leaves a partial result per piece - workgroup w and segment e meet in slot w + e, which no other pair has - and the
// join adds them; one that is not is finished where it was computed.  Lengths are only known on the device: each workgroup sums them up.
//   order 0: (sequence, kv head, column tile), neighbours read the same pages       order 1: (sequence, column tile, kv head), one look-up for all heads
struct Segment {
    int b, hk, ct, first, tiles;      // first tile, tiles
    Seq s;
};
__device__ __forceinline__ Segment segment_of(const AttnP& p, int order, int e) {
    Segment g;
    if (order) {
        g.hk = e % p.kv;
        e /= p.kv;
        g.ct = p.nct == 1 ? 0 : e % p.nct;
        g.b = p.nct == 1 ? e : e / p.nct;
    } else {
        g.ct = p.nct == 1 ? 0 : e % p.nct;
        e = p.nct == 1 ? e : e / p.nct;
        g.hk = e % p.kv;
        g.b = e / p.kv;
    }
    const Seq s = g.s = seq_of(p, g.b);
    const int cols = s.n * p.group, c0 = g.ct << p.cshift, cz = min(c0 + (1 << p.cshift), cols) - 1;
    g.first = g.tiles = 0;
    if (c0 < cols) {
        int lo, hi, dummy;
        sees(p, s.len, s.p0 + (c0 == 0 ? 0 : c0 / p.group), lo, dummy);
        sees(p, s.len, s.p0 + (cz == cols - 1 ? s.n - 1 : cz / p.group), dummy, hi);
        g.first = lo >> 6;
        g.tiles = max(((hi + 63) >> 6) - g.first, 0);
    }
    return g;
}
__device__ __forceinline__ Segment uni(const Segment& g) { return {uni(g.b), uni(g.hk), uni(g.ct), uni(g.first), uni(g.tiles), uni(g.s)}; }
// This workgroup's part [pos, end) of the line, the segment e that pos lies in and the line before that; false: nothing (all 64 * W threads;
// red: W + 2 ints).  In order 1 the kv heads of a column tile are counted at once.
template <int W, int ORDER>
__device__ __forceinline__ bool part_of(const AttnP& p, int wg, int& pos, int& end, int& e, int& before, int* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int entries = p.B * p.nct * (ORDER ? 1 : p.kv), mul = ORDER ? p.kv : 1;
    auto units = [&](int i) { return i < entries ? segment_of(p, ORDER, i * mul).tiles * mul : 0; };
    const int mine = units(tid);      // (up to 64 * W entries: looked up once)
    int all = mine;
    for (int i = tid + 64 * W; i < entries; i += 64 * W) all += units(i);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
    if (lane == 0) red[wave] = all;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) total += red[w];
    total = uni(total);
    const int share = uni(max((total + p.wgs - 1) / p.wgs, MIN_SHARE));
    pos = wg * share;
    end = min(pos + share, total);
    if (pos >= end) return false;
    int run = 0;
    for (int c = 0; c < entries; c += 64 * W) {
        const int u = c == 0 ? mine : units(c + tid);
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
    e = uni(red[W]) * mul;
    before = uni(red[W + 1]);
    __syncthreads();
    return true;
}

}  // namespace

// kv_attention_rows.hip: column tiles of 256, fp32 at hd 64 only; p is an AttnP
int pgt_kv_attention_rows_launch(const void* p, int dtype, int hd, unsigned groups, hipStream_t st);
