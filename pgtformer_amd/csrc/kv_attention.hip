// Attention over the paged 8-bit key / value cache (kv_cache.hip has the layouts and the scales).
//
//   out = softmax(scale * q K^T) V  per query row, K = ks * k8, V = vs * v8 with one power-of-two scale per page and kv head
//
// A page's scales never touch the elements: with t = (q . k8) * (scale * log2 e * ks) + log2 vs and a running reference m of each
// query, P = 2^(t - m) is the weight of the 8-bit V row, and the softmax sum takes P / vs.  Both products then run on the codes
// themselves, which 16-bit operands hold exactly (e4m3 has 4 significand bits): K in q's type, V in half.
//   P is rounded to half (2^-11; bf16 would leave 2^-8).  m is chosen so that the largest P is between 2^7 and 2^15: what underflows in
//   half is 2^-32 of the largest weight.  fp32 queries: q on three bf16 planes (all 24 bits), P on two half planes (22 bits).
//
// 16x16x32 MFMA, swapped:  S^T = K Q^T (rows = tokens, columns = queries),  O^T += V^T P^T.  A wave takes tiles of 64 tokens = four
// 16-token blocks; the rows of the four S^T tiles are a permutation of the tokens such that the 16 scores a lane ends up with all
// belong to block lane / 16 - one K and one V scale per lane - and are, in order, the 16 tokens that the lane's 16-byte load of V
// holds: P goes from the accumulators into the operand without an exchange, and nothing passes through LDS.
// The query columns are the group's heads times the tokens (column = token * group + head in group).
#include "kv_common.h"
#include "pgt_internal.h"

namespace {

typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

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
    float *po, *pml;                  // partial results of the splits: (slot, split, hd), (slot, split, {m, l})
    int64_t ldq, ldo;
    int pages, pshift, ldt, width, B, rows, max_new, heads, kv, group, nct, nsplit, chunk, causal, window;      // chunk: tiles of 64 tokens per split
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

constexpr int MAX_SPLIT = 256;
constexpr int NW = 4;      // waves per workgroup, each with its own share of the tokens

template <typename T, int HD, bool ONCE> __global__ __launch_bounds__(64 * NW, 2) void kv_attn_kernel(const AttnP p) {
    constexpr bool F32 = __is_same(T, float);
    constexpr bool HQ = __is_same(T, half_t);
    constexpr int QP = F32 ? 3 : 1;          // planes of q
    constexpr int KS = HD / 32;              // k-steps of S^T
    constexpr int ND = HD / 16;              // row tiles of O^T
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int col = lane & 15, g = lane >> 4;
    int id = blockIdx.x;
    const int split = id % p.nsplit; id /= p.nsplit;
    const int ct = id % p.nct; id /= p.nct;
    const int hk = id % p.kv, b = id / p.kv;
    const Seq s = seq_of(p, b);
    const int cols = s.n * p.group;
    if (ct * 16 >= cols) return;
    const int qc = ct * 16 + col;
    const int qi = min(qc, cols - 1) / p.group;
    const int head = hk * p.group + min(qc, cols - 1) % p.group;
    int lo, hi;
    sees(p, s.len, s.len - s.n + qi, lo, hi);
    // what the tile's first and last query see: the range to visit, and the part that every query sees
    int lo_a, hi_a, lo_z, hi_z;
    sees(p, s.len, s.len - s.n + ct * 16 / p.group, lo_a, hi_a);
    sees(p, s.len, s.len - s.n + min(ct * 16 + 15, cols - 1) / p.group, lo_z, hi_z);
    const int t_first = lo_a >> 6, t_end = (hi_z + 63) >> 6;
    const int t0 = t_first + split * p.chunk, te = min(t0 + p.chunk, t_end);
    if (p.nsplit > 1 && t0 >= te) return;      // the join does not look at it

    // Q^T operand: k-step 2 s + h covers dims 64 s + 16 g + 8 h .. + 7 of lane group g - the order of the K loads
    uint4 qf[QP][KS];
#pragma unroll
    for (int st = 0; st < KS; ++st) {
        const int d = 64 * (st >> 1) + 16 * g + 8 * (st & 1);
        const T* qp = (const T*)p.q + (s.r0 + qi) * p.ldq + head * HD + d;
        if constexpr (F32) {
            float f[8];
            *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(qp);
            *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(qp + 4);
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
                qf[pl][st] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            qf[0][st] = *reinterpret_cast<const uint4*>(qp);
        }
    }

    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int page = 1 << p.pshift, kblk = (lane >> 2) & 3;
    const size_t page_bytes = (size_t)page * HD, head_off = (size_t)hk * page_bytes, stride = (size_t)p.kv * page_bytes;
    const int32_t* tab = p.table + (size_t)b * p.ldt;

    // Loads run one tile ahead: K of tile t + NW is issued when the scores of t are done, V when its product is, page numbers two tiles ahead
    struct Page {
        int k, v;      // page of the block whose K rows this lane loads, and of its own block (V, scales)
    };
    auto pages_of = [&](int t) {
        const int ik = (t * 64 + 16 * kblk) >> p.pshift, iv = (t * 64 + 16 * g) >> p.pshift;
        return Page{t < te && ik < p.width ? tab[ik] : -1, t < te && iv < p.width ? tab[iv] : -1};
    };
    uint4 kr[4][HD / 64], vr[ND];
    float sk, sv;
    bool have;
    auto load_k = [&](int t, Page pg) {
        have = pg.v >= 0 && pg.v < p.pages;
        const int idv = have ? pg.v : 0, idk = pg.k >= 0 && pg.k < p.pages ? pg.k : 0;
        sk = p.ks[(size_t)idv * p.kv + hk];
        sv = p.vs[(size_t)idv * p.kv + hk];
        const uint8_t* kb = p.kp + idk * stride + head_off + (((t * 64 + 16 * kblk) & (page - 1)) + (lane & 3)) * 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) kr[r][c] = load16<ONCE>(kb + (size_t)(4 * c + g) * page * 16 + r * 64);
    };
    auto load_v = [&](int t, Page pg) {
        const int idv = pg.v >= 0 && pg.v < p.pages ? pg.v : 0;
        const uint8_t* vb = p.vp + idv * stride + head_off + (size_t)(((t * 64 + 16 * g) & (page - 1)) >> 4) * (HD * 16) + col * 16;
#pragma unroll
        for (int d = 0; d < ND; ++d) vr[d] = load16<ONCE>(vb + d * 256);
    };
    const Page pg = pages_of(t0 + wave);
    Page pn = pages_of(t0 + wave + NW);
    if (t0 + wave < te) {
        load_k(t0 + wave, pg);
        load_v(t0 + wave, pg);
    }
    for (int t = t0 + wave; t < te; t += NW) {
        const int tv = t * 64 + 16 * g;
        const bool more = t + NW < te;
        const Page p2 = pages_of(t + 2 * NW);
        f32x4 x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                const uint4 w = kr[r][c];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 a = HQ ? half8(h ? w.z : w.x, h ? w.w : w.y) : bfloat8(h ? w.z : w.x, h ? w.w : w.y);
#pragma unroll
                    for (int pl = QP - 1; pl >= 0; --pl)
                        x[r] = HQ ? mma_h(a, qf[pl][2 * c + h], x[r]) : mma_b(a, qf[pl][2 * c + h], x[r]);
                }
            }
        }
        const bool here = have;
        const float sk_t = sk, sv_t = sv;
        if (more) load_k(t + NW, pn);
        const float ev = (float)((int)((__float_as_uint(sv_t) >> 23) & 255) - 127), ck = p.c * sk_t;
        const bool masked = t * 64 < lo_z || t * 64 + 64 > hi_a || __any(!here);
        float y[16], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __builtin_fmaf(x[e >> 2][e & 3], ck, ev);
        if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!here || tv + e < lo || tv + e >= hi) y[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, y[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any(mx > m + 15.f)) {      // first tile: m = -inf
            const float mn = mx > m + 15.f ? mx - 7.f : m;      // each query by itself: its result does not depend on its neighbours
            const float al = m == -INFINITY ? 0.f : exp2_(m - mn);
            l *= al;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= al;
            m = mn;
        }
        const float mr = m == -INFINITY ? 0.f : m;      // nothing seen yet: every y is -inf
        float ls = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            y[e] = exp2_(y[e] - mr);
            ls += y[e];
        }
        l += ls * __uint_as_float((uint32_t)(127 - (int)ev) << 23);      // P / vs
        uint4 pf[2], pl2[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = f2h2_nosat(y[8 * h + 2 * e], y[8 * h + 2 * e + 1]);
            pf[h] = make_uint4(w[0], w[1], w[2], w[3]);
            if constexpr (F32) {
                x3_opaque(pf[h]);
                const uint32_t v[4] = {pf[h].x, pf[h].y, pf[h].z, pf[h].w};
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const halfx2 q2 = __builtin_bit_cast(halfx2, v[e]);
                    r[e] = f2h2_nosat(y[8 * h + 2 * e] - (float)q2.x, y[8 * h + 2 * e + 1] - (float)q2.y);
                }
                pl2[h] = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
        if (masked) {
            // 0 * NaN: a V code that stands for NaN must reach the queries that see its token, and only those
            uint32_t any = 0;
#pragma unroll
            for (int d = 0; d < ND; ++d) any |= nan_bytes(vr[d].x) | nan_bytes(vr[d].y) | nan_bytes(vr[d].z) | nan_bytes(vr[d].w);
            if (__any(any != 0)) {
                uint4 see[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t0 = tv + 8 * h + 2 * e;
                        w[e] = (here && t0 >= lo && t0 < hi ? 0x3c00u : 0u) | (here && t0 + 1 >= lo && t0 + 1 < hi ? 0x3c000000u : 0u);
                    }
                    see[h] = make_uint4(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t w[4] = {vr[d].x, vr[d].y, vr[d].z, vr[d].w}, one[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t nb = nan_bytes(w[e]) >> 7;      // 1 per NaN byte
                        w[e] &= ~(nb * 0xffu);
                        one[e] = nb * 0x38u;                            // e4m3 1.0
                    }
                    vr[d] = make_uint4(w[0], w[1], w[2], w[3]);
                    f32x4 cnt = f32x4{0.f, 0.f, 0.f, 0.f};
                    cnt = mma_h(half8(one[0], one[1]), see[0], cnt);
                    cnt = mma_h(half8(one[2], one[3]), see[1], cnt);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (cnt[e] > 0.f) o[d][e] = __builtin_nanf("");
                }
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const uint4 a0 = half8(vr[d].x, vr[d].y), a1 = half8(vr[d].z, vr[d].w);
            if constexpr (F32) {
                o[d] = mma_h(a0, pl2[0], o[d]);
                o[d] = mma_h(a1, pl2[1], o[d]);
            }
            o[d] = mma_h(a0, pf[0], o[d]);
            o[d] = mma_h(a1, pf[1], o[d]);
        }
        if (more) load_v(t + NW, pn);
        pn = p2;
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // join the waves: every one against the common reference
    __shared__ float sm[NW][16], sl[NW][16];
    __shared__ __attribute__((aligned(16))) float so[NW][16][HD + 4];
    if (g == 0) sm[wave][col] = m;
    __syncthreads();
    float mm = sm[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w][col]);
    const float al = m == -INFINITY ? 0.f : exp2_(m - mm);
    if (g == 0) sl[wave][col] = m == -INFINITY ? l : l * al;      // (an all-NaN column keeps its NaN sum)
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        const f32x4 v = m == -INFINITY ? o[d] : o[d] * al;
        *reinterpret_cast<f32x4*>(&so[wave][col][16 * d + 4 * g]) = v;
    }
    __syncthreads();
    // thread: column tid / 16, HD / 16 consecutive dims
    constexpr int PD = HD / 16;
    const int c2 = tid >> 4, d2 = (tid & 15) * PD, qc2 = ct * 16 + c2;
    if (qc2 >= cols) return;
    float f[PD], lt = 0.f;
#pragma unroll
    for (int e = 0; e < PD; ++e) f[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        lt += sl[w][c2];
#pragma unroll
        for (int e = 0; e < PD; ++e) f[e] += so[w][c2][d2 + e];
    }
    const int qi2 = qc2 / p.group, head2 = hk * p.group + qc2 % p.group;
    if (p.nsplit == 1) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;      // a row that sees nothing is zero
        T* op = (T*)p.out + (s.r0 + qi2) * p.ldo + head2 * HD + d2;
#pragma unroll
        for (int e = 0; e < PD; ++e) f[e] = lt == 0.f ? 0.f : f[e] * inv;
#pragma unroll
        for (int e = 0; e < PD; e += 4) store4(op + e, f + e);
    } else {
        const size_t slot = ((size_t)b * p.max_new + qi2) * p.heads + head2;
        float* w = p.po + (slot * p.nsplit + split) * HD + d2;
#pragma unroll
        for (int e = 0; e < PD; ++e) w[e] = f[e];
        if ((tid & 15) == 0) {
            float mm2 = sm[0][c2];
#pragma unroll
            for (int k = 1; k < NW; ++k) mm2 = fmaxf(mm2, sm[k][c2]);
            *reinterpret_cast<float2*>(p.pml + (slot * p.nsplit + split) * 2) = make_float2(mm2, lt);
        }
    }
}

// out = the splits' results against their common reference.  One workgroup per (sequence, token, head): HD / 4 threads hold the row, the
// rest of the 256 take other splits, four loads in flight each.
template <typename T, int HD> __global__ __launch_bounds__(256) void kv_attn_join_kernel(const AttnP p) {
    constexpr int LP = HD / 4, NS = 256 / LP;
    __shared__ float2 ml[MAX_SPLIT];
    __shared__ f32x4 so[NS][LP];
    __shared__ float sm[4], sl[4];
    int id = blockIdx.x;
    const int head = id % p.heads; id /= p.heads;
    const int qi = id % p.max_new, b = id / p.max_new, tid = threadIdx.x;
    const Seq s = seq_of(p, b);
    if (qi >= s.n) return;
    // the splits that hold tokens of this query's column tile
    const int col0 = (qi * p.group + head % p.group) & ~15, colz = min(col0 + 15, s.n * p.group - 1);
    int lo_a, hi_z, dummy;
    sees(p, s.len, s.len - s.n + col0 / p.group, lo_a, dummy);
    sees(p, s.len, s.len - s.n + colz / p.group, dummy, hi_z);
    const int tiles = ((hi_z + 63) >> 6) - (lo_a >> 6), n = tiles > 0 ? (tiles + p.chunk - 1) / p.chunk : 0;
    const size_t slot = ((size_t)b * p.max_new + qi) * p.heads + head;
    const float2 w = tid < n ? reinterpret_cast<const float2*>(p.pml)[slot * p.nsplit + tid] : make_float2(-INFINITY, 0.f);
    float m = wave_max(w.x);
    if ((tid & 63) == 0) sm[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float al = w.x == -INFINITY ? 1.f : exp2_(w.x - m);      // a split that saw nothing holds zeros (or NaN)
    if (tid < n) ml[tid] = make_float2(al, w.y * al);
    const float lw = wave_sum(tid < n ? w.y * al : 0.f);
    if ((tid & 63) == 0) sl[tid >> 6] = lw;
    __syncthreads();
    const float l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    const int c = tid % LP, k = tid / LP;
    const f32x4* po = reinterpret_cast<const f32x4*>(p.po + slot * p.nsplit * HD) + c;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = k; i < n; i += NS) o += po[(size_t)i * LP] * ml[i].x;
    so[k][c] = o;
    __syncthreads();
    if (k) return;
#pragma unroll
    for (int i = 1; i < NS; ++i) o += so[i][c];
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = l == 0.f ? 0.f : o[e] / l;
    store4((T*)p.out + (s.r0 + qi) * p.ldo + head * HD + 4 * c, f);
}

// Splits of the tokens, and tiles of 64 tokens in each: about 1024 workgroups of equal work (ragged lengths: what is past a sequence's
// end exits at once), at least a tile per wave, and one split where the whole length is short
struct Split {
    int n, chunk;
};
Split splits(int B, int max_new, int kv, int group, int width, int pshift, int causal, int window) {
    const int64_t base = (int64_t)B * kv * (((int64_t)max_new * group + 15) / 16);
    int64_t tiles = (((int64_t)width << pshift) + 63) / 64;
    if (causal && window) {      // a column tile's queries lie at most 15 tokens apart
        const int64_t w = ((int64_t)window + causal + 15 + 63) / 64 + 1;
        if (w < tiles) tiles = w;
    }
    if (tiles <= 4 * NW || base <= 0) return {1, (int)(tiles > 0 ? tiles : 1)};
    int64_t chunk = (tiles * base + 1023) / 1024;
    if (chunk < (tiles + MAX_SPLIT - 1) / MAX_SPLIT) chunk = (tiles + MAX_SPLIT - 1) / MAX_SPLIT;
    chunk = (chunk + NW - 1) / NW * NW;
    if (chunk >= tiles) return {1, (int)tiles};
    return {(int)((tiles + chunk - 1) / chunk), (int)chunk};
}

}  // namespace

extern "C" size_t pgt_kv_attention_workspace_bytes(int32_t B, int32_t max_new, int32_t heads, int32_t kv_heads, int32_t hd, int32_t width,
                                                   int32_t page, int32_t causal, int32_t window) {
    if (B <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || hd <= 0 || width <= 0 || kv_page_shift(page) < 0 || heads % kv_heads || causal < 0 || window < 0) return 0;
    const int n = splits(B, max_new, kv_heads, heads / kv_heads, width, kv_page_shift(page), causal, window).n;
    return n == 1 ? 0 : (size_t)B * max_new * heads * n * (hd + 2) * sizeof(float);
}

extern "C" int pgt_kv_attention(int32_t dtype, const void* q, int32_t ldq, const void* k_pages, const void* v_pages, const float* k_scale,
                                const float* v_scale, int32_t pages, int32_t page, int32_t kv_heads, int32_t hd, const int32_t* table,
                                int32_t ld_table, int32_t width, const int32_t* lens, const int32_t* cu, int32_t B, int32_t rows,
                                int32_t max_new, int32_t heads, float scale, int32_t causal, int32_t window, void* out, int32_t ldo,
                                void* workspace, size_t workspace_bytes, pgt_stream_t stream) {
    AttnP p = {};
    p.q = q; p.out = out; p.kp = (const uint8_t*)k_pages; p.vp = (const uint8_t*)v_pages; p.ks = k_scale; p.vs = v_scale;
    p.table = table; p.lens = lens; p.cu = cu; p.ldq = ldq; p.ldo = ldo; p.pages = pages; p.pshift = kv_page_shift(page);
    p.ldt = ld_table; p.width = width; p.B = B; p.rows = rows; p.max_new = max_new; p.heads = heads; p.kv = kv_heads;
    p.causal = causal; p.window = window; p.c = scale * 1.44269504088896340736f;
    PGT_CHECK(dtype == PGT_F32 || dtype == PGT_BF16 || dtype == PGT_F16, "kv_attention: bad dtype %d", dtype);
    PGT_CHECK(p.pshift > 0, "kv_attention: page=%d unsupported (16, 32, 64, 128)", page);
    PGT_CHECK(hd == 64 || hd == 128, "kv_attention: head_dim=%d unsupported (64, 128)", hd);
    PGT_CHECK(kv_heads > 0 && kv_heads <= 65536 && heads > 0 && heads <= 65536 && heads % kv_heads == 0,
              "kv_attention: %d heads over %d kv heads", heads, kv_heads);
    PGT_CHECK(pages > 0 && B >= 0 && rows >= 0 && max_new >= 0 && width >= 0 && ld_table >= width,
              "kv_attention: pages=%d B=%d rows=%d tokens per sequence=%d table width=%d", pages, B, rows, max_new, width);
    PGT_CHECK(causal >= 0 && window >= 0 && (causal > 0 || window == 0), "kv_attention: causal=%d window=%d", causal, window);
    PGT_CHECK(scale - scale == 0.f, "kv_attention: scale must be finite");
    PGT_CHECK(k_pages && v_pages && k_scale && v_scale, "kv_attention: null cache");
    PGT_CHECK((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "kv_attention: misaligned cache");
    if (B == 0 || rows == 0 || max_new == 0) return 0;
    PGT_CHECK(q && out && lens && (width == 0 || table), "kv_attention: null argument");
    PGT_CHECK(cu || (int64_t)B * max_new <= rows, "kv_attention: %d sequences of %d tokens in %d rows", B, max_new, rows);
    const int al = dtype == PGT_F32 ? 4 : 8;
    PGT_CHECK(ldq >= heads * hd && ldo >= heads * hd && ldq % al == 0 && ldo % al == 0,
              "kv_attention: row strides must cover heads * head_dim and be multiples of 16 bytes");
    PGT_CHECK((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "kv_attention: misaligned pointer");
    p.group = heads / kv_heads;
    p.nct = (int)(((int64_t)max_new * p.group + 15) / 16);
    const Split sp = splits(B, max_new, kv_heads, p.group, width, p.pshift, causal, window);
    p.nsplit = sp.n;
    p.chunk = sp.chunk;
    const int64_t wgs = (int64_t)B * kv_heads * p.nct * p.nsplit, slots = (int64_t)B * max_new * heads;
    PGT_CHECK((int64_t)max_new * p.group < (1 << 30) && wgs < (1LL << 31) && slots < (1LL << 31),
              "kv_attention: %d sequences of up to %d tokens exceed one launch", B, max_new);
    if (p.nsplit > 1) {
        const size_t need = (size_t)slots * p.nsplit * (hd + 2) * sizeof(float);
        PGT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                  "kv_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        p.po = (float*)workspace;
        p.pml = p.po + (size_t)slots * p.nsplit * hd;
    }
    hipStream_t st = (hipStream_t)stream;
#define ATTN_GO(TT, HD_)                                                                                              \
    do {                                                                                                              \
        if (p.nct == 1) hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, true>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p); \
        else hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, false>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p);      \
        if (p.nsplit > 1) hipLaunchKernelGGL((kv_attn_join_kernel<TT, HD_>), dim3((unsigned)slots), dim3(256), 0, st, p); \
    } while (0)
#define ATTN_HD(TT)                                                                                                   \
    do {                                                                                                              \
        if (hd == 64) ATTN_GO(TT, 64);                                                                                \
        else ATTN_GO(TT, 128);                                                                                        \
    } while (0)
    if (dtype == PGT_F32) ATTN_HD(float);
    else if (dtype == PGT_BF16) ATTN_HD(bf16_t);
    else ATTN_HD(half_t);
#undef ATTN_HD
#undef ATTN_GO
    PGT_LAUNCH_CHECK();
    return 0;
}
