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
    float *po, *pml;                  // partial results: (slot, 16 columns, hd), (slot, 16 columns, {m, l})
    int64_t ldq, ldo;
    int pages, pshift, ldt, width, B, rows, max_new, heads, kv, group, nct, wgs, causal, window;      // wgs: workgroups that share the work, 0 = one per column tile
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

constexpr int NW = 4;      // waves per workgroup, each with its own share of the tokens

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
    nct = (s.n * p.group + 15) >> 4;
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
// the whole line, and the part of it before sequence b (all 256 threads; red: 8 ints)
__device__ __forceinline__ Line line_of(const AttnP& p, int b, int& before, int* red) {
    int all = 0, pre = 0;
    for (int i = threadIdx.x; i < p.B; i += 64 * NW) {
        const int u = seq_units(p, i);
        all += u;
        if (i < b) pre += u;
    }
    all = wave_sum_i(all);
    pre = wave_sum_i(pre);
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = all;
        red[4 + (threadIdx.x >> 6)] = pre;
    }
    __syncthreads();
    Line l;
    l.total = red[0] + red[1] + red[2] + red[3];
    before = red[4] + red[5] + red[6] + red[7];
    l.share = max((l.total + p.wgs - 1) / p.wgs, NW);
    return l;
}
// the sequence that place `pos` of the line lies in, and the line before it
__device__ __forceinline__ void locate(const AttnP& p, int pos, int& b, int& before, int* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int run = 0;
    for (int c = 0; c < p.B; c += 64 * NW) {
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
            red[4] = c + tid;
            red[5] = e;
        }
        run += red[0] + red[1] + red[2] + red[3];
        if (run > pos) break;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(red[4]);
    before = __builtin_amdgcn_readfirstlane(red[5]);
    __syncthreads();
}

template <typename T, int HD, bool ONCE> __global__ __launch_bounds__(64 * NW, 2) void kv_attn_kernel(const AttnP p) {
    constexpr bool F32 = __is_same(T, float);
    constexpr bool HQ = __is_same(T, half_t);
    constexpr int QP = F32 ? 3 : 1;          // planes of q
    constexpr int KS = HD / 32;              // k-steps of S^T
    constexpr int ND = HD / 16;              // row tiles of O^T
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int col = lane & 15, g = lane >> 4;
    __shared__ int red[8];
    __shared__ float sm[NW][16], sl[NW][16];
    __shared__ __attribute__((aligned(16))) float so[NW][16][HD + 4];
    int b, before = 0, pos = 0, pos_end = 0;
    if (p.wgs == 0) {
        b = blockIdx.x / (p.nct * p.kv);
    } else {
        const Line line = line_of(p, 0, before, red);
        pos = blockIdx.x * line.share;
        pos_end = min(pos + line.share, line.total);
        if (pos >= pos_end) return;
        locate(p, pos, b, before, red);
    }
    for (;;) {      // the column tiles that this workgroup's part of the line touches
    const Seq s = seq_of(p, b);
    int ct, hk, t0, te, slot, units = 0;
    if (p.wgs == 0) {
        ct = blockIdx.x % p.nct;
        hk = blockIdx.x / p.nct % p.kv;
        t0 = te = slot = 0;
        if (ct * 16 >= s.n * p.group) return;
    } else {
        int nct, first;
        const int tiles = seq_tiles(p, s, first, nct);
        units = tiles * nct * p.kv;
        if (units == 0) { ++b; continue; }
        const int i = (pos - before) / tiles, off = pos - before - i * tiles;
        ct = i % nct;
        hk = i / nct;
        t0 = first + off;
        te = first + min(off + pos_end - pos, tiles);
        slot = blockIdx.x + (b * p.kv + hk) * p.nct + ct;
    }
    const int cols = s.n * p.group;
    const int qc = ct * 16 + col;
    const int qi = min(qc, cols - 1) / p.group;
    const int head = hk * p.group + min(qc, cols - 1) % p.group;
    int lo, hi;
    sees(p, s.len, s.len - s.n + qi, lo, hi);
    // what the tile's first and last query see: the range to visit, and the part that every query sees
    int lo_a, hi_a, lo_z, hi_z;
    sees(p, s.len, s.len - s.n + ct * 16 / p.group, lo_a, hi_a);
    sees(p, s.len, s.len - s.n + min(ct * 16 + 15, cols - 1) / p.group, lo_z, hi_z);
    if (p.wgs == 0) {
        t0 = lo_a >> 6;
        te = (hi_z + 63) >> 6;
    }

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
    float f[PD], lt = 0.f;
#pragma unroll
    for (int e = 0; e < PD; ++e) f[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        lt += sl[w][c2];
#pragma unroll
        for (int e = 0; e < PD; ++e) f[e] += so[w][c2][d2 + e];
    }
    if (p.wgs == 0) {
        if (qc2 < cols) {
            const int qi2 = qc2 / p.group, head2 = hk * p.group + qc2 % p.group;
            const float inv = lt == 0.f ? 0.f : 1.f / lt;      // a row that sees nothing is zero
            T* op = (T*)p.out + (s.r0 + qi2) * p.ldo + head2 * HD + d2;
#pragma unroll
            for (int e = 0; e < PD; ++e) f[e] = lt == 0.f ? 0.f : f[e] * inv;
#pragma unroll
            for (int e = 0; e < PD; e += 4) store4(op + e, f + e);
        }
        return;
    }
    if (qc2 < cols) {
        float* w = p.po + ((size_t)slot * 16 + c2) * HD + d2;
#pragma unroll
        for (int e = 0; e < PD; e += 4) store4(w + e, f + e);
        if ((tid & 15) == 0) {
            float mm2 = sm[0][c2];
#pragma unroll
            for (int k = 1; k < NW; ++k) mm2 = fmaxf(mm2, sm[k][c2]);
            store2(p.pml + ((size_t)slot * 16 + c2) * 2, mm2, lt);
        }
    }
    pos += te - t0;
    if (pos >= pos_end) return;
    if (pos - before >= units) {
        before += units;
        ++b;
    }
    __syncthreads();
    }
}

// out = the pieces' results against their common reference.  One workgroup per (sequence, token, head): HD / 4 threads hold the row, the
// rest of the 256 take other pieces, four loads in flight each.
constexpr int MAX_WGS = 768;
template <typename T, int HD> __global__ __launch_bounds__(64 * NW) void kv_attn_join_kernel(const AttnP p) {
    constexpr int LP = HD / 4, NS = 64 * NW / LP;
    __shared__ float al[MAX_WGS];
    __shared__ f32x4 so[NS][LP];
    __shared__ float sm[NW], sl[NW];
    __shared__ int red[8];
    int id = blockIdx.x;
    const int head = id % p.heads; id /= p.heads;
    const int qi = id % p.max_new, b = id / p.max_new, tid = threadIdx.x;
    const Seq s = seq_of(p, b);
    if (qi >= s.n) return;
    int before, first, nct;
    const Line line = line_of(p, b, before, red);
    const int tiles = seq_tiles(p, s, first, nct);
    const int qc = qi * p.group + head % p.group, ct = qc >> 4, hk = head / p.group;
    const int begin = before + (hk * nct + ct) * tiles;      // this column tile's part of the line, and the workgroups that hold some of it
    const int w0 = begin / line.share, n = tiles > 0 ? (begin + tiles - 1) / line.share - w0 + 1 : 0;
    const size_t slot = (size_t)w0 + (size_t)(b * p.kv + hk) * p.nct + ct;      // the next workgroup's is the next slot
    const float2* ml = reinterpret_cast<const float2*>(p.pml) + slot * 16 + (qc & 15);
    float m = -INFINITY, l = 0.f;
    for (int i = tid; i < n; i += 64 * NW) m = fmaxf(m, ml[i * 16].x);
    m = wave_max(m);
    if ((tid & 63) == 0) sm[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    for (int i = tid; i < n; i += 64 * NW) {
        const float2 w = ml[i * 16];
        const float a = w.x == -INFINITY ? 1.f : exp2_(w.x - m);      // a piece in which this query saw nothing holds zeros (or NaN)
        al[i] = a;
        l += w.y * a;
    }
    l = wave_sum(l);
    if ((tid & 63) == 0) sl[tid >> 6] = l;
    __syncthreads();
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    const int c = tid % LP, k = tid / LP;
    const f32x4* po = reinterpret_cast<const f32x4*>(p.po + (slot * 16 + (qc & 15)) * HD) + c;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = k; i < n; i += NS) o += po[(size_t)i * 16 * LP] * al[i];
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

// Workgroups that share the work: as many as run at once (hd 64: 3 per CU, 128: 2), or 0 = one per column tile, without a join, where no
// sequence can be longer than 16 tiles or there are so many column tiles that the chip is full anyway
int sharing(int B, int max_new, int kv, int group, int hd, int width, int pshift, int causal, int window) {
    const int64_t segs = (int64_t)B * kv * (((int64_t)max_new * group + 15) / 16);
    int64_t tiles = (((int64_t)width << pshift) + 63) / 64;
    if (causal && window) {      // from the first query's first token to the last one's last
        const int64_t w = ((int64_t)window + causal + max_new + 63) / 64 + 1;
        if (w < tiles) tiles = w;
    }
    if (tiles <= 4 * NW || segs <= 0 || segs >= 4096) return 0;
    return hd == 64 ? 768 : 512;
}
size_t slots_of(int B, int max_new, int kv, int group, int wgs) {
    return wgs ? (size_t)wgs + (size_t)B * kv * (((size_t)max_new * group + 15) / 16) : 0;
}

}  // namespace

extern "C" size_t pgt_kv_attention_workspace_bytes(int32_t B, int32_t max_new, int32_t heads, int32_t kv_heads, int32_t hd, int32_t width,
                                                   int32_t page, int32_t causal, int32_t window) {
    if (B <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || hd <= 0 || width <= 0 || kv_page_shift(page) < 0 || heads % kv_heads || causal < 0 || window < 0) return 0;
    const int group = heads / kv_heads, wgs = sharing(B, max_new, kv_heads, group, hd, width, kv_page_shift(page), causal, window);
    return slots_of(B, max_new, kv_heads, group, wgs) * 16 * (hd + 2) * sizeof(float);
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
    p.wgs = sharing(B, max_new, kv_heads, p.group, hd, width, p.pshift, causal, window);
    const int64_t segs = (int64_t)B * kv_heads * p.nct, wgs = p.wgs ? p.wgs : segs, rws = (int64_t)B * max_new * heads;
    PGT_CHECK((int64_t)max_new * p.group < (1 << 30) && segs < (1LL << 31) && rws < (1LL << 31),
              "kv_attention: %d sequences of up to %d tokens exceed one launch", B, max_new);
    if (p.wgs) {
        PGT_CHECK((double)segs * (((int64_t)width << p.pshift) / 64 + 1) < 2147483648.0,
                  "kv_attention: %d sequences of up to %d pages of %d tokens exceed one launch", B, width, page);
        const size_t slots = slots_of(B, max_new, kv_heads, p.group, p.wgs), need = slots * 16 * (hd + 2) * sizeof(float);
        PGT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                  "kv_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        p.po = (float*)workspace;
        p.pml = p.po + slots * 16 * hd;
    }
    hipStream_t st = (hipStream_t)stream;
#define ATTN_GO(TT, HD_)                                                                                              \
    do {                                                                                                              \
        if (p.nct == 1) hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, true>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p); \
        else hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, false>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p);      \
        if (p.wgs) hipLaunchKernelGGL((kv_attn_join_kernel<TT, HD_>), dim3((unsigned)rws), dim3(64 * NW), 0, st, p);   \
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
