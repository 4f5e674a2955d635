// Attention over the paged 8-bit cache for many query rows (a prompt's chunk, whole frames): kv_attention.hip has the mathematics.
//
// 32x32x16 MFMA, swapped (S^T = K Q^T, O^T += V^T P^T); a wave holds 64 query columns, a workgroup of 4 waves 256.  Per tile of 64 tokens the
// workgroup turns the codes into 16-bit operands ONCE, into LDS: 256 columns share one conversion, and every 1 KiB operand read feeds two
// matrix instructions (read per wave from the cache, conversion and loads cost as many cycles as the products).  The images are in operand
// order - K: 8 dims x 64 tokens, the tokens permuted so that a lane's 16 scores belong to one 16-token block (one scale) and are the 16
// tokens its V operand holds; V: 8 tokens x hd dims - all reads and writes are 16 bytes per lane without conflicts.  Three stages: the
// scores of the next 32 tokens are multiplied while the softmax of the current ones runs, across the tile boundary, one barrier per tile.
#include "kv_attention.h"

#include "pgt_internal.h"

namespace {

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}
// the larger of a lane's value and lane ^ 32's
__device__ __forceinline__ float max_of_halves(float v) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}

template <typename T, int HD, int NQ, int NW> __global__ __launch_bounds__(64 * NW, 2) void kv_attn_rows_kernel(const AttnP p) {
    constexpr bool HQ = __is_same(T, half_t);
    constexpr int KS = HD / 16, ND = HD / 32;              // k-steps of S^T, row blocks of O^T
    constexpr int CW = 32 * NQ, TH = 64 * NW, CT = CW * NW;      // columns of a wave; threads and columns of the workgroup
    constexpr int UN = HD / 64;                            // 16-byte units per thread of K (and of V) per tile
    static_assert(NW == 4, "a wave stages one of the four blocks of a tile");
    constexpr int KB = 64 * HD * 2, STAGE = 2 * KB;        // bytes of a K image; of a stage
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    __shared__ float2 sscale[2][4];                        // per 16-token block: score factor (negative: no page), log2 of the V scale
    __shared__ int nans;                                   // a V code in the range stands for NaN
    __shared__ int red[2 * NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, r = lane & 31;
    const int page = 1 << p.pshift;
    const size_t page_bytes = (size_t)page * HD, stride = (size_t)p.kv * page_bytes;

    int b, before = 0, pos = 0, pos_end = 0, id = 0;
    if (p.wgs == 0) {
        // column tiles of one (sequence, kv head) read the same pages: a contiguous run of ids per XCD (dispatch is round-robin over 8)
        const int nblk = gridDim.x, xcd = blockIdx.x & 7, q8 = nblk >> 3, r8 = nblk & 7;
        id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
        b = id / (p.nct * p.kv);
    } else {
        const Line line = line_of<NW>(p, 0, before, red);
        pos = blockIdx.x * line.share;
        pos_end = min(pos + line.share, line.total);
        if (pos >= pos_end) return;
        locate<NW>(p, pos, b, before, red);
    }
    for (;;) {
        const Seq s = seq_of(p, b);
        const int cols = s.n * p.group;
        int ct, hk, t0, te, slot = 0, units = 0;
        if (p.wgs == 0) {
            ct = p.nct - 1 - id % p.nct;      // the later queries see more: first
            hk = id / p.nct % p.kv;
            t0 = te = 0;
            if (ct * CT >= cols) return;
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
        const int shift = s.len - s.n;
        if (p.wgs == 0) {
            int lo, hi, dummy;
            sees(p, s.len, shift + ct * CT / p.group, lo, dummy);
            sees(p, s.len, shift + min(ct * CT + CT - 1, cols - 1) / p.group, dummy, hi);
            t0 = lo >> 6;
            te = (hi + 63) >> 6;
        }
        // this wave's columns: what every one of them sees, and what any of them does
        const int cw = ct * CT + wave * CW;
        int lo_a = 0, hi_a = 0, lo_z = 0, hi_z = 0;      // a wave without columns sees nothing
        if (cw < cols) {
            sees(p, s.len, shift + cw / p.group, lo_a, hi_a);
            sees(p, s.len, shift + min(cw + CW - 1, cols - 1) / p.group, lo_z, hi_z);
        }
        uint4 qf[NQ][KS];
        int lo[NQ], hi[NQ];
        const uint32_t flip = p.c < 0.f ? 0x80008000u : 0u;      // a negative scale goes into q: the largest score stays the largest weight
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int qc = min(cw + n * 32 + r, cols - 1), qi = qc / p.group;
            sees(p, s.len, shift + qi, lo[n], hi[n]);
            const T* qp = (const T*)p.q + (s.r0 + qi) * p.ldq + (hk * p.group + qc % p.group) * HD + 8 * h;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint4 w = *reinterpret_cast<const uint4*>(qp + 16 * k);
                w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
                qf[n][k] = w;
            }
        }
        f32x16 o[NQ][ND];
        float m[NQ], l[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[n][d][e] = 0.f;
        }

        // Staging: wave w brings block w (16 tokens) of a tile, so page and scales are the wave's: lane -> K (token lane & 15, chunks lane / 16
        // + 4 i), V (dims lane + 64 i).  Page numbers run one tile ahead of the loads, the loads one tile ahead of the conversion.
        const int32_t* tab = p.table + (size_t)b * p.ldt;
        uint4 rk[UN], rv[UN];
        int rpage, nextpage;
        float rsk, rsv;
        auto page_at = [&](int t, int blk) {
            const int i = (t * 64 + 16 * blk) >> p.pshift;
            return t < te && i < p.width ? tab[i] : -1;
        };
        auto ok = [&](int i) { return i >= 0 && i < p.pages; };
        const uint32_t k_at = (uint32_t)((lane >> 4) * page + (lane & 15)) * 16, k_step = (uint32_t)page * 64, v_at = (uint32_t)lane * 16;
        auto load_raw = [&](int t) {      // of page nextpage
            rpage = __builtin_amdgcn_readfirstlane(nextpage);
            const int id = ok(rpage) ? rpage : 0;
            const int tok = (t * 64 + 16 * wave) & (page - 1);
            const uint8_t *kb = p.kp + id * stride + hk * page_bytes + tok * 16, *vb = p.vp + id * stride + hk * page_bytes + (size_t)tok * HD;
#pragma unroll
            for (int i = 0; i < UN; ++i) rk[i] = *reinterpret_cast<const uint4*>(kb + (k_at + k_step * i));
#pragma unroll
            for (int i = 0; i < UN; ++i) rv[i] = *reinterpret_cast<const uint4*>(vb + (v_at + 1024u * i));
            rsk = p.ks[(size_t)id * p.kv + hk];
            rsv = p.vs[(size_t)id * p.kv + hk];
        };
        // token 16 hh + e of a 32-token half -> the row of S^T whose score ends up in register e of lane half hh
        const int k_to = (((lane >> 4) * 2) * 64 + 32 * (wave >> 1) + (lane & 3) + 8 * ((lane & 15) >> 2) + 4 * (wave & 1)) * 16;
        const int v_to = KB + (wave * 2 * HD + lane) * 16;
        auto store = [&](int st) {
            char* d = smem + st * STAGE;
#pragma unroll
            for (int i = 0; i < UN; ++i) {      // (opaque: or the compiler regroups the registers right behind the loads, and waits for them there)
                x3_opaque(rk[i]);
                x3_opaque(rv[i]);
            }
#pragma unroll
            for (int i = 0; i < UN; ++i) {
                const uint4 w = rk[i];
                *reinterpret_cast<uint4*>(d + k_to + i * 8192) = HQ ? half8(w.x, w.y) : bfloat8(w.x, w.y);
                *reinterpret_cast<uint4*>(d + k_to + i * 8192 + 1024) = HQ ? half8(w.z, w.w) : bfloat8(w.z, w.w);
            }
#pragma unroll
            for (int i = 0; i < UN; ++i) {
                const uint4 w = rv[i];
                *reinterpret_cast<uint4*>(d + v_to + i * 1024) = half8(w.x, w.y);
                *reinterpret_cast<uint4*>(d + v_to + i * 1024 + HD * 16) = half8(w.z, w.w);
            }
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < UN; ++i) bad |= nan_bytes(rv[i].x) | nan_bytes(rv[i].y) | nan_bytes(rv[i].z) | nan_bytes(rv[i].w);
            if (__any(bad != 0)) {      // NaN times the weight 0 of a query that does not see the token: zeros here, see the end
                nans = 1;
#pragma unroll
                for (int i = 0; i < UN; ++i) {
                    const uint4 w = rv[i];
                    auto clean = [](uint32_t v) { return v & ~((nan_bytes(v) >> 7) * 255u); };
                    *reinterpret_cast<uint4*>(d + v_to + i * 1024) = half8(clean(w.x), clean(w.y));
                    *reinterpret_cast<uint4*>(d + v_to + i * 1024 + HD * 16) = half8(clean(w.z), clean(w.w));
                }
            }
            if (lane == 0)      // (a factor of 0 would turn masked scores into NaN: 1e-30 is as flat)
                sscale[st][wave] = make_float2(ok(rpage) ? fmaxf(fabsf(p.c) * rsk, 1e-30f) : -1.f, (float)((int)((__float_as_uint(rsv) >> 23) & 255) - 127));
        };
        auto k_operand = [&](int st, int sb, int k) {
            return *reinterpret_cast<const uint4*>(smem + st * STAGE + (sb * 32 + r + 64 * h) * 16 + k * 2 * 64 * 16);
        };
        auto v_operand = [&](int st, int sb, int i) {      // i = k-step * ND + row block
            return *reinterpret_cast<const uint4*>(smem + st * STAGE + KB + ((sb * 2 + h) * 2 * HD + r) * 16 + ((i / ND) * HD + (i % ND) * 32) * 16);
        };
        float2 sc = make_float2(1.f, 0.f);      // of the current scores: factor and log2 of the V scale of this lane's 16 tokens
        float tm[NQ];                           // largest of a query's current scores, in units of the exponent
        auto top = [&](const f32x16 (&x)[NQ], int n) {
            float mx = x[n][0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, x[n][e]);
            return max_of_halves(__builtin_fmaf(mx, fabsf(sc.x), sc.y));
        };
        // the scores of half sb of stage st
        auto scores = [&](int st, int sb, f32x16 (&x)[NQ]) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint4 a = k_operand(st, sb, k);
#pragma unroll
                for (int n = 0; n < NQ; ++n) x[n] = mma16<T>(a, qf[n][k], k == 0 ? zero16() : x[n]);
            }
            sc = sscale[st][sb * 2 + h];
#pragma unroll
            for (int n = 0; n < NQ; ++n) tm[n] = top(x, n);
        };
        // softmax of the scores x of half sb of tile t (stage st) and their product with V; xn = the scores of half nsb of stage nst (behind
        // the last tile: of whatever is there, unused).  The order is fixed by hand (nothing moves over a SLICE): behind every product a slice of
        // vector work that takes about as long, operands read four products ahead.
#define SLICE() __builtin_amdgcn_sched_barrier(0)
        auto step = [&](int t, int st, int sb, int nst, int nsb, f32x16 (&x)[NQ], f32x16 (&xn)[NQ]) {
            const int tok = t * 64 + sb * 32;
            if (tok >= hi_z || tok + 32 <= lo_a) {
                scores(nst, nsb, xn);
                return;
            }
            const float ck = fabsf(sc.x), ev = sc.y;
            const int missing = __any(sc.x < 0.f);
            if ((tok < lo_z) | (tok + 32 > hi_a) | (missing != 0)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const uint32_t span = sc.x < 0.f ? 0u : (uint32_t)(hi[n] - lo[n]);
                    const int at = tok + 16 * h - lo[n];
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[n][e] = (uint32_t)(at + e) < span ? x[n][e] : -INFINITY;
                    tm[n] = top(x, n);
                }
            }
            bool up = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) up |= tm[n] > m[n] + 15.f;
            if (__any(up)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float mn = tm[n] > m[n] + 15.f ? tm[n] - 7.f : m[n];
                    const float al = m[n] == -INFINITY ? 0.f : exp2_(m[n] - mn);
                    l[n] *= al;
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[n][d] *= al;
                    m[n] = mn;
                }
            }
            const float back = __uint_as_float((uint32_t)(127 - (int)ev) << 23);      // 1 / vs
            float em[NQ], ls[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                em[n] = ev - (m[n] == -INFINITY ? 0.f : m[n]);
                ls[n] = 0.f;
            }
            uint32_t pw[NQ][8];
            auto weight2 = [&](int n, int i) {      // weights 2 i, 2 i + 1 of query block n
                const float a = exp2_(__builtin_fmaf(x[n][2 * i], ck, em[n])), b = exp2_(__builtin_fmaf(x[n][2 * i + 1], ck, em[n]));
                ls[n] += a;
                ls[n] += b;
                pw[n][i] = f2h2_nosat(a, b);
            };
            uint4 f[4];      // operands in flight
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = k_operand(nst, nsb, k);
            const float2 scn = sscale[nst][nsb * 2 + h];
            SLICE();
            // S^T of the next half; the weights of query block 0
#pragma unroll
            for (int i = 0; i < NQ * KS; ++i) {
                const int k = i / NQ, n = i % NQ;
                xn[n] = mma16<T>(f[k % 4], qf[n][k], k == 0 ? zero16() : xn[n]);
                if (n == NQ - 1) {
                    if (k + 4 < KS) f[k % 4] = k_operand(nst, nsb, k + 4);
                    else f[k % 4] = v_operand(st, sb, k + 4 - KS);
                }
                weight2(0, i);
                SLICE();
            }
            sc = scn;
            // O^T; the weights of query block 1, the largest of the next scores
            float mx[NQ];
            constexpr int NV = 2 * ND;      // products per query block
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int k = i / ND, d = i % ND;
                    o[n][d] = mma16<half_t>(f[i % 4], make_uint4(pw[n][4 * k], pw[n][4 * k + 1], pw[n][4 * k + 2], pw[n][4 * k + 3]), o[n][d]);
                    if (i + 4 < NV) f[i % 4] = v_operand(st, sb, i + 4);
                    if (NQ == 2 && n == 0) {
                        weight2(NQ - 1, 2 * i);
                        weight2(NQ - 1, 2 * i + 1);
                    } else {
                        constexpr int PER = 16 / NV;
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            if (i == 0) mx[q] = xn[q][0];
#pragma unroll
                            for (int e = 0; e < PER; ++e) mx[q] = fmaxf(mx[q], xn[q][PER * i + e]);
                        }
                    }
                    SLICE();
                }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                l[n] = __builtin_fmaf(ls[n], back, l[n]);
                tm[n] = max_of_halves(__builtin_fmaf(mx[n], fabsf(sc.x), sc.y));
            }
        };
#undef SLICE

        __syncthreads();      // the stages of the column tile before
        if (tid == 0) nans = 0;
        __syncthreads();
        if (t0 < te) {
            nextpage = page_at(t0, wave);
            load_raw(t0);
            nextpage = page_at(t0 + 1, wave);
            store(0);
            if (t0 + 1 < te) load_raw(t0 + 1);
            nextpage = page_at(t0 + 2, wave);
            __syncthreads();
            f32x16 xa[NQ], xb[NQ];
            scores(0, 0, xa);
            int st = 0;
            for (int t = t0; t < te; ++t, st ^= 1) {
                const bool more = t + 1 < te;
                step(t, st, 0, st, 1, xa, xb);
                __syncthreads();      // every wave is through with the other stage
                if (more) {
                    store(st ^ 1);
                    if (t + 2 < te) load_raw(t + 2);
                    nextpage = page_at(t + 3, wave);
                }
                __syncthreads();
                step(t, st, 1, st ^ 1, 0, xb, xa);
            }
        }

        // columns cw + 32 n + r: rows 32 d + 8 q + 4 h + 0..3 of O^T are in registers 4 q .. 4 q + 3
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float lt = l[n] + __shfl_xor(l[n], 32, 64);
            const int qc = cw + n * 32 + r;
            if (qc < cols) {
                if (p.wgs == 0) {
                    const float inv = lt == 0.f ? 0.f : 1.f / lt;
                    T* op = (T*)p.out + (s.r0 + qc / p.group) * p.ldo + (hk * p.group + qc % p.group) * HD + 4 * h;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            float f[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) f[e] = lt == 0.f ? 0.f : o[n][d][4 * q + e] * inv;
                            store4(op + 32 * d + 8 * q, f);
                        }
                } else {
                    const size_t at = (size_t)slot * CT + (qc & (CT - 1));
                    float* w = p.po + at * HD + 4 * h;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            float f[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) f[e] = o[n][d][4 * q + e];
                            store4(w + 32 * d + 8 * q, f);
                        }
                    if (h == 0) store2(p.pml + at * 2, m[n], lt);
                }
            }
        }
        // A V code that stands for NaN makes the outputs of exactly the queries that see its token NaN (and none by 0 * NaN)
        __threadfence();
        __syncthreads();
        if (nans) {
            for (int t = t0; t < te; ++t)
                for (int u = tid; u < 4 * HD; u += TH) {
                    const int blk = u / HD, dim = u % HD, tok = t * 64 + blk * 16, pg = page_at(t, blk);
                    if (!ok(pg)) continue;
                    const uint8_t* c = p.vp + pg * stride + hk * page_bytes + ((size_t)((tok & (page - 1)) >> 4) * HD + dim) * 16;
                    for (int e = 0; e < 16; ++e) {
                        if ((c[e] & 0x7f) != 0x7f) continue;
                        for (int qc = ct * CT; qc < min(ct * CT + CT, cols); ++qc) {
                            int lq, hq;
                            sees(p, s.len, shift + qc / p.group, lq, hq);
                            if (tok + e < lq || tok + e >= hq) continue;
                            if (p.wgs == 0) store_nan((T*)p.out + (s.r0 + qc / p.group) * p.ldo + (hk * p.group + qc % p.group) * HD + dim);
                            else p.po[((size_t)slot * CT + (qc & (CT - 1))) * HD + dim] = __builtin_nanf("");
                        }
                    }
                }
        }
        if (p.wgs == 0) return;
        pos += te - t0;
        if (pos >= pos_end) return;
        if (pos - before >= units) {
            before += units;
            ++b;
        }
    }
}

}  // namespace

int pgt_kv_attention_rows_launch(const void* pp, int bf16, int hd, unsigned groups, hipStream_t st) {
    const AttnP& p = *(const AttnP*)pp;
#define ROWS_GO(TT, HD_)                                                                                                          \
    hipLaunchKernelGGL((kv_attn_rows_kernel<TT, HD_, HD_ == 64 ? 2 : 1, 4>), dim3(groups), dim3(256), 0, st, p)
    if (bf16) {
        if (hd == 64) ROWS_GO(bf16_t, 64);
        else ROWS_GO(bf16_t, 128);
    } else {
        if (hd == 64) ROWS_GO(half_t, 64);
        else ROWS_GO(half_t, 128);
    }
#undef ROWS_GO
    PGT_LAUNCH_CHECK();
    return 0;
}
