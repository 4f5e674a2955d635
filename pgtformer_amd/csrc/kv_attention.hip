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
// holds: P goes from the accumulators into the operand without an exchange.
// The query columns are the group's heads times the tokens (column = token * group + head in group).
//
// Single tokens are bound by reading the cache once: 48 sequences of up to 8191 tokens, 32 / 8 heads of 128: 515 MB in 88 us, 5.9 TB/s (a plain
// streaming read: 7.1; fp32 queries, 48 of 8191: 6.0); one of 131071, 40 / 8 heads: 268 MB in 46 us, of which some 8 are start and end.
// Every wave has a tile in LDS and one in registers; the loads write LDS directly, since in registers the compiler waits for all of them
// wherever one is moved (113 us), and two tiles per wave in LDS leave half the waves (96).
#include "kv_attention.h"
#include "pgt_internal.h"

namespace {

constexpr int NW = 4;      // waves per workgroup, each with its own share of the tokens

template <typename T, int HD, bool ONCE> __global__ __launch_bounds__(64 * NW, 2) void kv_attn_kernel(const AttnP p) {
    constexpr bool F32 = __is_same(T, float);
    constexpr bool HQ = __is_same(T, half_t);
    constexpr int QP = F32 ? 3 : 1;          // planes of q
    constexpr int KS = HD / 32;              // k-steps of S^T
    constexpr int ND = HD / 16;              // row tiles of O^T
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    __shared__ int red[NW + 2];
    __shared__ float sm[NW][16], sl[NW][16];
    // per wave a tile: K (chunk of 16 dims, 64 slots, 16 bytes), V (dims / 16, 4 blocks, 16 dims, 16 bytes), and 64 words: the four blocks'
    // K scales, V scales, and pages of the next tile; afterwards the waves' results
    constexpr int KB = HD * 64, SET = 2 * KB + 256, NK = HD / 16;
    __shared__ __attribute__((aligned(16))) char rings[NW * SET];
    static_assert(16 * (HD + 4) * 4 <= SET, "the results fit");
    float (*so)[16][HD + 4] = reinterpret_cast<float (*)[16][HD + 4]>(rings);
    int e = blockIdx.x, before = 0, pos = 0, pos_end = 0;
    if (p.wgs && !part_of<NW, 1>(p, blockIdx.x, pos, pos_end, e, before, red)) return;
    for (;;) {      // the column tiles that this workgroup's part of the line touches
    const Segment sg = uni(segment_of(p, 1, e));
    const Seq& s = sg.s;
    const int cols = s.n * p.group, ct = sg.ct;
    if (p.wgs && sg.tiles == 0) { e += p.kv; continue; }
    if (ct * 16 >= cols) return;
    const int qc = min(ct * 16 + col, cols - 1), qi = qc / p.group, qg = qc - qi * p.group;
    int lo, hi;
    sees(p, s.len, s.p0 + qi, lo, hi);
    // what every query of the tile sees: from the last one's first token to the first one's last
    int hi_a, lo_z, dummy;
    sees_uni(p, s.len, s.p0 + ct * 16 / p.group, dummy, hi_a);
    sees_uni(p, s.len, s.p0 + min(ct * 16 + 15, cols - 1) / p.group, lo_z, dummy);
    int hk = sg.hk;
    if (p.wgs) {      // (the look-up gives the first kv head)
        hk = (pos - before) / sg.tiles;
        e += hk;
        before += hk * sg.tiles;
    }
    for (;;) {        // its kv heads
    const int t0 = sg.first + (p.wgs ? pos - before : 0), te = p.wgs ? sg.first + min(pos_end - before, sg.tiles) : sg.first + sg.tiles;
    const bool whole = te - t0 == sg.tiles;
    const int head = hk * p.group + qg;

    const int page = 1 << p.pshift, kblk = (lane >> 2) & 3;
    const size_t page_bytes = (size_t)page * HD, head_off = (size_t)hk * page_bytes, stride = (size_t)p.kv * page_bytes;
    const int32_t* tab = p.table + (size_t)sg.b * p.ldt;
    auto valid = [&](int t, int i, int k) { return i >= 0 && i < p.pages && ((t * 64 + 16 * k) >> p.pshift) < p.width; };
    auto page_slot = [&](int t, int k) { return tab + min((t * 64 + 16 * k) >> p.pshift, p.width - 1); };
    const int steps = (te - t0 - wave + NW - 1) / NW;      // this wave's tiles t0 + wave, + NW, ...
    // pages of the first tile: of the block whose K this lane brings, of the one whose scales it brings, and of its own (V, scores)
    int pk = -1, pm = -1, pv = -1;
    if (steps > 0) pk = *page_slot(t0 + wave, kblk), pm = *page_slot(t0 + wave, lane & 3), pv = *page_slot(t0 + wave, g);

    // Q^T operand: k-step 2 s + h covers dims 64 s + 16 g + 8 h .. + 7 of lane group g - the order of the K loads
    uint4 qf[QP][KS];
#pragma unroll
    for (int st = 0; st < KS; ++st) {
        const int d = 64 * (st >> 1) + 16 * g + 8 * (st & 1);
        const T* qp = (const T*)p.q + (s.r0 + qi) * p.ldq + head * HD + d;
        if constexpr (F32) {
            split3(qp, qf[0][st], qf[1][st], qf[2][st]);
        } else {
            qf[0][st] = *reinterpret_cast<const uint4*>(qp);
        }
    }
#pragma unroll
    for (int pl = 0; pl < QP; ++pl)
#pragma unroll
        for (int st = 0; st < KS; ++st) x3_opaque(qf[pl][st]);      // here, or the wait for them stands in the loop and drains the tiles' loads

    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEVER, l = 0.f;
    // Tiles come through LDS: the next K is asked for as soon as this one is in registers, the next V likewise, page numbers with the K of the
    // tile before.  Slot 16 r + i of a K chunk holds token 16 (i / 4) + 4 r + i % 4: row i of S^T tile r.
    char* ring = rings + wave * SET;
    const int k_tok = 16 * kblk + 4 * g + (lane & 3);      // lane -> slot lane
    // pages of tile t: of the block whose K this lane brings, and of its own block (V, scales, scores)
    auto ask_k = [&](int t, int pk) {
        const int id = valid(t, pk, kblk) ? pk : 0;
        const uint8_t* kb = p.kp + id * stride + head_off + ((t * 64 + k_tok) & (page - 1)) * 16;
        const uint32_t to = lds_address(ring);
#pragma unroll
        for (int c = 0; c < NK; ++c) lds_load16<ONCE>(kb + (size_t)c * page * 16, to + c * 1024);
    };
    auto ask_v = [&](int t, int pv) {
        const int id = valid(t, pv, g) ? pv : 0;
        const uint8_t* vb = p.vp + id * stride + head_off + (size_t)(((t * 64 + 16 * g) & (page - 1)) >> 4) * (HD * 16) + col * 16;
        const uint32_t to = lds_address(ring + KB);
#pragma unroll
        for (int d = 0; d < ND; ++d) lds_load16<ONCE>(vb + d * 256, to + d * 1024);
    };
    auto ask_m = [&](int t, int pm) {      // pm: the page of block lane & 3
        const size_t one = (size_t)(valid(t, pm, lane & 3) ? pm : 0) * p.kv + hk;
        const void* from = lane < 4 ? (const void*)(p.ks + one) : (const void*)(p.vs + one);
        if (lane >= 8) from = page_slot(t + NW, lane & 3);
        lds_load4(from, lds_address(ring + 2 * KB));
    };
    if (steps > 0) {
        ask_m(t0 + wave, pm);
        ask_k(t0 + wave, pk);
        ask_v(t0 + wave, pv);
    }
    for (int i = 0; i < steps; ++i) {
        const int t = t0 + wave + NW * i, tv = t * 64 + 16 * g;
        const bool more = i + 1 < steps, here = valid(t, pv, g);
        wait_loads<NK>();      // all but V
        uint4 kr[NK];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) kr[r * (HD / 64) + c] = *reinterpret_cast<const uint4*>(ring + ((4 * c + g) * 64 + 16 * r + col) * 16);
        const int* words = reinterpret_cast<const int*>(ring + 2 * KB);
        const float sk_t = __int_as_float(words[g]), sv_t = here ? __int_as_float(words[4 + g]) : 1.f;
        pk = words[8 + kblk], pv = words[8 + g], pm = words[8 + (lane & 3)];
        wait_lds();
        if (more) {
            ask_m(t + NW, pm);
            ask_k(t + NW, pk);
        }
        f32x4 x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                const uint4 w = kr[r * (HD / 64) + c];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 a = HQ ? half8(h ? w.z : w.x, h ? w.w : w.y) : bfloat8(h ? w.z : w.x, h ? w.w : w.y);
#pragma unroll
                    for (int pl = QP - 1; pl >= 0; --pl)
                        x[r] = HQ ? mma_h(a, qf[pl][2 * c + h], x[r]) : mma_b(a, qf[pl][2 * c + h], x[r]);
                }
            }
        }
        const float ev = log2_scale(sv_t), ck = p.c * sk_t;
        const bool masked = (t * 64 < lo_z) | (t * 64 + 64 > hi_a) | (__any(!here) != 0);
        float y[16], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __builtin_fmaf(x[e >> 2][e & 3], ck, ev);
        if (masked) {
            const uint32_t span = here ? (uint32_t)(hi - lo) : 0u;
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = (uint32_t)(tv + e - lo) < span ? y[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, y[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any(mx - m > 15.f)) {      // (a difference: m + 15 would be rounded, to m + 16 from 2^25 on, and 2^16 is no half)
            const float mn = mx - m > 15.f ? mx - 7.f : m;      // each query by itself: its result does not depend on its neighbours
            const float al = exp2_(m - mn);
            l *= al;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= al;
            m = mn;
        }
        float ls = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            y[e] = exp2_(y[e] - m);
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
        if (more) wait_loads<NK + 1>();      // all but the next tile's words and K
        else wait_loads<0>();
        uint4 vr[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) vr[d] = *reinterpret_cast<const uint4*>(ring + KB + d * 1024 + lane * 16);
        wait_lds();
        if (more) ask_v(t + NW, pv);
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
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // join the waves: every one against the common reference
    if (g == 0) sm[wave][col] = m;
    __syncthreads();      // (and every wave is through with its ring)
    float mm = sm[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w][col]);
    const float al = exp2_(m - mm);
    if (g == 0) sl[wave][col] = l * al;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        *reinterpret_cast<f32x4*>(&so[wave][col][16 * d + 4 * g]) = o[d] * al;
    }
    __syncthreads();
    // thread: column tid / (4 NW), HD / (4 NW) consecutive dims
    constexpr int PT = 4 * NW, PD = HD / PT;
    const int c2 = tid / PT, d2 = (tid % PT) * PD, qc2 = ct * 16 + c2;
    float f[PD], lt = 0.f;
#pragma unroll
    for (int e = 0; e < PD; ++e) f[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        lt += sl[w][c2];
#pragma unroll
        for (int e = 0; e < PD; ++e) f[e] += so[w][c2][d2 + e];
    }
    if (qc2 < cols && whole) {
        const int qi2 = qc2 / p.group, head2 = hk * p.group + qc2 % p.group;
        const float inv = lt == 0.f ? 0.f : 1.f / lt;      // a row that sees nothing is zero
        T* op = (T*)p.out + (s.r0 + qi2) * p.ldo + head2 * HD + d2;
#pragma unroll
        for (int e2 = 0; e2 < PD; ++e2) f[e2] = lt == 0.f ? 0.f : f[e2] * inv;
#pragma unroll
        for (int e2 = 0; e2 < PD; e2 += 4) store4(op + e2, f + e2);
    } else if (qc2 < cols) {
        const size_t at = ((size_t)blockIdx.x + e) * 16 + c2;
#pragma unroll
        for (int e2 = 0; e2 < PD; e2 += 4) store4(p.po + at * HD + d2 + e2, f + e2);
        if (tid % PT == 0) {
            float mm2 = sm[0][c2];
#pragma unroll
            for (int k = 1; k < NW; ++k) mm2 = fmaxf(mm2, sm[k][c2]);
            store2(p.pml + at * 2, mm2, lt);
        }
    }
    if (p.wgs && tid == 0) {
        if (t0 == sg.first) p.ends[e].x = blockIdx.x;
        if (te == sg.first + sg.tiles) p.ends[e].y = blockIdx.x;
    }
    pos += te - t0;
    if (pos >= pos_end) return;
    before += sg.tiles;
    ++e;
    __syncthreads();
    if (++hk == p.kv) break;
    }
    }
}

// out = the pieces' results against their common reference, for the segments that were cut (and zeros where nothing is seen).  HD / 4 threads
// hold a row.  Few pieces, many rows (the 256-column kernel: a segment is cut once or twice): a thread adds up ROWS rows at once, so that their
// loads are in flight together (one at a time: 30 us, four 18, eight 20 for 512 segments of 256 rows, hd 128).
constexpr int MAX_WGS = 768;
template <typename T, int HD> __device__ __forceinline__ void store_row(const AttnP& p, const Segment& sg, const Seq& s, int qc, int c, const f32x4& o, float l) {
    float f[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = l == 0.f ? 0.f : o[q] / l;
    store4((T*)p.out + (s.r0 + qc / p.group) * p.ldo + (sg.hk * p.group + qc % p.group) * HD + 4 * c, f);
}
template <typename T, int HD, int ROWS> __global__ __launch_bounds__(256) void kv_attn_join_rows_kernel(const AttnP p) {
    constexpr int LP = HD / 4, SIDE = 256 / LP, WG_ROWS = SIDE * ROWS;      // rows side by side, rows of a workgroup
    const int chunks = (1 << p.cshift) / WG_ROWS;
    const int e = blockIdx.x / chunks, r0 = blockIdx.x % chunks * WG_ROWS;
    const Segment sg = segment_of(p, 0, e);
    const Seq& s = sg.s;
    const int c0 = (sg.ct << p.cshift) + r0, cols = s.n * p.group;
    if (c0 >= cols) return;
    const int2 ends = sg.tiles > 0 ? p.ends[e] : make_int2(0, -1);
    const int w0 = ends.x, n = ends.y - w0 + 1;
    if (n == 1) return;
    const int c = threadIdx.x % LP, row = threadIdx.x / LP;
    size_t at = (((size_t)w0 + e) << p.cshift) + r0 + row;      // the next piece is in the next slot
    float l[ROWS], m[ROWS];
    f32x4 o[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) l[k] = 0.f, m[k] = NEVER, o[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n; ++i, at += (size_t)1 << p.cshift) {
        float2 w[ROWS];
        f32x4 x[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {      // (rows behind the last are slots nobody wrote: not stored)
            w[k] = reinterpret_cast<const float2*>(p.pml)[at + SIDE * k];
            x[k] = reinterpret_cast<const f32x4*>(p.po)[(at + SIDE * k) * LP + c];
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const float mn = fmaxf(m[k], w[k].x), a = exp2_(m[k] - mn), b = exp2_(w[k].x - mn);
            l[k] = l[k] * a + w[k].y * b;
            o[k] = o[k] * a + x[k] * b;
            m[k] = mn;
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int qc = c0 + row + SIDE * k;
        if (qc < cols) store_row<T, HD>(p, sg, s, qc, c, o[k], l[k]);
    }
}
// Many pieces, few rows: a workgroup per row, the pieces side by side, four loads in flight each.
template <typename T, int HD> __global__ __launch_bounds__(256) void kv_attn_join_kernel(const AttnP p) {
    constexpr int LP = HD / 4, NS = 256 / LP;
    const int tid = threadIdx.x, e = blockIdx.x / p.jrows, r0 = blockIdx.x % p.jrows;
    const Segment sg = segment_of(p, 1, e);
    const Seq& s = sg.s;
    const int qc = (sg.ct << 4) + r0;
    if (qc >= s.n * p.group) return;
    const int2 ends = sg.tiles > 0 ? p.ends[e] : make_int2(0, -1);
    const int w0 = ends.x, n = ends.y - w0 + 1;
    if (n == 1) return;
    const int c = tid % LP, k = tid / LP;
    const size_t at = (((size_t)w0 + e) << 4) + r0;
    const float2* ml = reinterpret_cast<const float2*>(p.pml) + at;
    const f32x4* po = reinterpret_cast<const f32x4*>(p.po + at * HD) + c;
    float l = 0.f, m = NEVER;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    __shared__ float al[MAX_WGS];
    __shared__ f32x4 so[NS][LP];
    __shared__ float sm[4], sl[4];
    for (int i = tid; i < n; i += 256) m = fmaxf(m, ml[(size_t)i << 4].x);
    m = wave_max(m);
    if ((tid & 63) == 0) sm[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    for (int i = tid; i < n; i += 256) {
        const float2 w = ml[(size_t)i << 4];
        const float a = exp2_(w.x - m);
        al[i] = a;
        l += w.y * a;
    }
    l = wave_sum(l);
    if ((tid & 63) == 0) sl[tid >> 6] = l;
    __syncthreads();
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
#pragma unroll 4
    for (int i = k; i < n; i += NS) o += po[((size_t)i << 4) * LP] * al[i];
    so[k][c] = o;
    __syncthreads();
    if (k) return;
#pragma unroll
    for (int i = 1; i < NS; ++i) o += so[i][c];
    store_row<T, HD>(p, sg, s, qc, c, o, l);
}

// How a call is run: column tiles of 16 (this file) or 256 (kv_attention_rows.hip), and the workgroups that share the work (0: one per column
// tile, no join).  Lengths are only known on the device; the table's width bounds them.
//
// 256 columns, in units of a tile's time (2.2 us at hd 128, 1.5 at 64): one workgroup per column tile takes ceil(segs / 256) * tiles + 4, of
// ragged lengths some 1.25 times that; shared, segs * tiles / 256 + 16 for the look-up, second segments and the join.  Shared against not, us, equal
// lengths: 64 segments of 60 tiles 52 / 97 (hd 64), 66 / 119 (128), of 28 tiles 39 / 52, 53 / 65; 256 of 12: 54 / 32, 74 / 44; 256 of 60: 120 / 101,
// 165 / 136; ragged, 256 of 160 and 512 of 128: 172 / 230, 437 / 559.  From 1024 segments on the dispatch evens lengths out by itself: 12 tiles 124 /
// 118, 175 / 158, 124 tiles 748 / 740, 1105 / 1039.
// 16 columns: the whole chip does a tile of 1024 segments in about that unit.  16 columns against 256, us: 1 sequence of 65536, 48 columns 35 / 60
// (hd 64), 71 / 73 (128), 64 columns 52 / 60, 49 / 73, 96 columns 44 / 62, 129 / 76, 128 columns 92 / 63, 78 / 77; 16 of 8192, 48 columns 52 / 80,
// 137 / 106, 64 columns 99 / 80, 86 / 106, 96 columns 85 / 85, 155 / 111, 128 columns 157 / 87, 163 / 115; 64 of 1024, 64 columns 33 / 44, 51 / 61,
// 128 columns 59 / 50, 96 / 67, 256 columns 114 / 64, 185 / 94; 4 of 700, 256 columns 10 / 29, 13 / 41.  The model does not see that the column tiles
// of a (sequence, kv head) read the same pages, which costs one reading where their pieces of the line run in step and several where they do not: of
// these it takes the slower kernel for 48 columns of 16 x 8192 and 96 of 65536 at hd 128, and for 64 of 16 x 8192 at hd 64.
// fp32 (hd 64; at 128 its three planes of q do not fit the registers of a wave of 32 columns): 2 of 8192, 8192 columns 764 / 552; 64 of 1024, 256
// columns 170 / 96; 4 of 2048, 512 columns 38 / 47.  At hd 128 the 16 columns take 1170 for 2 of 8192, 8192 columns, 1.13 times its five products.
struct Way {
    int cshift, wgs;
    size_t segs, slots;      // column tiles of the launch; slots of partial results
};
Way way_of(int dtype, int B, int max_new, int kv, int group, int hd, int width, int pshift, int causal, int window) {
    Way w;
    const int64_t cols = (int64_t)max_new * group;
    int64_t tiles = (((int64_t)width << pshift) + 63) / 64;
    if (causal && window) {      // from the first query's first token to the last one's last
        const int64_t n = ((int64_t)window + causal + max_new + 63) / 64 + 1;
        if (n < tiles) tiles = n;
    }
    const int64_t few = (int64_t)B * kv * ((cols + 15) >> 4), many = (int64_t)B * kv * ((cols + 255) >> 8);
    const double alone = 1.25 * ((many + 255) / 256) * tiles + 4, shared = (double)many * tiles / 256 + 16;
    const bool share = many < 1024 && shared < alone;
    if ((dtype != PGT_F32 || hd == 64) && (double)few * tiles / 1024 > (share ? shared : alone)) {
        w.cshift = 8;
        w.segs = many;
        w.wgs = share ? 256 : 0;
    } else {
        // Shared by as many as run at once (hd 64: 3 per CU, 128: 2), unless sequences are short or there are enough segments to even their
        // lengths out.  Shared against not, us: 8 segments of 16 tiles 12 / 8.5 (hd 64), 12 / 10 (128), of 64: 12 / 21, 13 / 27; 128 of 32: 20 / 13,
        // 19 / 17; 512 of 64: 54 / 43, 87 / 82, ragged 384 of 128: 95 / 106; 2048 of 32: 102 / 83, 180 / 165.
        w.cshift = 4;
        w.segs = few;
        w.wgs = hd == 64 ? 768 : 512;
        if (tiles <= (few >= 128 ? 32 : 16) || few >= 2048 || few == 0) w.wgs = 0;
    }
    w.slots = w.wgs ? w.wgs + w.segs : 0;
    return w;
}
size_t bytes_of(const Way& w, int hd) { return w.wgs ? ((w.slots << w.cshift) * (hd + 2) + w.segs * 2) * 4 : 0; }

}  // namespace

extern "C" size_t pgt_kv_attention_workspace_bytes(int32_t dtype, int32_t B, int32_t max_new, int32_t heads, int32_t kv_heads, int32_t hd, int32_t width,
                                                   int32_t page, int32_t causal, int32_t window) {
    if (B <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || hd <= 0 || width <= 0 || kv_page_shift(page) < 0 || heads % kv_heads || causal < 0 || window < 0) return 0;
    const Way w = way_of(dtype, B, max_new, kv_heads, heads / kv_heads, hd, width, kv_page_shift(page), causal, window);
    return bytes_of(w, hd);
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
    PGT_CHECK(((int64_t)width << p.pshift) <= 0x7fff0000, "kv_attention: %d pages of %d tokens: positions exceed 32 bits", width, page);      // (tiles are fetched ahead)
    PGT_CHECK(p.c - p.c == 0.f, "kv_attention: scale=%g must be finite, in units of log 2 too", scale);
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
    PGT_CHECK((int64_t)max_new * p.group < (1 << 30), "kv_attention: %d tokens per sequence exceed one launch", max_new);
    const Way w = way_of(dtype, B, max_new, kv_heads, p.group, hd, width, p.pshift, causal, window);
    p.cshift = w.cshift;
    p.nct = (max_new * p.group + (1 << w.cshift) - 1) >> w.cshift;
    p.wgs = w.wgs;
    p.jrows = w.cshift == 4 && max_new * p.group < 16 ? max_new * p.group : 1 << w.cshift;
    const size_t wgs = w.wgs ? w.wgs : w.segs;
    PGT_CHECK(w.segs < (1ULL << 31) && wgs * (w.cshift == 4 ? 256 : 512) < (1ULL << 32),      // (a grid's threads are counted in 32 bits)
              "kv_attention: %d sequences of up to %d tokens each exceed one launch", B, max_new);
    if (w.wgs) {
        PGT_CHECK((double)w.segs * (((int64_t)width << p.pshift) / 64 + 1) < 1073741824.0,
                  "kv_attention: %d sequences of up to %d pages of %d tokens exceed one launch", B, width, page);
        const size_t need = bytes_of(w, hd);
        PGT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                  "kv_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        p.po = (float*)workspace;
        p.pml = p.po + (w.slots << w.cshift) * hd;
        p.ends = (int2*)(p.pml + (w.slots << w.cshift) * 2);
    }
    hipStream_t st = (hipStream_t)stream;
    if (w.cshift != 4)
        if (const int rc = pgt_kv_attention_rows_launch(&p, dtype, hd, (unsigned)wgs, st)) return rc;
    constexpr int JR = 4;
#define ATTN_GO(TT, HD_)                                                                                              \
    do {                                                                                                              \
        if (w.cshift == 4) {                                                                                          \
            if (p.nct == 1) hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, true>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p);\
            else hipLaunchKernelGGL((kv_attn_kernel<TT, HD_, false>), dim3((unsigned)wgs), dim3(64 * NW), 0, st, p);  \
            const dim3 rows((unsigned)(w.segs * p.jrows));                                                            \
            if (p.wgs) hipLaunchKernelGGL((kv_attn_join_kernel<TT, HD_>), rows, dim3(256), 0, st, p);                 \
        } else if constexpr (!__is_same(TT, float) || HD_ == 64) {      /* the 256-column kernel has no other fp32 form */\
            const dim3 rows((unsigned)(w.segs * (HD_ / 4 / JR)));                                                     \
            if (p.wgs) hipLaunchKernelGGL((kv_attn_join_rows_kernel<TT, HD_, JR>), rows, dim3(256), 0, st, p);        \
        }                                                                                                             \
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
