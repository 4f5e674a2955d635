// Attention over the paged 8-bit cache for many query rows (a prompt's chunk, whole frames): kv_attention.hip has the mathematics.
//
// 32x32x16 MFMA, swapped (S^T = K Q^T, O^T += V^T P^T); a wave holds 32 query columns, a workgroup of 8 waves 256.  What bounds it is the
// vector work beside the products (per 32 x 32 scores: 512 cycles of products at hd 128, 256 at 64, and 62 vector instructions, 16 of them
// exponentials), so everything else is kept away from the waves: per tile of 64 tokens the workgroup turns the codes into 16-bit
// operands ONCE, into LDS, for all its columns.  The images are in operand order - K: 8 dims x 64 tokens, the tokens permuted so that a
// lane's 16 scores belong to one 16-token block (one scale) and are the 16 tokens its V operand holds; V: 8 tokens x hd dims - all reads
// and writes are 16 bytes per lane.  Three stages: the scores of the next 32 tokens are multiplied while the softmax of the current ones
// runs, across the tile boundary, one barrier per tile; every product has a slice of vector work behind it, fixed by hand.
// Per tile of 64 tokens x 256 columns: 2.2 us at hd 128 (970 TFLOP/s on the whole chip), 1.5 at 64 (720); two ragged chunks of 2047 rows over 8190
// tokens, 32 heads of 128: 360 us with the join, 860 TFLOP/s.  With 16 columns per wave and four waves the same took 590 us.
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

constexpr int NW = 8, TH = 64 * NW, CT = 32 * NW;      // waves, threads and columns of a workgroup

template <typename T> struct QType { typedef T type; };
template <> struct QType<float> { typedef bf16_t type; };

template <typename T, int HD> __global__ __launch_bounds__(TH, 2) void kv_attn_rows_kernel(const AttnP p) {
    constexpr bool HQ = __is_same(T, half_t), F32 = __is_same(T, float);
    constexpr int QP = F32 ? 3 : 1;                             // planes of q: fp32 as three bf16
    using Q = typename QType<T>::type;
    constexpr int KS = HD / 16, ND = HD / 32, NV = 2 * ND;      // k-steps of S^T; row blocks of O^T, its products
    constexpr int KB = 64 * HD * 2, STAGE = 2 * KB;             // bytes of a K image; of a stage
    __shared__ __attribute__((aligned(16))) char smem[3 * STAGE];
    constexpr int SET = (HD == 128 ? 2048 : 1024) + 256;        // bytes of a set of raw units of one wave
    __shared__ __attribute__((aligned(16))) char rings[NW * 3 * SET];
    __shared__ float2 sscale[3][4];                             // per 16-token block: score factor (negative: no page), log2 vs
    __shared__ int red[NW + 2];
    __shared__ int nans;                                        // a V code in the range stands for NaN
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, r = lane & 31;
    const int page = 1 << p.pshift;
    const size_t page_bytes = (size_t)page * HD, stride = (size_t)p.kv * page_bytes;

    // segments of one (sequence, kv head) read the same pages: a contiguous run of them per XCD (dispatch is round-robin over 8)
    const int nblk = gridDim.x, xcd = blockIdx.x & 7, q8 = nblk >> 3, r8 = nblk & 7;
    const int id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
    int e = id, before = 0, pos = 0, pos_end = 0;
    if (p.wgs) {
        if (!part_of<NW, 0>(p, id, pos, pos_end, e, before, red)) return;
    }
    for (;;) {      // the segments that this workgroup's part of the line touches
        const Segment sg = uni(segment_of(p, 0, e));
        if (p.wgs && sg.tiles == 0) { ++e; continue; }
        const int b = sg.b, hk = sg.hk, ct = sg.ct;
        const Seq& s = sg.s;
        const int cols = s.n * p.group, shift = s.p0;
        if (ct * CT >= cols) return;
        const int t0 = sg.first + (p.wgs ? pos - before : 0), te = p.wgs ? sg.first + min(pos_end - before, sg.tiles) : sg.first + sg.tiles;
        const bool whole = te - t0 == sg.tiles;

        // Staging: a unit is 64 lanes x 16 bytes of one block (16 tokens): K 4 chunks of 16 dims (lane -> token lane & 15, chunk lane / 16), V 64 dims.
        // hd 128: wave w brings unit w / 4 of K and of V of block w & 3; hd 64: waves 0-3 bring K, 4-7 V.  The loads go straight to LDS, into a
        // ring of three sets per wave, three tiles ahead of the conversion (in registers the compiler moved them, and waited for that); a set
        // also brings the block's scales and the page number of the tile three later.  Waits are by hand: NL loads per set, in order.
        constexpr bool BOTH = HD == 128;
        constexpr int NL = BOTH ? 3 : 2;
        const int blk = wave & 3, part = wave >> 2;
        const int32_t* tab = p.table + (size_t)b * p.ldt;
        auto page_index = [&](int t, int k) { return (t * 64 + 16 * k) >> p.pshift; };
        auto ok = [&](int i) { return i >= 0 && i < p.pages; };
        char* ring = rings + wave * 3 * SET;
        // where this lane's bytes of K, V and of the scales / the table (lanes 0, 1 / 2) lie in a page
        const uint32_t k_at = (uint32_t)((lane >> 4) * page + (lane & 15)) * 16 + (BOTH ? (uint32_t)(part * 4 * page * 16) : 0u);
        const uint32_t v_at = (uint32_t)(lane + (BOTH ? 64 * part : 0)) * 16;
        const uint8_t *kb = p.kp + hk * page_bytes + k_at, *vb = p.vp + hk * page_bytes + v_at;
        const uint8_t* base = BOTH || part == 0 ? kb : vb;
        const uint8_t* word = (const uint8_t*)((lane == 0 ? p.ks : p.vs) + hk);
        uint32_t word_step = (uint32_t)p.kv * 4;
        if (lane == 2) word = (const uint8_t*)tab, word_step = 4;
        auto fetch = [&](int slot, int t, int pg0, bool here) {      // block blk of tile t, in page pg0 (not here: page 0, not looked at)
            const uint32_t pg = here ? (uint32_t)pg0 : 0u;
            const uint32_t tok = (uint32_t)((t * 64 + 16 * blk) & (page - 1));
            const uint32_t to = lds_address(ring + slot * SET);
            const uint32_t k_off = tok * 16, v_off = tok * HD;
            lds_load16(base + (uint64_t)pg * (uint32_t)stride + (BOTH || part == 0 ? k_off : v_off), to);
            if constexpr (BOTH) lds_load16(vb + (uint64_t)pg * (uint32_t)stride + v_off, to + 1024);
            const uint32_t i = lane == 2 ? (uint32_t)min(page_index(t + 3, blk), p.width - 1) : pg;
            lds_load4(word + (uint64_t)i * word_step, to + SET - 256);
        };
        // whether the next three tiles have a page (kept in scalars: 150 instead of 153 us for the frames, 354 / 360 for the chunks)
        bool have0 = false, have1 = false, have2 = false;
        if (t0 < te) {      // the first three tiles are on their way while the columns are set up
            int pg[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) pg[i] = uni(tab[min(page_index(t0 + i, blk), p.width - 1)]);
            auto there = [&](int i) { return ok(pg[i]) & (t0 + i < te) & (page_index(t0 + i, blk) < p.width); };
            have0 = there(0);
            have1 = there(1);
            have2 = there(2);
            fetch(0, t0, pg[0], have0);
            fetch(1, t0 + 1, pg[1], have1);
            fetch(2, t0 + 2, pg[2], have2);
        }

        // this wave's columns: what every one of them sees, and what any of them does
        const int cw = ct * CT + wave * 32;
        int lo_a = 0, hi_a = 0, lo_z = 0, hi_z = 0;      // a wave without columns sees nothing
        if (cw < cols) {
            sees_uni(p, s.len, shift + cw / p.group, lo_a, hi_a);
            sees_uni(p, s.len, shift + min(cw + 31, cols - 1) / p.group, lo_z, hi_z);
        }
        int all_lo, all_hi, dummy;                       // what all columns of the workgroup see
        sees_uni(p, s.len, shift + ct * CT / p.group, dummy, all_hi);
        sees_uni(p, s.len, shift + min(ct * CT + CT - 1, cols - 1) / p.group, all_lo, dummy);
        const int qc = min(cw + r, cols - 1);
        int lo, hi;
        sees(p, s.len, shift + qc / p.group, lo, hi);
        uint4 qf[QP][KS];
        {
            const uint32_t flip = p.c < 0.f ? 0x80008000u : 0u;      // a negative scale goes into q: the largest score stays the largest weight
            const T* qp = (const T*)p.q + (s.r0 + qc / p.group) * p.ldq + (hk * p.group + qc % p.group) * HD + 8 * h;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if constexpr (F32) split3(qp + 16 * k, qf[0][k], qf[1][k], qf[2][k]);
                else qf[0][k] = *reinterpret_cast<const uint4*>(qp + 16 * k);
#pragma unroll
                for (int pl = 0; pl < QP; ++pl) {
                    uint4& w = qf[pl][k];
                    w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
                }
            }
        }
        auto mma_s = [&](const uint4& a, int k, f32x16 x) {      // the smallest plane first
#pragma unroll
            for (int pl = QP - 1; pl >= 0; --pl) x = mma16<Q>(a, qf[pl][k], x);
            return x;
        };
        f32x16 o[ND];
        float m = NEVER, l = 0.f;
        // most: what a lane's 16 weights may sum up to before the query's reference is looked at.  x ck + (ev - m) adds an unrounded product to a rounded
        // difference, which cancel to within the rounding of m only: from some 2^27 on that is more exponents than half has.  The weights of such a
        // query are always taken again, from the rounded score that m came from (most < 0; finite scores of any size: one weight of 1 is left)
        float most = 32768.f;
        auto far = [&]() { return fabsf(m) > 1048576.f && m != NEVER; };
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = zero16();

        // token 16 hh + e of a 32-token half -> the row of S^T whose score ends up in register e of lane half hh
        const int k_to = (((lane >> 4) + (BOTH ? 4 * part : 0)) * 128 + 32 * (blk >> 1) + (lane & 3) + 8 * ((lane & 15) >> 2) + 4 * (blk & 1)) * 16;
        const int v_to = KB + (blk * 2 * HD + lane + (BOTH ? 64 * part : 0)) * 16;
        uint4 ra, rb;      // a set, read before the product that hides its way
        float rscale;
        int rnext;
        auto take = [&](int set) {
            const char* in = ring + set * SET;
            ra = *reinterpret_cast<const uint4*>(in + lane * 16);
            if constexpr (BOTH) rb = *reinterpret_cast<const uint4*>(in + 1024 + lane * 16);
            rscale = *reinterpret_cast<const float*>(in + SET - 256 + (lane & 1) * 4);
            rnext = *reinterpret_cast<const int*>(in + SET - 256 + 8);
        };
        auto convert = [&](int st, int t) {      // the set taken, of tile t -> stage st; then the set is fetched again, for tile t + 3
            char* d = smem + st * STAGE;
            if (BOTH || part == 0) {
                *reinterpret_cast<uint4*>(d + k_to) = HQ ? half8(ra.x, ra.y) : bfloat8(ra.x, ra.y);
                *reinterpret_cast<uint4*>(d + k_to + 1024) = HQ ? half8(ra.z, ra.w) : bfloat8(ra.z, ra.w);
            }
            if (BOTH || part == 1) {
                uint4 w = BOTH ? rb : ra;
                if (!have0) w = make_uint4(0, 0, 0, 0);      // no page: page 0 was read in its place, and its NaN times the weight 0 would be one
                if (((t * 64 < all_lo) | (t * 64 + 64 > all_hi)) & (t < te)) {
                    // NaN times the weight 0 of a query that does not see the token: zeros here, see the end
                    const uint4 n = make_uint4(nan_bytes(w.x), nan_bytes(w.y), nan_bytes(w.z), nan_bytes(w.w));
                    if (__any((n.x | n.y | n.z | n.w) != 0)) nans = 1;
                    w.x &= ~((n.x >> 7) * 255u); w.y &= ~((n.y >> 7) * 255u); w.z &= ~((n.z >> 7) * 255u); w.w &= ~((n.w >> 7) * 255u);
                }
                *reinterpret_cast<uint4*>(d + v_to) = half8(w.x, w.y);
                *reinterpret_cast<uint4*>(d + v_to + HD * 16) = half8(w.z, w.w);
            }
            if (lane < 2 && part == 0) {      // (a factor of 0 would turn masked scores into NaN: the least normal number is as flat)
                const float factor = have0 ? fmaxf(fabsf(p.c) * rscale, 1.17549435e-38f) : -1.f, ev = log2_scale(rscale);
                reinterpret_cast<float*>(&sscale[st][blk])[lane] = lane ? ev : factor;
            }
            // pages of the tiles ahead, and whether they are there
            have0 = have1;
            have1 = have2;
            have2 = ok(uni(rnext)) & (t + 3 < te) & (page_index(t + 3, blk) < p.width);
            fetch(st, t + 3, rnext, have2);      // (the set is in registers: what is above needed them)
        };
        auto k_operand = [&](int st, int sb, int k) {
            return *reinterpret_cast<const uint4*>(smem + st * STAGE + (sb * 32 + r + 64 * h) * 16 + k * 2048);
        };
        auto v_operand = [&](int st, int sb, int i) {      // i = k-step * ND + row block
            return *reinterpret_cast<const uint4*>(smem + st * STAGE + KB + ((sb * 2 + h) * 2 * HD + r) * 16 + ((i / ND) * HD + (i % ND) * 32) * 16);
        };
        float2 sc = make_float2(1.f, 0.f);      // of the current scores: sscale of this lane's 16 tokens
        auto scores = [&](int st, int sb, f32x16& x) {
#pragma unroll
            for (int k = 0; k < KS; ++k) x = mma_s(k_operand(st, sb, k), k, k == 0 ? zero16() : x);
            sc = sscale[st][sb * 2 + h];
        };
        // softmax of the scores x of half sb of tile t (stage st) and their product with V; xn = the scores of half nsb of stage nst (behind the
        // last tile: of whatever is there, unused); half fsb of stage fst is what the step after this one begins with.  Nothing moves over a SLICE;
        // operands are read four products ahead, from one step into the next.  The barrier of a tile stands in the middle of its first step.
#define SLICE() __builtin_amdgcn_sched_barrier(0)
        uint4 f[4];      // operands in flight: the first of the step's S^T at its start
        auto ahead = [&](int st, int sb) {
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = k_operand(st, sb, k);
        };
        auto step = [&](int t, int st, int sb, int nst, int nsb, int fst, int fsb, f32x16& x, f32x16& xn) {
            const int tok = t * 64 + sb * 32;
            if (tok >= hi_z || tok + 32 <= lo_a) {
                if (cw < cols) scores(nst, nsb, xn);
                if (sb == 0) __syncthreads();
                ahead(fst, fsb);
                return;
            }
            const float ck = fabsf(sc.x), ev = sc.y;
            const float back = __uint_as_float((uint32_t)(127 - (int)ev) << 23);      // 1 / vs
            if ((tok < lo_z) | (tok + 32 > hi_a) | (__any(sc.x < 0.f) != 0)) {
                const uint32_t span = sc.x < 0.f ? 0u : (uint32_t)(hi - lo);
                const int at = tok + 16 * h - lo;
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = (uint32_t)(at + k) < span ? x[k] : -INFINITY;
            }
            float ls = 0.f;
            uint32_t pw[8], pl[F32 ? 8 : 1];      // weights in half; fp32: what is left of them, in half
            // weights 2 i, 2 i + 1; summed before they are rounded: in half, those of pages whose values are by far smaller than the others' - or
            // nothing but zeros - vanish, for the product as they should, but not for the sum
            float add = ev - m, less = 0.f;
            auto weight2 = [&](int i, bool again = false) {
                float a = __builtin_fmaf(x[2 * i], ck, add), b = __builtin_fmaf(x[2 * i + 1], ck, add);
                if (again) a -= less, b -= less;
                a = exp2_(a), b = exp2_(b);
                pw[i] = f2h2_nosat(a, b);
                if constexpr (F32) {
                    x3_opaque(pw[i]);
                    const halfx2 w = __builtin_bit_cast(halfx2, pw[i]);
                    pl[i] = f2h2_nosat(a - (float)w.x, b - (float)w.y);
                }
                ls += a + b;
            };
            const float2 scn = sscale[nst][nsb * 2 + h];
            SLICE();
#pragma unroll
            for (int k = 0; k < KS; ++k) {      // S^T of the next half, the weights
                xn = mma_s(f[k % 4], k, k == 0 ? zero16() : xn);
                if (k + 4 < KS) f[k % 4] = k_operand(nst, nsb, k + 4);
                else f[k % 4] = v_operand(st, sb, k + 4 - KS);
#pragma unroll
                for (int i = 0; i < 8 / KS; ++i) weight2(k * (8 / KS) + i);
                SLICE();
            }
            // A query whose weights passed 2^15 in sum (each fits half until then) takes a new reference, 7 under its largest score, and its weights
            // again - each query by itself: its result does not depend on its neighbours.  A maximum ahead of the weights would cost 12
            // instructions more, and its way from the products to the exponentials stands between the steps.
            if (__any(!(ls <= most))) {
                float mx = x[0];
#pragma unroll
                for (int k = 1; k < 16; ++k) mx = fmaxf(mx, x[k]);
                const float tm = max_of_halves(__builtin_fmaf(mx, ck, ev));
                const bool over = (max_of_halves(ls <= 32768.f ? 0.f : 1.f) > 0.f) | far();
                const float mn = over && tm - m > 10.f ? tm - 7.f : m;
                const float al = exp2_(m - mn);
                l *= al;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] *= al;
                m = mn;
                most = far() ? -1.f : 32768.f;
                add = far() ? ev : ev - m;
                less = far() ? m : 0.f;
                ls = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) weight2(i, true);
            }
            if (sb == 0) __syncthreads();      // the next tile's stage is written
            sc = scn;
#pragma unroll
            for (int i = 0; i < NV; ++i) {      // O^T
                const int k = i / ND, d = i % ND;
                if constexpr (F32) o[d] = mma16<half_t>(f[i % 4], make_uint4(pl[4 * k], pl[4 * k + 1], pl[4 * k + 2], pl[4 * k + 3]), o[d]);
                o[d] = mma16<half_t>(f[i % 4], make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]), o[d]);
                f[i % 4] = i + 4 < NV ? v_operand(st, sb, i + 4) : k_operand(fst, fsb, i + 4 - NV);
                SLICE();
            }
            l = __builtin_fmaf(ls, back, l);
        };
#undef SLICE

        __syncthreads();      // the stages of the segment before
        if (tid == 0) nans = 0;
        __syncthreads();
        if (t0 < te) {
            wait_loads<2 * NL>();
            take(0);
            convert(0, t0);
            wait_loads<2 * NL>();
            take(1);
            __syncthreads();
            f32x16 xa, xb;
            if (cw < cols) scores(0, 0, xa);
            ahead(0, 1);
            int st = 0;
            for (int t = t0; t < te; ++t) {
                const int nst = st == 2 ? 0 : st + 1;
                convert(nst, t + 1);      // (the stage was last read in tile t - 2, which every wave left before the last barrier)
                step(t, st, 0, st, 1, nst, 0, xa, xb);
                wait_loads<2 * NL>();      // the set of tile t + 2 is here, those of t + 3, t + 4 on the way
                take(nst == 2 ? 0 : nst + 1);
                step(t, st, 1, nst, 0, nst, 1, xb, xa);
                st = nst;
            }
            wait_loads<0>();
        }

        // column cw + r: rows 32 d + 8 q + 4 h + 0..3 of O^T are in registers 4 q .. 4 q + 3
        {
            const float lt = l + __shfl_xor(l, 32, 64);
            const int c = cw + r;
            if (c < cols && whole) {
                const float inv = lt == 0.f ? 0.f : 1.f / lt;      // a row that sees nothing is zero
                T* op = (T*)p.out + (s.r0 + c / p.group) * p.ldo + (hk * p.group + c % p.group) * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float f[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[k] = lt == 0.f ? 0.f : o[d][4 * q + k] * inv;
                        store4(op + 32 * d + 8 * q, f);
                    }
            } else if (c < cols) {
                const size_t at = ((size_t)id + e) * CT + (c & (CT - 1));
                float* w = p.po + at * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float f[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[k] = o[d][4 * q + k];
                        store4(w + 32 * d + 8 * q, f);
                    }
                if (h == 0) store2(p.pml + at * 2, m, lt);
            }
        }
        // A V code that stands for NaN, in a tile that not every column sees whole, makes the outputs of exactly the queries that see its token NaN
        if (nans) {      // (the same in every thread: last written before the last barrier of the tiles)
            __threadfence_block();
            __syncthreads();
            for (int t = t0; t < te; ++t) {
                if (t * 64 >= all_lo && t * 64 + 64 <= all_hi) continue;
                for (int u = tid; u < 4 * HD; u += TH) {
                    const int k = u / HD, dim = u % HD, tok = t * 64 + k * 16, pi = page_index(t, k), pg = pi < p.width ? tab[pi] : -1;
                    if (!ok(pg)) continue;
                    const uint8_t* c = p.vp + pg * stride + hk * page_bytes + ((size_t)((tok & (page - 1)) >> 4) * HD + dim) * 16;
                    for (int i = 0; i < 16; ++i) {
                        if ((c[i] & 0x7f) != 0x7f) continue;
                        for (int q = ct * CT; q < min(ct * CT + CT, cols); ++q) {
                            int lq, hq;
                            sees(p, s.len, shift + q / p.group, lq, hq);
                            if (tok + i < lq || tok + i >= hq) continue;
                            T* op = (T*)p.out + (s.r0 + q / p.group) * p.ldo + (hk * p.group + q % p.group) * HD + dim;
                            if constexpr (F32) { if (whole) *op = __builtin_nanf(""); }
                            else if (whole) store_nan(op);
                            if (!whole) p.po[(((size_t)id + e) * CT + (q & (CT - 1))) * HD + dim] = __builtin_nanf("");
                        }
                    }
                }
            }
        }
        if (p.wgs && tid == 0) {
            if (t0 == sg.first) p.ends[e].x = id;
            if (te == sg.first + sg.tiles) p.ends[e].y = id;
        }
        pos += te - t0;
        if (pos >= pos_end) return;
        before += sg.tiles;
        ++e;
    }
}

}  // namespace

int pgt_kv_attention_rows_launch(const void* pp, int dtype, int hd, unsigned groups, hipStream_t st) {
    const AttnP& p = *(const AttnP*)pp;
#define ROWS_GO(TT, HD_) hipLaunchKernelGGL((kv_attn_rows_kernel<TT, HD_>), dim3(groups), dim3(TH), 0, st, p)
    if (dtype == PGT_F32) {
        ROWS_GO(float, 64);
    } else if (dtype == PGT_BF16) {
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
