// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its gradient.
//
//   y = R(pos) (g * x * r),   r = 1 / sqrt(mean(x^2) + eps)      per head row x of hd elements, fp32 inside, one rounding at the store
//   R turns pair i of the first `rot` elements by the angle 2 pi * pos * freqs[i] (freqs in revolutions per position, fp64): pairs are
//   (i, i + rot / 2), or (2i, 2i + 1) in the interleaved form; the elements behind `rot` are not turned.
// gradient: z = R(-pos) dy, u = g * z, xh = x * r:   dx = r (u - xh * mean(xh * u)),   dg = sum over rows and heads of z * xh
//
// Memory bound: x is read once and y written once.  hd / 8 (or hd / 16) lanes hold a head row, two runs of 4 (8) elements each, picked so that
// both halves of every pair sit in one lane (a rotation needs no exchange; the mean is a few lane exchanges).  The angle is taken in fp64 and
// reduced to a fraction of a turn before it is rounded to fp32 - exact for any int32 position - once per token and pair, into
// LDS, for all heads of the token.  16411 tokens of 32 + 8 heads of 128 in bf16: 63 to 69 us, 5.3 to 4.8 TB/s (a copy: 5.1); the gradient of
// 8190: 49 to 52 us, 5.1 to 4.8 TB/s, and 4.7 for the sums of the gain gradients.  Issue counts: a division per row, selects between q and k and an
// exact root cost 10 us.
#include "kv_common.h"
#include "pgt_internal.h"

namespace {

// A run of 4 elements of a head row (16-bit: 8 bytes, fp32: 16 bytes).  ONCE: streaming loads, for the form that only reads
// and writes once (16411 tokens of 40 heads of 128: 74 instead of 77 us; the gradient, with twice the loads in flight, gains nothing).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool ONCE, typename T> __device__ __forceinline__ void ld4(const T* p, float* f) {
    if constexpr (__is_same(T, float)) {
        const f32x4* at = reinterpret_cast<const f32x4*>(p);
        const f32x4 w = ONCE ? __builtin_nontemporal_load(at) : *at;
        f[0] = w[0]; f[1] = w[1]; f[2] = w[2]; f[3] = w[3];
    } else {
        const u32x2* at = reinterpret_cast<const u32x2*>(p);
        const u32x2 v = ONCE ? __builtin_nontemporal_load(at) : *at;
        const uint32_t w[2] = {v.x, v.y};
        if constexpr (__is_same(T, bf16_t)) {
            f[0] = __uint_as_float(w[0] << 16); f[1] = __uint_as_float(w[0] & 0xffff0000u);
            f[2] = __uint_as_float(w[1] << 16); f[3] = __uint_as_float(w[1] & 0xffff0000u);
        } else {
            const halfx2 a = __builtin_bit_cast(halfx2, w[0]), b = __builtin_bit_cast(halfx2, w[1]);
            f[0] = (float)a.x; f[1] = (float)a.y; f[2] = (float)b.x; f[3] = (float)b.y;
        }
    }
}

// R elements: 4, or 8 of a 16-bit type (16 bytes)
template <int R, bool ONCE, typename T> __device__ __forceinline__ void ldr(const T* p, float* f) {
    if constexpr (R == 4) {
        ld4<ONCE>(p, f);
    } else {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4* at = reinterpret_cast<const u32x4*>(p);
        const u32x4 v = ONCE ? __builtin_nontemporal_load(at) : *at;
        Vec16<T>::unpack(make_uint4(v.x, v.y, v.z, v.w), f);
    }
}
template <int R, typename T> __device__ __forceinline__ void str(T* p, const float* f) {
    if constexpr (R == 4) store4(p, f);
    else *reinterpret_cast<uint4*>(p) = make_uint4(pair_of<T>(f[0], f[1]), pair_of<T>(f[2], f[3]), pair_of<T>(f[4], f[5]), pair_of<T>(f[6], f[7]));
}

struct RopeP {
    const void *q, *k, *dq, *dk;      // dq, dk: gradient form only
    void *qo, *ko;
    const int32_t* pos;
    const double* freqs;
    const float *qg, *kg;
    float* part;                      // gradient form: (workgroups, 2, hd) partial sums of dg
    int ldq, ldk, lddq, lddk, ldqo, ldko;
    int rows, heads, kv_heads, rot, inter, tok, run;
    float eps;
};

constexpr int MAXTOK = 4;

// sum over the N lanes of an aligned group, in all of them: lane exchanges that cost no instruction of their own
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int N> __device__ __forceinline__ float group_sum(float v) {
    static_assert(N == 2 || N == 4 || N == 8 || N == 16 || N == 32, "lanes of a head row");
    v = add_dpp<0xb1>(v);                            // lane ^ 1
    if constexpr (N >= 4) v = add_dpp<0x4e>(v);      // lane ^ 2
    if constexpr (N >= 8) v = add_dpp<0x141>(v);     // the other half of 8
    if constexpr (N >= 16) v = add_dpp<0x140>(v);    // the other half of 16
    if constexpr (N >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

// 1 / sqrt(v) to an ulp; the instruction takes subnormals for zero
__device__ __forceinline__ float rsqrt_(float v) {
    const bool small = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p60f : v);
    return small ? r * 0x1p30f : r;
}

template <typename T, int HD, bool BWD, int R> __global__ __launch_bounds__(256) void qk_rope_kernel(const RopeP p) {
    constexpr int LPH = HD / (2 * R), NG = 256 / LPH;      // lanes per head row, head rows in flight per workgroup
    __shared__ float2 turn[MAXTOK][HD / 2];
    const int tid = threadIdx.x, j = tid % LPH, grp = tid / LPH;
    const int nh = p.heads + p.kv_heads, half = p.rot >> 1;
    const bool turned = 2 * R * j < p.rot;
    // the two runs of 4 elements this lane holds, and its first pair (pairs pr .. pr + 3)
    const int lo = turned && !p.inter ? R * j : 2 * R * j;
    const int hi = turned && !p.inter ? half + R * j : 2 * R * j + R;
    const int pr = R * j;
    float gq[2 * R], gk[2 * R], sq[2 * R], sk[2 * R];
#pragma unroll
    for (int e = 0; e < 2 * R; ++e) {
        const int d = (e < R ? lo : hi - R) + e;
        gq[e] = p.qg ? p.qg[d] : 1.f;
        gk[e] = p.kg ? p.kg[d] : 1.f;
        sq[e] = sk[e] = 0.f;
    }
    // the workgroup's head rows: those of q, then those of k, tokens outermost; a group of lanes takes every step-th
    const int step = NG * gridDim.y, first = blockIdx.y * NG + grp;
    const int nblk = (p.rows + p.tok - 1) / p.tok;
    for (int blk = blockIdx.x; blk < nblk; blk += gridDim.x) {
        const int t0 = blk * p.tok, nt = min(p.tok, p.rows - t0);
        for (int i = tid; i < nt * half; i += 256) {
            const int t = i / half, c = i - t * half;
            const double rev = (double)p.pos[t0 + t] * p.freqs[c];
            float s, cs;
            sincospif((float)(2.0 * (rev - rint(rev))), &s, &cs);
            turn[t][c] = make_float2(cs, s);
        }
        __syncthreads();
        auto rows_of = [&](const void* xp, int ldx, const void* dyp, int lddy, void* yp, int ldy, int heads, int from, const float* gain, float* sum) {
            const int dt = step / heads, dh = step - dt * heads;
            int t = from / heads, h = from - t * heads;
            for (; t < nt;) {
                const size_t row = t0 + t;
                const T* x = (const T*)xp + row * ldx + h * HD;
                float f[2 * R], z[2 * R];
                ldr<R, !BWD>(x + lo, f);
                ldr<R, !BWD>(x + hi, f + R);
                if constexpr (BWD) {
                    const T* dy = (const T*)dyp + row * lddy + h * HD;
                    ldr<R, !BWD>(dy + lo, z);
                    ldr<R, !BWD>(dy + hi, z + R);
                }
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 2 * R; ++e) ss += f[e] * f[e];
                const float r = rsqrt_(group_sum<LPH>(ss) * (1.f / HD) + p.eps);
                float* v = BWD ? z : f;
                if constexpr (!BWD) {
#pragma unroll
                    for (int e = 0; e < 2 * R; ++e) f[e] = f[e] * r * gain[e];
                }
                if (turned) {
#pragma unroll
                    for (int e = 0; e < R; ++e) {
                        const float2 cs = turn[t][pr + e];
                        const float s = BWD ? -cs.y : cs.y;
                        if (p.inter) {
                            const float a = v[2 * e], b = v[2 * e + 1];
                            v[2 * e] = a * cs.x - b * s;
                            v[2 * e + 1] = b * cs.x + a * s;
                        } else {
                            const float a = v[e], b = v[R + e];
                            v[e] = a * cs.x - b * s;
                            v[R + e] = b * cs.x + a * s;
                        }
                    }
                }
                if constexpr (BWD) {
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 2 * R; ++e) {
                        f[e] *= r;
                        sum[e] += z[e] * f[e];
                        z[e] *= gain[e];
                        dot += f[e] * z[e];
                    }
                    dot = group_sum<LPH>(dot) * (1.f / HD);
#pragma unroll
                    for (int e = 0; e < 2 * R; ++e) z[e] = r * (z[e] - f[e] * dot);
                }
                T* y = (T*)yp + row * ldy + h * HD;
                str<R>(y + lo, v);
                str<R>(y + hi, v + R);
                t += dt;
                h += dh;
                if (h >= heads) h -= heads, ++t;
            }
        };
        if (p.heads) rows_of(p.q, p.ldq, p.dq, p.lddq, p.qo, p.ldqo, p.heads, first, gq, sq);
        const int past = nt * p.heads - first;      // the head rows of q behind this group's first, to the next multiple of step
        if (p.kv_heads) rows_of(p.k, p.ldk, p.dk, p.lddk, p.ko, p.ldko, p.kv_heads, past > 0 ? (past + step - 1) / step * step - past : -past, gk, sk);
        __syncthreads();
    }
    if constexpr (BWD) {      // the workgroup's share of dg: head rows in flight added in order
        __shared__ float red[2][NG][HD];
#pragma unroll
        for (int e = 0; e < 2 * R; ++e) {
            const int d = (e < R ? lo : hi - R) + e;
            red[0][grp][d] = sq[e];
            red[1][grp][d] = sk[e];
        }
        __syncthreads();
        for (int i = tid; i < 2 * HD; i += 256) {
            const int w = i / HD, d = i - w * HD;
            float s = 0.f;
            for (int g = 0; g < NG; ++g) s += red[w][g][d];
            p.part[(size_t)blockIdx.x * (2 * HD) + i] = s;
        }
    }
}

// dg[i] = sum over the n workgroups of part[w][i], in a fixed order (fp64: up to 1024 terms).  16 outputs per workgroup, 64 threads each, so
// that a thread's share of the terms is loaded at once.
__global__ __launch_bounds__(1024) void qk_rope_gain_kernel(const float* __restrict__ part, int n, int hd, float* __restrict__ dqg,
                                                            float* __restrict__ dkg) {
    __shared__ double red[64][17];
    const int c = threadIdx.x & 15, s = threadIdx.x >> 4, i = blockIdx.x * 16 + c;
    double a = 0;
    for (int w = s; w < n; w += 64 * 8) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = part[(size_t)min(w + 64 * k, n - 1) * (2 * hd) + i];
#pragma unroll
        for (int k = 0; k < 8; ++k) a += w + 64 * k < n ? f[k] : 0.f;
    }
    red[s][c] = a;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        __syncthreads();
        if (s < o) red[s][c] = a += red[s + o][c];
    }
    if (s == 0) {
        float* out = i < hd ? dqg : dkg;
        if (out) out[i < hd ? i : i - hd] = (float)a;
    }
}

// Tokens per workgroup that share one pass over the angles.  1 / 2 / 4 of them, us: 128 tokens 3.7 / 5.0 / 6.4 (40 heads of 128, bf16), 3.1 / 3.1 / 3.9
// (16 of 64, fp32); 1024: 9.6 / 6.9 / 8.1, 4.5 / 3.9 / 4.5; 4096: 32.7 / 18.5 / 16.6, 11.8 / 9.1 / 8.1; the gradient's are closer together.
int rope_tok(int rows) { return rows >= 2500 ? MAXTOK : rows >= 512 ? 2 : 1; }
int rope_bwd_groups(int rows) {
    const int n = (rows + rope_tok(rows) - 1) / rope_tok(rows);
    return n < 1024 ? n : 1024;
}

int check(int dtype, const RopeP& p, int hd, bool bwd) {
    PGT_CHECK(dtype == PGT_F32 || dtype == PGT_BF16 || dtype == PGT_F16, "qk_norm_rope: bad dtype %d", dtype);
    PGT_CHECK(hd == 32 || hd == 64 || hd == 128 || hd == 256, "qk_norm_rope: head_dim=%d unsupported (32, 64, 128, 256)", hd);
    PGT_CHECK(p.rows >= 0 && p.heads >= 0 && p.kv_heads >= 0 && p.heads + p.kv_heads > 0 && (int64_t)p.heads * hd < (1 << 30) &&
              (int64_t)p.kv_heads * hd < (1 << 30), "qk_norm_rope: rows=%d heads=%d kv_heads=%d", p.rows, p.heads, p.kv_heads);
    PGT_CHECK(p.rot >= 0 && p.rot <= hd && p.rot % 8 == 0, "qk_norm_rope: %d rotated elements of %d (a multiple of 8)", p.rot, hd);
    PGT_CHECK(p.eps >= 0.f, "qk_norm_rope: eps=%g", p.eps);
    PGT_CHECK(!p.heads || p.rows == 0 || (p.q && p.qo && (!bwd || p.dq)), "qk_norm_rope: null argument");
    PGT_CHECK(!p.kv_heads || p.rows == 0 || (p.k && p.ko && (!bwd || p.dk)), "qk_norm_rope: null argument");
    PGT_CHECK(!p.rot || p.rows == 0 || (p.pos && p.freqs), "qk_norm_rope: a rotation needs positions and freqs");
    const int al = dtype == PGT_F32 ? 4 : 8;      // elements of 16 bytes
    const int nq = p.heads ? 1 : 0, nk = p.kv_heads ? 1 : 0;
    PGT_CHECK((!nq || (p.ldq >= p.heads * hd && p.ldqo >= p.heads * hd && (!bwd || p.lddq >= p.heads * hd))) &&
              (!nk || (p.ldk >= p.kv_heads * hd && p.ldko >= p.kv_heads * hd && (!bwd || p.lddk >= p.kv_heads * hd))),
              "qk_norm_rope: a row stride is shorter than its row");
    PGT_CHECK(nq * (p.ldq | p.ldqo | (bwd ? p.lddq : 0)) % al == 0 && nk * (p.ldk | p.ldko | (bwd ? p.lddk : 0)) % al == 0,
              "qk_norm_rope: row strides must be multiples of 16 bytes");
    const uintptr_t a = nq * ((uintptr_t)p.q | (uintptr_t)p.qo | (uintptr_t)p.dq) | nk * ((uintptr_t)p.k | (uintptr_t)p.ko | (uintptr_t)p.dk);
    PGT_CHECK((a & 15) == 0, "qk_norm_rope: misaligned pointer");
    return 0;
}

template <bool BWD> void launch(int dtype, int hd, const RopeP& p, dim3 grid, hipStream_t st) {
#define ROPE_GO(TT, HD)                                                                                                   \
    do {                                                                                                                  \
        if constexpr (!BWD && !__is_same(TT, float)) {                                                                    \
            if (p.run == 8) {                                                                                             \
                hipLaunchKernelGGL((qk_rope_kernel<TT, HD, false, 8>), grid, dim3(256), 0, st, p);                        \
                break;                                                                                                    \
            }                                                                                                             \
        }                                                                                                                 \
        hipLaunchKernelGGL((qk_rope_kernel<TT, HD, BWD, 4>), grid, dim3(256), 0, st, p);                                  \
    } while (0)
#define ROPE_HD(TT)                                                                                                       \
    do {                                                                                                                  \
        if (hd == 32) ROPE_GO(TT, 32);                                                                                    \
        else if (hd == 64) ROPE_GO(TT, 64);                                                                               \
        else if (hd == 128) ROPE_GO(TT, 128);                                                                             \
        else ROPE_GO(TT, 256);                                                                                            \
    } while (0)
    if (dtype == PGT_F32) ROPE_HD(float);
    else if (dtype == PGT_BF16) ROPE_HD(bf16_t);
    else ROPE_HD(half_t);
#undef ROPE_HD
#undef ROPE_GO
}

}  // namespace

extern "C" int pgt_qk_norm_rope(int32_t dtype, const void* q, int32_t ldq, const void* k, int32_t ldk, int32_t rows, int32_t heads,
                                int32_t kv_heads, int32_t hd, const int32_t* positions, const double* freqs, int32_t rot,
                                int32_t interleaved, const float* q_gain, const float* k_gain, float eps, void* q_out, int32_t ldqo,
                                void* k_out, int32_t ldko, pgt_stream_t stream) {
    RopeP p = {};
    p.q = q; p.k = k; p.qo = q_out; p.ko = k_out; p.pos = positions; p.freqs = freqs; p.qg = q_gain; p.kg = k_gain;
    p.ldq = ldq; p.ldk = ldk; p.ldqo = ldqo; p.ldko = ldko;
    p.rows = rows; p.heads = heads; p.kv_heads = kv_heads; p.rot = rot; p.inter = interleaved != 0; p.eps = eps;
    if (const int rc = check(dtype, p, hd, false)) return rc;
    if (rows == 0) return 0;
    p.tok = rope_tok(rows);
    // runs of 16 bytes of a 16-bit type where the pairs allow it: 16411 tokens 65 instead of 74 us; with a token per workgroup the longer way of a
    // lane costs more (4 tokens: 4.7 instead of 3.9)
    p.run = dtype != PGT_F32 && rot % 16 == 0 && p.tok > 1 ? 8 : 4;
    const int ng = 256 / (hd / (2 * p.run)), nh = heads + kv_heads;
    const int nblk = (rows + p.tok - 1) / p.tok;      // (a grid's threads are counted in 32 bits: a workgroup takes every 2^22-th block of tokens)
    const dim3 grid(nblk < (1 << 22) ? nblk : 1 << 22, p.tok == 1 ? (nh + ng - 1) / ng : 1);
    PGT_CHECK(grid.y <= 65535, "qk_norm_rope: %d heads", nh);
    launch<false>(dtype, hd, p, grid, (hipStream_t)stream);
    PGT_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t pgt_qk_norm_rope_backward_workspace_bytes(int32_t rows, int32_t hd) {
    return rows <= 0 || hd <= 0 ? 0 : (size_t)rope_bwd_groups(rows) * 2 * hd * sizeof(float);
}

extern "C" int pgt_qk_norm_rope_backward(int32_t dtype, const void* dq, int32_t lddq, const void* dk, int32_t lddk, const void* q,
                                         int32_t ldq, const void* k, int32_t ldk, int32_t rows, int32_t heads, int32_t kv_heads,
                                         int32_t hd, const int32_t* positions, const double* freqs, int32_t rot, int32_t interleaved,
                                         const float* q_gain, const float* k_gain, float eps, void* dq_in, int32_t lddqi, void* dk_in,
                                         int32_t lddki, float* dq_gain, float* dk_gain, void* workspace, size_t workspace_bytes,
                                         pgt_stream_t stream) {
    RopeP p = {};
    p.q = q; p.k = k; p.dq = dq; p.dk = dk; p.qo = dq_in; p.ko = dk_in; p.pos = positions; p.freqs = freqs; p.qg = q_gain; p.kg = k_gain;
    p.ldq = ldq; p.ldk = ldk; p.lddq = lddq; p.lddk = lddk; p.ldqo = lddqi; p.ldko = lddki;
    p.rows = rows; p.heads = heads; p.kv_heads = kv_heads; p.rot = rot; p.inter = interleaved != 0; p.eps = eps;
    if (const int rc = check(dtype, p, hd, true)) return rc;
    const size_t need = pgt_qk_norm_rope_backward_workspace_bytes(rows, hd);
    PGT_CHECK(workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0)),
              "qk_norm_rope_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    p.part = (float*)workspace;
    p.tok = rope_tok(rows);
    hipStream_t st = (hipStream_t)stream;
    const int groups = rows ? rope_bwd_groups(rows) : 0;
    if (rows) launch<true>(dtype, hd, p, dim3(groups), st);
    PGT_LAUNCH_CHECK();
    if (dq_gain || dk_gain)
        hipLaunchKernelGGL(qk_rope_gain_kernel, dim3(2 * hd / 16), dim3(1024), 0, st, p.part, groups, hd, dq_gain, dk_gain);
    PGT_LAUNCH_CHECK();
    return 0;
}
