// The 8-bit key-value cache: quantising tokens into its pages, reading them back, and attention over
// them. Layout and index arithmetic: onpu_kv8.h.
#include <algorithm>

#include "onpu_launch.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int KT = 256;                       // threads per workgroup

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// 16 (8) consecutive values, fp32 or bf16, as they lie
template <bool F32> struct Raw16 { uint4 u[F32 ? 4 : 2]; };
template <bool F32> struct Raw8 { uint4 u[F32 ? 2 : 1]; };
template <bool F32, class R> __device__ __forceinline__ R load_raw(const void * base, int64_t at) {
    const uint4 * p = F32 ? (const uint4 *) ((const float *) base + at) : (const uint4 *) ((const uint16_t *) base + at);
    R r;
#pragma unroll
    for (size_t i = 0; i < sizeof(R) / 16; i++) r.u[i] = p[i];
    return r;
}
template <bool F32, class R> __device__ __forceinline__ float raw_at(const R & r, int e) {
    const uint4 u = r.u[F32 ? e >> 2 : e >> 3];
    const int w = F32 ? e & 3 : (e >> 1) & 3;
    const uint32_t x = w == 0 ? u.x : (w == 1 ? u.y : (w == 2 ? u.z : u.w));
    return F32 ? __uint_as_float(x) : (e & 1 ? bf_hi(x) : bf_lo(x));
}
template <bool F32> __device__ __forceinline__ void load16(const void * base, int64_t at, float (&x)[16]) {
    const Raw16<F32> r = load_raw<F32, Raw16<F32>>(base, at);
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = raw_at<F32>(r, e);
}

// ------------------------------------------------------------------ write
// A workgroup per (touched page, kv head, sequence). Per K and V: a = max |x| of the new values, s = max(a, 2^-96) / 127
// (and the page's own scale, where it holds earlier tokens, if that is larger; their codes are then
// rescaled when s grew), code = x / s to the nearest, ties to even, of the exact quotient: with c the
// nearest integer of x * (1 / s), x - c s is exact in one fma (a multiple of half an ulp of s and below s), so that
// a c one off near a border is put right by comparing it with s / 2. A value that is not finite makes
// the page's scale NaN, and all that is read of it. Bound by the bytes for prompts: each value is read once
// and stays in registers across the maximum (a lane has 16 d of a K token and 8 d of 4 V tokens, so that
// V's bytes of 4 tokens are whole words); K's codes go out from there, V's through LDS in the page's
// order. A page with earlier tokens is changed in place, its new bytes alone unless the scale grows.
// 8192 tokens x 8 x 128 bf16: 17.0 us for 50 MB, 3.0 TB/s (all pages are on the card at once, so the loads, the
// codes' arithmetic and the stores follow one another: 44 % of the waves' cycles wait); one token: 4.4 us, the latency
// of position, table, scale and row in turn.
struct WriteArgs {
    Kv8Cache c;
    Kv8Table t;
    const void * x[2];
    int64_t rs[2], hs[2];
    int W;                                    // pages a sequence can touch
};

__device__ __forceinline__ int quant(float x, float s, float inv) {
    float c = rintf(x * inv);
    const float e = fmaf(-c, s, x), h = 0.5f * s;
    const bool odd = ((int) c) & 1;
    if (e > h || (e == h && odd)) c += 1.f;
    if (e < -h || (e == -h && odd)) c -= 1.f;
    return (int) fminf(fmaxf(c, -127.f), 127.f);
}
// The codes of four values, their lowest bytes: c = x / s + 1.5 2^23 in one fma has the nearest integer of x * (1 / s) in
// its last bits, right unless x - c s is all but s / 2. For fp32 `far`, the largest |x - c s| so far, tells (within
// 2^-16 s of s / 2, three values of 10^5): then quant decides. bf16 values of a page whose largest is bf16 as well fall
// there in almost every wave, so each is put right at once by comparing with s / 2, and far is s / 2 after an exact tie.
// (8192 tokens x 8 x 128 bf16, K and V: 19.5 us with far alone, 17.8 with this.)
template <bool F32> __device__ __forceinline__ uint32_t near4(const float (&x)[4], float s, float inv, float & far) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float c = fmaf(x[e], inv, 12582912.f), r = fmaf(-(c - 12582912.f), s, x[e]);
        if (F32) {
            far = fmaxf(far, fabsf(r));
            y[e] = __float_as_uint(c);
        } else {
            const float h = 0.5f * s;
            far = fabsf(r) == h ? h : far;
            y[e] = __float_as_uint(fabsf(r) > h ? c + copysignf(1.f, r) : c);
        }
    }
    return __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u) | __builtin_amdgcn_perm(y[3], y[2], 0x04000c0cu);
}
// the largest |value| of raw words, as bits (NaN the largest)
template <bool F32> __device__ __forceinline__ uint32_t raw_max(uint32_t m, uint4 u) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
        m = F32 ? max(m, w[e] & 0x7fffffffu)
                : __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                         __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu)));
    return m;
}
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
    return (uint32_t) (a & 255) | (uint32_t) (b & 255) << 8 | (uint32_t) (c & 255) << 16 | (uint32_t) d << 24;
}

template <bool F32> __device__ __forceinline__ float one_at(const void * x, int64_t at) {
    return F32 ? ((const float *) x)[at] : bf16_to_f32(((const uint16_t *) x)[at]);
}

// the scale of values whose largest magnitude has these bits
__device__ __forceinline__ float scale_for(uint32_t bits) {
    return bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(bits), KV8_TINY) / 127.f;
}

// Where word w of V's codes is in LDS: a lane turns the words of 4 or 8 d, lanes differ in 16 d and in the token's quad,
// which are 256 and 64 words apart; 4 words between every 256 leave 16 banks of 64 to them instead of 2
// (8192 tokens x 8 x 128 bf16 written in 17.0 us, read in 10.6; without 17.8, 11.9).
__device__ __forceinline__ int vt_at(int w) { return w + (w >> 8) * 4; }

// NQ: D up to 128 NQ
template <bool F32, int NQ>
__global__ __launch_bounds__(KT) void k_kv8_write(WriteArgs a) {
    constexpr int NK = 2 * NQ, NV = NQ;       // units of a lane: 16 d of one K token, 8 d of 4 V tokens
    extern __shared__ __align__(16) uint32_t vt[];               // V's 64 D codes (vt_at)
    __shared__ uint32_t wmax[2][KT / 64];
    const int D = a.c.D, NC = D / 16, t = threadIdx.x, g = blockIdx.x % a.c.Hkv, w = blockIdx.x / a.c.Hkv, i = blockIdx.y;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int64_t p0 = a.t.pos[i], pg = (p0 < 0 ? 0 : p0) / KV8_PAGE + w, base = pg * KV8_PAGE;
    if (p0 < 0 || base >= p0 + r.n) return;
    const int id = kv8_page(a.t.table + i * a.t.tld, pg, a.t.P, a.c.pages);
    if (id < 0) return;
    const int s0 = p0 > base ? (int) (p0 - base) : 0, s1 = p0 + r.n - base < KV8_PAGE ? (int) (p0 + r.n - base) : KV8_PAGE;
    const int64_t row0 = r.row + (base - p0);                    // the row of slot 0 (below the sequence's for s0 > 0)
    int8_t * out = a.c.codes + ((int64_t) id * a.c.Hkv + g) * 2 * KV8_PAGE * D;
    float * sc = a.c.scales + ((int64_t) id * a.c.Hkv + g) * 2;
    const float so[2] = {s0 > 0 ? sc[0] : 0.f, s0 > 0 ? sc[1] : 0.f};
    const bool some = s1 - s0 < 8;            // few tokens: a lane has one value at a time
    uint32_t m[2] = {0, 0};
    Raw16<F32> xk[NK];
    Raw8<F32> xv[NV][4];
    if (some) {
        for (int kv = 0; kv < 2; kv++)
            for (int u = t; u < (s1 - s0) * D; u += KT) {
                const int64_t at = (row0 + s0 + u / D) * a.rs[kv] + g * a.hs[kv] + u % D;
                m[kv] = max(m[kv], __float_as_uint(fabsf(one_at<F32>(a.x[kv], at))));
            }
    } else {
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int u = t + KT * k, tok = u / NC, ok = tok >= s0 && tok < s1;
            xk[k] = load_raw<F32, Raw16<F32>>(a.x[0], (row0 + (ok ? tok : s0)) * a.rs[0] + g * a.hs[0] + u % NC * 16);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int u = t + KT * k, q = u / (2 * NC), d = u % (2 * NC) * 8;      // tokens 4 q .. 4 q + 3
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int tok = 4 * q + e, ok = tok >= s0 && tok < s1;
                xv[k][e] = load_raw<F32, Raw8<F32>>(a.x[1], (row0 + (ok ? tok : s0)) * a.rs[1] + g * a.hs[1] + d);
            }
        }
#pragma unroll
        for (int k = 0; k < NK; k++)          // (slots outside repeat slot s0: the maximum is of the new values)
#pragma unroll
            for (size_t e = 0; e < sizeof(xk[0]) / 16; e++) m[0] = raw_max<F32>(m[0], xk[k].u[e]);
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (size_t e = 0; e < sizeof(xv[0][0]) / 16; e++) m[1] = raw_max<F32>(m[1], xv[k][n].u[e]);
        if (!F32)                             // (two bf16 maxima a word)
#pragma unroll
            for (int kv = 0; kv < 2; kv++) m[kv] = max(m[kv] << 16, m[kv] & 0xffff0000u);
    }
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        for (int o = 32; o > 0; o >>= 1) m[kv] = max(m[kv], (uint32_t) __shfl_xor((int) m[kv], o));       // (NaN is the largest)
        if ((t & 63) == 0) wmax[kv][t >> 6] = m[kv];
    }
    __syncthreads();
    float s[2], inv[2];
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        uint32_t b = wmax[kv][0];
#pragma unroll
        for (int k = 1; k < KT / 64; k++) b = max(b, wmax[kv][k]);
        s[kv] = scale_for(b);
        if (s0 > 0 && !(so[kv] <= s[kv])) s[kv] = s[kv] != s[kv] ? s[kv] : so[kv];          // (a NaN stays)
        inv[kv] = 1.f / s[kv];
        if (s0 > 0 && s[kv] > so[kv]) {       // the earlier codes in the new scale
            const double f = (double) so[kv] / (double) s[kv];
            uint4 * p = (uint4 *) (out + kv * KV8_PAGE * D);
            for (int u = t; u < 4 * D; u += KT) {
                uint32_t y[4] = {p[u].x, p[u].y, p[u].z, p[u].w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[e] = bytes4((int) rint((int8_t) y[e] * f), (int) rint((int8_t) (y[e] >> 8) * f),
                                  (int) rint((int8_t) (y[e] >> 16) * f), (int) rint((int8_t) (y[e] >> 24) * f));
                p[u] = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
    }
    if (s0 > 0) __syncthreads();              // the new bytes go on top (and so has been read by all)
    if (t < 2) sc[t] = t ? s[1] : s[0];
    const float lim[2] = {s[0] * 0.4999847f, s[1] * 0.4999847f};
    if (some && s0 > 0) {
        for (int kv = 0; kv < 2; kv++)
            for (int u = t; u < (s1 - s0) * D; u += KT) {
                const int tok = s0 + u / D, d = u % D;
                const int64_t at = (row0 + tok) * a.rs[kv] + g * a.hs[kv] + d;
                const float x = one_at<F32>(a.x[kv], at);
                out[kv ? KV8_PAGE * D + kv8_v_at(D, tok, d) : kv8_k_at(D, tok, d)] = (int8_t) quant(x, s[kv], inv[kv]);
            }
        return;
    }
    if (some) {                               // a page begun by a few tokens
        for (int u = t; u < 16 * D; u += KT) {
            const int tok = u / (D / 4), d = u % (D / 4) * 4;
            uint32_t y = 0;
            if (tok < s1) {
                int q[4];
                for (int e = 0; e < 4; e++) {
                    const int64_t at = (row0 + tok) * a.rs[0] + g * a.hs[0] + d + e;
                    q[e] = quant(one_at<F32>(a.x[0], at), s[0], inv[0]);
                }
                y = bytes4(q[0], q[1], q[2], q[3]);
            }
            *(uint32_t *) (out + kv8_k_at(D, tok, d)) = y;
            const int vq = u / D, vd = u % D;                    // tokens 4 vq .. 4 vq + 3
            y = 0;
            for (int e = 0; e < 4; e++)
                if (4 * vq + e < s1) {
                    const int64_t at = (row0 + 4 * vq + e) * a.rs[1] + g * a.hs[1] + vd;
                    y |= (uint32_t) (quant(one_at<F32>(a.x[1], at), s[1], inv[1]) & 255) << (8 * e);
                }
            *(uint32_t *) (out + KV8_PAGE * D + kv8_v_at(D, 4 * vq, vd)) = y;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const int u = t + KT * k, tok = u / NC, d = u % NC * 16;
        if (tok >= KV8_PAGE || tok < s0 || (s0 > 0 && tok >= s1)) continue;
        uint32_t y[4];
        float far = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x[4] = {raw_at<F32>(xk[k], 4 * e), raw_at<F32>(xk[k], 4 * e + 1), raw_at<F32>(xk[k], 4 * e + 2),
                                raw_at<F32>(xk[k], 4 * e + 3)};
            y[e] = near4<F32>(x, s[0], inv[0], far);
        }
        if (far > lim[0])
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] = bytes4(quant(raw_at<F32>(xk[k], 4 * e), s[0], inv[0]), quant(raw_at<F32>(xk[k], 4 * e + 1), s[0], inv[0]),
                              quant(raw_at<F32>(xk[k], 4 * e + 2), s[0], inv[0]), quant(raw_at<F32>(xk[k], 4 * e + 3), s[0], inv[0]));
        if (tok >= s1) y[0] = y[1] = y[2] = y[3] = 0;
        *(uint4 *) (out + kv8_k_at(D, tok, d)) = make_uint4(y[0], y[1], y[2], y[3]);
    }
    const bool merge = s0 > 0;                // V's words of the page as they are below the new bytes
    int8_t * ov = out + KV8_PAGE * D;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int u = t + KT * k, q = u / (2 * NC), d = u % (2 * NC) * 8;
        if (q >= 16) continue;
        uint32_t keep = 0;                    // bytes of tokens that are not new
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (4 * q + e < s0 || 4 * q + e >= s1) keep |= 255u << (8 * e);
        if (merge && keep == 0xffffffffu) continue;
        uint32_t y[8];
        float far = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x[4] = {raw_at<F32>(xv[k][0], e), raw_at<F32>(xv[k][1], e), raw_at<F32>(xv[k][2], e),
                                raw_at<F32>(xv[k][3], e)};
            y[e] = near4<F32>(x, s[1], inv[1], far);
        }
        if (far > lim[1])
#pragma unroll
            for (int e = 0; e < 8; e++)
                y[e] = bytes4(quant(raw_at<F32>(xv[k][0], e), s[1], inv[1]), quant(raw_at<F32>(xv[k][1], e), s[1], inv[1]),
                              quant(raw_at<F32>(xv[k][2], e), s[1], inv[1]), quant(raw_at<F32>(xv[k][3], e), s[1], inv[1]));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int at = kv8_v_at(D, 4 * q, d + e);
            if (merge) *(uint32_t *) (ov + at) = (y[e] & ~keep) | (keep ? *(uint32_t *) (ov + at) & keep : 0);
            else vt[vt_at(at / 4)] = y[e] & ~keep;
        }
    }
    if (merge) return;
    __syncthreads();
    for (int u = t; u < 4 * D; u += KT) ((uint4 *) ov)[u] = *(const uint4 *) (vt + vt_at(4 * u));
}

// ------------------------------------------------------------------ read
// A workgroup per (page, kv head, sequence): value = code * scale, rounded once (bf16: that rounded
// again); code + 128 by an unsigned byte's conversion, less 128 in the product's fma, whose one rounding is
// the product's. A page that the table does not have reads as NaN. Bound by the bytes: a lane writes 16 bytes of a
// K row or of 4 V rows, so that a wave's stores are whole lines (16 d a lane, fp32: 16 prompts of up to 1500 of
// 4 x 96 15.9 us, so 11.6), V's words turned through LDS. 8192 tokens x 8 x 128 to bf16: 10.6 us for 50 MB, 4.7 TB/s.
struct ReadArgs {
    Kv8Cache c;
    Kv8Table t;
    void * y[2];
    int W;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// N values (fp32 4, bf16 8: 16 bytes) to `at` of y
template <bool F32, int N> __device__ __forceinline__ void put(void * y, int64_t at, const float (&v)[N]) {
    if (F32) {
#pragma unroll
        for (int e = 0; e < N; e += 4) *(float4 *) ((float *) y + at + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 8)
            *(uint4 *) ((uint16_t *) y + at + e) = make_uint4(pack_bf16(v[e], v[e + 1]), pack_bf16(v[e + 2], v[e + 3]),
                                                              pack_bf16(v[e + 4], v[e + 5]), pack_bf16(v[e + 6], v[e + 7]));
    }
}

template <bool F32>
__global__ __launch_bounds__(KT) void k_kv8_read(ReadArgs a) {
    extern __shared__ __align__(16) uint32_t vt[];               // V's 64 D codes (vt_at)
    const int D = a.c.D, t = threadIdx.x, g = blockIdx.x % a.c.Hkv, w = blockIdx.x / a.c.Hkv, i = blockIdx.y;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int64_t p0 = a.t.pos[i], pg = (p0 - (p0 & (KV8_PAGE - 1))) / KV8_PAGE + w, base = pg * KV8_PAGE;
    if (base >= p0 + r.n) return;
    const int id = kv8_page(a.t.table + i * a.t.tld, pg, a.t.P, a.c.pages);
    const int s0 = p0 > base ? (int) (p0 - base) : 0, s1 = p0 + r.n - base < KV8_PAGE ? (int) (p0 + r.n - base) : KV8_PAGE;
    const int64_t row0 = r.row + (base - p0);
    const int8_t * in = a.c.codes + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2 * KV8_PAGE * D;
    const float * sc = a.c.scales + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2;
    for (int u = t; u < 4 * D; u += KT) *(uint4 *) (vt + vt_at(4 * u)) = ((const uint4 *) (in + KV8_PAGE * D))[u];
    const float nan = __uint_as_float(0x7fc00000u), sk = id < 0 ? nan : sc[0], sv = id < 0 ? nan : sc[1];
    constexpr int E = F32 ? 4 : 8;            // 16 bytes of a row a lane, so that a wave's stores are whole lines
    const int per = D / E;
    for (int u = s0 * per + t; u < s1 * per; u += KT) {
        const int tok = u / per, d = u % per * E;
        const uint32_t * p = (const uint32_t *) (in + kv8_k_at(D, tok, d));
        float v[E];
#pragma unroll
        for (int k = 0; k < E / 4; k++) {
            const uint32_t x = p[k] ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * k + e] = fmaf((float) (x >> (8 * e) & 255), sk, -128.f * sk);
        }
        put<F32, E>(a.y[0], ((row0 + tok) * a.c.Hkv + g) * D + d, v);
    }
    __syncthreads();
    for (int u = (s0 >> 2) * per + t; u < ((s1 + 3) >> 2) * per; u += KT) {
        const int q = u / per, d = u % per * E;
        uint32_t x[E];
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = vt[vt_at(kv8_v_at(D, 4 * q, d + e) / 4)] ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (4 * q + k < s0 || 4 * q + k >= s1) continue;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = fmaf((float) (x[e] >> (8 * k) & 255), sv, -128.f * sv);
            put<F32, E>(a.y[1], ((row0 + 4 * q + k) * a.c.Hkv + g) * D + d, v);
        }
    }
}

// ------------------------------------------------------------------ attention
struct Kv8AttnArgs {
    Kv8Cache c;
    Kv8Table t;                               // t.pos: tokens of each sequence, the new ones among them
    const void * q;
    void * out;
    const float * mask, * sinks;
    float * ws;                               // partials of C-token chunks: o [T Hq][nch][D], then (max, sum) [T Hq][nch]
    int64_t qrs, qhs, mld;
    float scale;
    int Hq, rep, max_len, window, f32, C, nch, fold;
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
constexpr float LOG2E = 1.44269504088896341f;

// a workgroup barrier that orders LDS accesses only: global loads stay in flight across it
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// values [at, at + 4) of a page's mask, of which the first `have` exist (uniform); 0 for the others
__device__ __forceinline__ f32x4 mask4(const float * page, int at, int have) {
    struct __attribute__((packed, aligned(4))) V { f32x4 v; };   // (rows start anywhere)
    if (have >= KV8_PAGE) return ((const V *) (page + at))->v;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *) page, (short) 0, 4 * have, 0x00020000);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, 4 * (at + e), 0, 0));
    return v;
}

template <bool NT> __device__ __forceinline__ uint4 load_code(const int8_t * p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return NT ? __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u4 *) p)) : *(const uint4 *) p;
}

// the larger (or the sum) of x and the lane 32, then 16 away
template <bool MAX> __device__ __forceinline__ float across_quads(float x) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = MAX ? fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)) : __uint_as_float(r.x) + __uint_as_float(r.y);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return MAX ? fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)) : __uint_as_float(r.x) + __uint_as_float(r.y);
}
// the sum over the 4 lanes of a quad permute, the same bits in each
__device__ __forceinline__ float quad_sum(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, false));
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, false));
}

// Few query rows (a decode token, a verification): bound by the cache's bytes, so the codes go to the int8
// matrix instructions as they lie in memory, with nothing converted, and the fp32 side is cut into int8
// instead. A row of q is a fixed-point number of 31 bits below its largest |q| (to 2^-31 of it: more than
// fp32's own), in four signed bytes; the four are rows 4 h + part of a 16-row operand that holds 4 heads, their
// integer sums exact. The scores come out as lane (row 4 h + part, quad), token 16 a + 4 quad + c: the
// order of V's bytes, so the lane's weights, cut the same way (weight e^(x - m) <= 1 to 2^-31), are the other
// product's operand without a move across lanes. A wave takes every SW-th page, K of its next one loading
// once this one's scores are out, V after its products; waves meet in LDS, chunks in k_kv8_join or k_kv8_combine.
// RS sets of 4 rows; NC: chunks of 16 d (D / 16 or more); NT: non-temporal loads of the codes.
// 32 / 8 heads of 128: 65536 tokens 24.7 us (134 MB, 5.4 TB/s); 64 sequences of up to 8192 107 us (578 MB, 5.4 TB/s
// of the 7.07 that streaming reads reach; FETCH_SIZE 1.014 times the codes). 200 tokens 6.2 us, the latency of lens,
// table and codes in turn and the waves' joint. 64 / 8 heads of 64, a window of 4000 of 16 sequences: 17.8 us
// (66 MB, 3.7 TB/s: two sets' cuts and softmax on half the bytes a page).
template <int NC, int RS, int SW, bool MASK, bool NT>
__global__ __launch_bounds__(64 * SW, SW == 8 ? 2 : (RS == 1 ? (NC <= 4 ? 4 : (NC <= 8 ? 3 : (NC <= 12 ? 2 : 1)))
                                                             : (RS * NC <= 16 ? 2 : 1))) void k_kv8_step(Kv8AttnArgs a) {
    constexpr int KS = (NC + 3) / 4, HG = 4 * RS;
    extern __shared__ __align__(16) float lds[];                 // red [SW][HG][D], ml [SW][HG][2], the rows' bytes for RS > 1
    const int D = a.c.D, nc = D / 16, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = blockIdx.x % a.c.Hkv, z = blockIdx.x / a.c.Hkv, c = blockIdx.y, i = blockIdx.z;
    const int quad = lane >> 4, part = lane & 3;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int rows = r.n * a.rep, R0 = z * HG;                   // this group's rows: token R / rep, head g rep + R % rep
    if (R0 >= rows) return;
    const int nrow = rows - R0 < HG ? rows - R0 : HG;
    const int full = a.t.pos[i] < 0 ? 0 : a.t.pos[i], len = full < a.max_len ? full : a.max_len;
    const int64_t at0 = (int64_t) full - r.all;
    const Kv8Seen first = kv8_seen(at0 + R0 / a.rep, len, a.window);
    const Kv8Seen last = kv8_seen(at0 + (R0 + nrow - 1) / a.rep, len, a.window);
    const int64_t c0 = kv8_start(at0, len, a.window) + (int64_t) c * a.C, c1 = c0 + a.C;
    const int lo = first.lo > c0 ? first.lo : (int) (c0 < last.hi ? c0 : last.hi), hi = last.hi < c1 ? last.hi : (int) c1;
    if (a.nch > 1 && lo >= hi) return;
    const int pend = (hi + KV8_PAGE - 1) / KV8_PAGE;
    const int32_t * tab = a.t.table + i * a.t.tld;
    const float nan = __uint_as_float(0x7fc00000u);

    // a lane's row of set k: which positions it sees, where its q is
    auto row_of = [&](int k, Kv8Seen & sees) {
        const int rr = 4 * k + ((lane & 15) >> 2) < nrow ? 4 * k + ((lane & 15) >> 2) : nrow - 1;
        const int R = R0 + rr, j = R / a.rep, h = g * a.rep + (R - j * a.rep);
        sees = kv8_seen(at0 + j, len, a.window);
        return (r.row + j) * a.qrs + h * a.qhs;
    };
    int rlo[RS], rhi[RS];
    int64_t qat[RS];
#pragma unroll
    for (int k = 0; k < RS; k++) {
        Kv8Seen sees;
        qat[k] = row_of(k, sees);
        rlo[k] = sees.lo;
        rhi[k] = sees.hi;
    }
    uint4 kr[4][KS], vr[NC];
    const uint32_t lane16 = 16 * lane;
    float sk, sv;
    auto page_base = [&](int id) { return a.c.codes + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2 * KV8_PAGE * D; };
    auto load_k = [&](int id) {               // (steps past D meet zeros of q; they read on into V's codes)
        const int8_t * p = page_base(id);     // (uniform: the lane's offset stays one register)
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int s = 0; s < KS; s++) kr[t][s] = load_code<NT>(p + t * nc * 256 + s * 1024 + lane16);
    };
    auto load_v = [&](int id) {               // (chunks past D re-read the last: not stored)
        const int8_t * p = page_base(id) + KV8_PAGE * D;
#pragma unroll
        for (int n = 0; n < NC; n++) vr[n] = load_code<NT>(p + (n < nc ? n : nc - 1) * 1024 + lane16);
    };
    auto load_s = [&](int id) {
        const float * p = a.c.scales + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2;
        const bool bad = id < 0 || full > a.max_len;
        sk = bad ? nan : p[0];
        sv = bad ? nan : p[1];
    };
    int pg = lo / KV8_PAGE + w;
    if (pg < pend) {
        const int id = kv8_page(tab, pg, a.t.P, a.c.pages);
        load_k(id);
        load_v(id);
        load_s(id);
    }
    // the rows' bytes
    const uint32_t b = 3 - part, flip = part ? 0x80808080u : 0u;
    const uint32_t sel01 = 0x0c0c0000u | (4 + b) << 8 | b, sel23 = 0x00000c0cu | (4 + b) << 24 | b << 16;
    constexpr int bias = 0x00808080;          // makes the lower three bytes' signed digits unsigned
    auto cut = [&](uint32_t y0, uint32_t y1, uint32_t y2, uint32_t y3) {           // byte `part` of four biased numbers
        return (__builtin_amdgcn_perm(y1, y0, sel01) | __builtin_amdgcn_perm(y3, y2, sel23)) ^ flip;
    };
    auto cut_row = [&](int64_t base, i32x4 (&y)[KS]) {           // the bytes of a lane's row, and what a unit of them is worth
        float q[KS][16];
        uint32_t mq = 0;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int d = 64 * s + 16 * quad;
            if (a.f32) load16<true>(a.q, base + (d < D ? d : 0), q[s]);
            else load16<false>(a.q, base + (d < D ? d : 0), q[s]);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                if (d >= D) q[s][e] = 0.f;
                mq = max(mq, __float_as_uint(q[s][e]) & 0x7fffffffu);            // (a NaN is the largest)
            }
        }
        mq = max(mq, (uint32_t) __shfl_xor((int) mq, 16));
        mq = max(mq, (uint32_t) __shfl_xor((int) mq, 32));
        const int e2 = mq >= 0x7f800000u ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(mq));     // the largest < 2^e2
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                uint32_t x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = (uint32_t) (int) rintf(ldexpf(q[s][4 * u + e], 30 - e2)) + bias;
                y[s][u] = cut(x[0], x[1], x[2], x[3]);
            }
        return mq >= 0x7f800000u ? nan : ldexpf(MASK ? a.scale : a.scale * LOG2E, e2 - 30);
    };
    i32x4 qa[RS][KS];
    float rowf[RS];
    if (RS == 1) {
        rowf[0] = cut_row(qat[0], qa[0]);
    } else {                                                     // a set a wave, shared through LDS
        i32x4 * fq = (i32x4 *) (lds + SW * HG * (D + 2));
        float * ff = (float *) (fq + RS * KS * 64);
        if (w < RS) {
            int64_t at = qat[0];
#pragma unroll
            for (int k = 1; k < RS; k++) at = w == k ? qat[k] : at;
            i32x4 y[KS];
            ff[w * 64 + lane] = cut_row(at, y);
#pragma unroll
            for (int s = 0; s < KS; s++) fq[(w * KS + s) * 64 + lane] = y[s];
        }
        lds_barrier();
#pragma unroll
        for (int k = 0; k < RS; k++) {
            rowf[k] = ff[k * 64 + lane];
#pragma unroll
            for (int s = 0; s < KS; s++) qa[k][s] = fq[(k * KS + s) * 64 + lane];
        }
    }
    const float pw = __uint_as_float((127u + 8 * b) << 23);      // 256^(3 - part)
    float m[RS], l[RS], acc[RS][NC];
#pragma unroll
    for (int k = 0; k < RS; k++) {
        m[k] = -__builtin_inff();
        l[k] = 0.f;
#pragma unroll
        for (int n = 0; n < NC; n++) acc[k][n] = 0.f;
    }
    for (; pg < pend; pg += SW) {
        const int t0 = pg * KV8_PAGE, next = pg + SW < pend ? kv8_page(tab, pg + SW, a.t.P, a.c.pages) : -1;
        const float skc = sk, svc = sv;
        f32x4 mk[4];
        if (MASK)                             // (ahead of the next page's loads, which would be waited for with it)
#pragma unroll
            for (int t = 0; t < 4; t++) mk[t] = mask4(a.mask + i * a.mld + t0, 16 * t + 4 * quad, hi - t0);
        const bool edge = t0 < last.lo || t0 + KV8_PAGE > first.hi || t0 < lo || t0 + KV8_PAGE > hi;
        i32x4 pa[RS];
        float al[RS];
        bool up = false;
#pragma unroll
        for (int k = 0; k < RS; k++) {
            if (RS * NC > 16) __builtin_amdgcn_sched_barrier(0);             // (a set at a time, or its registers are not enough)
            const float f = rowf[k] * skc * pw;              // of this lane's byte
            float x[16];
            i32x4 sc[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                sc[t] = (i32x4){0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; s++)
                    sc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, kr[t][s]), qa[k][s], sc[t], 0, 0, 0);
            }
            if (k == RS - 1 && pg + SW < pend) { load_k(next); load_s(next); }
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float y = (float) sc[t][e] * f;
                    asm("" : "+v"(y));        // (fused with the sum's first addition, the four lanes would round apart, and
                    y = quad_sum(y);          // the bytes that each cuts from its weight would not belong together)
                    if (MASK) y += mk[t][e];
                    x[4 * t + e] = y;
                }
            if (edge) {
                const int l0 = (rlo[k] > lo ? rlo[k] : lo) - t0 - 4 * quad, h0 = (rhi[k] < hi ? rhi[k] : hi) - t0 - 4 * quad;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int n = 16 * (e >> 2) + (e & 3);
                    x[e] = n >= l0 && n < h0 ? x[e] : -__builtin_inff();
                }
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 16; e++) mx = fmaxf(mx, x[e]);
            mx = fmaxf(m[k], across_quads<true>(mx));
            const float base = mx == -__builtin_inff() ? 0.f : mx;
            al[k] = m[k] == mx ? 1.f : __builtin_amdgcn_exp2f(MASK ? (m[k] - base) * LOG2E : m[k] - base);
            up = up || m[k] != mx;
            m[k] = mx;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = __builtin_amdgcn_exp2f(MASK ? (x[4 * t + e] - base) * LOG2E : x[4 * t + e] - base);
                    sum += p;
                    y[e] = (uint32_t) (int) fmaf(p, 1073741824.f, (float) bias);        // (past 2^23: rounded to a whole number)
                }
                pa[k][t] = cut(y[0], y[1], y[2], y[3]);
            }
            l[k] = fmaf(l[k], al[k], sum);
        }
        if (__any(up)) {
#pragma unroll
            for (int k = 0; k < RS; k++) {
                const float f = __shfl(al[k], 4 * quad);         // of the head whose o this lane holds
#pragma unroll
                for (int n = 0; n < NC; n++) acc[k][n] *= f;
            }
        }
        float fh[RS], fl[RS];                                    // the value of a step of o's upper and lower bytes
#pragma unroll
        for (int k = 0; k < RS; k++) {
            fh[k] = svc * 6.103515625e-05f;                      // 2^-14, 2^-30
            fl[k] = svc * 9.31322574615478515625e-10f;
            if (svc != svc && !__shfl((int) (rlo[k] < t0 + KV8_PAGE && rhi[k] > t0), 4 * quad)) fh[k] = fl[k] = 0.f;
        }                                                        // (NaN only where a row sees the page)
#pragma unroll
        for (int n = 0; n < NC; n++) {
            if (n * RS % 4 == 0) __builtin_amdgcn_sched_barrier(0);          // (four products' results at a time)
#pragma unroll
            for (int k = 0; k < RS; k++) {
                const i32x4 v = __builtin_bit_cast(i32x4, vr[n]);
                const i32x4 d = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa[k], v, (i32x4){0, 0, 0, 0}, 0, 0, 0);
                acc[k][n] = fmaf((float) ((d[0] << 8) + d[1]), fh[k], acc[k][n]);
                acc[k][n] = fmaf((float) ((d[2] << 8) + d[3]), fl[k], acc[k][n]);
            }
        }
        if (pg + SW < pend) load_v(next);
    }
    // the waves' rows meet
    float * red = lds, * ml = lds + SW * HG * D;
#pragma unroll
    for (int k = 0; k < RS; k++) {
        const float sum = across_quads<false>(l[k]);
        if (part == 0 && quad == 0) {
            ml[(w * HG + 4 * k + (lane >> 2)) * 2] = m[k];
            ml[(w * HG + 4 * k + (lane >> 2)) * 2 + 1] = sum;
        }
#pragma unroll
        for (int n = 0; n < NC; n++)
            if (n < nc) red[(w * HG + 4 * k + quad) * D + 16 * n + (lane & 15)] = acc[k][n];
    }
    __syncthreads();
    const float unit = MASK ? LOG2E : 1.f;                       // (maxima are in powers of 2 without a mask)
    float * wml = a.ws + a.t.T * a.Hq * a.nch * D;
    for (int u = threadIdx.x; u < nrow * D; u += 64 * SW) {
        const int rr = u / D, d = u - rr * D;
        const int R = R0 + rr, j = R / a.rep, h = g * a.rep + (R - j * a.rep);
        const int64_t o = (r.row + j) * a.Hq + h;
        const float sink = a.sinks && a.nch == 1 ? a.sinks[h] * (MASK ? 1.f : LOG2E) : -__builtin_inff();
        float M = sink, L = 0.f, y = 0.f;
#pragma unroll
        for (int k = 0; k < SW; k++) M = fmaxf(M, ml[(k * HG + rr) * 2]);
        const float base = M == -__builtin_inff() ? 0.f : M;
#pragma unroll
        for (int k = 0; k < SW; k++) {
            const float f = __builtin_amdgcn_exp2f((ml[(k * HG + rr) * 2] - base) * unit);
            L = fmaf(f, ml[(k * HG + rr) * 2 + 1], L);
            if (ml[(k * HG + rr) * 2 + 1] != ml[(k * HG + rr) * 2 + 1]) L = nan;     // no score but NaN
            y = fmaf(f, red[(k * HG + rr) * D + d], y);
        }
        if (a.nch == 1) {
            if (a.sinks) L += __builtin_amdgcn_exp2f((sink - base) * unit);
            y = L == 0.f ? 0.f : y / L;
            if (a.f32) ((float *) a.out)[o * D + d] = y;
            else ((uint16_t *) a.out)[o * D + d] = f32_to_bf16(y);
        } else {
            a.ws[(o * a.nch + c) * D + d] = y;
            if (d == 0) {
                wml[(o * a.nch + c) * 2] = M;
                wml[(o * a.nch + c) * 2 + 1] = L;
            }
        }
    }
}

// Many query rows (prompts): bound by the matrix cores and the softmax's vector work together: the products of
// a page and 32 rows take 1024 cycles of a SIMD (D = 128), the rest of it 1150, and two waves of a SIMD take the
// sum of both, in whatever order they are run (alternating them by barriers: 397 us where this takes 352).
// A workgroup takes 32 WR rows (token, head of the kv head g), 32 a wave, and goes through the pages
// that they see; a page's codes become fp16 (exact) in LDS once for its waves, in the order that the
// matrix instructions take them, two pages deep with the next one's codes in registers: they are converted and stored
// between the products of the scores, whose time hides it (by themselves after them: 512 tokens of 40 / 8 heads over
// 32768 371 us, so 352; 8 prompts at D = 256 242, 212). WV waves: 8 share a page's conversion, and with KS = 2 are two
// groups of 4 with every second page each, joined at the end; which of them is taken where is attn_plan's rule.
// A wave forms S^T = K q^T: lane (row n, half) then holds tokens 32 T + 8 i + 4 half + c, which, V's tokens being
// taken in the same order, is the operand of O^T = V^T P^T without a move across lanes. Rounding: q (bf16) is
// exact in fp16 after scaling its row by a power of two (to 2^-32 of the largest); the weights are
// rounded to fp16 (half a step 2^-12 of each, and the row's sum adds the rounded ones), below the
// output's bf16; F32: q and the weights in two fp16 parts each, to 2^-22, twice the products. Sums, maxima and o are
// fp32. The V scale rides on the weights, relative to a power of two 2^eref that follows it; a row's reference maximum
// moves only when a score passes it by 2^3.
// 32 / 8 heads of 128 bf16: 2048 tokens on themselves 61 us (560 TFLOP/s), 8192 620 us (885), 512 of 40 / 8 over
// 32768 352 us (950; a large bf16 product reaches 1372). 2048 in fp32: 114 us.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// four codes -> fp16, exactly: 1024 + (code + 128) by its bits, less 1152
__device__ __forceinline__ void codes_f16(uint32_t u, uint32_t & lo, uint32_t & hi) {
    u ^= 0x80808080u;
    const f16x2 k = {(_Float16) -1152.f, (_Float16) -1152.f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + k);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + k);
}

template <int NC, int WV, int KS, bool MASK, bool F32>
__global__ __launch_bounds__(64 * WV, NC <= 8 && !F32 ? 8 / WV : 1) void k_kv8_tile(Kv8AttnArgs a) {
    constexpr int PARTS = F32 ? 2 : 1;        // fp16 parts of q and of a weight
    constexpr bool ACC = NC > 8 || F32;       // more than 256 registers: o stays in accumulation registers
    constexpr int WR = WV / KS, TR = 32 * WR, NU = 2 * NC / WR, ND = NC / 2;         // waves over the rows, rows, a wave's load
    constexpr int FRAGS = 4 * NC;                                                    // units, d tiles of 32, KiB of a page
    static_assert(NU * WR == 2 * NC, "the waves share a page's units evenly");
    extern __shared__ __align__(16) uint4 lds4[];                // [KS][2][FRAGS][64], MASK: [KS][2][64] floats
    const int D = a.c.D, nc = D / 16, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // of KS groups of waves, each with every KS-th page; waves 4 apart share a SIMD: the first 64 rows' are on all four
    const int grp = wave / WR, w = (wave % WR) ^ (2 * grp);
    uint4 * page = lds4 + grp * 2 * FRAGS * 64;
    float * masks = (float *) (lds4 + KS * 2 * FRAGS * 64) + grp * 2 * KV8_PAGE;                 // the pages' mask values
    const int c = blockIdx.y, i = blockIdx.z, half = lane >> 5, n31 = lane & 31;
    const int g = blockIdx.x % a.c.Hkv;
    int z = blockIdx.x / a.c.Hkv;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int rows = r.n * a.rep, ngrp = (rows + TR - 1) / TR;
    if (z >= ngrp) return;
    // the longest first; with no more workgroups than run at once, the second half the shortest first, so that
    // what two workgroups of a CU have adds to the same
    z = a.fold && z >= ngrp / 2 ? z - ngrp / 2 : ngrp - 1 - z;
    const int R0 = z * TR, nrow = rows - R0 < TR ? rows - R0 : TR;
    const int full = a.t.pos[i] < 0 ? 0 : a.t.pos[i], len = full < a.max_len ? full : a.max_len;
    const int64_t at0 = (int64_t) full - r.all;
    const Kv8Seen first = kv8_seen(at0 + R0 / a.rep, len, a.window);
    const Kv8Seen last = kv8_seen(at0 + (R0 + nrow - 1) / a.rep, len, a.window);
    const int64_t c0 = kv8_start(at0, len, a.window) + (int64_t) c * a.C, c1 = c0 + a.C;
    const int lo = first.lo > c0 ? first.lo : (int) (c0 < last.hi ? c0 : last.hi), hi = last.hi < c1 ? last.hi : (int) c1;
    if (a.nch > 1 && lo >= hi) return;
    const int pbeg = lo / KV8_PAGE, pend = (hi + KV8_PAGE - 1) / KV8_PAGE;
    const int32_t * tab = a.t.table + i * a.t.tld;
    const float nan = __uint_as_float(0x7fc00000u), inf = __builtin_inff();

    // this wave's share of a page: where each unit's 16 bytes are, and the fragments that they make
    uint32_t src[NU];
    int dst[NU][2];
#pragma unroll
    for (int u = 0; u < NU; u++) {
        const int k = w + WR * u;
        if (k < NC) {                                            // K: tokens 32 T + n31, chunk 2 s + half
            const int T = k / (NC / 2), s2 = k % (NC / 2), ch = 2 * s2 + half < nc ? 2 * s2 + half : nc - 1;
            src[u] = ((2 * T + (n31 >> 4)) * nc + ch) * 256 + (lane & 15) * 16;
            dst[u][0] = (T * NC + 2 * s2) * 64 + lane;
            dst[u][1] = dst[u][0] + 64;
        } else {                                                 // V: d 32 dt + n31, tokens' quad 2 v + half
            const int dt = (k - NC) >> 1, v = (k - NC) & 1, ch = 2 * dt + (n31 >> 4) < nc ? 2 * dt + (n31 >> 4) : nc - 1;
            src[u] = KV8_PAGE * D + ch * 1024 + (2 * v + half) * 256 + (lane & 15) * 16;
            dst[u][0] = (2 * NC + dt * 4 + v) * 64 + lane;
            dst[u][1] = dst[u][0] + 128;
        }
    }
    uint4 raw[NU], piece;
    auto load_unit = [&](int u, int64_t at) { raw[u] = *(const uint4 *) (a.c.codes + at + src[u]); };
    auto load = [&](int64_t at) {
#pragma unroll
        for (int u = 0; u < NU; u++) load_unit(u, at);
    };
    float mraw = 0.f;                         // the mask of the page in registers, a token a lane
    auto load_mask = [&](int pg) {
        const int64_t at = (int64_t) pg * KV8_PAGE + lane;
        if (MASK) mraw = at < hi ? a.mask[i * a.mld + at] : 0.f;
    };
    auto store_piece = [&](int k, uint4 * to) {                  // a quarter of a unit: 4 codes of a lane
        const int u = k >> 2, e = k & 3;
        const uint32_t x = e == 0 ? raw[u].x : (e == 1 ? raw[u].y : (e == 2 ? raw[u].z : raw[u].w));
        codes_f16(x, e & 1 ? piece.z : piece.x, e & 1 ? piece.w : piece.y);
        if (e & 1) to[dst[u][e >> 1]] = piece;
    };
    auto store = [&](uint4 * to) {
#pragma unroll
        for (int k = 0; k < 4 * NU; k++) store_piece(k, to);
    };
    // ids and scales of 64 pages at a time, a page a lane: no load to wait for in the loop
    int64_t lat = 0;                          // where its codes begin
    float lsk = 0.f, lls = 0.f;               // K's scale, log2 of V's
    auto fetch = [&](int p0) {
        const int at = p0 + KS * lane, id = at < pend ? kv8_page(tab, at, a.t.P, a.c.pages) : -1;
        const float * p = a.c.scales + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2;
        const bool bad = id < 0 || full > a.max_len;
        lat = ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2 * KV8_PAGE * D;
        lsk = bad ? nan : p[0];
        lls = bad ? nan : __builtin_amdgcn_logf(p[1] < 1e-36f ? 1e-36f : p[1]);
    };
    auto lane_at = [&](int n) {
        const uint32_t hi = __builtin_amdgcn_readlane((int) (lat >> 32), n), lo = __builtin_amdgcn_readlane((int) lat, n);
        return (int64_t) ((uint64_t) hi << 32 | lo);
    };
    auto lane_f = [&](float v, int n) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), n)); };

    const int p0 = pbeg + grp, np = pend > p0 ? (pend - p0 + KS - 1) / KS : 0;
    const int rounds = pend > pbeg ? (pend - pbeg + KS - 1) / KS : 0;
    float qk[3] = {0.f, 0.f, 0.f}, qs[3] = {0.f, 0.f, 0.f};      // scales of pages n .. n + 2
    int64_t next = 0;                         // where page n + 2 is
    if (np > 0) {                             // (the first page's codes are on their way while q is prepared)
        fetch(p0);
        load(lane_at(0));
        load_mask(p0);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            qk[k] = lane_f(lsk, k);
            qs[k] = lane_f(lls, k);
        }
        next = lane_at(0);
    }

    // this lane's row
    const int rr = w * 32 + n31 < nrow ? w * 32 + n31 : nrow - 1, j = (R0 + rr) / a.rep, h = g * a.rep + (R0 + rr - j * a.rep);
    const Kv8Seen mine = kv8_seen(at0 + j, len, a.window);
    const bool live = w * 32 < nrow;                             // a wave behind the last row only loads
    const int wl = live ? w * 32 : nrow - 1, wh = w * 32 + 31 < nrow ? w * 32 + 31 : nrow - 1;
    const Kv8Seen wfirst = kv8_seen(at0 + (R0 + wl) / a.rep, len, a.window);
    const Kv8Seen wlast = kv8_seen(at0 + (R0 + wh) / a.rep, len, a.window);
    f16x8 q[PARTS][NC];
    float rowf;
    {
        const int64_t base = (r.row + j) * a.qrs + h * a.qhs;
        Raw8<F32> u[NC];
        uint32_t mq = 0;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int d = 16 * (k / 2 * 2 + half) + 8 * (k & 1);
            u[k] = load_raw<F32, Raw8<F32>>(a.q, base + (d < D ? d : 0));
#pragma unroll
            for (size_t e = 0; e < sizeof(u[0]) / 16; e++) {
                if (d >= D) u[k].u[e] = make_uint4(0, 0, 0, 0);
                mq = raw_max<F32>(mq, u[k].u[e]);
            }
        }
        if (!F32) mq = max(mq << 16, mq & 0xffff0000u);
        mq = max(mq, (uint32_t) __shfl_xor((int) mq, 32));
        const int e2 = mq >= 0x7f800000u ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(mq));     // the largest < 2^e2, to 2^8
        rowf = mq >= 0x7f800000u ? nan : ldexpf(fabsf(a.scale) * (MASK ? 1.f : LOG2E), e2 - 8);
        const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = ldexpf(sign * raw_at<F32>(u[k], e), 8 - e2);
                q[0][k][e] = (_Float16) x;
                if (F32) q[PARTS - 1][k][e] = (_Float16) (x - (float) q[0][k][e]);
            }
    }
    f32x16 o[ND];
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[t][e] = 0.f;
    float m = -inf, l = 0.f;
    int eref = -1000, emax = -1000;                              // no page yet

    auto buffer = [&](int n) { return page + (n & 1) * FRAGS * 64; };
    if (np > 0) {
        store(page);
        if (MASK) masks[lane] = mraw;
        load(lane_at(np > 1 ? 1 : 0));
        load_mask(p0 + KS);
    }
    f32x16 sc[2];
    f16x2 p[PARTS][2][8];
    // step k of the scores' products, of a page's K in LDS
    const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    auto k_step = [&](int k, uint4 fr) {
#pragma unroll
        for (int y = 0; y < PARTS; y++)
            sc[k / NC] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fr), q[y][k % NC],
                                                                k % NC || y ? sc[k / NC] : zero, 0, 0, 0);
    };
    // ... and of o's, of V: 16 tokens (T, v), 32 d each
    auto v_frag = [&](int k) { return 2 * NC + k % ND * 4 + k / ND; };
    auto v_step = [&](int k, uint4 fr) {
        const int T = k / ND >> 1, v = k / ND & 1, t = k % ND;
#pragma unroll
        for (int y = 0; y < PARTS; y++) {
            f16x8 b;
#pragma unroll
            for (int e = 0; e < 8; e++) b[e] = p[y][T][2 * (v + 2 * (e >> 2)) + ((e & 3) >> 1)][e & 1];
            o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fr), b, o[t], 0, 0, 0);
        }
    };
    // the scores of page n; between the products the codes that are in registers go to LDS as page n + 1, and the loads of
    // those of page n + 2 are issued
    auto scores = [&](int n) {
        const uint4 * cur = buffer(n);
        uint4 * to = buffer(n + 1);
        if (MASK) masks[(~n & 1) * KV8_PAGE + lane] = mraw;
        // fragments four products ahead of their use, held in this order (the scheduler would read each just before it)
        uint4 fr[4];
#pragma unroll
        for (int k = 0; k < 4; k++) fr[k] = cur[k * 64 + lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2 * NC; k++) {
            k_step(k, fr[k & 3]);
            if (k + 4 < 2 * NC) fr[k & 3] = cur[(k + 4) * 64 + lane];
#pragma unroll
            for (int e = k * 4 * NU / (2 * NC); e < (k + 1) * 4 * NU / (2 * NC); e++) {
                store_piece(e, to);
                if ((e & 3) == 3) load_unit(e >> 2, next);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        load_mask(p0 + (n + 2) * KS);
    };
    auto pass_on = [&](int n) {               // the codes alone
        store(buffer(n + 1));
        load(next);
        if (MASK) masks[(~n & 1) * KV8_PAGE + lane] = mraw;
        load_mask(p0 + (n + 2) * KS);
    };
    auto look_up = [&](int n) {               // page n + 2 (past the last: it again, unused)
        const int n2 = n + 2;
        if (n2 < np) {
            if ((n2 & 63) == 0) fetch(p0 + n2 * KS);
            next = lane_at(n2 & 63);
            qk[2] = lane_f(lsk, n2 & 63);
            qs[2] = lane_f(lls, n2 & 63);
        }
    };
    auto weights = [&](int n, float skc, float lsc) {
        const int t0 = (p0 + n * KS) * KV8_PAGE;
        // a page of a NaN scale: rows that see it become NaN at its end; with the scale in their scores the others would, too
        const bool poison = !(lsc < 128.f) || skc != skc;
        if (skc != skc) skc = 1.f;
        const float cs0 = rowf * skc, cs = cs0 < 1e-35f ? 1e-35f : cs0;      // (above 0, so that -inf stays -inf; a NaN stays)
        const bool edge = t0 < wlast.lo || t0 + KV8_PAGE > wfirst.hi || t0 < lo || t0 + KV8_PAGE > hi;
        if (MASK) {
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f32x4 mk = *(const f32x4 *) (masks + (n & 1) * KV8_PAGE + 32 * T + 8 * e + 4 * half);
#pragma unroll
                    for (int v = 0; v < 4; v++) sc[T][4 * e + v] = fmaf(sc[T][4 * e + v], cs, mk[v]);
                }
        }
        if (edge) {
            const int l0 = (mine.lo > lo ? mine.lo : lo) - t0 - 4 * half, h0 = (mine.hi < hi ? mine.hi : hi) - t0 - 4 * half;
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int n = 32 * T + 8 * (e >> 2) + (e & 3);
                    sc[T][e] = n >= l0 && n < h0 ? sc[T][e] : -inf;
                }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, sc[T][e]);
        {
            typedef unsigned u2 __attribute__((ext_vector_type(2)));
            const u2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(x.x), __uint_as_float(x.y));
        }
        if (!MASK) mx *= cs;
        // V's scale as a power of two within 2^4 of the reference, which moves otherwise (never 2^60 below the largest)
        if (!(lsc < 128.f)) lsc = eref > -1000 ? (float) eref : 0.f;
        const float step = MASK ? 3.f / LOG2E : 3.f;
        const bool move = mx > m + step;      // (m = -inf: any score)
        const bool shift_v = fabsf(lsc - (float) eref) > 4.f;
        if (__any(move) || shift_v) {
            const float mn = move ? mx : m, base = mn == -inf ? 0.f : mn;
            float f = m == -inf ? 0.f : __builtin_amdgcn_exp2f(MASK ? (m - base) * LOG2E : m - base);
            l *= f;
            m = mn;
            if (shift_v) {
                int e = (int) rintf(lsc);
                emax = e > emax ? e : emax;
                e = e < emax - 60 ? emax - 60 : e;
                f = ldexpf(f, eref - e > 200 ? 200 : (eref - e < -200 ? -200 : eref - e));
                eref = e;
            }
#pragma unroll
            for (int t = 0; t < ND; t++) {
                if (ACC) asm volatile("" : "+a"(o[t]));       // (o stays in accumulation registers but here, where it is
#pragma unroll                                                   //  read and written back; without this each page copied it)
                for (int e = 0; e < 16; e++) o[t][e] *= f;
                if (ACC) asm volatile("" : "+a"(o[t]));
            }
        }
        // weights: 2^8 e^(x - m) sv 2^-eref in fp16
        const float base = m == -inf ? 0.f : m, lr = 8.f + (lsc - (float) eref);
        float k = cs, off = lr - base;
        if (!MASK && __any(fabsf(base) > 65536.f)) {             // there a score's own rounding counts, as m has it
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float x = sc[T][e] * cs;
                    asm volatile("" : "+v"(x));                  // (not fused with the difference)
                    sc[T][e] = x - base;
                }
            k = 1.f;
            off = lr;
        }
        float sum = 0.f;
        const f16x2 one = {(_Float16) 1.f, (_Float16) 1.f};
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f32x2 y;
#pragma unroll
                for (int v = 0; v < 2; v++)
                    y[v] = __builtin_amdgcn_exp2f(MASK ? fmaf(sc[T][2 * e + v] - base, LOG2E, lr)
                                                       : fmaf(sc[T][2 * e + v], k, off));
                p[0][T][e] = __builtin_convertvector(y, f16x2);
                sum = __builtin_amdgcn_fdot2(p[0][T][e], one, sum, false);
                if (F32) {
                    p[PARTS - 1][T][e] = __builtin_convertvector(y - __builtin_convertvector(p[0][T][e], f32x2), f16x2);
                    sum = __builtin_amdgcn_fdot2(p[PARTS - 1][T][e], one, sum, false);
                }
            }
        l = fmaf(sum, __builtin_amdgcn_exp2f(-lr), l);
        if (poison && mine.lo < t0 + KV8_PAGE && mine.hi > t0) l = nan;
    };
    auto values = [&](int n) {
        const uint4 * cur = buffer(n);
#pragma unroll
        for (int k = 0; k < 2 * NC; k++) v_step(k, cur[v_frag(k) * 64 + lane]);
    };
    auto shift = [&] {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            qk[k] = qk[k + 1];
            qs[k] = qs[k + 1];
        }
    };
    for (int n = 0; n < rounds; n++) {
        look_up(n);
        lds_barrier();                        // page n is whole, the other buffer is read
        const int t0 = (p0 + n * KS) * KV8_PAGE;
        if (live && n < np && t0 < wlast.hi && t0 + KV8_PAGE > wfirst.lo) {
            scores(n);
            weights(n, qk[0], qs[0]);
            values(n);
        } else pass_on(n);
        shift();
    }
    if (KS > 1) {                             // the groups meet in the first, through LDS, in units of 2^m and 2^eref
        lds_barrier();
        float * ex = (float *) lds4 + w * (16 * ND + 2) * 64 + lane;
        const float unit = MASK ? LOG2E : 1.f;
#pragma unroll
        for (int k = 1; k < KS; k++) {
            if (grp == k && live) {
                const float f = ldexpf(1.f, eref <= -1000 ? 0 : eref);
                ex[0] = m;
                ex[64] = l;
#pragma unroll
                for (int t = 0; t < ND; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) ex[(2 + 16 * t + e) * 64] = o[t][e] * f;
            }
            lds_barrier();
            if (grp == 0 && live) {
                const float mo = ex[0], lo2 = ex[64], mn = fmaxf(m, mo), base = mn == -inf ? 0.f : mn;
                float f = __builtin_amdgcn_exp2f((m - base) * unit);
                const float fo = __builtin_amdgcn_exp2f((mo - base) * unit);
                l = l * f + lo2 * fo;
                f = ldexpf(f, eref <= -1000 ? 0 : eref);
#pragma unroll
                for (int t = 0; t < ND; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[t][e] = fmaf(o[t][e], f, ex[(2 + 16 * t + e) * 64] * fo);
                m = mn;
                eref = 0;
            }
            if (k + 1 < KS) lds_barrier();
        }
        if (grp > 0) return;
    }
    if (!live || w * 32 + n31 >= nrow) return;
    {
        typedef unsigned u2 __attribute__((ext_vector_type(2)));
        const u2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(x.x) + __uint_as_float(x.y);
    }
    const int64_t at = (r.row + j) * a.Hq + h;
    float f = ldexpf(1.f, eref <= -1000 ? 0 : eref - 8);
    if (a.nch == 1) {
        if (a.sinks) {
            const float base = m == -inf ? 0.f : m;
            l += __builtin_amdgcn_exp2f(MASK ? (a.sinks[h] - base) * LOG2E : a.sinks[h] * LOG2E - base);
        }
        f = l == 0.f ? 0.f : f / l;
    } else if (half == 0) {
        float * wml = a.ws + a.t.T * a.Hq * a.nch * D + (at * a.nch + c) * 2;
        wml[0] = m;
        wml[1] = l;
    }
#pragma unroll
    for (int t = 0; t < ND; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (32 * t + 8 * e >= D) continue;
            const int d = 32 * t + 8 * e + 4 * half;
            const float4 y = make_float4(o[t][4 * e] * f, o[t][4 * e + 1] * f, o[t][4 * e + 2] * f, o[t][4 * e + 3] * f);
            if (F32 && a.nch == 1) *(float4 *) ((float *) a.out + at * D + d) = y;
            else if (a.nch > 1) *(float4 *) (a.ws + (at * a.nch + c) * D + d) = y;
            else *(uint2 *) ((uint16_t *) a.out + at * D + d) =
                make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
        }
}

// The chunks of a row joined: W waves per (row, head), W | 4. A wave finds the largest maximum and the weights,
// a chunk a lane; then D / 4 lanes (rounded up to 16, 32 or 64) add 4 columns each over every (64 / lanes W)th
// chunk, 8 loads in flight. Bound by latency for few rows of many chunks, by the bytes of the partials for many
// rows of few.
template <int W>
__global__ __launch_bounds__(KT) void k_kv8_combine(Kv8AttnArgs a) {
    constexpr int CW = KT / 64;
    __shared__ float sw[CW][64];
    __shared__ f32x4 sred[CW][64];
    const int D = a.c.D, i = blockIdx.y, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rh = blockIdx.x * (CW / W) + w / W, h = rh % a.Hq, j = rh / a.Hq, part = w % W;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const bool live = j < r.n;
    if (W == 1 ? !live : (blockIdx.x * (CW / W)) / a.Hq >= r.n) return;       // (W > 1 meets at a barrier: leave together)
    const int full = a.t.pos[i] < 0 ? 0 : a.t.pos[i], len = full < a.max_len ? full : a.max_len;
    const Kv8Seen s = kv8_seen((int64_t) full - r.all + j, len, a.window);
    const int at = kv8_start((int64_t) full - r.all, len, a.window);
    const int ca = (s.lo - at) / a.C, cb = live && s.hi > s.lo ? (s.hi - 1 - at) / a.C + 1 : ca;             // this row's chunks
    const int64_t o = (r.row + (live ? j : 0)) * a.Hq + h;
    const float * wo = a.ws + o * a.nch * D, * wml = a.ws + a.t.T * a.Hq * a.nch * D + o * a.nch * 2;
    // (maxima are in powers of 2 without a mask, in powers of e with one: its lowest value has to fit)
    const float unit = a.mask ? LOG2E : 1.f, sink = a.sinks ? a.sinks[h] * (a.mask ? 1.f : LOG2E) : -__builtin_inff();
    float M = sink;
    for (int c = ca + lane; c < cb; c += 64) M = fmaxf(M, wml[2 * c]);
    M = wave_max(M);
    const float base = M == -__builtin_inff() ? 0.f : M;
    const int DL = D <= 64 ? 16 : (D <= 128 ? 32 : 64), G = 64 / DL * W, d = lane % DL * 4, gr = part * (64 / DL) + lane / DL;
    float den = 0.f;
    f32x4 y = {0, 0, 0, 0};
    for (int b = ca; b < cb; b += 64) {
        const int n = cb - b < 64 ? cb - b : 64, c = b + (lane < n ? lane : n - 1);
        const float f = __builtin_amdgcn_exp2f((wml[2 * c] - base) * unit), lc = wml[2 * c + 1];
        if (lane < n) den = lc != lc ? lc : fmaf(f, lc, den);
        sw[w][lane] = f;
        __builtin_amdgcn_wave_barrier();
        for (int k = gr; k < n; k += 8 * G) {
            f32x4 x[8];
            const float * p = wo + (int64_t) b * D + (d < D ? d : 0);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = *(const f32x4 *) (p + (int64_t) (k + G * e < n ? k + G * e : k) * D);
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k + G * e < n) y += sw[w][k + G * e] * x[e];
        }
        __builtin_amdgcn_wave_barrier();
    }
    den = wave_sum(den) + (a.sinks ? __builtin_amdgcn_exp2f((sink - base) * unit) : 0.f);
    sred[w][lane] = y;
    if (W > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    if (live && part == 0 && lane < DL && d < D) {
        for (int k = 1; k < G; k++) y += sred[w + k / (64 / DL)][(k % (64 / DL)) * DL + lane];
        const float f = 1.f / den;
        const float4 v = den == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
        if (a.f32) *(float4 *) ((float *) a.out + o * D + d) = v;
        else *(uint2 *) ((uint16_t *) a.out + o * D + d) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    }
}

// ... and of few chunks (up to J): D / 4 lanes a row, 4 columns each, every chunk's maximum, sum and columns loaded at
// once. (512 x 40 rows of 3 chunks: 15.5 us by the kernel above, which goes through LDS and two more latencies.)
template <int J>
__global__ __launch_bounds__(KT) void k_kv8_join(Kv8AttnArgs a) {
    const int D = a.c.D, DL = D / 4, i = blockIdx.y, u = blockIdx.x * KT + threadIdx.x, rh = u / DL, d = (u - rh * DL) * 4;
    const int h = rh % a.Hq, j = rh / a.Hq;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    if (j >= r.n) return;
    const int full = a.t.pos[i] < 0 ? 0 : a.t.pos[i], len = full < a.max_len ? full : a.max_len;
    const Kv8Seen s = kv8_seen((int64_t) full - r.all + j, len, a.window);
    const int at = kv8_start((int64_t) full - r.all, len, a.window);
    const int ca = (s.lo - at) / a.C, n = s.hi > s.lo ? (s.hi - 1 - at) / a.C + 1 - ca : 0;        // this row's chunks
    const int64_t o = (r.row + j) * a.Hq + h;
    const float * wo = a.ws + (o * a.nch + ca) * D + d, * wml = a.ws + a.t.T * a.Hq * a.nch * D + (o * a.nch + ca) * 2;
    const float unit = a.mask ? LOG2E : 1.f, sink = a.sinks ? a.sinks[h] * (a.mask ? 1.f : LOG2E) : -__builtin_inff();
    float mc[J], lc[J];
    f32x4 x[J];
#pragma unroll
    for (int k = 0; k < J; k++) {             // (past the row's chunks its first again, unused; none: nothing is read)
        const int c = k < n ? k : 0;
        mc[k] = n > 0 ? wml[2 * c] : -__builtin_inff();
        lc[k] = n > 0 ? wml[2 * c + 1] : 0.f;
        x[k] = n > 0 ? *(const f32x4 *) (wo + (int64_t) c * D) : (f32x4){0, 0, 0, 0};
    }
    float M = sink, den = 0.f;
#pragma unroll
    for (int k = 0; k < J; k++) M = k < n ? fmaxf(M, mc[k]) : M;
    const float base = M == -__builtin_inff() ? 0.f : M;
    f32x4 y = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < J; k++)
        if (k < n) {
            const float f = __builtin_amdgcn_exp2f((mc[k] - base) * unit);
            den += f * lc[k];
            y += f * x[k];
        }
    if (a.sinks) den += __builtin_amdgcn_exp2f((sink - base) * unit);
    const float f = 1.f / den;
    const float4 v = den == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
    if (a.f32) *(float4 *) ((float *) a.out + o * D + d) = v;
    else *(uint2 *) ((uint16_t *) a.out + o * D + d) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// tile: k_kv8_tile's plan, else k_kv8_step's
struct AttnPlan { bool tile; int RS, ngrp, C, nch, fold, wv, ks, sw; bool nt; };

AttnPlan attn_plan(int f32, int Hq, int D, int Hkv, int nseq, int max_n, int max_len, int window) {
    AttnPlan p;
    const int64_t rows = (int64_t) max_n * (Hq / Hkv);
    p.tile = rows > 16 && (!f32 || D <= 128);                    // (fp32 at D > 128 has no registers for two parts of q)
    p.RS = rows <= 4 ? 1 : (rows <= 8 || D > 64 ? 2 : 4);        // (four sets' registers fit beside the codes of D = 64)
    // The prompt kernel's workgroups: 8 waves over 256 rows where every row sees nearly the same tokens (512 over 32768: 352
    // us, in two groups 396); 8 waves in two groups of every second page over 128 rows where there are no more, or no
    // more of these than CUs (1024 on themselves 34.7 -> 29.5 us, 1024 behind 1024 54.9 -> 46.8; of 320 such workgroups
    // 20.2 -> 25.2); else 4 waves over 128 rows, which balance a causal triangle better (2048: 61 us, 256 rows 83).
    // (8 waves need whole units of a page: D up to 64 and from 97 to 128.)
    const bool eight = !f32 && (D <= 64 || (D > 96 && D <= 128));
    p.wv = eight && (rows <= 128 || (int64_t) max_n * 4 <= max_len) ? 8 : 4;
    const bool two = eight && (rows <= 128 || ((int64_t) max_n * 4 > max_len && (rows + 127) / 128 * Hkv * nseq <= 256));
    if (two) p.wv = 8;
    p.ks = two ? 2 : 1;
    const int group = p.tile ? 32 * p.wv / p.ks : 4 * p.RS;
    p.ngrp = (int) ((rows + group - 1) / group);
    const int64_t wgs = (int64_t) Hkv * p.ngrp * nseq;
    // the most tokens of a sequence that the call's rows see, from the page of the first (kv8_start)
    const int64_t eff = window > 0 ? std::min<int64_t>(max_len, (int64_t) window + max_n + KV8_PAGE - 2) : max_len;
    int64_t C;
    if (p.tile) {
        // Split along the tokens where the workgroups leave CUs without, in chunks of 512 tokens or more; where every row
        // sees nearly the same tokens, of 256 up to 16 chunks and of 128 up to 8 (32 rows of 8 heads at D = 256 over 2000 in 4
        // chunks 36.8 us, in 8 27.8; 17 tokens over 1000 whole 23.6, in 8 16.0; but 32 tokens over 8000 in 16 25.2, in 32
        // 28.0: the partials). 2048 tokens or more for a twofold split, whose gain the partials and the join cost again.
        // And further where whole rounds of the workgroups come out fuller.
        const int64_t slots = p.wv == 8 || D > 128 || f32 ? 256 : 512;
        auto used = [&](int64_t n) { return (double) (wgs * n) / (double) ((wgs * n + slots - 1) / slots * slots); };
        const bool flat = (int64_t) max_n * 4 <= eff;
        int64_t most = (eff + 511) / 512;
        if (flat) most = std::max(most, std::max(std::min<int64_t>((eff + 255) / 256, 16), std::min<int64_t>((eff + 127) / 128, 8)));
        int64_t nch = std::min(std::max<int64_t>(slots / wgs, 1), most);
        if (nch == 2 && eff < 4096) nch = 1;
        if (flat)
            for (int64_t n = nch + 1; n <= 8 && eff / n >= 2048; n++)
                if (used(n) > 1.15 * used(nch)) nch = n;
        C = ((eff + nch - 1) / nch + KV8_PAGE - 1) / KV8_PAGE * KV8_PAGE;
    } else {
        // whole up to 2048 tokens (2000 of one sequence: 11.0 us; 4000 in 8 chunks 7.4, the join 3.3 and its launch), then in
        // chunks of 512 to 2048 tokens, so that the workgroups go around the 256 CUs twice
        C = eff <= 2048 ? eff : std::min<int64_t>(std::max<int64_t>(eff * wgs / 512, 512), 2048);
        // eight waves a workgroup where the workgroups leave CUs without
        p.sw = wgs * ((eff + C - 1) / C) <= 256 && D <= 128 ? 8 : 4;
        // non-temporal loads where the codes are more than the caches would keep for another call (MB, us without -> with: 1070
        // 187 -> 170, 578 116 -> 103, 245 64 -> 57, 134 27.4 -> 24.1, 67 15.3 -> 15.4, 33 13.6 -> 15.8, 4 11.0 -> 13.6)
        p.nt = p.ngrp == 1 && 2 * eff * nseq * Hkv * D >= 100000000;
        const int64_t round = p.sw * KV8_PAGE;
        C = (C + round - 1) / round * round;
    }
    p.C = (int) (C > (1 << 30) ? 1 << 30 : C);
    p.nch = (int) ((eff + (int64_t) p.C - 1) / p.C);
    p.fold = p.wv == 4 && wgs * p.nch <= 512;
    return p;
}

template <int NC, int RS, int SW> hipError_t run_step(const Kv8AttnArgs & a, const AttnPlan & p, hipStream_t s) {
    const dim3 grid((unsigned) (a.c.Hkv * p.ngrp), (unsigned) p.nch, (unsigned) a.t.nseq);
    const size_t lds = sizeof(float) * SW * 4 * RS * (a.c.D + 2) + (RS > 1 ? RS * ((NC + 3) / 4 * 1024 + 256) : 0);
    if (a.mask) k_kv8_step<NC, RS, SW, true, false><<<grid, 64 * SW, lds, s>>>(a);
    else if (SW == 4 && RS <= 2 && p.nt) k_kv8_step<NC, RS, SW, false, SW == 4 && RS <= 2><<<grid, 64 * SW, lds, s>>>(a);
    else k_kv8_step<NC, RS, SW, false, false><<<grid, 64 * SW, lds, s>>>(a);
    return hipGetLastError();
}

template <int NC> hipError_t run_attn(const Kv8AttnArgs & a, const AttnPlan & p, hipStream_t s) {
    if (!p.tile) {
        if constexpr (NC <= 4)
            if (p.RS == 4) return p.sw == 8 ? run_step<NC, 4, 8>(a, p, s) : run_step<NC, 4, 4>(a, p, s);
        if constexpr (NC <= 8)
            if (p.sw == 8) return p.RS == 1 ? run_step<NC, 1, 8>(a, p, s) : run_step<NC, 2, 8>(a, p, s);
        return p.RS == 1 ? run_step<NC, 1, 4>(a, p, s) : run_step<NC, 2, 4>(a, p, s);
    }
    const dim3 grid((unsigned) (a.c.Hkv * p.ngrp), (unsigned) p.nch, (unsigned) a.t.nseq);
    const size_t lds = 2 * 4 * NC * 1024 + (a.mask ? 2 * KV8_PAGE * sizeof(float) : 0);
    if constexpr (NC <= 8 && NC % 4 == 0)
        if (p.wv == 8) {
            if (p.ks == 2 && a.mask) k_kv8_tile<NC, 8, 2, true, false><<<grid, 512, 2 * lds, s>>>(a);
            else if (p.ks == 2) k_kv8_tile<NC, 8, 2, false, false><<<grid, 512, 2 * lds, s>>>(a);
            else if (a.mask) k_kv8_tile<NC, 8, 1, true, false><<<grid, 512, lds, s>>>(a);
            else k_kv8_tile<NC, 8, 1, false, false><<<grid, 512, lds, s>>>(a);
            return hipGetLastError();
        }
    if constexpr (NC <= 8)
        if (a.f32) {
            if (a.mask) k_kv8_tile<NC, 4, 1, true, true><<<grid, KT, lds, s>>>(a);
            else k_kv8_tile<NC, 4, 1, false, true><<<grid, KT, lds, s>>>(a);
            return hipGetLastError();
        }
    if (a.mask) k_kv8_tile<NC, 4, 1, true, false><<<grid, KT, lds, s>>>(a);
    else k_kv8_tile<NC, 4, 1, false, false><<<grid, KT, lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace

// workgroups per sequence and sequences that a launch of KT threads takes
static bool grid_fits(int64_t x, int nseq) { return x <= (int64_t) 0xffffffffu / KT && nseq <= 65535; }

hipError_t launch_kv8_write(const Kv8Cache & c, const Kv8Table & t, const void * k, const void * v, int f32, int64_t krs,
                            int64_t khs, int64_t vrs, int64_t vhs, hipStream_t s) {
    WriteArgs a{c, t, {k, v}, {krs, vrs}, {khs, vhs}, (int) (((int64_t) t.max_n + KV8_PAGE - 2) / KV8_PAGE + 1)};
    if (!grid_fits((int64_t) a.W * c.Hkv, t.nseq)) return hipErrorInvalidValue;
    const dim3 grid((unsigned) (a.W * c.Hkv), (unsigned) t.nseq);
    const size_t lds = (KV8_PAGE + 1) * c.D;
    if (f32 && c.D <= 128) k_kv8_write<true, 1><<<grid, KT, lds, s>>>(a);
    else if (f32) k_kv8_write<true, 2><<<grid, KT, lds, s>>>(a);
    else if (c.D <= 128) k_kv8_write<false, 1><<<grid, KT, lds, s>>>(a);
    else k_kv8_write<false, 2><<<grid, KT, lds, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8Cache & c, const Kv8Table & t, void * k, void * v, int f32, hipStream_t s) {
    ReadArgs a{c, t, {k, v}, (int) (((int64_t) t.max_n + KV8_PAGE - 2) / KV8_PAGE + 1)};
    if (!grid_fits((int64_t) a.W * c.Hkv, t.nseq)) return hipErrorInvalidValue;
    const dim3 grid((unsigned) (a.W * c.Hkv), (unsigned) t.nseq);
    if (f32) k_kv8_read<true><<<grid, KT, (KV8_PAGE + 1) * c.D, s>>>(a);
    else k_kv8_read<false><<<grid, KT, (KV8_PAGE + 1) * c.D, s>>>(a);
    return hipGetLastError();
}

int64_t kv8_attn_ws_bytes(int f32, int Hq, int D, int Hkv, int nseq, int64_t T, int max_n, int max_len, int window) {
    const AttnPlan p = attn_plan(f32, Hq, D, Hkv, nseq, max_n, max_len, window);
    return p.nch == 1 ? 0 : T * Hq * p.nch * (D + 2) * (int64_t) sizeof(float);
}

hipError_t launch_kv8_attn(const Kv8Cache & c, const Kv8Table & t, const void * q, int f32, int Hq, int64_t qrs, int64_t qhs,
                           int max_len, const float * mask, int64_t mld, const float * sinks, int window, float scale,
                           void * out, void * ws, hipStream_t s) {
    const AttnPlan p = attn_plan(f32, Hq, c.D, c.Hkv, t.nseq, t.max_n, max_len, window);
    Kv8AttnArgs a{c, t, q, out, mask, sinks, (float *) ws, qrs, qhs, mld, scale, Hq, Hq / c.Hkv, max_len, window, f32, p.C,
                  p.nch, p.fold};
    // (rows times heads within a grid keeps the join's thread index, D / 4 times that, below 2^31)
    if (!grid_fits((int64_t) Hq * t.max_n, t.nseq) || !grid_fits((int64_t) c.Hkv * p.ngrp, t.nseq) || p.nch > 65535)
        return hipErrorInvalidValue;
    const int nc = c.D / 16;
    hipError_t e = nc <= 4 ? run_attn<4>(a, p, s) : (nc <= 6 ? run_attn<6>(a, p, s) : (nc <= 8 ? run_attn<8>(a, p, s) :
                   (nc <= 12 ? run_attn<12>(a, p, s) : run_attn<16>(a, p, s))));
    if (e != hipSuccess || p.nch == 1) return e;
    const int64_t rh = (int64_t) Hq * t.max_n;
    const dim3 join((unsigned) ((rh * (c.D / 4) + KT - 1) / KT), (unsigned) t.nseq);
    if (p.nch <= 4) k_kv8_join<4><<<join, KT, 0, s>>>(a);
    else if (p.nch <= 8) k_kv8_join<8><<<join, KT, 0, s>>>(a);
    else if (p.nch > 16) k_kv8_combine<4><<<dim3((unsigned) rh, (unsigned) t.nseq), KT, 0, s>>>(a);
    else k_kv8_combine<1><<<dim3((unsigned) ((rh + KT / 64 - 1) / (KT / 64)), (unsigned) t.nseq), KT, 0, s>>>(a);
    return hipGetLastError();
}
