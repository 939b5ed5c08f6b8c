// The 8-bit key-value cache: quantising tokens into its pages, reading them back, and attention over
// them. Layout and index arithmetic: onpu_kv8.h.
#include <algorithm>

#include "onpu_launch.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int KT = 256;                       // threads per workgroup

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// 16 consecutive values, fp32 or bf16
template <bool F32> __device__ __forceinline__ void load16(const void * base, int64_t at, float (&x)[16]) {
    if (F32) {
        const uint4 * p = (const uint4 *) ((const float *) base + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 u = p[i];
            x[4 * i] = __uint_as_float(u.x); x[4 * i + 1] = __uint_as_float(u.y);
            x[4 * i + 2] = __uint_as_float(u.z); x[4 * i + 3] = __uint_as_float(u.w);
        }
    } else {
        const uint4 * p = (const uint4 *) ((const uint16_t *) base + at);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 u = p[i];
            x[8 * i] = bf_lo(u.x); x[8 * i + 1] = bf_hi(u.x); x[8 * i + 2] = bf_lo(u.y); x[8 * i + 3] = bf_hi(u.y);
            x[8 * i + 4] = bf_lo(u.z); x[8 * i + 5] = bf_hi(u.z); x[8 * i + 6] = bf_lo(u.w); x[8 * i + 7] = bf_hi(u.w);
        }
    }
}

// ------------------------------------------------------------------ write
// A workgroup per (touched page, kv head, sequence). Per K and V: a = max |x| of the new values, s = max(a, 2^-96) / 127
// (and the page's own scale, where it holds earlier tokens, if that is larger; their codes are then
// rescaled when s grew), code = x / s to the nearest, ties to even, of the exact quotient: with c the
// nearest integer of x * (1 / s), x - c s is exact in one fma (a multiple of half an ulp of s and below s), so that
// a c one off near a border is put right by comparing it with s / 2. A value that is not finite makes
// the page's scale NaN, and all that is read of it.
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

template <bool F32>
__global__ __launch_bounds__(KT) void k_kv8_write(WriteArgs a) {
    extern __shared__ __align__(16) int8_t tile[];               // K's 64 D codes, then V's
    __shared__ uint32_t wmax[2][KT / 64];
    const int D = a.c.D, NC = D / 16, t = threadIdx.x, g = blockIdx.x % a.c.Hkv, w = blockIdx.x / a.c.Hkv, i = blockIdx.y;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int64_t p0 = a.t.pos[i], pg = (p0 < 0 ? 0 : p0) / KV8_PAGE + w, base = pg * KV8_PAGE;
    if (p0 < 0 || base >= p0 + r.n) return;
    const int id = kv8_page(a.t.table + i * a.t.tld, pg, a.t.P, a.c.pages);
    if (id < 0) return;
    const int s0 = p0 > base ? (int) (p0 - base) : 0, s1 = p0 + r.n - base < KV8_PAGE ? (int) (p0 + r.n - base) : KV8_PAGE;
    const int64_t row0 = r.row + (base + s0 - p0);               // the row of slot s0
    const int units = (s1 - s0) * NC;
    int8_t * out = a.c.codes + ((int64_t) id * a.c.Hkv + g) * 2 * KV8_PAGE * D;
    float * sc = a.c.scales + ((int64_t) id * a.c.Hkv + g) * 2;
    float x[16];
    uint32_t m[2] = {0, 0};
    for (int u = t; u < units; u += KT)
        for (int kv = 0; kv < 2; kv++) {
            load16<F32>(a.x[kv], (row0 + u / NC) * a.rs[kv] + g * a.hs[kv] + u % NC * 16, x);
            for (int e = 0; e < 16; e++) m[kv] = max(m[kv], __float_as_uint(x[e]) & 0x7fffffffu);    // NaN the largest
        }
    for (int kv = 0; kv < 2; kv++) {
        for (int o = 32; o > 0; o >>= 1) m[kv] = max(m[kv], (uint32_t) __shfl_xor((int) m[kv], o));
        if ((t & 63) == 0) wmax[kv][t >> 6] = m[kv];
    }
    float s[2], so[2];
    for (int kv = 0; kv < 2; kv++) so[kv] = s0 > 0 ? sc[kv] : 0.f;
    // the page as it is (zeros for a new one)
    uint4 * tl = (uint4 *) tile;
    for (int u = t; u < 8 * D; u += KT) tl[u] = s0 > 0 ? ((const uint4 *) out)[u] : make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int kv = 0; kv < 2; kv++) {
        uint32_t b = wmax[kv][0];
        for (int k = 1; k < KT / 64; k++) b = max(b, wmax[kv][k]);
        s[kv] = b >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(b), KV8_TINY) / 127.f;
        if (s0 > 0 && !(so[kv] <= s[kv])) s[kv] = s[kv] != s[kv] ? s[kv] : so[kv];          // (a NaN stays)
        if (s0 > 0 && s[kv] > so[kv]) {
            const double f = (double) so[kv] / (double) s[kv];
            for (int u = t; u < KV8_PAGE * D; u += KT) {
                int8_t * p = tile + kv * KV8_PAGE * D + u;
                *p = (int8_t) rint(*p * f);
            }
        }
    }
    __syncthreads();
    for (int u = t; u < units; u += KT)
        for (int kv = 0; kv < 2; kv++) {
            load16<F32>(a.x[kv], (row0 + u / NC) * a.rs[kv] + g * a.hs[kv] + u % NC * 16, x);
            const float inv = 1.f / s[kv];
            const int token = s0 + u / NC, d = u % NC * 16;
            for (int e = 0; e < 16; e++)
                tile[kv ? KV8_PAGE * D + kv8_v_at(D, token, d + e) : kv8_k_at(D, token, d + e)] = (int8_t) quant(x[e], s[kv], inv);
        }
    __syncthreads();
    for (int u = t; u < 8 * D; u += KT) ((uint4 *) out)[u] = tl[u];
    if (t < 2) sc[t] = s[t];
}

// ------------------------------------------------------------------ read
// A workgroup per (page, kv head, sequence): value = code * scale, one rounding (two for bf16: to fp32
// and then to bf16). A page that the table does not have reads as NaN.
struct ReadArgs {
    Kv8Cache c;
    Kv8Table t;
    void * y[2];
    int W;
};

template <bool F32>
__global__ __launch_bounds__(KT) void k_kv8_read(ReadArgs a) {
    const int D = a.c.D, NC = D / 16, t = threadIdx.x, g = blockIdx.x % a.c.Hkv, w = blockIdx.x / a.c.Hkv, i = blockIdx.y;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    const int64_t p0 = a.t.pos[i], pg = (p0 - (p0 & (KV8_PAGE - 1))) / KV8_PAGE + w, base = pg * KV8_PAGE;
    if (base >= p0 + r.n) return;
    const int id = kv8_page(a.t.table + i * a.t.tld, pg, a.t.P, a.c.pages);
    const int s0 = p0 > base ? (int) (p0 - base) : 0, s1 = p0 + r.n - base < KV8_PAGE ? (int) (p0 + r.n - base) : KV8_PAGE;
    const int64_t row0 = r.row + (base + s0 - p0);
    const int8_t * in = a.c.codes + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2 * KV8_PAGE * D;
    const float * sc = a.c.scales + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2;
    for (int kv = 0; kv < 2; kv++) {
        const float s = id < 0 ? __uint_as_float(0x7fc00000u) : sc[kv];
        for (int u = t; u < (s1 - s0) * NC; u += KT) {
            const int token = s0 + u / NC, d = u % NC * 16;
            const int64_t at = ((row0 + u / NC) * a.c.Hkv + g) * D + d;
            for (int e = 0; e < 16; e++) {
                const float v = in[kv ? KV8_PAGE * D + kv8_v_at(D, token, d + e) : kv8_k_at(D, token, d + e)] * s;
                if (F32) ((float *) a.y[kv])[at + e] = v;
                else ((uint16_t *) a.y[kv])[at + e] = f32_to_bf16(v);
            }
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
    float * ws;
    int64_t qrs, qhs, mld;
    float scale;
    int Hq, rep, max_len, window;
};

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A workgroup per (query row, head); its 4 waves take every fourth page, a lane per token for the scores
// and a lane per 4 columns for the products, with a running maximum and sum per wave.
template <bool F32>
__global__ __launch_bounds__(KT) void k_kv8_attn(Kv8AttnArgs a) {
    __shared__ float qs[KV8_MAX_D], ps[KT], ml[KT / 64][2], red[KT / 64][KV8_MAX_D];
    const int D = a.c.D, NC = D / 16, t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int h = blockIdx.x % a.Hq, j = blockIdx.x / a.Hq, i = blockIdx.y, g = h / a.rep;
    const Kv8Rows r = kv8_rows(a.t.off, i, a.t.T, a.t.max_n);
    if (j >= r.n) return;
    const int64_t row = r.row + j;
    const int full = a.t.pos[i] < 0 ? 0 : a.t.pos[i], len = full < a.max_len ? full : a.max_len;
    const Kv8Seen seen = kv8_seen((int64_t) full - r.n + j, len, a.window);
    for (int d = t; d < D; d += KT)
        qs[d] = F32 ? ((const float *) a.q)[row * a.qrs + h * a.qhs + d] : bf16_to_f32(((const uint16_t *) a.q)[row * a.qrs + h * a.qhs + d]);
    __syncthreads();
    float m = -__builtin_inff(), l = 0.f, o[4] = {0, 0, 0, 0};
    for (int pg = seen.lo / KV8_PAGE + w; pg * KV8_PAGE < seen.hi; pg += KT / 64) {
        const int id = kv8_page(a.t.table + i * a.t.tld, pg, a.t.P, a.c.pages), token = pg * KV8_PAGE + lane;
        const int8_t * kc = a.c.codes + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2 * KV8_PAGE * D, * vc = kc + KV8_PAGE * D;
        const float * sc = a.c.scales + ((int64_t) (id < 0 ? 0 : id) * a.c.Hkv + g) * 2;
        const bool bad = id < 0 || full > a.max_len;
        const float sk = bad ? __uint_as_float(0x7fc00000u) : sc[0], sv = bad ? __uint_as_float(0x7fc00000u) : sc[1];
        float x = 0.f;
        for (int d = 0; d < D; d++) x += qs[d] * kc[kv8_k_at(D, lane, d)];
        x = x * (sk * a.scale);
        const bool see = token >= seen.lo && token < seen.hi;
        if (a.mask && see) x += a.mask[i * a.mld + token];
        if (!see) x = -__builtin_inff();
        const float mn = fmaxf(m, wave_max(x)), base = mn == -__builtin_inff() ? 0.f : mn;
        const float p = x == -__builtin_inff() ? 0.f : expf(x - base), f = m == -__builtin_inff() ? 0.f : expf(m - base);
        l = l * f + p;
        ps[t] = p;
        __builtin_amdgcn_wave_barrier();
        for (int k = 0; k < 4; k++) {
            const int d = lane + 64 * k;
            if (d >= D) continue;
            float y = 0.f;
            for (int n = 0; n < KV8_PAGE; n++) y += ps[64 * w + n] * vc[kv8_v_at(D, n, d)];
            o[k] = o[k] * f + y * sv;
        }
        __builtin_amdgcn_wave_barrier();
        m = mn;
    }
    l = wave_sum(l);
    if (lane == 0) { ml[w][0] = m; ml[w][1] = l; }
    for (int k = 0; k < 4; k++)
        if (lane + 64 * k < D) red[w][lane + 64 * k] = o[k];
    __syncthreads();
    float M = a.sinks ? a.sinks[h] : -__builtin_inff(), L = 0.f;
    for (int k = 0; k < KT / 64; k++) M = fmaxf(M, ml[k][0]);
    const float base = M == -__builtin_inff() ? 0.f : M;
    float f[KT / 64];
    for (int k = 0; k < KT / 64; k++) {
        f[k] = ml[k][0] == -__builtin_inff() ? (ml[k][1] != 0.f ? ml[k][1] : 0.f) : expf(ml[k][0] - base);    // (NaN stays)
        L += f[k] * ml[k][1];
    }
    if (a.sinks) L += expf(a.sinks[h] - base);
    for (int d = t; d < D; d += KT) {
        float y = 0.f;
        for (int k = 0; k < KT / 64; k++) y += f[k] == 0.f ? 0.f : f[k] * red[k][d];
        y = L == 0.f ? 0.f : y / L;
        const int64_t at = (row * a.Hq + h) * D + d;
        if (F32) ((float *) a.out)[at] = y;
        else ((uint16_t *) a.out)[at] = f32_to_bf16(y);
    }
}

}  // namespace

// workgroups per sequence and sequences that a launch of KT threads takes
static bool grid_fits(int64_t x, int nseq) { return x <= (int64_t) 0xffffffffu / KT && nseq <= 65535; }

hipError_t launch_kv8_write(const Kv8Cache & c, const Kv8Table & t, const void * k, const void * v, int f32, int64_t krs,
                            int64_t khs, int64_t vrs, int64_t vhs, hipStream_t s) {
    WriteArgs a{c, t, {k, v}, {krs, vrs}, {khs, vhs}, (int) (((int64_t) t.max_n + KV8_PAGE - 2) / KV8_PAGE + 1)};
    if (!grid_fits((int64_t) a.W * c.Hkv, t.nseq)) return hipErrorInvalidValue;
    const dim3 grid((unsigned) (a.W * c.Hkv), (unsigned) t.nseq);
    if (f32) k_kv8_write<true><<<grid, KT, 2 * KV8_PAGE * c.D, s>>>(a);
    else k_kv8_write<false><<<grid, KT, 2 * KV8_PAGE * c.D, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8Cache & c, const Kv8Table & t, void * k, void * v, int f32, hipStream_t s) {
    ReadArgs a{c, t, {k, v}, (int) (((int64_t) t.max_n + KV8_PAGE - 2) / KV8_PAGE + 1)};
    if (!grid_fits((int64_t) a.W * c.Hkv, t.nseq)) return hipErrorInvalidValue;
    const dim3 grid((unsigned) (a.W * c.Hkv), (unsigned) t.nseq);
    if (f32) k_kv8_read<true><<<grid, KT, 0, s>>>(a);
    else k_kv8_read<false><<<grid, KT, 0, s>>>(a);
    return hipGetLastError();
}

int64_t kv8_attn_ws_bytes(int, int, int, int, int64_t, int, int, int) { return 0; }

hipError_t launch_kv8_attn(const Kv8Cache & c, const Kv8Table & t, const void * q, int f32, int Hq, int64_t qrs, int64_t qhs,
                           int max_len, const float * mask, int64_t mld, const float * sinks, int window, float scale,
                           void * out, void * ws, hipStream_t s) {
    Kv8AttnArgs a{c, t, q, out, mask, sinks, (float *) ws, qrs, qhs, mld, scale, Hq, Hq / c.Hkv, max_len, window};
    if (!grid_fits((int64_t) Hq * t.max_n, t.nseq)) return hipErrorInvalidValue;
    const dim3 grid((unsigned) (Hq * t.max_n), (unsigned) t.nseq);
    if (f32) k_kv8_attn<true><<<grid, KT, 0, s>>>(a);
    else k_kv8_attn<false><<<grid, KT, 0, s>>>(a);
    return hipGetLastError();
}
