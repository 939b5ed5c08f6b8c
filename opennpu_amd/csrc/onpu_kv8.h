// The 8-bit key-value cache's layout and the index arithmetic that its kernels share (host and
// device; the host form is what the CPU tests compile).
//
// A page holds KV8_PAGE tokens of one layer. codes int8 [pages][Hkv][2][64 D] (K, then V of a head),
// scales fp32 [pages][Hkv][2]; a value is code * scale. Within a head's K: [4][D / 16][16 tokens]
// [16 d], token 16 a + b at [a][.][b][.]; V: [D / 16][4][16 d][4][4], token 16 a + 4 b + c at
// [.][b][.][a][c]. These are the operands of the matrix instructions as their lanes hold them: 16
// bytes of a lane are 16 d of one K token, or one d of the 16 V tokens whose weights the lane has
// from the scores' result, so that the kernels load them as they lie and need no transposition.
#pragma once
#include <stdint.h>

#ifndef ONPU_HD
#ifdef __HIPCC__
#define ONPU_HD __host__ __device__ __forceinline__
#else
#define ONPU_HD inline
#endif
#endif

constexpr int KV8_PAGE = 64, KV8_MAX_D = 256;
constexpr float KV8_TINY = 1.262177448e-29f;                     // 2^-96: the least maximum a scale is made of

ONPU_HD int kv8_k_at(int D, int token, int d) { return ((token >> 4) * (D >> 4) + (d >> 4)) * 256 + (token & 15) * 16 + (d & 15); }
ONPU_HD int kv8_v_at(int D, int token, int d) {
    (void) D;
    return (d >> 4) * 1024 + (token >> 2 & 3) * 256 + (d & 15) * 16 + (token >> 4) * 4 + (token & 3);
}

// The tokens of sequence i of a call: rows [row, row + n) of its T. off may hold anything: rows stay
// inside [0, T) and n inside [0, max_n]; all: the sequence's rows, also where they are more than max_n.
// Without off every sequence has max_n rows.
struct Kv8Rows { int64_t row, all; int n; };
ONPU_HD Kv8Rows kv8_rows(const int32_t * off, int i, int64_t T, int max_n) {
    Kv8Rows r;
    if (!off) { r.row = (int64_t) i * max_n; r.all = r.n = max_n; return r; }
    int64_t a = off[i], b = off[i + 1];
    a = a < 0 ? 0 : (a > T ? T : a);
    b = b < a ? a : (b > T ? T : b);
    r.row = a;
    r.all = b - a;
    r.n = (int) (b - a > max_n ? max_n : b - a);
    return r;
}

// the page of positions [64 p, 64 p + 64) by a sequence's table of P entries; -1: none
ONPU_HD int kv8_page(const int32_t * table, int64_t p, int P, int pages) {
    if (p < 0 || p >= P) return -1;
    const int id = table[p];
    return id >= 0 && id < pages ? id : -1;
}

// positions [lo, hi) that the query at position `at` sees of a cache of len tokens
struct Kv8Seen { int lo, hi; };
ONPU_HD Kv8Seen kv8_seen(int64_t at, int len, int window) {
    Kv8Seen s;
    s.hi = at + 1 < len ? (int) (at + 1 < 0 ? 0 : at + 1) : len;
    const int64_t lo = window > 0 ? at + 1 - window : 0;
    s.lo = lo < 0 ? 0 : (lo > s.hi ? s.hi : (int) lo);
    return s;
}
// the page-aligned position from which a sequence's chunks count: its first query at `at` sees nothing before it
// (with a window the chunks are as many as the window needs, wherever it lies)
ONPU_HD int kv8_start(int64_t at, int len, int window) {
    const int lo = kv8_seen(at, len, window).lo;
    return lo - lo % KV8_PAGE;
}

struct Kv8Cache {
    int8_t * codes;
    float * scales;
    int pages, Hkv, D;
};
struct Kv8Table {
    const int32_t * table, * pos, * off;      // pos: write, read: first position; attention: tokens in all
    int64_t tld, T;
    int P, nseq, max_n;
};
