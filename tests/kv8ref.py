"""The 8-bit key-value cache from its definition, in numpy and 64 bits (test infrastructure): pages as
codes by token, written and read by plain loops, attention as a softmax in float64."""
import numpy as np

PAGE = 64
TINY = 2.0 ** -96


def places(D):
    """the byte of (token, d) in a head's K and V tiles"""
    t, d = np.arange(PAGE)[:, None], np.arange(D)[None]
    return (((t // 16) * (D // 16) + d // 16) * 256 + t % 16 * 16 + d % 16,
            d // 16 * 1024 + t // 4 % 4 * 256 + d % 16 * 16 + t // 16 * 4 + t % 4)


class Cache:
    """codes int8 [pages][Hkv][2][64 D] and scales fp32 [pages][Hkv][2], in the library's layout"""

    def __init__(self, codes, scales):
        self.codes, self.scales = codes.copy(), scales.copy()
        self.D = codes.shape[3] // PAGE
        self.at = places(self.D)

    def page(self, table, p):
        return int(table[p]) if 0 <= p < len(table) and 0 <= table[p] < len(self.codes) else -1

    def tokens(self, page, g, kv):
        """codes [64][D]"""
        return self.codes[page, g, kv][self.at[kv]]

    def put(self, page, g, kv, c):
        self.codes[page, g, kv][self.at[kv]] = c

    def write(self, k, v, table, pos):
        """one sequence: k, v float [n][Hkv][D] at positions pos .."""
        n = len(k)
        if pos < 0 or n == 0:
            return
        for p in range(pos // PAGE, (pos + n - 1) // PAGE + 1):
            page = self.page(table, p)
            if page < 0:
                continue
            a, b = max(pos - p * PAGE, 0), min(pos + n - p * PAGE, PAGE)
            for kv, x in ((0, k), (1, v)):
                for g in range(self.codes.shape[1]):
                    new = x[p * PAGE + a - pos:p * PAGE + b - pos, g].astype(np.float64)
                    s = np.float32(max(np.abs(new).max(), TINY) / 127) if np.isfinite(new).all() else np.float32(np.nan)
                    c = self.tokens(page, g, kv).astype(np.float64) if a else np.zeros((PAGE, self.D))
                    if a:
                        old = self.scales[page, g, kv]
                        s = old if old > s or np.isnan(old) else s
                        if s > old:
                            c = np.rint(c * (np.float64(old) / np.float64(s)))
                    c[a:b] = 0 if np.isnan(s) else np.rint(new / np.float64(s))
                    self.put(page, g, kv, c.astype(np.int8))
                    self.scales[page, g, kv] = s

    def read(self, table, pos, n):
        """k, v float64 [n][Hkv][D], exact"""
        out = np.full((2, n, self.codes.shape[1], self.D), np.nan)
        for j in range(n):
            page = self.page(table, (pos + j) // PAGE)
            if page < 0:
                continue
            for g in range(self.codes.shape[1]):
                for kv in range(2):
                    out[kv, j, g] = self.codes[page, g, kv][self.at[kv][(pos + j) % PAGE]] * np.float64(self.scales[page, g, kv])
        return out

    def attn(self, q, table, length, mask=None, sinks=None, window=0, scale=None):
        """one sequence: q float64 [n][Hq][D] -> (out [n][Hq][D], the largest sum_d |scale q_d K_td| seen, and
        the largest |V| of a kv head)"""
        n, Hq, D = q.shape
        Hkv = self.codes.shape[1]
        scale = D ** -0.5 if scale is None else scale
        out, big = np.zeros((n, Hq, D)), 0.0
        if length <= 0:
            return out, big, 0.0
        K, V = self.read(table, 0, length)
        for j in range(n):
            p = length - n + j
            lo = max(0, p + 1 - window) if window else 0
            if p < 0 or lo > p:
                continue
            for h in range(Hq):
                g = h // (Hq // Hkv)
                x = K[lo:p + 1, g] @ q[j, h] * scale
                big = max(big, np.nan_to_num(np.abs(K[lo:p + 1, g]) @ np.abs(q[j, h]) * abs(scale)).max())
                if mask is not None:
                    # (in fp32, as a mask of the type's lowest value is meant: it swallows the score)
                    with np.errstate(over="ignore"):
                        x = np.where(np.abs(mask[lo:p + 1]) > 1e30, (x.astype(np.float32) + mask[lo:p + 1]).astype(np.float64),
                                     x + mask[lo:p + 1])
                m = x.max() if sinks is None else max(x.max(), sinks[h])
                if m == -np.inf:
                    continue
                e = np.exp(x - m)
                l = e.sum() + (0 if sinks is None else np.exp(np.float64(sinks[h]) - m))
                out[j, h] = e @ V[lo:p + 1, g] / l if l != 0 else 0
        return out, big, float(np.nan_to_num(np.abs(V)).max())
