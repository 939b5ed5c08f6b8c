"""The calls of the 8-bit key-value cache that are timed: tokens quantised into pages and read back
(kv8_write, kv8_read), and attention over those pages (kv8_attn), from one token of one sequence to
batches, speculative verification and prompts.

A page holds 64 tokens of one layer for all its kv heads, per head the K codes and the V codes
(int8, values code * scale, one fp32 scale per page, head and K | V). codes [pages][Hkv][2][64 D]:
K as [4][D / 16][16 tokens][16 d], token 16 a + b at [a][.][b][.]; V as [D / 16][4][16 d][4][4], token
16 a + 4 b + c at [.][b][.][a][c]. table [B][P]: the page of each sequence's positions 64 p .. 64 p + 63.

Lengths follow from the case alone (so that work() can count them); everything else from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64
TINY = 2.0 ** -96


def listed():
    return [
        # one token of one sequence appended, its page read back: the smallest call, all latency
        {"name": "append_b1", "kind": "append", "B": 1, "n": 1, "ragged": False, "start": 1000, "Hkv": 8, "D": 128,
         "dt": "f32"},
        # a decode step of 64 sequences at odd lengths
        {"name": "append_b64", "kind": "append", "B": 64, "n": 1, "ragged": False, "start": 4000, "Hkv": 8, "D": 128,
         "dt": "bf16"},
        # a prompt of 8192 tokens written from the start
        {"name": "append_prompt_8192", "kind": "append", "B": 1, "n": 8192, "ragged": False, "start": 0, "Hkv": 8,
         "D": 128, "dt": "bf16"},
        # prompts of several lengths behind cached prefixes, fp32, a head size that is no power of two
        {"name": "append_ragged", "kind": "append", "B": 16, "n": 1500, "ragged": True, "start": 500, "Hkv": 4, "D": 96,
         "dt": "f32"},
        # one decode token early in a conversation: latency
        {"name": "decode_b1_s200", "kind": "attn", "B": 1, "n": 1, "ragged": False, "S": 200, "Hq": 32, "Hkv": 8, "D": 128,
         "dt": "f32", "window": 0, "sinks": False, "mask": False},
        # one decode token at a long context
        {"name": "decode_b1_s65536", "kind": "attn", "B": 1, "n": 1, "ragged": False, "S": 65536, "Hq": 32, "Hkv": 8,
         "D": 128, "dt": "f32", "window": 0, "sinks": False, "mask": False},
        # a batch of 64 sequences of mixed lengths decoded together
        {"name": "decode_b64_ragged", "kind": "attn", "B": 64, "n": 1, "ragged": True, "S": 8192, "Hq": 32, "Hkv": 8,
         "D": 128, "dt": "bf16", "window": 0, "sinks": False, "mask": False},
        # a layer with sinks and a sliding window, 64-wide heads
        {"name": "decode_window_sinks", "kind": "attn", "B": 16, "n": 1, "ragged": True, "S": 20000, "Hq": 64, "Hkv": 8,
         "D": 64, "dt": "bf16", "window": 4000, "sinks": True, "mask": False},
        # speculative verification: 8 tokens each of 4 left-padded sequences
        {"name": "verify_m8", "kind": "attn", "B": 4, "n": 8, "ragged": True, "S": 8000, "Hq": 32, "Hkv": 4, "D": 128,
         "dt": "bf16", "window": 0, "sinks": False, "mask": True},
        # a prompt attending to itself
        {"name": "prompt_2048", "kind": "attn", "B": 1, "n": 2048, "ragged": False, "S": 2048, "Hq": 32, "Hkv": 8, "D": 128,
         "dt": "bf16", "window": 0, "sinks": False, "mask": False},
        # a chunk of a long prompt over the 32768 tokens cached up to its end
        {"name": "chunk_512_s32768", "kind": "attn", "B": 1, "n": 512, "ragged": False, "S": 32768, "Hq": 40, "Hkv": 8,
         "D": 128, "dt": "bf16", "window": 0, "sinks": False, "mask": False},
        # prompts of several lengths in one call, wide heads
        {"name": "prompts_ragged_d256", "kind": "attn", "B": 8, "n": 1500, "ragged": True, "S": 2500, "Hq": 16, "Hkv": 2,
         "D": 256, "dt": "bf16", "window": 0, "sinks": False, "mask": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 4, 128), (64, 8, 64), (16, 2, 256), (40, 8, 128), (8, 8, 64), (12, 2, 96), (16, 1, 128),
         (6, 2, 192), (28, 4, 128), (10, 10, 80), (4, 2, 48)]


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "verify", "prompt"])
    Hq, Hkv, D = rng.choice(HEADS)
    if kind == "append":
        B, n = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 8192)])
        n = max(1, min(n, 8192 * 8 * 128 // (B * Hkv * D)))
        return {"kind": kind, "B": B, "n": n, "ragged": rng.random() < 0.5, "start": _log(rng, 1, 4000) - 1, "Hkv": Hkv,
                "D": D, "dt": rng.choice(["bf16", "f32"])}
    B, S, n = _log(rng, 1, 64), _log(rng, 1, 65536), 1
    if kind == "verify":
        n = rng.randint(2, 16)
    if kind == "prompt":
        B, n = _log(rng, 1, 16), _log(rng, 17, 4096)
        S = n + rng.choice([0, _log(rng, 1, 32768)])
    S = max(n, min(S, 64 * 8192 * 8 * 128 // (B * Hkv * D)))
    while 4 * D * Hq * B * n * S > 3e11 and n > 1:
        n, S = max(1, n // 2), max(n // 2, S - (n - n // 2))
    return {"kind": "attn", "B": B, "n": n, "ragged": rng.random() < 0.6, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D,
            "dt": rng.choice(["bf16", "bf16", "f32"]), "window": rng.choice([0, 0, 0, _log(rng, 16, 8192)]),
            "sinks": rng.random() < 0.3, "mask": kind != "prompt" and rng.random() < 0.3}


def _lengths(c):
    """(tokens before the call, new tokens) of every sequence; the first is the longest"""
    r = random.Random(c["B"] * 1000003 + c["n"] * 1009 + c.get("S", c.get("start")))
    new = [c["n"]] + [r.randint(1, c["n"]) if c["ragged"] else c["n"] for _ in range(c["B"] - 1)]
    if c["kind"] == "append":
        return [r.randint(0, c["start"]) for _ in new], new
    total = [c["S"]] + [max(n, r.randint(1, c["S"])) if c["ragged"] else c["S"] for n in new[1:]]
    return [t - n for t, n in zip(total, new)], new


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    old, new = (np.array(v, np.int32) for v in _lengths(c))
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    P = int(((old + new + PAGE - 1) // PAGE).max())
    pages = int(((old + new + PAGE - 1) // PAGE).sum()) + 3
    # pages handed out in no order; past a sequence's own pages the table holds -1
    free, at = rng.permutation(pages).astype(np.int32), 0
    table = np.full((B, P), -1, np.int32)
    for i, k in enumerate((old + new + PAGE - 1) // PAGE):
        table[i, :k] = free[at:at + k]
        at += k
    codes = torch.empty((pages, Hkv, 2, PAGE * D), dtype=torch.int8, device="cuda")
    for part in codes.split(max(1, (1 << 27) // (Hkv * 2 * PAGE * D))):
        part.copy_((32 * torch.randn(part.shape, device="cuda", generator=g)).round_().clamp_(-127, 127))
    scales = torch.exp(0.25 * torch.randn((pages, Hkv, 2), device="cuda", generator=g)) / 32
    dt = torch.float32 if c["dt"] == "f32" else torch.bfloat16
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    st = {"codes": codes, "scales": scales, "table": dev(table), "off": dev(_offsets(new)), "T": int(new.sum()),
          "max_n": int(new.max()), "case": c}
    if c["kind"] == "append":
        # what comes back: each sequence's positions from the start of its first touched page
        first = old // PAGE * PAGE
        back = old + new - first
        st.update(pos=dev(old), k=torch.randn((st["T"], Hkv, D), device="cuda", generator=g).to(dt),
                  v=torch.randn((st["T"], Hkv, D), device="cuda", generator=g).to(dt), rpos=dev(first),
                  roff=dev(_offsets(back)), rows=int(back.sum()), max_back=int(back.max()), dt=dt)
        return st
    st.update(lens=dev(old + new), max_len=int((old + new).max()), window=c["window"], scale=D ** -0.5,
              q=(2 * torch.randn((st["T"], c["Hq"], D), device="cuda", generator=g)).to(dt), sinks=None, mask=None)
    if c["sinks"]:
        st["sinks"] = torch.randn((c["Hq"],), device="cuda", generator=g)
    if c["mask"]:
        # a bias per position, and left padding of up to a quarter of a sequence's earlier tokens
        m = 0.5 * torch.randn((B, P * PAGE), device="cuda", generator=g)
        pad = torch.from_numpy(rng.integers(0, old // 4 + 1)).cuda()
        st["mask"] = m.masked_fill_(torch.arange(P * PAGE, device="cuda")[None] < pad[:, None], -math.inf)
    return st


# ---------------------------------------------------------------- the plain form
def _k_tokens(c):
    """K codes of pages [..., 64 D] -> [..., 64, D]"""
    t = c.unflatten(-1, (4, -1, 16, 16)).transpose(-3, -2)
    return t.flatten(-2).flatten(-3, -2)


def _v_tokens(c):
    """V codes of pages [..., 64 D] -> [..., 64, D]"""
    t = c.unflatten(-1, (-1, 4, 16, 4, 4))
    return t.movedim((-2, -4, -1, -5, -3), (-5, -4, -3, -2, -1)).flatten(-2).flatten(-4, -2)


def _k_tiles(t):
    return t.unflatten(-1, (-1, 16)).unflatten(-3, (4, 16)).transpose(-3, -2).flatten(-4)


def _v_tiles(t):
    x = t.unflatten(-1, (-1, 16)).unflatten(-3, (4, 4, 4))
    return x.movedim((-2, -4, -1, -5, -3), (-5, -4, -3, -2, -1)).flatten(-5)


def _rows(off, T):
    """sequence and index within it of each of T rows"""
    t = torch.arange(T, device=off.device)
    i = torch.searchsorted(off[1:].long(), t, right=True)
    return i, t - off.long()[i]


def _append(st):
    c = st["case"]
    table, pos, off = st["table"].long(), st["pos"].long(), st["off"].long()
    n = off[1:] - off[:-1]
    W = (c["n"] + PAGE - 2) // PAGE + 1                                   # pages a sequence can touch
    page = pos[:, None] // PAGE + torch.arange(W, device=pos.device)[None]
    idx = page[:, :, None] * PAGE + torch.arange(PAGE, device=pos.device) - pos[:, None, None]    # [B][W][64]
    live = (page * PAGE < (pos + n)[:, None]) & (page < table.shape[1])
    ids = torch.gather(table, 1, page.clamp(max=table.shape[1] - 1))[live]
    idx = idx[live]                                                       # [touched][64]: index of the new token
    is_new = (idx >= 0) & (idx < n[:, None].expand(-1, W)[live][:, None])
    row = (off[:-1, None].expand(-1, W)[live][:, None] + idx).clamp(0, st["T"] - 1)
    had = idx[:, 0] < 0                                                   # earlier tokens in the page
    sel = is_new[:, :, None, None]
    for part, x, tokens, tiles in ((0, st["k"], _k_tokens, _k_tiles), (1, st["v"], _v_tokens, _v_tiles)):
        x = x[row].float().masked_fill(~sel, 0.0)                         # [touched][64][Hkv][D]
        amax = x.abs().amax((1, 3)).clamp(min=TINY)
        # (quotients in 64 bits: values next to a border between two codes)
        s_old = st["scales"][ids, :, part]
        s = (amax.double() / 127).float()
        s = torch.where(had[:, None], torch.maximum(s, s_old), s)
        old = tokens(st["codes"][ids, :, part]).transpose(1, 2)           # [touched][64][Hkv][D]
        ratio = (s_old.double() / s.double())[:, None, :, None]
        kept = torch.where(had[:, None, None, None] & ~sel & (idx < 0)[:, :, None, None], (old * ratio).round(), 0.0)
        new = (x.double() / s.double()[:, None, :, None]).round()
        both = torch.where(sel, new, kept).to(torch.int8)
        st["codes"][ids, :, part] = tiles(both.transpose(1, 2))
        st["scales"][ids, :, part] = s
    # read back
    i, j = _rows(st["roff"], st["rows"])
    p = st["rpos"].long()[i] + j
    pid = table[i, p // PAGE]
    out = []
    for part, tokens in ((0, _k_tokens), (1, _v_tokens)):
        held = tokens(st["codes"][:, :, part])                            # [pages][Hkv][64][D]
        out.append((held[pid, :, p % PAGE].float() * st["scales"][pid, :, part][:, :, None]).to(st["dt"]))
    return out


def _visible(st, pos, t):
    """whether positions t (last axis) are seen from query positions pos"""
    seen = t <= pos[..., None]
    return seen & (t > pos[..., None] - st["window"]) if st["window"] else seen


def _attend(st):
    c = st["case"]
    B, Hq, Hkv, D, n = c["B"], c["Hq"], c["Hkv"], c["D"], c["n"]
    table, rep = st["table"].long().clamp(min=0), Hq // Hkv
    S = table.shape[1] * PAGE
    kv = []
    for part, tokens in ((0, _k_tokens), (1, _v_tokens)):
        x = tokens(st["codes"][table, :, part]).float() * st["scales"][table, :, part][..., None, None]    # [B][P][Hkv][64][D]
        kv.append(x.transpose(1, 2).reshape(B * Hkv, S, D))
    i, j = _rows(st["off"], st["T"])
    q = torch.zeros((B, n, Hq, D), device=i.device)
    q[i, j] = st["q"].float()
    q = q.view(B, n, Hkv, rep, D).permute(0, 2, 1, 3, 4).reshape(B * Hkv, n * rep, D)
    x = torch.matmul(q, kv[0].transpose(1, 2).contiguous()).view(B, Hkv, n, rep, S) * st["scale"]
    if st["mask"] is not None:
        x = x + st["mask"][:, None, None, None, :]
    cnt = st["off"][1:].long() - st["off"][:-1].long()
    pos = (st["lens"].long() - cnt)[:, None] + torch.arange(n, device=i.device)
    see = _visible(st, pos, torch.arange(S, device=i.device))             # [B][n][S]
    x = x.masked_fill_(~see[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    sink = None
    if st["sinks"] is not None:
        sink = st["sinks"].view(1, Hkv, 1, rep, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    p = (x - m).exp_()
    l = p.sum(-1, keepdim=True)
    if sink is not None:
        l = l + (sink - m).exp()
    o = torch.matmul(p.view(B * Hkv, n * rep, S), kv[1]).view(B, Hkv, n, rep, D)
    o = torch.where(l > 0, o / l, 0.0).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)
    return o[i, j].to(st["q"].dtype)


# ---------------------------------------------------------------- one pass
def run(st):
    if own:
        from opennpu_amd.device import kv8_attn, kv8_read, kv8_write
        if "k" in st:
            kv8_write(st["codes"], st["scales"], st["k"], st["v"], st["table"], st["pos"], st["off"], st["max_n"])
            return kv8_read(st["codes"], st["scales"], st["table"], st["rpos"], st["rows"], st["roff"], st["max_back"],
                            dtype=st["dt"])
        return kv8_attn(st["q"], st["codes"], st["scales"], st["table"], st["lens"], st["off"], st["max_n"],
                        st["max_len"], mask=st["mask"], sinks=st["sinks"], window=st["window"], scale=st["scale"])
    return _append(st) if "k" in st else _attend(st)


def work(case):
    c = case
    old, new = _lengths(c)
    size, vec = 4 if c["dt"] == "f32" else 2, c["Hkv"] * c["D"]
    if c["kind"] == "append":
        T, back = sum(new), sum(o + n - o // PAGE * PAGE for o, n in zip(old, new))
        touched = sum((o + n - 1) // PAGE - o // PAGE + 1 for o, n in zip(old, new))
        # k and v in, codes and scales out; codes and scales in again, values out
        return {"bytes": 2 * vec * (T * (size + 1) + back * (1 + size)) + 3 * 8 * c["Hkv"] * touched,
                "flops": 2 * vec * (3 * T + back)}
    seen = pairs = 0
    for o, n in zip(old, new):
        w = c["window"] or o + n
        seen += o + n - max(0, o + 1 - w)
        # query token j sees min(o + j + 1, w) positions
        k = max(0, min(n, w - o))                                         # tokens that see less than the window
        pairs += k * o + k * (k + 1) // 2 + (n - k) * w
    T = sum(new)
    return {"bytes": 2 * vec * seen + 8 * c["Hkv"] * (seen // PAGE) + 2 * size * T * c["Hq"] * c["D"] +
            (4 * seen if c["mask"] else 0), "flops": 4 * c["D"] * c["Hq"] * pairs}


# ---------------------------------------------------------------- from the definition, in 64 bits
def _held(codes, D):
    """codes [pages][Hkv][2][64 D] -> the place of (token, d) in a page's K and V tiles, as index arrays"""
    t, d = np.arange(PAGE)[:, None], np.arange(D)[None]
    k = ((t // 16) * (D // 16) + d // 16) * 256 + t % 16 * 16 + d % 16
    v = (d // 16) * 1024 + (t // 4 % 4) * 256 + d % 16 * 16 + t // 16 * 4 + t % 4
    return [torch.from_numpy(a).to(codes.device) for a in (k, v)]


def exact(case, seed):
    st = prepare(case, seed)
    D, Hkv = case["D"], case["Hkv"]
    place = _held(st["codes"], D)
    old, new = _lengths(case)
    table, off = st["table"].cpu().numpy(), _offsets(new)
    if case["kind"] == "append":
        outs = ([], [])
        for i, (o, n) in enumerate(zip(old, new)):
            pages = torch.from_numpy(table[i, o // PAGE:(o + n - 1) // PAGE + 1].astype(np.int64)).cuda()
            first = o - o // PAGE * PAGE                                  # slots held before
            for part, x in enumerate((st["k"], st["v"])):
                x = x[int(off[i]):int(off[i + 1])].double()
                z = torch.zeros((len(pages) * PAGE, Hkv, D), dtype=torch.float64, device="cuda")
                z[first:first + n] = x
                z = z.view(len(pages), PAGE, Hkv, D)
                s = (z.abs().amax(dim=(1, 3)).clamp(min=TINY) / 127).float().double()    # a scale is held in 32 bits
                before = st["scales"][pages[0], :, part].double()
                if first:
                    s[0] = torch.maximum(s[0], before)
                value = torch.round(z / s[:, None, :, None]) * s[:, None, :, None]
                if first:
                    held = st["codes"][pages[0], :, part][:, place[part]].double()    # [Hkv][64][D]
                    kept = torch.round(held * (before / s[0])[:, None, None]) * s[0][:, None, None]
                    value[0, :first] = kept[:, :first].transpose(0, 1)
                outs[part].append(value.view(-1, Hkv, D)[:first + n])
        return [torch.cat(o) for o in outs]
    Hq, rep = case["Hq"], case["Hq"] // Hkv
    outs = []
    for i, (o, n) in enumerate(zip(old, new)):
        P = (o + n + PAGE - 1) // PAGE
        pages = torch.from_numpy(table[i, :P].astype(np.int64)).cuda()
        q = st["q"][int(off[i]):int(off[i + 1])].double()
        res = torch.zeros((n, Hq, D), dtype=torch.float64, device="cuda")
        t = torch.arange(o + n, device="cuda")
        for g in range(Hkv):
            K, V = (st["codes"][pages, g, part][:, place[part]].double().mul_(st["scales"][pages, g, part].double()[:, None, None])
                    .view(P * PAGE, D)[:o + n] for part in (0, 1))
            for a in range(0, n, 256):
                b = min(n, a + 256)
                at = torch.arange(o + a, o + b, device="cuda")[:, None]
                dead = t[None] > at
                if st["window"]:
                    dead |= t[None] <= at - st["window"]
                y = torch.einsum("jrd,td->jrt", q[a:b, g * rep:(g + 1) * rep], K) * st["scale"]
                if st["mask"] is not None:
                    y = y + st["mask"][i, :o + n].double()
                y.masked_fill_(dead[:, None], -math.inf)
                if st["sinks"] is not None:
                    sk = st["sinks"][g * rep:(g + 1) * rep].double()[None, :, None].expand(b - a, -1, 1)
                    w = torch.softmax(torch.cat([y, sk], -1), -1)[..., :-1]
                else:
                    w = torch.softmax(y, -1)
                res[a:b, g * rep:(g + 1) * rep] = torch.einsum("jrt,td->jrd", w, V)
        outs.append(res)
    return torch.cat(outs)
