"""The 8-bit key-value cache on the GPU (kv8_write, kv8_read, kv8_attn) against its definition in
64 bits (tests/kv8ref.py): codes, scales and fp32 values bit for bit, attention within bounds that are
worked out from the arithmetic (see _bound)."""
import numpy as np
import pytest

from kv8ref import PAGE, Cache

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _dt(name):
    import torch
    return torch.float32 if name == "f32" else torch.bfloat16


def _i32(a):
    return _dev(np.asarray(a, np.int32))


def _off(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _rand_cache(rng, pages, Hkv, D):
    codes = np.clip(np.rint(32 * rng.standard_normal((pages, Hkv, 2, PAGE * D))), -127, 127).astype(np.int8)
    return codes, (np.exp(0.3 * rng.standard_normal((pages, Hkv, 2))) / 32).astype(np.float32)


def _table(rng, totals, extra=2):
    """(table [n][P] of pages handed out in no order, -1 past a sequence's own, pages in all)"""
    need = [(t + PAGE - 1) // PAGE for t in totals]
    pages = sum(need) + extra
    free, table, at = rng.permutation(pages), np.full((len(totals), max(max(need), 1)), -1, np.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = free[at:at + k]
        at += k
    return table, pages


def _rows(rng, T, heads, D, dt):
    """random rows: a tensor on the GPU, and the same values in float64"""
    t = _dev(rng.standard_normal((T, heads, D)).astype(np.float32), _dt(dt))
    return t, t.float().cpu().numpy().astype(np.float64)


WRITES = [
    (1, 16, [0], [1]), (2, 48, [63], [1]), (8, 128, [64], [1]), (8, 128, [0], [64]), (4, 96, [5], [200]),
    (2, 256, [130, 0, 64, 127, 1], [1, 65, 63, 2, 128]), (3, 80, [10, 700, 33], [0, 5, 90]), (1, 64, [191], [66]),
]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hkv,D,pos,n", WRITES)
def test_write_equals_the_definition(gpu, dt, Hkv, D, pos, n):
    """codes and scales bit for bit, pages that the call does not touch as they were; twice, the second
    time with larger values (the scale grows and the earlier codes are rescaled)"""
    from opennpu_amd.device import kv8_write
    rng = np.random.default_rng(D + sum(pos) + sum(n))
    table, pages = _table(rng, [p + 2 * k for p, k in zip(pos, n)])
    codes, scales = _rand_cache(rng, pages, Hkv, D)
    ref, gc, gs = Cache(codes, scales), _dev(codes), _dev(scales)
    off = _off(n)
    print(f"kv8_write {dt} Hkv={Hkv} D={D} pos={pos} n={n}", flush=True)
    for again in range(2):
        at = [p + again * k for p, k in zip(pos, n)]
        k, kf = _rows(rng, off[-1], Hkv, D, dt)
        v, vf = _rows(rng, off[-1], Hkv, D, dt)
        k, kf, v, vf = k * (1 + again), kf * (1 + again), v * (1 + 3 * again), vf * (1 + 3 * again)
        kv8_write(gc, gs, k, v, _i32(table), _i32(at), _i32(off), max(n))
        for i in range(len(n)):
            ref.write(kf[off[i]:off[i + 1]], vf[off[i]:off[i + 1]], table[i], at[i])
        assert np.array_equal(gs.cpu().numpy(), ref.scales)
        assert np.array_equal(gc.cpu().numpy(), ref.codes)


def test_write_token_by_token(gpu):
    """150 tokens one at a time with growing and shrinking values, a window of them in bulk: every state
    equals the definition's, and reading back gives its values"""
    import torch
    from opennpu_amd.device import kv8_cache, kv8_read, kv8_write
    rng = np.random.default_rng(5)
    Hkv, D, T = 2, 64, 150
    table = np.array([[2, 0, 3]], np.int32)
    gc, gs = kv8_cache(4, Hkv, D)
    ref = Cache(gc.cpu().numpy(), gs.cpu().numpy())
    x = (rng.standard_normal((T, Hkv, D)) * np.exp(rng.standard_normal((T, 1, 1)))).astype(np.float32)
    gx, p = _dev(x), 0
    while p < T:
        n = 1 if p % 50 else 7
        n = min(n, T - p)
        kv8_write(gc, gs, gx[p:p + n], gx[p:p + n].neg(), _i32(table), _i32([p]))
        ref.write(x[p:p + n].astype(np.float64), -x[p:p + n].astype(np.float64), table[0], p)
        p += n
        assert np.array_equal(gs.cpu().numpy(), ref.scales) and np.array_equal(gc.cpu().numpy(), ref.codes), p
    k, v = kv8_read(gc, gs, _i32(table), _i32([0]), T, dtype=torch.float32)
    want = ref.read(table[0], 0, T).astype(np.float32)
    assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


def test_write_borders_between_codes(gpu):
    """values at and one step beside every border between two codes, for scales that are no power of two"""
    from opennpu_amd.device import kv8_write
    D, n = 128, 64
    codes, scales = np.zeros((2, 1, 2, 64 * D), np.int8), np.zeros((2, 1, 2), np.float32)
    gc, gs, ref = _dev(codes), _dev(scales), Cache(codes, scales)
    for amax in (127.0, 1.0, 3.7, 1e-20, 5e20, 2.0 ** -97):
        s = np.float32(np.maximum(np.float32(amax), np.float32(2.0 ** -96)) / np.float32(127))
        b = ((np.arange(-126, 127) - 0.5) * np.float64(s)).astype(np.float32)
        x = np.concatenate([b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf)), [np.float32(amax)]])
        x = np.clip(x, -np.float32(amax), np.float32(amax))
        x = np.resize(x, (n, 1, D)).astype(np.float32)
        kv8_write(gc, gs, _dev(x), _dev(x[::-1]), _i32([[1]]), _i32([0]))
        ref.write(x.astype(np.float64), x[::-1].astype(np.float64), [1], 0)
        assert np.array_equal(gs.cpu().numpy(), ref.scales)
        assert np.array_equal(gc.cpu().numpy(), ref.codes), amax


def test_write_bf16_ties_and_near_ties(gpu):
    """the bf16 values below a page's largest, down to its 2^-9: a scale of few bits makes exact ties of many, any
    other quotients within a rounding of one"""
    import torch
    from opennpu_amd.device import kv8_write
    D, n = 128, 64
    codes, scales = np.zeros((2, 1, 2, 64 * D), np.int8), np.zeros((2, 1, 2), np.float32)
    gc, gs, ref = _dev(codes), _dev(scales), Cache(codes, scales)
    for bits in [0x42fe, 0x3f80, 0x3fc8, 0x4049, 0x0301, 0x7f7f] + list(range(0x4080, 0x4100, 5)):
        top = np.arange(max(bits - 9 * 128, 0), bits + 1, dtype=np.uint32)
        x = np.concatenate([top << 16, (top << 16) | np.uint32(1 << 31)]).view(np.float32)
        x = np.resize(x, (n, 1, D))
        t = _dev(x).to(torch.bfloat16)
        assert np.array_equal(t.float().cpu().numpy(), x)
        kv8_write(gc, gs, t, t.flip(0), _i32([[1]]), _i32([0]))
        ref.write(x.astype(np.float64), x[::-1].astype(np.float64), [1], 0)
        assert np.array_equal(gs.cpu().numpy(), ref.scales)
        assert np.array_equal(gc.cpu().numpy(), ref.codes), hex(bits)


def test_write_values_that_are_not_finite(gpu):
    """the page, head and K | V that got one reads as NaN, nothing else does; beginning the page anew clears it"""
    import torch
    from opennpu_amd.device import kv8_cache, kv8_read, kv8_write
    rng = np.random.default_rng(2)
    gc, gs = kv8_cache(3, 2, 64)
    table = _i32([[2, 0]])
    for bad in (NAN, float("inf"), -float("inf")):
        x = rng.standard_normal((100, 2, 64)).astype(np.float32)
        y = x.copy()
        y[70, 1, 5] = bad
        kv8_write(gc, gs, _dev(x), _dev(y), table, _i32([0]))
        k, v = kv8_read(gc, gs, table, _i32([0]), 100, dtype=torch.float32)
        assert torch.isfinite(k).all() and torch.isfinite(v[:64]).all() and torch.isfinite(v[64:, 0]).all()
        assert torch.isnan(v[64:, 1]).all()
        kv8_write(gc, gs, _dev(x[:1]), _dev(x[:1]), table, _i32([100]))           # it stays with a later token
        assert torch.isnan(kv8_read(gc, gs, table, _i32([64]), 37)[1][:, 1]).all()
        kv8_write(gc, gs, _dev(x[:9]), _dev(x[:9]), table, _i32([64]))
        assert torch.isfinite(kv8_read(gc, gs, table, _i32([64]), 9)[1]).all()


def test_write_and_read_pages_that_do_not_exist(gpu):
    """entries outside [0, pages), positions past the table and below 0: nothing written, NaN read, every
    other byte as it was"""
    import torch
    from opennpu_amd.device import kv8_read, kv8_write
    rng = np.random.default_rng(3)
    codes, scales = _rand_cache(rng, 4, 2, 64)
    table = np.array([[1, -1, 4, 2], [2 ** 31 - 1, 0, -2 ** 31, 9], [3, 3, 3, 3]], np.int32)
    pos, n = [10, 60, -5], [300, 70, 3]
    off = _off(n)
    gc, gs, ref = _dev(codes), _dev(scales), Cache(codes, scales)
    k, kf = _rows(rng, off[-1], 2, 64, "f32")
    v, vf = _rows(rng, off[-1], 2, 64, "f32")
    kv8_write(gc, gs, k, v, _i32(table), _i32(pos), _i32(off), 300)
    for i in range(3):
        ref.write(kf[off[i]:off[i + 1]], vf[off[i]:off[i + 1]], table[i], pos[i])
    assert np.array_equal(gs.cpu().numpy(), ref.scales) and np.array_equal(gc.cpu().numpy(), ref.codes)
    out = kv8_read(gc, gs, _i32(table), _i32(pos), int(off[-1]), _i32(off), dtype=torch.float32)
    want = np.concatenate([ref.read(table[i], pos[i], n[i]) for i in range(3)], 1).astype(np.float32)
    assert np.array_equal(out[0].cpu().numpy(), want[0], equal_nan=True)
    assert np.array_equal(out[1].cpu().numpy(), want[1], equal_nan=True)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hkv,D,pos,n", WRITES)
def test_read_equals_the_definition(gpu, dt, Hkv, D, pos, n):
    """fp32: code * scale rounded once; bf16: that rounded again. Rows behind the last sequence as they were"""
    import torch
    from opennpu_amd.device import kv8_read
    rng = np.random.default_rng(D)
    table, pages = _table(rng, [p + k for p, k in zip(pos, n)])
    codes, scales = _rand_cache(rng, pages, Hkv, D)
    ref, off = Cache(codes, scales), _off(n)
    T = int(off[-1]) + 3
    out = tuple(torch.full((T, Hkv, D), 7.0, dtype=_dt(dt), device="cuda") for _ in range(2))
    kv8_read(_dev(codes), _dev(scales), _i32(table), _i32(pos), T, _i32(off), max(n), out=out)
    for kv in range(2):
        want = np.concatenate([ref.read(table[i], pos[i], n[i])[kv] for i in range(len(n))]).astype(np.float32)
        got = out[kv].float().cpu().numpy()
        assert np.array_equal(got[:-3], torch.from_numpy(want).to(_dt(dt)).float().numpy())
        assert (got[-3:] == 7).all()


def test_write_strided_rows_other_stream_and_replay(gpu):
    """k and v as views into one projection's output, on a stream of their own, then captured and replayed
    with other positions and values in the same buffers, eager calls between the replays"""
    import torch
    from opennpu_amd.device import kv8_read, kv8_write
    rng = np.random.default_rng(8)
    Hkv, D, B = 4, 64, 3
    codes, scales = _rand_cache(rng, 12, Hkv, D)
    table = np.arange(12).reshape(3, 4)[:, ::-1]
    wide = np.full((3, 9), -1, np.int32)
    wide[:, :4] = table
    gt = _i32(wide)[:, :4]                                       # rows further apart than columns
    gc, gs, ref = _dev(codes), _dev(scales), Cache(codes, scales)
    qkv = torch.zeros((B, (8 + 2 * Hkv) * D), dtype=torch.bfloat16, device="cuda")
    k, v = qkv[:, 8 * D:(8 + Hkv) * D].view(B, Hkv, D), qkv[:, (8 + Hkv) * D:].view(B, Hkv, D)
    pos = _i32([0, 0, 0])

    def step(write, at):
        x = _dev(rng.standard_normal(qkv.shape).astype(np.float32)).to(torch.bfloat16)
        qkv.copy_(x)
        pos.copy_(_i32(at))
        write()
        for i in range(B):
            ref.write(k[i:i + 1].double().cpu().numpy(), v[i:i + 1].double().cpu().numpy(), table[i], at[i])
        torch.cuda.synchronize()
        assert np.array_equal(gc.cpu().numpy(), ref.codes) and np.array_equal(gs.cpu().numpy(), ref.scales), at

    call = lambda: kv8_write(gc, gs, k, v, gt, pos)              # noqa: E731
    side = torch.cuda.Stream()

    def on_side():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
    step(call, [5, 64, 200])
    step(on_side, [6, 65, 201])
    g = torch.cuda.CUDAGraph()
    out = [torch.empty((B, Hkv, D), device="cuda") for _ in range(2)]
    with torch.cuda.graph(g):
        call()
        kv8_read(gc, gs, gt, pos, B, out=out)
    for at in ([7, 66, 202], [63, 127, 255], [64, 128, 0]):
        step(g.replay, at)
        want = np.stack([ref.read(table[i], at[i], 1)[:, 0] for i in range(B)], 1).astype(np.float32)
        assert np.array_equal(torch.stack(out).cpu().numpy(), want)
        step(call, [a + 1 if (a + 1) % 64 else a for a in at])


# ---------------------------------------------------------------- attention
def _bound(dt, ref, big, vmax, length):
    """How far an output may be off. e bounds a score's error: at most D + 8 roundings (of 2^-24 each) of terms
    that add to big = max sum |scale q K|; a softmax weight is then off by a factor e^(2 e), and by 8
    roundings of its exponential, scale and share; sums over the tokens, 64 of a page and then a page at a
    time, round 64 + pages + 16 times. All weights add to 1, so the output is off by that times 2 max |V| at
    most. bf16 outputs: the weights may be held in fp16 for the products (half a step 2^-11), and the
    result is rounded to bf16 (half a step, 2^-8)."""
    e = (256 + 8) * 2.0 ** -24 * big
    rel = np.expm1(2 * e) + (8 + 64 + length / 64 + 16) * 2.0 ** -24
    tol = 2 * vmax * rel
    return tol + 2.0 ** -22 * np.abs(ref) if dt == "f32" else tol + vmax * 2.0 ** -11 + 2.0 ** -8 * np.abs(ref)


def _attn_case(rng, dt, Hq, Hkv, D, lens, n, window=0, sinks=False, mask=None, scale=None, cache=None, loud=2.0):
    """(got [T][Hq][D] float64, want, bound) of one call over a random cache"""
    from opennpu_amd.device import kv8_attn
    table, pages = _table(rng, lens)
    codes, scales = _rand_cache(rng, pages, Hkv, D)
    if cache is not None:
        cache(table, codes, scales)
    off = _off(n)
    q = _dev((loud * rng.standard_normal((off[-1], Hq, D))).astype(np.float32), _dt(dt))
    qf = q.double().cpu().numpy()
    sk = rng.standard_normal(Hq).astype(np.float32) if sinks else None
    P = table.shape[1] * PAGE
    m = None
    if mask is not None:
        m = (0.5 * rng.standard_normal((len(n), P))).astype(np.float32)
        mask(m)
    got = kv8_attn(q, _dev(codes), _dev(scales), _i32(table), _i32(lens), _i32(off), max(n), max(max(lens), 1),
                   mask=None if m is None else _dev(m), sinks=None if sk is None else _dev(sk), window=window, scale=scale)
    ref = Cache(codes, scales)
    want, tol = np.zeros(qf.shape), np.zeros(qf.shape)
    for i, length in enumerate(lens):
        o, big, vmax = ref.attn(qf[off[i]:off[i + 1]], table[i], length, None if m is None else m[i], sk, window, scale)
        want[off[i]:off[i + 1]] = o
        tol[off[i]:off[i + 1]] = _bound(dt, o, big, vmax, length)
    return got.double().cpu().numpy(), want, tol


def _close(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    d = np.nan_to_num(np.abs(got - want))
    assert (d <= np.nan_to_num(tol)).all(), (d.max(), np.unravel_index((d - np.nan_to_num(tol)).argmax(), d.shape))


HEADS = [(1, 1, 16), (2, 2, 32), (6, 3, 48), (4, 2, 64), (10, 2, 80), (12, 2, 96), (16, 1, 128), (32, 8, 128), (7, 1, 192), (4, 2, 256),
         (20, 1, 64), (5, 5, 112)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_attn_decode(gpu, dt, Hq, Hkv, D):
    """one token of sequences of 0 to 1000 tokens, at and beside the ends of pages"""
    rng = np.random.default_rng(Hq * 1000 + D)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 0, 320]
    print(f"kv8_attn decode {dt} {Hq}/{Hkv}/{D}", flush=True)
    _close(*_attn_case(rng, dt, Hq, Hkv, D, lens, [1] * len(lens)))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_attn_several_tokens(gpu, dt, Hq, Hkv, D):
    """2 to 90 query tokens beside a decode token and a sequence without any, sinks"""
    rng = np.random.default_rng(Hq * 77 + D)
    print(f"kv8_attn tokens {dt} {Hq}/{Hkv}/{D}", flush=True)
    _close(*_attn_case(rng, dt, Hq, Hkv, D, [300, 64, 90, 9, 130, 70, 200], [2, 64, 90, 8, 1, 0, 33], sinks=True))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,lens,n", [
    (8, 2, 128, [700, 450, 128], [300, 450, 128]), (8, 2, 64, [2000], [257]), (2, 1, 256, [300, 260], [129, 260]),
    (4, 4, 96, [513], [513]), (16, 1, 80, [400], [31])])
@pytest.mark.parametrize("window,sinks", [(0, False), (100, True), (1, False)])
def test_attn_prompts(gpu, dt, Hq, Hkv, D, lens, n, window, sinks):
    rng = np.random.default_rng(D + window)
    print(f"kv8_attn prompts {dt} {Hq}/{Hkv}/{D} {lens} {n} window={window}", flush=True)
    _close(*_attn_case(rng, dt, Hq, Hkv, D, lens, n, window=window, sinks=sinks))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,S", [(8, 2, 128, 9000), (64, 8, 64, 5000), (4, 1, 256, 4100), (3, 3, 48, 12345)])
@pytest.mark.parametrize("window", [0, 1500])
def test_attn_long(gpu, dt, Hq, Hkv, D, S, window):
    """long caches beside short ones, split over many workgroups and joined"""
    rng = np.random.default_rng(S)
    print(f"kv8_attn long {dt} {Hq}/{Hkv}/{D} {S} window={window}", flush=True)
    _close(*_attn_case(rng, dt, Hq, Hkv, D, [S, 70, S // 2 + 1], [1, 1, 3], window=window, sinks=window > 0))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,n", [(8, 2, 128, 1), (4, 2, 64, 3), (8, 2, 128, 12), (4, 1, 256, 40), (6, 3, 96, 70), (2, 2, 64, 300)])
def test_attn_windows_of_several_chunks(gpu, dt, Hq, Hkv, D, n):
    """windows that are split over workgroups, beginning anywhere in a page and in any place of the sequence,
    beside sequences shorter than the window"""
    rng = np.random.default_rng(D + n)
    lens = [9001, 2564 + n, 70 + n, 5555, n, 6016]
    print(f"kv8_attn window chunks {dt} {Hq}/{Hkv}/{D} n={n}", flush=True)
    for window in (2500, 4097):
        _close(*_attn_case(rng, dt, Hq, Hkv, D, lens, [n, 1, n, 2, n, 1], window=window, sinks=window == 2500))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_attn_prompts_of_many_workgroups(gpu, dt, D, masked):
    """more prompts than the card runs at once, on themselves and behind a few tokens"""
    rng = np.random.default_rng(D)
    n = [130, 129, 1, 77, 130, 128, 64, 130, 33]
    print(f"kv8_attn many prompts {dt} D={D} masked={masked}", flush=True)

    def mask(m):
        m[2, :64] = -np.inf
        m[4, 100:] = -np.inf
    _close(*_attn_case(rng, dt, 32, 16, D, [k + 9 * i for i, k in enumerate(n)], n, mask=mask if masked else None))


@pytest.mark.parametrize("dt,D,n,masked", [("bf16", 64, 20, False), ("bf16", 128, 20, True), ("bf16", 128, 130, False),
                                           ("f32", 96, 70, False), ("f32", 128, 20, True)])
def test_attn_many_pages_of_one_workgroup(gpu, dt, D, n, masked):
    """so many sequences and heads that none is split, one of them of 150 pages, masked in places"""
    rng = np.random.default_rng(D + n)
    lens = [9601] + [n + 40 * i for i in range(15)]
    print(f"kv8_attn many pages {dt} D={D} n={n} masked={masked}", flush=True)

    def mask(m):
        m[0, 3000:7000] = -np.inf
    _close(*_attn_case(rng, dt, 16, 16, D, lens, [n] + [3] * 14 + [n], mask=mask if masked else None))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 5, 150])
@pytest.mark.parametrize("sinks", [False, True])
def test_attn_masks(gpu, dt, n, sinks):
    """left padding by -inf that leaves query rows without a position, a sequence masked whole, a mask of the
    type's lowest value (on some positions, and on all: then it counts as a constant), a NaN behind the
    sequence's last token"""
    rng = np.random.default_rng(n)
    low = np.finfo(np.float32).min
    lens = [400, 333, 200, 200, 700]

    def mask(m):
        m[0, :330] = -np.inf
        m[1] = -np.inf
        m[2, :150] = low
        m[3] = low
        m[4, 100:500] = -np.inf
        for i, s in enumerate(lens):
            m[i, s:] = np.nan
    print(f"kv8_attn masks {dt} n={n}", flush=True)
    got, want, tol = _attn_case(rng, dt, 8, 2, 128, lens, [n] * 5, mask=mask, sinks=sinks)
    _close(got, want, tol)
    assert (got[n:2 * n] == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 100])
def test_attn_pages_that_do_not_exist_and_poisoned_pages(gpu, dt, n):
    """a sequence that needs a page which its table does not have, or whose page holds a NaN, gives NaN where
    it sees that page; others are right; query rows before the first token give zeros"""
    rng = np.random.default_rng(4)
    lens, ns = [500, 500, 300, max(n - 2, 1), 400], [n, n, n, n, n]

    def spoil(table, codes, scales):
        table[0, 2] = -1
        table[1, 7] = 10 ** 6
        scales[table[2, 1], 1, 0] = np.nan
    got, want, tol = _attn_case(rng, dt, 4, 2, 64, lens, ns, cache=spoil)
    assert np.isnan(got[:n]).all() and np.isnan(got[2 * n - 1]).all()
    assert np.isnan(got[3 * n - 1, 2:]).all() and np.isfinite(got[3 * n - 1, :2]).all()
    assert np.isfinite(got[3 * n:]).all()
    ok = np.isfinite(want)
    assert (np.abs(got - want)[ok] <= tol[ok]).all() if np.isfinite(got[ok]).all() else False


@pytest.mark.parametrize("n", [1, 4, 130])
def test_attn_lengths_past_max_len(gpu, n):
    """a sequence longer than the bound that the caller gave: NaN, and the others are right"""
    import torch
    from opennpu_amd.device import kv8_attn
    rng = np.random.default_rng(6)
    table, pages = _table(rng, [400, 200])
    codes, scales = _rand_cache(rng, pages, 2, 64)
    q = torch.randn((2 * n, 4, 64), device="cuda")
    args = (q, _dev(codes), _dev(scales), _i32(table), _i32([400, 200]))
    full, cut = kv8_attn(*args), kv8_attn(*args, max_len=200)
    assert torch.isnan(cut[:n]).all() and torch.isfinite(full).all()
    assert torch.allclose(cut[n:], full[n:], rtol=0, atol=1e-4)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 40])
def test_attn_scales_far_apart(gpu, dt, n):
    """pages whose values are 2^-20 and 2^20 of their neighbours', weights that hold on to the small ones, a
    negative and a zero score scale"""
    rng = np.random.default_rng(9)

    def spread(table, codes, scales):
        scales[:, :, 1] *= (2.0 ** rng.integers(-20, 20, scales[:, :, 1].shape)).astype(np.float32)
    for scale in (0.125, -0.125, 0.0):
        _close(*_attn_case(rng, dt, 4, 2, 64, [700, 130], [n, n], cache=spread, scale=scale))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("loud", [0.0, 1e-30, 60.0, 3e30])
def test_attn_quiet_and_loud_queries(gpu, dt, n, loud):
    """queries of zeros (plain means), of tiny values, so loud that one position takes all, and so loud
    that scores pass the range of half precision"""
    rng = np.random.default_rng(10)
    got, want, tol = _attn_case(rng, dt, 4, 2, 64, [300, 65], [n, n], loud=loud)
    if loud < 1e20:
        _close(got, want, tol)
    else:                                                        # ties aside, one position has all the weight
        assert np.isfinite(got).all()
        hit = np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 1e-5
        assert hit.mean() > 0.99


@pytest.mark.parametrize("n", [1, 2, 70])
def test_attn_nan_queries_stay_in_their_row(gpu, n):
    import torch
    from opennpu_amd.device import kv8_attn
    rng = np.random.default_rng(11)
    table, pages = _table(rng, [300])
    codes, scales = _rand_cache(rng, pages, 2, 64)
    for dt in ("f32", "bf16"):
        q = torch.randn((n, 4, 64), device="cuda").to(_dt(dt))
        args = (_dev(codes), _dev(scales), _i32(table), _i32([300]))
        good = kv8_attn(q, *args)
        for bad in (NAN, float("inf")):
            q2 = q.clone()
            q2[n // 2, 1, 3] = bad
            got = kv8_attn(q2, *args)
            assert torch.isnan(got[n // 2, 1]).all()
            good2, got2 = good.clone(), got.clone()
            good2[n // 2, 1] = got2[n // 2, 1] = 0
            assert torch.equal(good2, got2)


@pytest.mark.parametrize("B,n,S", [(2, 1, 3000), (1, 1, 50), (2, 6, 2000), (1, 200, 900)])
def test_attn_replay_streams_and_repeats(gpu, B, n, S):
    """the same bits again, on another stream, and from a graph replayed with other lengths and queries in its
    buffers, eager calls between; two graphs with a workspace each, replayed in turn"""
    import torch
    from opennpu_amd.device import kv8_attn
    rng = np.random.default_rng(S)
    table, pages = _table(rng, [S] * B)
    codes, scales = _rand_cache(rng, pages, 2, 128)
    gc, gs, gt = _dev(codes), _dev(scales), _i32(table)
    for dt in (torch.float32, torch.bfloat16):
        q = torch.randn((B * n, 8, 128), device="cuda").to(dt)
        lens = _i32([S] * B)
        call = lambda o: kv8_attn(q, gc, gs, gt, lens, max_len=S, out=o)        # noqa: E731
        first = call(None)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call(None)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, call(None)) and torch.equal(first, other)
        outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
        for o in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call(o)
            graphs.append(g)
        for r in range(3):
            q.copy_(torch.randn(q.shape, device="cuda"))
            lens.copy_(_i32(rng.integers(n, S + 1, B)))
            for o in outs:
                o.zero_()
            for g in graphs:
                g.replay()
            want = call(None)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want), r


@pytest.mark.parametrize("n", [1, 12, 60])
def test_attn_replay_of_windows_and_masks(gpu, n):
    """a graph of a window's chunks and one of a masked call, replayed with lengths that move the window and with
    another mask in the buffers"""
    import torch
    from opennpu_amd.device import kv8_attn
    rng = np.random.default_rng(n)
    table, pages = _table(rng, [9000, 9000])
    codes, scales = _rand_cache(rng, pages, 2, 64)
    gc, gs, gt, lens = _dev(codes), _dev(scales), _i32(table), _i32([9000, 8000])
    q, mask = torch.randn((2 * n, 8, 64), device="cuda").bfloat16(), torch.zeros((2, 9000), device="cuda")
    calls = [lambda o: kv8_attn(q, gc, gs, gt, lens, max_len=9000, window=2500, out=o),         # noqa: E731
             lambda o: kv8_attn(q, gc, gs, gt, lens, max_len=9000, mask=mask, out=o)]           # noqa: E731
    graphs, outs = [], []
    for call in calls:
        call(None)
        outs.append(torch.zeros_like(q))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(outs[-1])
        graphs.append(g)
    for at in ([9000, 63 + n], [2500, 2564], [6401, 8999]):
        lens.copy_(_i32(at))
        mask.copy_(torch.where(torch.rand(mask.shape, device="cuda") < 0.5, -float("inf"), 0.0))
        for g, o, call in zip(graphs, outs, calls):
            o.zero_()
            g.replay()
            want = call(None)
            torch.cuda.synchronize()
            assert torch.equal(o, want), at


def test_attn_strided_queries_and_untouched_rows(gpu):
    """q as a view into a projection's output; rows behind the last sequence, and a sequence's rows past
    max_n, as they were"""
    import torch
    from opennpu_amd.device import kv8_attn
    rng = np.random.default_rng(12)
    table, pages = _table(rng, [100, 90])
    codes, scales = _rand_cache(rng, pages, 2, 64)
    qkv = torch.randn((9, 10 * 64), device="cuda")
    q = qkv[:, 64:64 * 9].view(9, 8, 64)
    args = (_dev(codes), _dev(scales), _i32(table), _i32([100, 90]), _i32([0, 2, 5]))
    out = torch.full((9, 8, 64), 7.0, device="cuda")
    kv8_attn(q, *args, max_n=3, out=out)
    want = kv8_attn(q.contiguous(), *args, max_n=3)
    assert torch.equal(out[:5], want[:5]) and (out[5:] == 7).all()
    out.fill_(7)
    kv8_attn(q, *args, max_n=2, out=out)                         # (the positions stay those of all three rows)
    assert torch.equal(out[:4], want[:4]) and (out[4:] == 7).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attn_many_pages_in_one_workgroup(gpu, dt):
    """a sequence of more than 64 pages that is not split, beside short ones; one of its late pages holds a NaN
    that the rows before it do not see, also where they share a wave with rows that do"""
    rng = np.random.default_rng(21)
    lens, n = [4500] + [30] * 39, [20] * 40

    def spoil(table, codes, scales):
        scales[table[0, 70], 3, 0] = np.nan                      # tokens 4480 ..: rows 0 .. of the last 20 do not see it
        scales[table[0, 70], 5, 1] = np.nan
    got, want, tol = _attn_case(rng, dt, 8, 8, 64, lens, n)
    _close(got, want, tol)
    for length, first in ((4490, 10), (4485, 15)):               # rows from `first` on see page 70
        got, want, tol = _attn_case(rng, dt, 8, 8, 64, [length] + lens[1:], n, cache=spoil)
        bad = np.isnan(got).any(-1)
        assert bad[first:20, [3, 5]].all() and bad.sum() == 2 * (20 - first)
        ok = ~np.isnan(got)
        assert (np.abs(got - want)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 40])
def test_empty_calls(gpu, dt, n):
    """no sequences, and no rows, are no error"""
    import torch
    from opennpu_amd.device import kv8_attn, kv8_cache, kv8_read, kv8_write
    c, s = kv8_cache(2, 2, 64)
    t, p = torch.empty((0, 3), dtype=torch.int32, device="cuda"), _i32([])
    k = torch.empty((0, 2, 64), dtype=_dt(dt), device="cuda")
    kv8_write(c, s, k, k, t, p)
    assert kv8_read(c, s, t, p, 0)[0].shape == (0, 2, 64)
    assert kv8_attn(torch.empty((0, 4, 64), dtype=_dt(dt), device="cuda"), c, s, t, p).shape == (0, 4, 64)
    t, p, off = _i32([[0, 1]] * 2), _i32([0, 5]), _i32([0, 0, 0])
    kv8_write(c, s, k, k, t, p, off, n)
    out = torch.full((3, 4, 64), 7.0, dtype=_dt(dt), device="cuda")
    kv8_attn(torch.zeros_like(out), c, s, t, p, off, n, out=out)
    assert (out == 7).all() and (c == 0).all()


def test_a_run_of_the_three(gpu):
    """a prompt written and attended, then decoded token by token for a batch, as a serving loop does it, with a
    verification of three tokens at the end: against the definition at every step"""
    from opennpu_amd.device import kv8_attn, kv8_cache, kv8_read, kv8_write
    import torch
    rng = np.random.default_rng(13)
    Hq, Hkv, D, prompt = 8, 2, 64, [70, 5, 128]
    B = len(prompt)
    table, pages = _table(rng, [p + 12 for p in prompt])
    gt = _i32(table)
    gc, gs = kv8_cache(pages, Hkv, D)
    ref = Cache(gc.cpu().numpy(), gs.cpu().numpy())
    have = np.zeros(B, np.int32)
    for n in (prompt, [1] * B, [1] * B, [3] * B):
        off = _off(n)
        q, qf = _rows(rng, off[-1], Hq, D, "bf16")
        k, kf = _rows(rng, off[-1], Hkv, D, "bf16")
        v, vf = _rows(rng, off[-1], Hkv, D, "bf16")
        kv8_write(gc, gs, k, v, gt, _i32(have), _i32(off), max(n))
        got = kv8_attn(q, gc, gs, gt, _i32(have + n), _i32(off), max(n), int((have + n).max())).double().cpu().numpy()
        for i in range(B):
            a, b = off[i], off[i + 1]
            ref.write(kf[a:b], vf[a:b], table[i], int(have[i]))
            o, big, vmax = ref.attn(qf[a:b], table[i], int(have[i]) + n[i])
            assert (np.abs(got[a:b] - o) <= _bound("bf16", o, big, vmax, 200)).all()
        have = have + np.array(n, np.int32)
    assert np.array_equal(gc.cpu().numpy(), ref.codes) and np.array_equal(gs.cpu().numpy(), ref.scales)
    k, v = kv8_read(gc, gs, gt, _i32([0] * B), int(have.sum()), _i32(_off(have)), dtype=torch.float32)
    want = np.concatenate([ref.read(table[i], 0, int(have[i])) for i in range(B)], 1).astype(np.float32)
    assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


def test_argument_errors(gpu):
    """refused with ValueError or RuntimeError before anything is launched"""
    import torch
    from opennpu_amd.device import kv8_attn, kv8_cache, kv8_read, kv8_write
    c, s = kv8_cache(3, 2, 64)
    t, p = _i32([[0, 1], [2, 2]]), _i32([0, 0])
    k = torch.zeros((4, 2, 64), device="cuda")
    q = torch.zeros((4, 8, 64), device="cuda")
    kv8_write(c, s, k, k, t, p)
    kv8_attn(q, c, s, t, p)
    for bad in ((c.float(), s, k, k, t, p), (c, s.double(), k, k, t, p), (c[:, :1], s, k, k, t, p), (c, s, k.half(), k.half(), t, p),
                (c, s, k, k.bfloat16(), t, p), (c, s, k[:, :1], k[:, :1], t, p), (c, s, k.cpu(), k, t, p), (c, s, k, k, t.long(), p),
                (c, s, k, k, t, p[:1]), (c, s, k, k, t.cpu(), p), (c, s, k[:3], k[:3], t, p), (c, s, k, k, t, p, _i32([0, 4])),
                (c, s, k.transpose(1, 2).contiguous().transpose(1, 2), k, t, p)):
        with pytest.raises(ValueError):
            kv8_write(*bad)
    with pytest.raises(RuntimeError, match="16 bytes"):
        odd = torch.zeros((4 * 2 * 64 + 1,), device="cuda")[1:].view(4, 2, 64)
        kv8_write(c, s, odd, k, t, p)
    for kw in (dict(dtype=torch.float16), dict(out=(k, k[:2])), dict(out=(k, k.bfloat16())), dict(out=(k, k), dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            kv8_read(c, s, t, p, 4, **kw)
    for kw in (dict(mask=torch.zeros((2, 100), device="cuda")), dict(mask=torch.zeros((1, 128), device="cuda")),
               dict(sinks=torch.zeros((4,), device="cuda")), dict(sinks=torch.zeros((8,))), dict(out=q.bfloat16()),
               dict(out=torch.zeros((4, 8, 128), device="cuda")[:, :, :64])):
        with pytest.raises(ValueError):
            kv8_attn(q, c, s, t, p, **kw)
    for kw in (dict(window=-1), dict(max_len=0)):
        with pytest.raises(RuntimeError, match="window >= 0"):
            kv8_attn(q, c, s, t, p, **kw)
    with pytest.raises(RuntimeError, match="multiple of Hkv"):
        kv8_attn(q[:, :7], c, s, t, p)
    for bad in ([None, c, s, t, p], [q, [1], s, t, p], [q, c, s, None, p], [q, c, s, t, 5], [q.cpu(), c, s, t, p]):
        with pytest.raises(ValueError):
            kv8_attn(*bad)
    for kw in (dict(window=1.5), dict(max_len="9"), dict(scale="x")):
        with pytest.raises(TypeError):
            kv8_attn(q, c, s, t, p, **kw)
    for kw in (dict(window=2 ** 40), dict(off=_i32([0, 2, 4]), max_n=2 ** 40), dict(ws=3), dict(out=1)):
        with pytest.raises(ValueError):
            kv8_attn(q, c, s, t, p, **kw)
    with pytest.raises(RuntimeError, match="workspace"):
        kv8_attn(q, c, s, _i32(np.zeros((2, 200))), p, ws=torch.empty((16,), dtype=torch.uint8, device="cuda"))
