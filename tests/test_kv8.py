"""The 8-bit key-value cache on the CPU: its layout and index arithmetic (onpu_kv8.h compiled for the
host), among them pages and row ranges that do not exist, and what the C entries refuse."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from opennpu_amd import _lib
from kv8ref import PAGE, Cache, places

CSRC = Path(__file__).resolve().parents[1] / "opennpu_amd" / "csrc"
SRC = """
#include "onpu_kv8.h"
extern "C" {
int at(int kv, int D, int token, int d) { return kv ? kv8_v_at(D, token, d) : kv8_k_at(D, token, d); }
void rows(const int32_t * off, int i, int64_t T, int max_n, int64_t * o) { Kv8Rows r = kv8_rows(off, i, T, max_n); o[0] = r.row; o[1] = r.n; o[2] = r.all; }
int page(const int32_t * table, int64_t p, int P, int pages) { return kv8_page(table, p, P, pages); }
void seen(int64_t at, int len, int window, int * o) { Kv8Seen s = kv8_seen(at, len, window); o[0] = s.lo; o[1] = s.hi; }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv8")
    (d / "h.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "h.so"), str(d / "h.cpp")],
                   check=True)
    L = C.CDLL(str(d / "h.so"))
    L.rows.argtypes = [C.c_void_p, C.c_int, C.c_int64, C.c_int, C.c_void_p]
    L.page.argtypes = [C.c_void_p, C.c_int64, C.c_int, C.c_int]
    L.seen.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_void_p]
    return L


@pytest.mark.parametrize("D", [16, 48, 80, 96, 128, 256])
def test_layout(host, D):
    for kv, at in enumerate(places(D)):
        assert sorted(at.reshape(-1)) == list(range(PAGE * D))           # every byte once
        got = [[host.at(kv, D, t, d) for d in range(D)] for t in range(PAGE)]
        assert np.array_equal(np.array(got), at)


def test_row_ranges_stay_inside(host):
    """whatever off holds, rows [row, row + n) lie in [0, T) and n in [0, max_n]"""
    out = (C.c_int64 * 3)()
    big = 2 ** 31 - 1
    for T in (1, 7, 100):
        for a in (-big - 1, -1, 0, 3, 7, 100, big):
            for b in (-big - 1, -1, 0, 4, 7, 100, big):
                off = np.array([a, b], np.int32)
                for max_n in (1, 5, big):
                    host.rows(off.ctypes.data, 0, T, max_n, out)
                    row, n, every = out
                    assert 0 <= row <= T and 0 <= n <= max_n and row + every <= T and n == min(every, max_n)
                    if 0 <= a <= b <= T:
                        assert row == a and n == min(b - a, max_n)
    host.rows(None, 3, 20, 5, out)
    assert tuple(out) == (15, 5, 5)


def test_pages_that_do_not_exist(host):
    table = np.array([3, -1, 7, 2 ** 31 - 1, -2 ** 31, 0], np.int32)
    got = [host.page(table.ctypes.data, p, 6, 7) for p in range(-2, 8)]
    assert got == [-1, -1, 3, -1, -1, -1, -1, 0, -1, -1]
    assert host.page(table.ctypes.data, 2 ** 40, 6, 7) == -1


def test_seen_positions(host):
    out = (C.c_int * 2)()
    for at in (-2 ** 31, -5, -1, 0, 1, 63, 64, 99, 100, 2 ** 31 + 5):
        for length in (0, 1, 64, 100):
            for window in (0, 1, 2, 64, 2 ** 31 - 1):
                host.seen(at, length, window, out)
                lo, hi = out
                want = [t for t in range(length) if t <= at and (window == 0 or t > at - window)]
                assert 0 <= lo <= hi <= length
                assert list(range(lo, hi)) == want


def test_reference_quantiser():
    """the reference's own step: a value is off by at most half a step, two where a page was rescaled"""
    rng = np.random.default_rng(0)
    c = Cache(np.zeros((2, 1, 2, 64 * 32), np.int8), np.zeros((2, 1, 2), np.float32))
    x = rng.standard_normal((100, 1, 32)).astype(np.float32)
    c.write(x[:70], x[:70] * 2, [1, 0], 0)
    c.write(x[70:], x[70:] * 3, [1, 0], 70)
    k, v = c.read([1, 0], 0, 100)
    assert np.abs(k[:64] - x[:64]).max() <= 0.5001 * c.scales[1, 0, 0]
    assert np.abs(k[64:] - x[64:]).max() <= 1.0001 * c.scales[0, 0, 0]
    assert np.abs(v[70:] - 3 * x[70:]).max() <= 0.5001 * c.scales[0, 0, 1]


class _Args:
    """a call's arguments that the host accepts, with one changed; pointers are never read by the host"""
    BASE = {
        "write": dict(codes=1 << 20, scales=1 << 20, pages=4, Hkv=2, D=64, k=1 << 20, v=1 << 20, bf16=1, krs=128, khs=64,
                      vrs=128, vhs=64, table=1 << 20, tld=3, P=3, pos=1 << 20, off=1 << 20, nseq=2, T=5, max_n=4, stream=None),
        "read": dict(codes=1 << 20, scales=1 << 20, pages=4, Hkv=2, D=64, table=1 << 20, tld=3, P=3, pos=1 << 20, off=1 << 20,
                     nseq=2, T=5, max_n=4, k=1 << 20, v=1 << 20, bf16=1, stream=None),
        "attn": dict(q=1 << 20, bf16=1, Hq=4, qrs=256, qhs=64, codes=1 << 20, scales=1 << 20, pages=4, Hkv=2, D=64,
                     table=1 << 20, tld=3, P=3, lens=1 << 20, off=1 << 20, nseq=2, T=5, max_n=4, max_len=100, mask=None, mld=0,
                     sinks=None, window=0, scale=0.1, out=1 << 20, ws=1 << 20, ws_bytes=1 << 40, stream=None),
    }


CACHE = [dict(codes=None), dict(scales=None), dict(table=None), dict(D=0), dict(D=24), dict(D=272), dict(Hkv=0), dict(pages=0),
         dict(pages=1 << 31), dict(codes=(1 << 20) + 8), dict(scales=(1 << 20) + 4), dict(P=0), dict(tld=2), dict(nseq=-1),
         dict(nseq=0), dict(T=-1), dict(max_n=0), dict(off=None), dict(max_n=-1), dict(bf16=2), dict(nseq=65536, tld=3)]
MORE = {
    "write": [dict(k=None), dict(v=None), dict(pos=None), dict(k=(1 << 20) + 8), dict(krs=132), dict(khs=4), dict(vrs=1), dict(vhs=12),
              dict(bf16=0, krs=130), dict(max_n=2 ** 31 - 1)],
    "read": [dict(k=None), dict(v=None), dict(pos=None), dict(v=(1 << 20) + 4), dict(max_n=2 ** 31 - 1)],
    "attn": [dict(q=None), dict(out=None), dict(lens=None), dict(Hq=3), dict(Hq=0), dict(qrs=4), dict(qhs=2), dict(max_len=0), dict(max_len=2 ** 31 - 64),
             dict(window=-1), dict(mask=1 << 20, mld=99), dict(out=(1 << 20) + 4)],
}


@pytest.mark.parametrize("name", ["write", "read", "attn"])
def test_refusals(name):
    """each refused on the host with a reason, before anything is launched"""
    L = _lib.lib()
    fn = getattr(L, f"onpu_kv8_{name}_dev")
    for change in CACHE + MORE[name]:
        args = dict(_Args.BASE[name], **change)
        assert fn(*args.values()) == -1, change
        assert f"onpu_kv8_{name}_dev".encode() in L.onpu_last_error(), change
    # nothing to do is no error
    assert fn(*dict(_Args.BASE[name], T=0, nseq=0, max_n=0).values()) == 0


def test_short_workspace_is_refused():
    L = _lib.lib()
    need = L.onpu_kv8_attn_ws_bytes(1, 4, 64, 2, 2, 5, 4, 100000, 0)
    if need:
        args = dict(_Args.BASE["attn"], max_len=100000)
        for bad in (dict(ws_bytes=need - 1), dict(ws=None), dict(ws=(1 << 20) + 4)):
            assert L.onpu_kv8_attn_dev(*dict(args, **bad).values()) == -1
            assert b"workspace" in L.onpu_last_error()
