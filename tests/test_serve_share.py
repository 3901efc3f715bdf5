"""Each attention workgroup's search for its share of the work, on the host: the
functions that the kernels call (csrc/serve_batch.hpp), for every workgroup of
a launch.  None of this reaches a GPU."""
import ctypes as C
import os

import numpy as np
import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "c", "libserve_share.so")


class HostShare(C.Structure):
    _fields_ = [("page_table", C.c_void_p), ("kv_len", C.c_void_p), ("q_start", C.c_void_p),
                ("table_stride", C.c_longlong)] + [(n, C.c_int) for n in (
                    "T", "B", "max_pages", "page_log2", "n_pages", "prefix_len", "G", "Hkv", "rows", "keys_log2",
                    "pre_blocks", "stacked", "pause", "long_groups")]


@pytest.fixture(scope="module")
def host():
    assert os.path.exists(LIB), "build tests/c first (__graft_entry__.build())"
    h = C.CDLL(LIB)
    h.serve_shares.restype = C.c_longlong
    return h


def _shares(host, lens, start, T, cap, launched, by_xcd=False, G=1, Hkv=1, rows=16, keys_log2=7, pre=0, stacked=0,
            pause=0, long_groups=0):
    keep = [np.ascontiguousarray(x, np.int32) if x is not None else None for x in (np.zeros((len(lens), cap)), lens, start)]
    h = HostShare(*[None if x is None else x.ctypes.data for x in keep], cap, T, len(lens), cap, 4, 1, 0, G, Hkv, rows,
                  keys_log2, pre, stacked, pause, long_groups)
    most = 1 << 16
    out, ranges, units = np.zeros((most, 9), np.int64), np.zeros((launched, 2), np.int64), C.c_longlong()
    n = host.serve_shares(C.byref(h), launched, int(by_xcd), C.c_void_p(out.ctypes.data), C.c_longlong(most),
                          C.c_void_p(ranges.ctypes.data), C.byref(units))
    assert n >= 0, n
    return out[:n], ranges, units.value


def _groups(news, lens, cap, G, Hkv, rows, keys, pre):
    """Blocks of every (sequence, tile, head), from their definition."""
    want = {}
    for s, n in enumerate(news):
        for tile in range(-(-n * G // rows)):
            last = min(n - 1, ((tile + 1) * rows - 1) // G)
            seen = min(max(lens[s] - n + last + 1, 0), max(min(lens[s], cap * 16), 0))
            for h in range(Hkv):
                want[(s, tile, h)] = max(1, pre + -(-seen // keys))
    return want


BATCHES = [
    # news, lens, G, Hkv, rows, keys, prefix blocks
    ([1], [1], 1, 1, 16, 128, 0),
    ([1] * 9, [0, 1, 127, 128, 129, 1000, 5, 0, 300], 4, 8, 16, 128, 0),
    ([1] * 300, [17 * (i % 50) for i in range(300)], 6, 2, 16, 128, 0),
    ([i % 3 for i in range(700)], [40 * (i % 7) for i in range(700)], 2, 2, 16, 128, 1),
    ([40, 0, 7, 1], [10, 12, 500, 3], 40, 1, 128, 64, 0),
    ([200, 3], [200, 900], 4, 2, 128, 64, 1),
    ([0, 0, 1100, 0], [0, 0, 1100, 0], 1, 2, 16, 128, 0),  # more tiles than a wave's lanes
    ([0] * 20 + [9000] + [1] * 40, [0] * 20 + [9000] + [300] * 40, 1, 1, 128, 64, 0),
    ([1] * 30 + [1500] + [0] * 270, [500] * 30 + [1500] + [0] * 270, 1, 1, 16, 128, 0),
    ([500, 700, 300], [900, 700, 2000], 4, 2, 128, 64, 0),
]


@pytest.mark.parametrize("news,lens,G,Hkv,rows,keys,pre", BATCHES)
@pytest.mark.parametrize("launched,by_xcd", [(512, False), (512, True), (24, True), (7, True)])
@pytest.mark.parametrize("pause,long_groups", [(0, 0), (3, 0), (3, 1), (3, 20), (1, 400)])
def test_every_block_is_in_one_share(host, news, lens, G, Hkv, rows, keys, pre, launched, by_xcd, pause, long_groups):
    cap, start = -(-max(max(lens), 1) // 16), np.concatenate([[0], np.cumsum(news)])
    segs, ranges, units = _shares(host, lens, start, sum(news), cap, launched, by_xcd, G, Hkv, rows,
                                  keys.bit_length() - 1, pre, 0, pause, long_groups)
    want = _groups(news, lens, cap, G, Hkv, rows, keys, pre)
    # the units, and how many workgroups have some: fewer where groups are long
    assert units == sum(nb + pause for nb in want.values())
    W = units
    if long_groups:
        W >>= sum(units >= (n + pause) * long_groups for n in (8, 16))
    W = min(W, launched)
    assert [tuple(r) for r in ranges.tolist()] == [(units * w // W, units * (w + 1) // W) if w < W else (0, 0)
                                                   for w in range(launched)]
    # every block once, a group's parts those of consecutive workgroups, in their order
    seen, last = {}, {}
    for w, s, tile, h, b0, b1, nb, st, base in segs[np.argsort(segs[:, 0], kind="stable")].tolist():
        group = (s, tile, h)
        assert nb == want[group] and b0 == seen.get(group, 0) < b1 <= nb and st == sum(news[:s])
        assert b0 == 0 or last[group] == w - 1
        assert ranges[w, 0] <= base + pause + b0 and base + pause + b1 <= ranges[w, 1]
        seen[group], last[group] = b1, w
    assert seen == want


def test_a_stacked_prefix_is_one_sequence(host):
    segs, _, units = _shares(host, [3] * 5, None, 5, 1, 6, G=4, Hkv=2, pre=9, stacked=1)
    assert set(map(tuple, segs[:, 1:4].tolist())) == {(0, t, h) for t in (0, 1) for h in (0, 1)} and units == 36


@pytest.mark.parametrize("seed", range(60))
def test_any_contents_are_searched_within_bounds(host, seed):
    """Lengths and starts of any kind: the search ends, at rows of T and at blocks of
    keys inside the table."""
    r = np.random.default_rng(seed)
    B, T, cap = int(r.integers(1, 400)), int(r.integers(1, 3000)), int(r.integers(1, 5))
    wild = lambda lo, hi, n: np.where(r.random(n) < 0.3, r.choice([-2 ** 31, -1, 0, 2 ** 31 - 1], n), r.integers(lo, hi, n))
    start = np.sort(wild(-5, T + 5, B + 1)) if seed % 2 else wild(-5, T + 5, B + 1) if B < 20 else np.clip(
        np.arange(B + 1) * 2 - 7 + r.integers(-3, 4, B + 1), -9, 2 ** 31 - 1)
    G, rows = int(r.integers(1, 9)), (16, 128)[seed % 3 == 0]
    segs, _, _ = _shares(host, wild(-20, 120, B), start, T, cap, int(r.integers(1, 600)), True, G, 2, rows, 6,
                         pause=int(r.integers(0, 4)), long_groups=int(r.integers(0, 50)))
    for w, s, tile, h, b0, b1, nb, st, base in segs.tolist():
        assert 0 <= st < T and 0 <= s < B and 0 <= h < 2 and (tile * rows) // G + st < T
        assert nb <= max(1, -(-cap * 16 // 64)) and 0 <= b0 < b1 <= nb
