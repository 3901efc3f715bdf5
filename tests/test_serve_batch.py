"""The serving kernels' index functions on the host (csrc/serve_batch.hpp built
for the CPU), and the entry points' refusals: none of these reach a GPU."""
import ctypes as C
import os

import numpy as np
import pytest

import npu_amd
from npu_amd import _lib
from npu_amd.memref import BF16, F32, I32
from test_abi import _err, _mr

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "c", "libserve_batch.so")


class HostBatch(C.Structure):
    _fields_ = [("page_table", C.c_void_p), ("kv_len", C.c_void_p), ("q_start", C.c_void_p),
                ("table_stride", C.c_longlong), ("T", C.c_int), ("B", C.c_int), ("max_pages", C.c_int),
                ("page_log2", C.c_int), ("n_pages", C.c_int), ("prefix_len", C.c_int)]


@pytest.fixture(scope="module")
def host():
    assert os.path.exists(LIB), "build tests/c first (__graft_entry__.build())"
    h = C.CDLL(LIB)
    h.serve_segments.restype = C.c_longlong
    h.serve_segments.argtypes = [C.POINTER(HostBatch)] + [C.c_int] * 7 + [C.c_void_p, C.c_longlong]
    return h


def _batch(table, lens, start, T, page_log2, n_pages, prefix=0):
    keep = [np.ascontiguousarray(a, np.int32) if a is not None else None for a in (table, lens, start)]
    ptr = [None if a is None else a.ctypes.data for a in keep]
    b = HostBatch(ptr[0], ptr[1], ptr[2], keep[0].shape[1], T, keep[0].shape[0], keep[0].shape[1], page_log2, n_pages,
                  prefix)
    b.keep = keep
    return b


def _places(host, b):
    out = np.zeros((b.T, 4), np.int32)
    host.serve_places(C.byref(b), out.ctypes.data_as(C.c_void_p))
    return out


def test_places_of_tokens(host):
    table = np.array([[4, 2, 0], [1, 3, 9], [5, -1, 2 ** 31 - 1]])
    b = _batch(table, [20, 33, 40], [0, 3, 4, 9], 11, 4, 6, prefix=7)
    got = _places(host, b)
    want = [(7 + j, table[s][j // 16], j % 16, 1) for s, j in
            [(0, 17), (0, 18), (0, 19), (1, 32), (2, 35), (2, 36), (2, 37), (2, 38), (2, 39)]]
    want = [(p, q if 0 <= q < 6 else -1, i, v) for p, q, i, v in want]
    assert [tuple(r) for r in got[:9]] == want
    assert not got[9:, 3].any() and (got[9:, 1] == -1).all()  # rows of no sequence


@pytest.mark.parametrize("lens", [[0, -5, 2 ** 31 - 1], [48, 49, -2 ** 31]])
def test_places_stay_inside_the_table(host, lens):
    for start in ([0, 2, 4, 6], [0, 0, 0, 6], [0, 6, 6, 6], [-3, 2, 100, 2 ** 31 - 1], [5, 1, 3, 0],
                  [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 7], None):
        T = 3 if start is None else 6
        b = _batch(np.arange(9).reshape(3, 3), lens, start, T, 4, 9)
        got = _places(host, b)
        live = got[got[:, 3] == 1]
        assert (live[:, 0] >= 0).all() and (live[:, 0] < 48).all() and (live[:, 2] < 16).all()
        assert ((live[:, 1] >= 0) & (live[:, 1] < 9)).all()
        assert (got[got[:, 3] == 0][:, 1] == -1).all()


def _segments(host, b, G, Hkv, rows, keys, pre, stacked, W):
    most = 1 << 16
    out = np.zeros((most, 8), np.int32)
    n = host.serve_segments(C.byref(b), G, Hkv, rows, keys, pre, stacked, W, out.ctypes.data, most)
    assert n >= 0, n
    return out[:n]


SPLITS = [
    # news, lens, G, Hkv, rows, keys, prefix blocks, W
    ([1], [1], 1, 1, 16, 128, 0, 1),
    ([1] * 9, [0, 1, 127, 128, 129, 1000, 5, 0, 300], 4, 8, 16, 128, 0, 512),
    ([1] * 9, [0, 1, 127, 128, 129, 1000, 5, 0, 300], 4, 8, 16, 128, 0, 7),
    ([1] * 300, [17 * (i % 50) for i in range(300)], 6, 2, 16, 128, 0, 512),
    ([40, 0, 7, 1], [40, 12, 500, 3], 3, 2, 16, 128, 2, 64),
    ([40, 0, 7, 1], [10, 12, 500, 3], 40, 1, 128, 64, 0, 33),
    ([0, 0, 5], [9, 0, 5], 1, 3, 64, 32, 0, 512),
]


@pytest.mark.parametrize("news,lens,G,Hkv,rows,keys,pre,W", SPLITS)
@pytest.mark.parametrize("ragged", [True, False])
def test_every_block_of_every_tile_is_one_workgroups(host, news, lens, G, Hkv, rows, keys, pre, W, ragged):
    if not ragged and set(news) != {1}:
        pytest.skip("without starts each sequence has one token")
    start = np.concatenate([[0], np.cumsum(news)]) if ragged else None
    cap = -(-max(max(lens), 1) // 16)
    b = _batch(np.zeros((len(news), cap)), lens, start, sum(news), 4, 1)
    segs = _segments(host, b, G, Hkv, rows, keys, pre, 0, W)
    want = {}
    for s, n in enumerate(news):
        for tile in range(-(-n * G // rows)):
            last = min(n - 1, ((tile + 1) * rows - 1) // G)
            vis = min(max(lens[s] - n + last + 1, 0), max(lens[s], 0))
            for h in range(Hkv):
                want[(s, tile, h)] = max(1, pre + -(-vis // keys))
    seen = {}
    for w, s, tile, h, b0, b1, nb, st in segs.tolist():
        assert nb == want[(s, tile, h)] and b0 == seen.get((s, tile, h), 0) < b1
        assert st == sum(news[:s])
        seen[(s, tile, h)] = b1
    assert seen == want
    # equal shares, at most one cut at each end of a workgroup
    per = np.bincount(segs[:, 0], (segs[:, 5] - segs[:, 4]).astype(float), minlength=segs[:, 0].max() + 1)
    assert per.max() - per.min() <= 1
    assert (np.unique(segs[:, 0]) == np.arange(min(W, int(per.sum())))).all()
    for w in np.unique(segs[:, 0]):
        mine = segs[segs[:, 0] == w]
        assert (mine[1:, 4] == 0).all() and (mine[:-1, 5] == mine[:-1, 6]).all()


@pytest.mark.parametrize("news,lens,G,Hkv,rows,keys,pre,W", SPLITS + [
    ([200, 3], [200, 900], 4, 2, 128, 64, 1, 50), ([1] * 50, [1] * 50, 1, 2, 128, 64, 0, 130)])
@pytest.mark.parametrize("pause", [1, 3])
def test_every_block_is_one_workgroups_with_pauses_between_groups(host, news, lens, G, Hkv, rows, keys, pre, W, pause):
    cap = -(-max(max(lens), 1) // 16)
    b = _batch(np.zeros((len(news), cap)), lens, np.concatenate([[0], np.cumsum(news)]), sum(news), 4, 1)
    most = 1 << 16
    out = np.zeros((most, 8), np.int32)
    host.serve_segments_paused.restype = C.c_longlong
    n = host.serve_segments_paused(C.byref(b), G, Hkv, rows, keys, pre, pause, W, C.c_void_p(out.ctypes.data),
                                   C.c_longlong(most))
    assert n >= 0, n
    segs, seen, last = out[:n], {}, {}
    want = {(s, t, h): nb for _, s, t, h, _, _, nb, _ in _segments(host, b, G, Hkv, rows, keys, pre, 0, W).tolist()}
    for w, s, tile, h, b0, b1, nb, st in segs.tolist():
        assert nb == want[(s, tile, h)] and b0 == seen.get((s, tile, h), 0) < b1 and st == sum(news[:s])
        assert b0 == 0 or last[(s, tile, h)] == w - 1  # parts of consecutive workgroups
        seen[(s, tile, h)], last[(s, tile, h)] = b1, w
    assert seen == want
    # shares equal in blocks and pauses, but for what is cut at their ends
    cost = np.zeros(W)
    for w, s, tile, h, b0, b1, nb, st in segs.tolist():
        cost[w] += b1 - b0 + (pause if b0 == 0 else 0)
    units = sum(nb + pause for nb in want.values())
    assert cost.max() <= -(-units // min(W, units)) + pause


def test_the_stacked_prefix_is_one_sequence(host):
    b = _batch(np.zeros((5, 1)), [3] * 5, None, 5, 4, 1)
    segs = _segments(host, b, 4, 2, 16, 128, 9, 1, 6)
    assert set(map(tuple, segs[:, 1:4].tolist())) == {(0, t, h) for t in (0, 1) for h in (0, 1)}
    assert (segs[:, 6] == 9).all() and (segs[:, 5] - segs[:, 4]).sum() == 36


@pytest.mark.parametrize("seed", range(40))
def test_any_contents_divide_within_bounds(host, seed):
    """Lengths and starts of any kind: every segment's rows are rows of T, and
    its blocks reach no key past the table."""
    r = np.random.default_rng(seed)
    B, T, cap = int(r.integers(1, 6)), int(r.integers(1, 30)), int(r.integers(1, 5))
    wild = lambda lo, hi, n: np.where(r.random(n) < 0.3, r.choice([-2 ** 31, -1, 0, 2 ** 31 - 1], n), r.integers(lo, hi, n))
    b = _batch(np.zeros((B, cap)), wild(-20, 120, B), wild(-5, T + 5, B + 1), T, 4, 1)
    G, rows, keys = int(r.integers(1, 9)), 16, 32
    segs = _segments(host, b, G, 2, rows, keys, 0, 0, int(r.integers(1, 40)))
    for w, s, tile, h, b0, b1, nb, st in segs.tolist():
        assert 0 <= st < T and 0 <= s < B and (tile * rows) // G + st < T
        assert nb <= max(1, -(-cap * 16 // keys)) and 0 <= b0 < b1 <= nb


# ---- refusals ------------------------------------------------------------------------
def _call(fn, ms, *rest):
    return getattr(npu_amd.lib(), fn)(*[None if m is None else C.byref(m) for m in ms], *rest, None)


def _append(prefix=0, pairs=0, **over):
    a = {"Q": _mr([2, 512], BF16), "K": _mr([2, 256], BF16), "V": _mr([2, 256], BF16), "cos": _mr([64, 64]),
         "sin": _mr([64, 64]), "kp": _mr([5, 2, 16, 128], BF16), "vp": _mr([5, 2, 16, 128], BF16),
         "table": _mr([2, 4], I32), "lens": _mr([2], I32), "start": None, "Qo": _mr([2, 512], BF16)}
    a.update(over)
    return _call("fused_llama_rope_append", a.values(), prefix, pairs)


APPEND_REFUSALS = [
    (dict(Q=None), 1, "Q: null"), (dict(Q=_mr([2, 512])), 1, "element type"), (dict(Q=_mr([2, 520], BF16)), 1, "Q: rows of 520"),
    (dict(Q=_mr([2, 384], BF16)), 1, "multiple of 2"), (dict(Q=_mr([3, 512], BF16)), 1, "without q_start"),
    (dict(Q=_mr([2, 512], BF16, ptr=0x10008)), 2, "16-byte"), (dict(Q=_mr([2, 512], BF16, strides=[516, 1])), 2, "stride of 516"),
    (dict(Q=_mr([2, 512], BF16, strides=[256, 1])), 2, "overlap"), (dict(Q=_mr([2, 512], BF16, strides=[1, 2])), 2, "contiguous"),
    (dict(K=_mr([2, 128], BF16)), 1, "K: [2,128]"), (dict(V=_mr([1, 256], BF16)), 1, "V: [1,256]"),
    (dict(Qo=_mr([2, 256], BF16)), 1, "Qo"), (dict(cos=_mr([64, 60])), 2, "multiple of 8"), (dict(cos=_mr([64, 72])), 2, "up to 64"),
    (dict(cos=_mr([63, 64]), sin=_mr([63, 64])), 1, "63 positions"), (dict(sin=_mr([64, 32])), 1, "sin_t"),
    (dict(cos=_mr([64, 64], strides=[128, 1])), 2, "cos_t: must be contiguous"), (dict(prefix=1), 1, "reach 65"),
    (dict(prefix=-1), 1, "negative"), (dict(pairs=2), 1, "pairs 2"), (dict(vp=_mr([5, 2, 32, 128], BF16)), 1, "v_pages: size[2]"),
    (dict(kp=_mr([5, 2, 24, 128], BF16)), 2, "power of two"), (dict(kp=_mr([5, 2, 8, 128], BF16)), 2, "power of two"),
    (dict(kp=_mr([5, 2, 16, 96], BF16)), 2, "head dim 96"), (dict(kp=_mr([5, 2, 16, 128], BF16, strides=[4096, 128, 256, 1])), 2, "contiguous"),
    (dict(kp=_mr([5, 2, 16, 128], BF16, strides=[4000, 2048, 128, 1])), 2, "overlap"),
    (dict(kp=_mr([5, 2, 16, 128])), 1, "element type"), (dict(table=_mr([2, 4])), 1, "page_table"),
    (dict(table=_mr([2, 0], I32)), 1, "positive"), (dict(table=_mr([2, 2 ** 28], I32)), 2, "2^31"),
    (dict(lens=_mr([3], I32)), 1, "kv_len: size 3"), (dict(start=_mr([2], I32)), 1, "q_start: size 2"),
    (dict(lens=_mr([2], I32, strides=[2])), 2, "contiguous"), (dict(lens=_mr([2], I32, ptr=0x10002)), 2, "4-byte"),
]


def _attend(prefix=0, scale=0.1, **over):
    a = {"Q": _mr([2, 512], BF16), "kp": _mr([5, 2, 16, 128], BF16), "vp": _mr([5, 2, 16, 128], BF16),
         "table": _mr([2, 4], I32), "lens": _mr([2], I32), "start": None, "pre": None, "A": _mr([2, 512], BF16),
         "ws": _mr([1 << 27])}
    a.update(over)
    return _call("fused_llama_paged_attention", a.values(), prefix, C.c_float(scale))


ATTEND_REFUSALS = [
    (dict(A=_mr([2, 256], BF16)), 1, "A: [2,256]"), (dict(A=_mr([2, 512])), 1, "element type"),
    (dict(Q=_mr([2, 640], BF16)), 1, "multiple of 2"), (dict(prefix=17), 1, "prefix_table: absent"),
    (dict(prefix=17, pre=_mr([1], I32)), 1, "needs 2"), (dict(pre=_mr([1], I32)), 1, "prefix_len is 0"),
    (dict(scale=0.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
    (dict(ws=_mr([64])), 1, "workspace: 64"), (dict(ws=None), 1, "workspace"), (dict(ws=_mr([1 << 27], ptr=0x10008)), 2, "16-byte"),
    (dict(vp=_mr([4, 2, 16, 128], BF16)), 1, "v_pages"), (dict(table=_mr([2, 4], I32, strides=[3, 1])), 2, "overlap"),
]


@pytest.mark.parametrize("over,status,text", ATTEND_REFUSALS)
def test_attention_refuses(over, status, text):
    over = dict(over)
    assert _attend(over.pop("prefix", 0), over.pop("scale", 0.1), **over) == status and text in _err(), _err()


def test_attention_workspace_sizes():
    f = npu_amd.lib().npu_paged_attention_workspace
    assert f(2, 2, 4, 2, 128, 0) > 0 and f(64, 64, 32, 8, 128, 6000) > 0
    for bad in ((0, 1, 4, 2, 128, 0), (1, 1, 4, 3, 128, 0), (1, 1, 4, 2, 96, 0), (1, 1, 4, 2, 64, -1), (1, 0, 4, 2, 64, 0),
                (2 ** 30, 1, 4, 4, 64, 0), (1, 1, 2048, 1, 64, 0)):
        assert f(*bad) == -1, bad


@pytest.mark.parametrize("over,status,text", APPEND_REFUSALS)
def test_append_refuses(over, status, text):
    over = dict(over)
    assert _append(over.pop("prefix", 0), over.pop("pairs", 0), **over) == status and text in _err(), _err()


def _sample(**over):
    a = {"logits": _mr([3, 100]), "u": _mr([3]), "temperature": _mr([3]), "top_k": _mr([3], I32), "top_p": _mr([3]),
         "min_p": _mr([3]), "tokens": _mr([3], I32), "probs": _mr([3]), "ws": _mr([1 << 27])}
    a.update(over)
    return _call("fused_sample_tokens", a.values())


SAMPLE_REFUSALS = [
    (dict(logits=None), 1, "logits: null"), (dict(logits=_mr([3, 100], I32)), 1, "element type"),
    (dict(logits=_mr([300])), 1, "rank"), (dict(logits=_mr([3, (1 << 20) + 1])), 2, "2^20"),
    (dict(logits=_mr([3, 100], strides=[1, 3])), 2, "contiguous"), (dict(logits=_mr([3, 100], strides=[90, 1])), 2, "overlap"),
    (dict(logits=_mr([3, 100], ptr=0x10002)), 2, "4-byte"), (dict(u=None), 1, "u: null"), (dict(u=_mr([4])), 1, "u: size 4"),
    (dict(temperature=_mr([1])), 1, "temperature"), (dict(top_k=_mr([3])), 1, "top_k"), (dict(top_p=_mr([3], BF16)), 1, "top_p"),
    (dict(min_p=_mr([3], strides=[2])), 2, "min_p"), (dict(tokens=None), 1, "tokens"), (dict(tokens=_mr([3])), 1, "tokens"),
    (dict(probs=_mr([2])), 1, "probs"), (dict(ws=None), 1, "workspace"), (dict(ws=_mr([1])), 1, "workspace: 1"),
]


@pytest.mark.parametrize("over,status,text", SAMPLE_REFUSALS)
def test_sampling_refuses(over, status, text):
    assert _sample(**over) == status and text in _err(), _err()


def test_sampling_workspace_sizes():
    f = npu_amd.lib().npu_sample_workspace
    assert f(1, 1) > 0 and f(256, 1 << 20) > 0
    assert [f(0, 5), f(5, 0), f(1, (1 << 20) + 1), f(-1, 5)] == [-1] * 4


def test_wrappers_refuse_host_tensors():
    import torch
    from npu_amd import groups
    t = lambda *s, d=torch.bfloat16: torch.zeros(s, dtype=d)
    i = lambda *s: t(*s, d=torch.int32)
    with pytest.raises(ValueError, match="Q: expected a tensor on the GPU"):
        groups.fused_llama_rope_append(t(1, 64), t(1, 64), t(1, 64), t(16, 32, d=torch.float32),
                                       t(16, 32, d=torch.float32), t(1, 1, 16, 64), t(1, 1, 16, 64), i(1, 1), i(1),
                                       t(1, 64))


def _fake(number):
    """sample_tokens' operands as tensors without memory on a device of any number."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, d=torch.float32: torch.empty(s, dtype=d, device="cuda:0")
        args = {"logits": e(2, 64), "u": e(2), "tokens": e(2, d=torch.int32), "workspace": e(4)}
    for t in args.values():
        t.fake_device = torch.device("cuda", number)
    return args


def test_wrappers_refuse_tensors_of_several_devices():
    from npu_amd import groups
    for name in ("u", "tokens", "workspace"):
        args = dict(_fake(0), **{name: _fake(1)[name]})
        with pytest.raises(ValueError, match=f"{name}: on cuda:1, logits on cuda:0"):
            groups.fused_sample_tokens(**args)


@pytest.mark.gpu
def test_wrappers_refuse_tensors_of_another_than_the_current_device(cuda):
    from npu_amd import groups
    with pytest.raises(ValueError, match="logits: on cuda:1, the current device is cuda:0"):
        groups.fused_sample_tokens(**_fake(1))


# ---- the build -----------------------------------------------------------------------
@pytest.mark.parametrize("python,built", [("python3", True), ("false", False)])
def test_the_python_binding_is_built_where_there_is_a_torch_to_bind_to(python, built):
    """The library itself needs hipcc and g++ alone."""
    import subprocess
    said = subprocess.run(["make", "-n", "-B", "-C", _lib.SRC_DIR, f"PYTHON={python}"], check=True, capture_output=True,
                          text=True).stdout
    assert "libnpu_amd.so" in said and "libnpu_host.so" in said and "npu_calibrate" in said
    assert ("serve_bind.cpp" in said) == built
