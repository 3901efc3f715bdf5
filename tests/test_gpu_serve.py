"""The serving operators on the GPU against their plain 64-bit forms
(serve_refs.py)."""
import math

import numpy as np
import pytest
import torch

import serve_refs as R

pytestmark = pytest.mark.gpu

BF16_HALF_STEP = 2.0 ** -8  # finfo(bfloat16).eps / 2


# ---- append ------------------------------------------------------------------------
def _append_bound(exact, mag):
    """Two products and a sum in f32 (three roundings of at most 2^-24 of the
    products' magnitudes), then one rounding to bf16."""
    return BF16_HALF_STEP * exact.abs() + (1 + BF16_HALF_STEP) * 3 * 2.0 ** -24 * mag


def _check_append(bt, Q, K, V, cos, sin, Qo, pairs, **kw):
    from npu_amd import groups
    ref = R.append64(bt, Q, K, V, cos, sin, pairs)
    groups.fused_llama_rope_append(Q, K, V, cos, sin, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, Qo,
                                   q_start=bt.q_start, prefix_len=bt.prefix, pairs=pairs, **kw)
    torch.cuda.synchronize()
    q, k, v = (t.cpu().double() for t in (Qo, bt.k_pages, bt.v_pages))
    assert ((q - ref[0]).abs() <= _append_bound(ref[0], ref[1])).all()
    assert ((k - ref[2]).abs() <= _append_bound(ref[2], ref[3])).all()
    assert torch.equal(v, ref[4])


APPEND = [
    # news, lens, H, Hkv, Dh, page, prefix, pairs, width, kind
    ([1], [1], 8, 8, 64, 16, 0, "interleaved", 32, {}),
    ([1] * 7, [1, 16, 17, 32, 33, 100, 15], 32, 8, 128, 16, 0, "interleaved", 64, {"ragged": False}),
    ([1] * 70, list(range(1, 71)), 4, 1, 64, 32, 5, "halves", 32, {"ragged": False}),
    ([5, 0, 37, 1], [5, 3, 90, 64], 6, 2, 128, 64, 100, "halves", 64, {}),
    ([33, 2], [33, 40], 5, 5, 64, 16, 7, "interleaved", 8, {}),      # the first 16 entries of a head
    ([33, 2], [33, 40], 3, 3, 128, 32, 0, "halves", 24, {}),         # 48 of 128
    ([4, 3], [2, 0], 4, 2, 64, 16, 0, "interleaved", 32, {}),        # tokens before their table
    ([6, 1], [50, 1], 4, 2, 64, 16, 0, "halves", 32, {"max_pages": 3}),   # tokens past it
    ([3, 2], [9, 20], 4, 2, 64, 16, 3, "interleaved", 32, {"extra": 4}),  # rows of no sequence
]


@pytest.mark.parametrize("news,lens,H,Hkv,Dh,page,prefix,pairs,width,kind", APPEND)
def test_append(cuda, news, lens, H, Hkv, Dh, page, prefix, pairs, width, kind):
    bt = R.Batch(news, lens, Hkv, Dh, page, prefix, seed=len(news) + H, **kind)
    cos, sin = (t.cuda() for t in R.rope_tables(prefix + bt.max_pages * page, width))
    Q, K, V = bt.rnd(bt.T, H * Dh), bt.rnd(bt.T, Hkv * Dh), bt.rnd(bt.T, Hkv * Dh)
    _check_append(bt, Q, K, V, cos, sin, torch.full_like(Q, 7.0), pairs)


def test_append_slices_in_place_and_strided_pages(cuda):
    """Q, K, V as slices of one buffer, Qo = Q, and a cache whose keys and
    values share one allocation page by page."""
    bt = R.Batch([3, 9, 1], [30, 9, 17], 2, 64, 16, 4, seed=5)
    H, Hkv, Dh = 6, 2, 64
    buf = bt.rnd(bt.T, (H + 2 * Hkv) * Dh + 16)
    Q, K, V = (buf[:, a * Dh:b * Dh] for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
    both = bt.rnd(bt.P, 2, Hkv, 16, Dh)
    bt.k_pages, bt.v_pages = both[:, 0], both[:, 1]
    cos, sin = (t.cuda() for t in R.rope_tables(4 + bt.max_pages * 16, 32))
    rest = buf[:, (H + 2 * Hkv) * Dh:].clone()
    ref = R.append64(bt, Q, K, V, cos, sin, "interleaved")
    from npu_amd import groups
    groups.fused_llama_rope_append(Q, K, V, cos, sin, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, Q,
                                   q_start=bt.q_start, prefix_len=4)
    assert ((Q.cpu().double() - ref[0]).abs() <= _append_bound(ref[0], ref[1])).all()
    assert ((bt.k_pages.cpu().double() - ref[2]).abs() <= _append_bound(ref[2], ref[3])).all()
    assert torch.equal(bt.v_pages.cpu().double(), ref[4]) and torch.equal(buf[:, (H + 2 * Hkv) * Dh:], rest)


def test_append_bad_pages_store_nothing(cuda):
    bt = R.Batch([2, 1, 1], [20, 5, 5], 2, 64, 16, seed=6)
    bt.page_table[0, 1], bt.page_table[1, 0], bt.page_table[2, 0] = bt.P, -5, 2 ** 31 - 1
    Q, K, V = bt.rnd(bt.T, 128), bt.rnd(bt.T, 128), bt.rnd(bt.T, 128)
    cos, sin = (t.cuda() for t in R.rope_tables(bt.max_pages * 16, 32))
    before = bt.k_pages.clone(), bt.v_pages.clone()
    _check_append(bt, Q, K, V, cos, sin, torch.empty_like(Q), "halves")
    assert torch.equal(bt.k_pages, before[0]) and torch.equal(bt.v_pages, before[1])


def test_append_to_a_cache_past_32_bits(cuda):
    """A cache of more than 2^31 elements: the last pages are written, and the
    places that a 32-bit offset would name are not."""
    Hkv, page, Dh, P = 8, 64, 128, 33000
    assert P * Hkv * page * Dh > 2 ** 31
    k, v = (torch.zeros((P, Hkv, page, Dh), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[P - 1], [P - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([64, 3], dtype=torch.int32, device="cuda")
    bt = R.Batch([1, 1], [1, 1], Hkv, Dh, page)
    Q, K, V = bt.rnd(2, Hkv * Dh), bt.rnd(2, Hkv * Dh), bt.rnd(2, Hkv * Dh)
    from npu_amd import groups
    cos, sin = (t.cuda() for t in R.rope_tables(page, 64))
    groups.fused_llama_rope_append(Q, K, V, cos, sin, k, v, table, lens, torch.empty_like(Q))
    assert torch.equal(v[P - 1, :, 63].reshape(-1), V[0]) and torch.equal(v[P - 2, :, 2].reshape(-1), V[1])
    assert int(torch.count_nonzero(v)) == int(torch.count_nonzero(V))
    assert int(torch.count_nonzero(k[:P - 2])) == 0


def test_append_on_another_stream_and_captured(cuda):
    """The call on a side stream, and captured: a replay appends at the lengths
    that the device arrays then hold."""
    from npu_amd import groups
    bt = R.Batch([1, 1], [3, 18], 2, 64, 16, ragged=False, max_pages=2, seed=8)
    cos, sin = (t.cuda() for t in R.rope_tables(32, 32))
    Q, K, V = bt.rnd(2, 256), bt.rnd(2, 128), bt.rnd(2, 128)
    Qo = torch.empty_like(Q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = lambda st: groups.fused_llama_rope_append(Q, K, V, cos, sin, bt.k_pages, bt.v_pages, bt.page_table,
                                                     bt.kv_len, Qo, stream=st)
    ref = R.append64(bt, Q, K, V, cos, sin, "interleaved")
    call(side)
    side.synchronize()
    assert ((Qo.cpu().double() - ref[0]).abs() <= _append_bound(ref[0], ref[1])).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(torch.cuda.current_stream())
    for step in range(3):
        bt.kv_len += 1
        bt.lens = [n + 1 for n in bt.lens]
        Q.copy_(bt.rnd(2, 256))
        ref = R.append64(bt, Q, K, V, cos, sin, "interleaved")
        g.replay()
        torch.cuda.synchronize()
        assert ((Qo.cpu().double() - ref[0]).abs() <= _append_bound(ref[0], ref[1])).all(), step
        assert ((bt.k_pages.cpu().double() - ref[2]).abs() <= _append_bound(ref[2], ref[3])).all(), step
        assert torch.equal(bt.v_pages.cpu().double(), ref[4]), step


# ---- attention -----------------------------------------------------------------------
def _attend_bound(bt, Q, scale, exact, mag, seen):
    """|A - exact| at most: the output's rounding, 2^-8 |exact|; the
    probabilities', 2^-8 of every term; the logits' f32 sums, Dh + 4 roundings of
    the products' magnitudes (at most |q| |k| scale), an error of the exponent and
    so of p, above and below the line; and the f32 sums over the keys, above and
    below, whose rescalings cost no more than as many terms again."""
    norm = lambda t: float(torch.nan_to_num(t.detach().cpu().double(), nan=0.0, posinf=0.0, neginf=0.0)
                           .reshape(-1, bt.Dh).norm(dim=1).max())
    logit = norm(Q) * norm(bt.k_pages) * scale
    per_term = 2.0 ** -8 + 2 * (bt.Dh + 4) * 2.0 ** -24 * logit + 4 * (seen[:, None] + 64) * 2.0 ** -24
    return BF16_HALF_STEP * exact.abs() + (1 + BF16_HALF_STEP) * per_term * mag


def _attend(bt, Q, A=None, scale=None, stream=None):
    from npu_amd import groups
    A = torch.full_like(Q, 3.0) if A is None else A
    ws = groups.paged_attention_workspace(Q, bt.k_pages, bt.page_table, bt.prefix)
    ws.fill_(float("nan"))
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    groups.fused_llama_paged_attention(Q, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, A,
                                       scale or bt.Dh ** -0.5, ws, q_start=bt.q_start,
                                       prefix_table=bt.prefix_table, prefix_len=bt.prefix, stream=stream)
    torch.cuda.synchronize()
    return A


def _check_attend(bt, Q, A=None, scale=None, stream=None):
    A = _attend(bt, Q, A, scale, stream)
    scale = scale or bt.Dh ** -0.5
    exact, mag, seen = R.attend64(bt, Q, scale)
    got = A.cpu().double()
    assert torch.isfinite(got).all()
    bad = (got - exact).abs() > _attend_bound(bt, Q, scale, exact, mag, seen)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"
    return A


ATTEND = [
    # news, lens, H, Hkv, Dh, page, prefix, kind
    ([1], [1], 1, 1, 64, 16, 0, {"ragged": False}),
    ([1], [500], 8, 8, 64, 16, 0, {"ragged": False}),
    ([1], [5000], 8, 2, 128, 64, 0, {"ragged": False}),
    ([1] * 12, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 700], 6, 2, 128, 16, 0, {"ragged": False}),
    ([1] * 9, [0, 1, 100, 0, 0, 3, 257, 64, 65], 16, 1, 64, 32, 0, {"ragged": False}),
    ([1] * 5, [3, 40, 0, 1, 90], 34, 2, 64, 16, 0, {"ragged": False}),   # 17 rows a key head
    ([1] * 300, [(37 * i) % 90 for i in range(300)], 4, 2, 64, 16, 0, {"ragged": False}),
    ([1] * 6, [0, 1, 100, 30, 0, 3], 8, 2, 128, 16, 1, {"ragged": False}),     # a prefix of one key
    ([1] * 40, [(13 * i) % 70 for i in range(40)], 8, 2, 64, 32, 333, {"ragged": False}),
    ([1] * 3, [0, 0, 0], 4, 4, 64, 16, 129, {"ragged": False}),                # the prefix alone
    ([1], [77], 6, 3, 128, 16, 140, {"ragged": False}),
    ([5, 0, 37, 1], [5, 3, 90, 64], 6, 2, 128, 64, 0, {}),
    ([5, 0, 37, 1], [5, 3, 90, 64], 6, 2, 64, 16, 100, {}),
    ([1, 2, 0, 1], [9, 2, 1, 40], 4, 2, 64, 16, 50, {}),                       # few rows, ragged, shared prefix
    ([150, 65], [150, 400], 3, 1, 128, 32, 0, {}),
    ([300], [300], 4, 4, 64, 16, 20, {}),
    ([700], [900], 10, 2, 128, 16, 0, {}),
    ([4, 3], [2, 0], 4, 2, 64, 16, 0, {}),                # tokens that see nothing
    ([4, 3], [2, 0], 4, 2, 64, 16, 9, {}),                # or the prefix alone
    ([6, 1], [50, 1], 4, 2, 64, 16, 0, {"max_pages": 3}),  # keys past the table
    ([3, 2], [9, 20], 4, 2, 64, 16, 0, {"extra": 4}),      # rows of no sequence
    ([1, 2], [9, 20], 4, 2, 64, 16, 40, {"extra": 4}),
    ([257, 0, 90], [300, 7, 90], 4, 1, 64, 64, 33, {"extra": 3}),
    ([128], [128], 1, 1, 128, 16, 0, {}),
    ([129], [2], 2, 1, 128, 16, 65, {}),                   # most tokens see the prefix alone
    ([200], [50], 1, 1, 64, 16, 0, {}),                    # most tokens see nothing
    ([64], [2000], 3, 3, 128, 32, 0, {}),
    ([1] * 90, [i % 7 for i in range(90)], 6, 2, 128, 16, 500, {"ragged": False}),
    ([3] * 30, [3 + i for i in range(30)], 4, 4, 64, 16, 257, {}),
    # tables that reach past 1024 keys, whatever the lengths: divided over workgroups
    ([1] * 12, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 700], 6, 2, 128, 16, 0, {"ragged": False, "max_pages": 70}),
    ([1] * 5, [3, 40, 0, 1, 90], 34, 2, 64, 16, 0, {"ragged": False, "max_pages": 70}),
    ([1] * 300, [(37 * i) % 90 for i in range(300)], 4, 2, 64, 16, 0, {"ragged": False, "max_pages": 70}),
    ([1] * 6, [0, 1, 100, 30, 0, 3], 8, 2, 128, 16, 1, {"ragged": False, "max_pages": 70}),
    ([1] * 40, [(13 * i) % 70 for i in range(40)], 8, 2, 64, 32, 333, {"ragged": False, "max_pages": 70}),
    # and ones that do not: whole groups to a workgroup, of four waves and of eight
    ([1] * 5, [1024, 1023, 0, 513, 257], 8, 4, 128, 32, 0, {"ragged": False}),
    ([1] * 70, [(97 * i) % 1025 for i in range(70)], 8, 4, 64, 256, 0, {"ragged": False}),
    ([1] * 70, [(97 * i) % 1025 for i in range(70)], 12, 4, 128, 32, 700, {"ragged": False}),
    ([1], [900], 5, 5, 64, 16, 100, {"ragged": False}),
]


@pytest.mark.parametrize("news,lens,H,Hkv,Dh,page,prefix,kind", ATTEND)
def test_attention(cuda, news, lens, H, Hkv, Dh, page, prefix, kind):
    bt = R.Batch(news, lens, Hkv, Dh, page, prefix, seed=len(news) + H, **kind)
    A = _check_attend(bt, bt.rnd(bt.T, H * Dh))
    spare = bt.T - sum(news)
    assert not spare or not A[-spare:].any()


# A prefix long enough to have a product of its own, under few rows and many, short own
# keys and (by the table's width) long ones, one token a sequence and several, some of
# which see the prefix alone, and rows of no sequence.
STACKED = [
    ([1] * 12, [0, 1, 100, 30, 0, 3, 64, 65, 15, 16, 17, 257], 16, 8, 128, 16, 3000, {"ragged": False}),
    ([1] * 40, [(13 * i) % 70 for i in range(40)], 4, 2, 64, 32, 1111, {"ragged": False}),
    ([1] * 150, [i % 7 for i in range(150)], 8, 8, 64, 64, 900, {"ragged": False}),
    ([1] * 12, [0, 1, 1100, 30, 0, 3, 64, 65, 15, 16, 17, 257], 16, 8, 128, 16, 3000, {"ragged": False}),
    ([1] * 30, [(97 * i) % 1500 for i in range(30)], 34, 2, 64, 16, 6000, {"ragged": False}),
    ([3] * 30, [(5 * i) % 40 for i in range(30)], 4, 4, 64, 16, 9001, {}),
    ([5, 0, 37, 1] * 4, [5, 3, 90, 64] * 4, 16, 8, 128, 64, 4400, {}),
    ([1, 2] * 10, [9, 20] * 10, 8, 8, 64, 16, 6950, {"extra": 4}),
    ([20] * 8, [20, 400, 3, 77, 0, 19, 21, 1000], 16, 4, 128, 16, 18500, {"extra": 1}),
]


@pytest.mark.parametrize("news,lens,H,Hkv,Dh,page,prefix,kind", STACKED)
def test_attention_over_a_long_prefix(cuda, news, lens, H, Hkv, Dh, page, prefix, kind):
    from npu_amd import groups
    bt = R.Batch(news, lens, Hkv, Dh, page, prefix, seed=len(news) + H, **kind)
    # and bad pages and what no token sees, in the prefix's and the own keys'
    bt.prefix_table[2], bt.prefix_table[-2] = bt.P, -1
    last = prefix % page
    if last:
        bt.v_pages[int(bt.prefix_table[-1]), :, last:] = math.nan
        bt.k_pages[int(bt.prefix_table[-1]), :, last:] = math.inf
    for b, n in enumerate(lens):
        if n % page:
            bt.v_pages[int(bt.table[b, n // page]), :, n % page:] = math.inf
    with groups.collect_plans() as cp:
        A = _check_attend(bt, bt.rnd(bt.T, H * Dh))
    assert cp.plans[0].kernel.decode().startswith("llama_paged_attention_prefix")
    spare = bt.T - sum(news)
    assert not spare or not A[-spare:].any()


@pytest.mark.parametrize("news,H,Hkv,prefix,names", [
    ([1] * 8, 8, 2, 0, ["_whole"]), ([1] * 8, 8, 2, 20, ["_whole"]), ([1] * 7, 8, 2, 6000, ["_prefix", "_whole"]),
    ([1] * 32, 8, 2, 3000, ["_prefix_tiles", "_whole"]), ([400], 4, 2, 20, ["_tiles", "_join"]),
    ([1], 8, 2, 1025, ["", "_join"]), ([1, 2], 8, 2, 0, ["", "_join"]), ([1, 2], 8, 2, 20, ["", "_join"]),
    ([1, 1, 2] * 5, 6, 2, 40000, ["_prefix", "", "_join"]),
    ([40] * 20, 4, 2, 28000, ["_prefix_tiles", "_tiles", "_join"]), ([15] * 30, 4, 2, 0, ["", "_join"]),
    ([16] * 30, 4, 2, 0, ["_tiles", "_join"]), ([16] * 2, 4, 2, 0, ["", "_join"]),
])
def test_attention_kernels_by_rows(cuda, news, H, Hkv, prefix, names):
    """Few rows a sequence: the kernel that divides keys over waves, whole groups
    to a workgroup where histories are short; many rows, or a prefix under many
    rows of a batch: the kernel that divides rows."""
    from npu_amd import groups
    bt = R.Batch(news, [n + 3 for n in news], Hkv, 64, 16, prefix, ragged=set(news) != {1})
    with groups.collect_plans() as cp:
        _attend(bt, bt.rnd(bt.T, H * 64))
    assert [p.kernel.decode() for p in cp.plans] == ["llama_paged_attention" + n for n in names]


def test_attention_large_logits(cuda):
    """Logits of hundreds, rising and falling along the keys: maxima that move
    in every block."""
    bt = R.Batch([1, 30], [900, 700], 2, 64, 16, 50, seed=3)
    ramp = torch.linspace(-8, 8, bt.P, device="cuda").to(torch.bfloat16)
    bt.k_pages *= ramp[:, None, None, None]
    _check_attend(bt, bt.rnd(bt.T, 4 * 64) * 6)
    bt = R.Batch([90, 130], [900, 130], 2, 128, 16, 50, seed=3)
    bt.k_pages *= torch.linspace(-8, 8, bt.P, device="cuda").to(torch.bfloat16)[:, None, None, None]
    _check_attend(bt, bt.rnd(bt.T, 4 * 128) * 4)


@pytest.mark.parametrize("prefix", [0, 70])
def test_attention_ignores_what_masked_places_hold(cuda, prefix):
    """NaN and Inf past a sequence's last key, past the prefix's and in pages
    that no table names."""
    bt = R.Batch([1, 1, 1, 1], [0, 1, 45, 130], 2, 64, 32, prefix, ragged=False, seed=4)
    used = torch.zeros(bt.P, 32, dtype=torch.bool)
    for b, n in enumerate(bt.lens):
        for j in range(n):
            used[bt.table[b, j // 32], j % 32] = True
    for j in range(prefix):
        used[bt.pre[j // 32], j % 32] = True
    free = (~used).nonzero()
    for x, fill in ((bt.k_pages, (float("nan"), float("inf"))), (bt.v_pages, (float("inf"), float("nan")))):
        x[free[0::2, 0].cuda(), :, free[0::2, 1].cuda()] = fill[0]
        x[free[1::2, 0].cuda(), :, free[1::2, 1].cuda()] = fill[1]
    _check_attend(bt, bt.rnd(4, 4 * 64))


@pytest.mark.parametrize("news,lens,Dh,prefix", [
    ([5, 0, 12, 1], [9, 4, 300, 64], 64, 0), ([3, 2], [9, 40], 128, 30), ([31], [2500], 128, 0),
    ([150, 65], [150, 400], 128, 0), ([70, 40], [71, 3000], 64, 20), ([1, 200], [5, 200], 64, 0)])
def test_attention_ignores_what_later_tokens_hold(cuda, news, lens, Dh, prefix):
    """NaN and Inf in new tokens' keys and values: the tokens before do not see
    them, and the others' entries are what any weight makes of them."""
    H, Hkv, page = 4, 2, 16
    bt = R.Batch(news, lens, Hkv, Dh, page, prefix, seed=9)
    Q = bt.rnd(bt.T, H * Dh)
    want, some = torch.zeros(bt.T, H, Dh, dtype=torch.float64), torch.zeros(bt.T, H, Dh, dtype=torch.bool)
    for t, b, j in bt.tokens():
        if t % 3 == 0 or j < 0:
            continue
        first, rows = t - int(bt.start[b]), slice(t, int(bt.start[b + 1]))
        at, head, entry = (int(bt.table[b, j // page]), j % page), t % Hkv, (7 * t) % Dh
        value = (math.nan, math.inf, -math.inf)[first % 7 % 3]
        bt.v_pages[at[0], head, at[1], entry] = value
        heads = slice(head * (H // Hkv), (head + 1) * (H // Hkv))
        want[rows, heads, entry] += value
        some[rows, heads, entry] = True
        if rows.stop - t <= 2:  # a key too, of the last tokens
            bt.k_pages[at[0], 1 - head, at[1], 3] = math.nan
            heads = slice((1 - head) * (H // Hkv), (2 - head) * (H // Hkv))
            want[rows, heads] = math.nan
            some[rows, heads] = True
    assert some.any()
    got = _attend(bt, Q).cpu().double()
    exact, mag, seen = R.attend64(bt, Q, Dh ** -0.5)
    want, some = want.view(bt.T, -1), some.view(bt.T, -1)
    assert torch.equal(torch.nan_to_num(got[some], nan=7.0), torch.nan_to_num(want[some], nan=7.0))
    assert torch.isfinite(got[~some]).all()
    bad = ((got - exact).abs() > _attend_bound(bt, Q, Dh ** -0.5, exact, mag, seen)) & ~some
    assert not bad.any(), f"{int(bad.sum())} outside, first at {bad.nonzero()[0].tolist()}"


def test_attention_bad_pages_are_masked(cuda):
    bt = R.Batch([1, 1, 1], [100, 40, 20], 2, 128, 16, 40, ragged=False, seed=6)
    bt.page_table[0, 2], bt.page_table[0, 6], bt.page_table[1, 0] = bt.P, -1, 2 ** 31 - 1
    bt.page_table[2, 0] = bt.page_table[2, 1] = -2 ** 31
    bt.prefix_table[1] = bt.P + 7
    _check_attend(bt, bt.rnd(3, 8 * 128))
    bt = R.Batch([70], [200], 2, 64, 16, 40, seed=7)
    bt.page_table[0, 2], bt.page_table[0, 9], bt.prefix_table[0] = -1, bt.P, -7
    bt.table = bt.page_table.cpu().numpy()
    _check_attend(bt, bt.rnd(70, 4 * 64))


def test_attention_strides_streams_and_repeats(cuda):
    """Query rows inside a wider buffer, a strided output, strided pages, a side
    stream; the same call gives the same bits."""
    bt = R.Batch([3, 9, 1], [30, 200, 17], 2, 64, 16, 4, seed=5)
    both = bt.rnd(bt.P, 2, 2, 16, 64)
    bt.k_pages, bt.v_pages = both[:, 0], both[:, 1]
    wide = bt.rnd(bt.T, 6 * 64 + 40)
    out = torch.zeros((bt.T, 6 * 64 + 8), dtype=torch.bfloat16, device="cuda")
    A = _check_attend(bt, wide[:, 8:8 + 6 * 64], out[:, :6 * 64], stream=torch.cuda.Stream())
    first = A.clone()
    assert torch.equal(_attend(bt, wide[:, 8:8 + 6 * 64], out[:, :6 * 64]), first) and not out[:, 6 * 64:].any()


def test_attention_over_a_cache_past_32_bits(cuda):
    Hkv, page, Dh, P = 8, 64, 128, 33000
    k, v = (torch.zeros((P, Hkv, page, Dh), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = R.Batch([1, 1], [100, 64], Hkv, Dh, page, 70, ragged=False, seed=9)
    move = torch.arange(P - small.P, P, device="cuda")
    k[move], v[move] = small.k_pages, small.v_pages
    Q = small.rnd(2, 16 * Dh)
    want = _check_attend(small, Q)
    shift = lambda t: torch.where(t >= 0, t + (P - small.P), t)
    small.k_pages, small.v_pages = k, v
    small.page_table, small.prefix_table = shift(small.page_table), shift(small.prefix_table)
    assert torch.equal(_attend(small, Q), want)


@pytest.mark.parametrize("prefix", [0, 100])
def test_attention_captured(cuda, prefix):
    """A captured call attends to what the device arrays say at each replay."""
    from npu_amd import groups
    bt = R.Batch([1, 1, 1], [3, 118, 0], 2, 64, 16, prefix, ragged=False, max_pages=9, seed=8)
    bt.page_table.copy_(torch.arange(27, device="cuda", dtype=torch.int32).view(3, 9) % bt.P)
    Q = bt.rnd(3, 4 * 64)
    A = torch.empty_like(Q)
    ws = groups.paged_attention_workspace(Q, bt.k_pages, bt.page_table, prefix)
    call = lambda: groups.fused_llama_paged_attention(Q, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, A, 0.125,
                                                      ws, prefix_table=bt.prefix_table, prefix_len=prefix,
                                                      stream=torch.cuda.current_stream())
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for step in range(4):
        bt.kv_len += 5
        Q.copy_(bt.rnd(3, 4 * 64) * (step + 1))
        g.replay()
        torch.cuda.synchronize()
        replayed = A.clone()
        A.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(A, replayed), step
        bt.lens = [n + 5 for n in bt.lens]
        bt.table = bt.page_table.cpu().numpy()
        exact, mag, seen = R.attend64(bt, Q, 0.125)
        assert ((A.cpu().double() - exact).abs() <= _attend_bound(bt, Q, 0.125, exact, mag, seen)).all(), step


# ---- sampling ------------------------------------------------------------------------
def _sample(x, u, temperature=None, top_k=None, top_p=None, min_p=None, probs=True, stream=None):
    from npu_amd import groups
    B = x.shape[0]
    f = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32, device="cuda")
    i = None if top_k is None else torch.tensor(top_k, dtype=torch.int32, device="cuda")
    tokens = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((B,), -7.0, device="cuda") if probs else None
    ws = groups.sample_workspace(x)
    ws.fill_(float("nan"))
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    groups.fused_sample_tokens(x, f(u), tokens, ws, temperature=f(temperature), top_k=i, top_p=f(top_p),
                               min_p=f(min_p), probs=pr, stream=stream)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), None if pr is None else pr.cpu().double().numpy()


def _check_sample(x, u, **kw):
    """Tokens equal; probabilities within f32's rounding (2^-24) and the
    weights' (2^-43 of the largest weight each, above and below the line)."""
    u = np.asarray(u, np.float32)
    kw = {n: None if v is None else np.asarray(v, np.int32 if n == "top_k" else np.float32) for n, v in kw.items()}
    tokens, probs = _sample(x, u, **kw)
    host = x.double().cpu().numpy()
    for b in range(x.shape[0]):
        row = {n: None if v is None else v[b] for n, v in kw.items()}
        tok, pr = R.sample64(host[b], u[b], **row)
        assert tokens[b] == tok, (b, tokens[b], tok, row)
        assert abs(probs[b] - pr) <= 2.0 ** -24 * pr + (x.shape[1] + 1) * 2.0 ** -42, (b, probs[b], pr)


def _logits(B, V, seed, spread=2.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, V), generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (B, 6), generator=g), torch.rand((B, 6), generator=g) * 8)
    return x.to(dtype).cuda()


SETTINGS = {
    "none": lambda r, B: {},
    "temperature": lambda r, B: {"temperature": r.uniform(0.1, 3, B)},
    "top_k": lambda r, B: {"top_k": r.integers(1, 200, B)},
    "top_p": lambda r, B: {"top_p": r.uniform(0.05, 1, B)},
    "min_p": lambda r, B: {"min_p": r.uniform(0.001, 0.9, B)},
    "all": lambda r, B: {"temperature": r.uniform(0.1, 3, B), "top_k": r.integers(-1, 3000, B),
                         "top_p": r.uniform(0.3, 1.2, B), "min_p": r.uniform(-0.1, 0.1, B)},
}


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("B,V,dtype", [(3, 1, "f32"), (4, 2, "bf16"), (5, 7, "f32"), (9, 100, "bf16"), (6, 1023, "f32"),
                                       (7, 2049, "f32"), (5, 32000, "f32"), (4, 50257, "bf16"), (3, 128000, "f32"),
                                       (2, 300001, "bf16"), (300, 517, "f32")])
def test_sample(cuda, B, V, dtype, setting):
    r = np.random.default_rng(B * V)
    x = _logits(B, V, B + V, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32)
    _check_sample(x, r.random(B, np.float32), **SETTINGS[setting](r, B))


def test_sample_flat_and_steep(cuda):
    """Spreads from almost equal logits to one that has all the mass."""
    r = np.random.default_rng(1)
    for spread in (1e-6, 0.01, 0.3, 30.0, 1e4, 1e30):
        x = _logits(4, 40000, 3, spread)
        _check_sample(x, r.random(4, np.float32), temperature=[1, 1, 0.3, 2])
        _check_sample(x, r.random(4, np.float32), top_p=[0.9, 0.5, 0.999, 0.1], top_k=[0, 30000, 5, 0])


@pytest.mark.parametrize("V", [5, 4096, 100000])
def test_sample_ties_go_to_the_lowest_index(cuda, V):
    """Equal logits, and logits of few values: more in one bin than are ranked
    at once."""
    u = np.linspace(0, 0.999, 8, dtype=np.float32)
    same = torch.full((8, V), 1.5, device="cuda")
    same[1::2] = -0.0
    same[1::4, ::2] = 0.0
    _check_sample(same, u)
    _check_sample(same, u, top_k=[1, 2, 3, V // 2, V - 1, V, 0, V + 7])
    _check_sample(same, u, top_p=[0.5, 0.25, 1e-6, 0.75, 0.125, 1.0, 2.0, 0.0])
    few = torch.from_numpy(np.random.default_rng(2).integers(-3, 3, (8, V)).astype(np.float32)).cuda()
    _check_sample(few, u, top_k=[0, 1, 2, V // 3, V // 2, V, 0, 7], top_p=[0.9] * 8)
    _check_sample(few, u, min_p=[np.exp(np.float32(-1)) * 1.001, 0.5, 1.0, 3.0, 1e-30, 0.0, 0.3, 0.01])


def test_sample_at_the_borders_of_u(cuda):
    """Eight equal weights: u = i / 8 is the first number of entry i."""
    x = torch.zeros((8, 8), device="cuda")
    tokens, _ = _sample(x, [i / 8 for i in range(8)])
    assert tokens.tolist() == list(range(8))
    tokens, _ = _sample(x, [float(np.nextafter(np.float32(i / 8), np.float32(0))) for i in range(1, 9)])
    assert tokens.tolist() == list(range(8))
    tokens, _ = _sample(x, [-1.0, 0.0, 1.0, 2.0, float("inf"), -float("inf"), float("nan"), 0.99])
    assert tokens.tolist() == [0, 0, 7, 7, 7, 0, 0, 7]


def test_sample_masked_and_infinite_logits(cuda):
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    rows = [[-inf] * 6, [nan] * 6, [-inf, nan, -inf, 2.0, -inf, nan], [inf, 1, inf, nan, -inf, inf],
            [low] * 6, [low, low, -3.0, low, -3.0, low], [nan, 1.0, 1.0, -inf, 0.5, inf], [3e38, -3e38, 3e38, 0, low, 1]]
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.tensor(rows, device="cuda").to(dtype)
        for u in (0.0, 0.4, 0.7, 0.999):
            _check_sample(x, [u] * 8)
            _check_sample(x, [u] * 8, top_k=[2] * 8, top_p=[0.8] * 8, min_p=[0.1] * 8)
            _check_sample(x, [u] * 8, temperature=[1e-44] * 8)
            _check_sample(x, [u] * 8, temperature=[1e30] * 8)
    wide = torch.full((2, 70000), -inf, device="cuda")
    wide[0, 69999] = -50.0
    _check_sample(wide, [0.5, 0.5], top_p=[0.9, 0.9])


def test_sample_greedy(cuda):
    x = _logits(6, 3000, 4)
    x[0, 7] = x[0, 2900] = 50.0
    tokens, probs = _sample(x, [0.9] * 6, temperature=[0.0, -1.0, float("nan"), 0.0, 1.0, 1.0],
                            top_k=[0, 0, 0, 5, 1, 0], top_p=[1, 1, 1, 1, 1, -0.5])
    assert tokens.tolist() == x.argmax(1).tolist() and tokens[0] == 7 and (probs == 1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_strided_rows(cuda, dtype):
    """Rows at every alignment, inside a wider buffer whose other columns would
    win; without probs; on another stream; the same call gives the same answer."""
    buf = torch.full((9, 5021), 100.0, device="cuda", dtype=dtype)
    x = buf[:, 3:4999]
    x.copy_(_logits(9, 4996, 5))
    u = np.random.default_rng(3).random(9, np.float32)
    _check_sample(x, u, top_p=[0.9] * 9)
    want, _ = _sample(x, u, top_p=[0.9] * 9)
    got, _ = _sample(x, u, top_p=[0.9] * 9, probs=False, stream=torch.cuda.Stream())
    assert (got == want).all()


def test_sample_captured(cuda):
    from npu_amd import groups
    x = _logits(4, 9000, 6)
    u = torch.rand(4, device="cuda")
    tokens, probs = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda")
    ws = groups.sample_workspace(x)
    p = torch.full((4,), 0.9, device="cuda")
    call = lambda: groups.fused_sample_tokens(x, u, tokens, ws, top_p=p, probs=probs, stream=torch.cuda.current_stream())
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for step in range(4):
        x.copy_(_logits(4, 9000, 60 + step))
        u.copy_(torch.rand(4))
        g.replay()
        torch.cuda.synchronize()
        got = tokens.clone(), probs.clone()
        tokens.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(tokens, got[0]) and torch.equal(probs, got[1]), step
        host = x.double().cpu().numpy()
        assert tokens.tolist() == [R.sample64(host[b], float(u[b]), top_p=np.float32(0.9))[0] for b in range(4)], step


# ---- together ------------------------------------------------------------------------
def _model64(model, H, tokens, eps=1e-5):
    """Logits of every position in f64, from host copies of the weights."""
    layers, embed, g_out, w_out = model
    f = lambda t: t.detach().cpu().double()
    norm = lambda x, g: x * (x.square().mean(1, keepdim=True) + eps).rsqrt() * f(g)
    x = f(embed)[tokens]
    n, D = x.shape
    dh = D // H
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64) / dh)
    hid = torch.ones(n, n, dtype=torch.bool).triu(1)
    for p in layers:
        xn = norm(x, p["g1"])
        q, k, v = (xn @ f(p[w]) for w in ("wq", "wk", "wv"))
        out = torch.empty_like(q)
        for h in range(H):
            c = slice(h * dh, (h + 1) * dh)
            rot = lambda t: torch.stack([t[:, 0::2] * angle.cos() - t[:, 1::2] * angle.sin(),
                                         t[:, 0::2] * angle.sin() + t[:, 1::2] * angle.cos()], 2).reshape(n, dh)
            s = (rot(q[:, c]) @ rot(k[:, c]).T * dh ** -0.5).masked_fill(hid, -math.inf)
            out[:, c] = s.softmax(1) @ v[:, c]
        x = x + out @ f(p["wo"])
        hn = norm(x, p["g2"])
        g = hn @ f(p["wg"])
        x = x + (g * torch.sigmoid(g) * (hn @ f(p["wu"]))) @ f(p["wd"])
    return norm(x, g_out) @ f(w_out)


@pytest.mark.parametrize("prefix", [0, 37])
def test_serving(cuda, prefix):
    """Prompts of several lengths, then drawn tokens, eager and replayed from a
    graph, with a sequence leaving and another taking its slot: each step's logits
    against the whole sequence's in f64, each drawn token against its logits.
    The logits are off by a rounding of 2^-8 at nine places a layer (the
    normalised rows twice, QKV, the rotated, the probabilities, A, h, the gated
    and the layer's output) and two after: at most so many of the row's norm."""
    from npu_amd import serving
    H, V, L = 2, 448, 2
    model = serving.random_model(L, 128, H, 192, V, seed=5)
    s = serving.Server(*model, n_heads=H, slots=4, pages=40, page=16, max_pages=10)
    g = torch.Generator().manual_seed(2)
    draw = lambda n: torch.randint(0, V, (n,), generator=g).tolist()
    pre = draw(prefix)
    if prefix:
        s.set_prefix(pre)
    live, setting = {}, {0: {"temperature": 0.7, "top_k": 40}, 1: {"top_p": 0.9}, 2: {"min_p": 0.05}, 3: {"temperature": 0.0}}

    def add(slot, n):
        live[slot] = draw(n)
        s.add(slot, live[slot], **setting[slot])

    def check(slots):
        logits, tokens = s.logits.cpu(), s.tokens.tolist()
        for b in slots:
            exact = _model64(model, H, pre + live[b])[-1]
            assert float((logits[b].double() - exact).norm()) <= (9 * L + 2) * BF16_HALF_STEP * float(exact.norm()), b
            kw = {k: v[b].item() for k, v in s.settings.items()}
            assert tokens[b] == R.sample64(logits[b].double().numpy(), s.u[b].item(), **kw)[0], b
            live[b].append(tokens[b])

    def numbers():
        s.u.copy_(torch.rand(4, generator=g))

    add(0, 5), add(1, 1), add(3, 40)
    numbers()
    s.prefill()
    check([0, 1, 3])
    for _ in range(3):
        numbers()
        s.step()
        check([0, 1, 3])
    s.remove(1)
    del live[1]
    add(2, 70)
    numbers()
    s.prefill()
    check([2])
    graph = s.capture()
    for _ in range(13):
        s.make_room()
        numbers()
        graph.replay()
        torch.cuda.synchronize()
        check([0, 2, 3])
    with pytest.raises(RuntimeError, match="is taken"):
        s.add(0, [1])
    with pytest.raises(ValueError, match="0 .. 447"):
        s.add(1, [448])


def test_a_prefix_is_refused_while_a_captured_step_lives(cuda):
    """...and the step goes on as captured; without it the prefix is taken."""
    from npu_amd import serving
    s = serving.Server(*serving.random_model(1, 128, 2, 192, 64, seed=6), n_heads=2, slots=2, pages=8, page=16, max_pages=3)
    s.add(0, [1, 2, 3], temperature=0.0)
    first = s.prefill().tolist()[0]
    graph = s.capture()
    s.make_room()
    graph.replay()
    torch.cuda.synchronize()
    second = s.tokens.tolist()[0]
    s.remove(0)
    with pytest.raises(RuntimeError, match="captured"):
        s.set_prefix([5] * 20)
    s.add(0, [1, 2, 3], temperature=0.0)
    assert s.prefill().tolist()[0] == first
    s.make_room()
    graph.replay()
    torch.cuda.synchronize()
    assert s.tokens.tolist()[0] == second
    s.remove(0)
    del graph
    s.set_prefix([5] * 20)
    assert s.prefix_len == 20


def test_empty_tensors_are_refused_not_taken_as_absent(cuda):
    from npu_amd import groups
    from npu_amd.groups import NpuError
    x, u = torch.zeros((2, 8), device="cuda"), torch.zeros(2, device="cuda")
    tokens, ws = torch.full((2,), -7, dtype=torch.int32, device="cuda"), groups.sample_workspace(x)
    empty = lambda d: torch.empty(0, dtype=d, device="cuda")
    for name in ("temperature", "top_k", "top_p", "min_p", "probs"):
        kw = {name: empty(torch.int32 if name == "top_k" else torch.float32)}
        with pytest.raises(NpuError, match=rf"{name}: size\[0\] = 0 must be positive"):
            groups.fused_sample_tokens(x, u, tokens, ws, **kw)
    with pytest.raises(NpuError, match=r"u: size\[0\] = 0"):
        groups.fused_sample_tokens(x, empty(torch.float32), tokens, ws)
    bt = R.Batch([1, 1], [3, 20], 2, 64, 16, 0, ragged=False, seed=4)
    Q = bt.rnd(2, 4 * 64)
    A = torch.zeros_like(Q)
    ws = groups.paged_attention_workspace(Q, bt.k_pages, bt.page_table, 0)
    attend = lambda **kw: groups.fused_llama_paged_attention(Q, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, A,
                                                             0.125, ws, **kw)
    for name, kw in (("q_start", {}), ("prefix_table", {"prefix_len": 3})):
        with pytest.raises(NpuError, match=rf"{name}: size\[0\] = 0"):
            attend(**{name: empty(torch.int32)}, **kw)
    torch.cuda.synchronize()
    assert (tokens == -7).all() and not A.any()
    want = attend().clone()
    assert torch.equal(attend(prefix_table=empty(torch.int32)), want)  # a prefix of no keys has no pages


@pytest.mark.parametrize("news,lens,G,Hkv,Dh,kind,names", [
    # a prompt in one of many slots, and pieces of prompts among sequences of one token
    ([0] * 30 + [700] + [0] * 9, [0] * 30 + [700] + [50] * 9, 1, 4, 64, {}, ["_tiles", "_join"]),
    ([0] * 290 + [5000], [0] * 290 + [5020], 1, 1, 64, {}, ["_tiles", "_join"]),
    ([1] * 60 + [300] + [1] * 20, [30 * (i % 9) for i in range(60)] + [900] + [40] * 20, 4, 2, 128, {}, ["_tiles", "_join"]),
    ([1] * 100 + [240], [7 * i for i in range(100)] + [1000], 4, 2, 64, {}, ["_tiles", "_join"]),
    ([1] * 100 + [220], [7 * i for i in range(100)] + [1000], 4, 2, 64, {}, ["", "_join"]),
    # as many rows each: one 16-row tile, two
    ([4] * 64, [11 * i for i in range(64)], 4, 2, 64, {}, ["", "_join"]),
    ([5] * 64, [11 * i for i in range(64)], 4, 2, 64, {}, ["_tiles", "_join"]),
    ([1] * 60, [13 * i for i in range(60)], 20, 2, 64, {"ragged": False, "max_pages": 70}, ["_tiles", "_join"]),
    ([1] * 60, [13 * i for i in range(60)], 20, 2, 64, {"ragged": False, "max_pages": 64}, ["_whole"]),
])
def test_attention_of_uneven_batches(cuda, news, lens, G, Hkv, Dh, kind, names):
    """Tokens spread over the sequences in any way: no long one in small tiles."""
    from npu_amd import groups
    bt = R.Batch(news, lens, Hkv, Dh, 16, 0, seed=len(news) + G, **kind)
    with groups.collect_plans() as cp:
        _check_attend(bt, bt.rnd(bt.T, G * Hkv * Dh))
    assert [p.kernel.decode() for p in cp.plans] == ["llama_paged_attention" + n for n in names]


def test_two_threads_on_two_streams(cuda):
    """Each of the serving calls on two streams at the same time, with workspaces of their own:
    the bits of the same calls alone, and each thread's own errors and plans."""
    import threading

    from npu_amd import _lib, groups
    batches = [R.Batch([1] * 40, [97 * i % 1500 for i in range(40)], 2, 128, 16, 0, ragged=False, max_pages=96, seed=11),
               R.Batch([200, 0, 90], [260, 5, 400], 2, 128, 16, 40, seed=12)]
    logits = [_logits(20, 40000, 13), _logits(9, 50001, 14, dtype=torch.bfloat16)]

    def prepare(i):
        bt, x = batches[i], logits[i]
        cos, sin = (t.cuda() for t in R.rope_tables(bt.prefix + bt.max_pages * bt.page, 64))
        Q = bt.rnd(bt.T, 8 * 128)
        K, V, B = bt.rnd(bt.T, 256), bt.rnd(bt.T, 256), x.shape[0]
        Qo, A = torch.zeros_like(Q), torch.zeros_like(Q)
        tokens = torch.zeros(B, dtype=torch.int32, device="cuda")
        ws, sws = groups.paged_attention_workspace(Q, bt.k_pages, bt.page_table, bt.prefix), groups.sample_workspace(x)
        u, p = torch.linspace(0, 0.99, B, device="cuda"), torch.full((B,), 0.9, device="cuda")

        def run(stream):
            groups.fused_llama_rope_append(Q, K, V, cos, sin, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, Qo,
                                           q_start=bt.q_start, prefix_len=bt.prefix, stream=stream)
            groups.fused_llama_paged_attention(Qo, bt.k_pages, bt.v_pages, bt.page_table, bt.kv_len, A, 0.09, ws,
                                               q_start=bt.q_start, prefix_table=bt.prefix_table, prefix_len=bt.prefix,
                                               stream=stream)
            groups.fused_sample_tokens(x, u, tokens, sws, top_p=p, stream=stream)

        return run, (Qo, A, bt.k_pages, bt.v_pages, tokens)

    prepared = [prepare(i) for i in range(2)]
    alone = []
    for run, outs in prepared:
        run(None)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in outs])
        for t in (outs[0], outs[1], outs[4]):
            t.zero_()
    torch.cuda.synchronize()
    errors, plans, together = [], [set(), set()], threading.Barrier(2)

    def worker(i):
        try:
            stream = torch.cuda.Stream()
            together.wait()
            for n in range(6):
                prepared[i][0](stream)
                plans[i].add(tuple(bytes(p.kernel) for p in _lib.last_launch_plans()))
                if i == 0:
                    try:
                        groups.fused_sample_tokens(logits[0], logits[0][0], prepared[0][1][4], logits[0][0])
                    except groups.NpuError as e:
                        assert "u: size 40000" in str(e), e
            if i == 1:
                assert _lib.lib().npu_last_error() == b""
            stream.synchronize()
        except Exception as e:  # raised below, in the test's own thread
            errors.append(repr(e))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    torch.cuda.synchronize()
    assert plans == [{(b"sample_tokens",)}] * 2
    for (_, outs), want in zip(prepared, alone):
        for got, w in zip(outs, want):
            assert torch.equal(got, w)
