"""The serving operators on the GPU against their plain 64-bit forms
(serve_refs.py)."""
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
]


@pytest.mark.parametrize("news,lens,H,Hkv,Dh,page,prefix,kind", ATTEND)
def test_attention(cuda, news, lens, H, Hkv, Dh, page, prefix, kind):
    bt = R.Batch(news, lens, Hkv, Dh, page, prefix, seed=len(news) + H, **kind)
    A = _check_attend(bt, bt.rnd(bt.T, H * Dh))
    spare = bt.T - sum(news)
    assert not spare or not A[-spare:].any()


def test_attention_large_logits(cuda):
    """Logits of hundreds, rising and falling along the keys: maxima that move
    in every block."""
    bt = R.Batch([1, 30], [900, 700], 2, 64, 16, 50, seed=3)
    ramp = torch.linspace(-8, 8, bt.P, device="cuda").to(torch.bfloat16)
    bt.k_pages *= ramp[:, None, None, None]
    _check_attend(bt, bt.rnd(bt.T, 4 * 64) * 6)


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


def test_attention_bad_pages_are_masked(cuda):
    bt = R.Batch([1, 1, 1], [100, 40, 20], 2, 128, 16, 40, ragged=False, seed=6)
    bt.page_table[0, 2], bt.page_table[0, 6], bt.page_table[1, 0] = bt.P, -1, 2 ** 31 - 1
    bt.page_table[2, 0] = bt.page_table[2, 1] = -2 ** 31
    bt.prefix_table[1] = bt.P + 7
    _check_attend(bt, bt.rnd(3, 8 * 128))


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
