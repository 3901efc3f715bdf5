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
