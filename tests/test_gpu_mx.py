"""The operators in microscaled floats, and the log probabilities, on the GPU against
their plain 64-bit forms (mx_refs.py)."""
import math

import numpy as np
import pytest
import torch

import mx_refs as R

pytestmark = pytest.mark.gpu

BF16_HALF_STEP = 2.0 ** -8  # finfo(bfloat16).eps / 2
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def _rnd(*shape, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * spread


def _mx(R_, K, kind, fill=0x55, stride=None):
    """Buffers for a quantised [R, K], filled with what a kernel has to overwrite."""
    w = K if kind == "e4m3" else K // 2
    q = torch.full((R_, stride or w), fill, dtype=U8, device="cuda")[:, :w]
    return (q.view(torch.float8_e4m3fn) if kind == "e4m3" else q), torch.full((R_, K // 32), fill, dtype=U8, device="cuda")


def _np64(t):
    return t.detach().cpu().double().numpy()


# ---- quantisation --------------------------------------------------------------------
def _wild(R_, K, seed, dtype=BF16):
    """Blocks of every size: normal, tiny, huge, zeros, subnormal, ties, one entry."""
    x = _rnd(R_, K, seed=seed).double()
    b = x.view(R_, -1, 32)
    r = np.random.default_rng(seed)
    for i in range(b.shape[0]):
        for j in range(b.shape[1]):
            pick = int(r.integers(0, 9))
            if pick == 0:
                b[i, j] = 0.0
            elif pick == 1:
                b[i, j] *= 2.0 ** float(r.integers(-125, 120))
            elif pick == 2:
                b[i, j] *= 2.0 ** -130
            elif pick == 3:  # ties of both formats
                b[i, j] = torch.from_numpy(r.integers(-48, 49, 32) / 8.0)
            elif pick == 4:
                b[i, j, 1:] = 0.0
            elif pick == 5:
                b[i, j, 0] = 7.99
            elif pick == 6:
                b[i, j] = -b[i, j].abs() * 0.01
    return x.to(dtype)


def _check_quantize(x, kind, values=True, stream=None, **kw):
    from npu_amd import groups
    R_, K = x.shape
    q, s = _mx(R_, K, kind)
    v = torch.full((R_, K), 9.0, dtype=BF16, device="cuda") if values else None
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    groups.fused_mx_quantize(x, q, s, values=v, stream=stream, **kw)
    torch.cuda.synchronize()
    c, sc = R.quantize(_np64(x), kind)
    assert np.array_equal(s.cpu().numpy(), sc)
    assert np.array_equal(R.codes(q, kind), c)
    if values:
        want = torch.from_numpy(R.values(q, s, kind)).float().to(BF16)
        assert torch.equal(torch.nan_to_num(v.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    return q, s


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R_,K", [(1, 32), (1, 64), (3, 96), (5, 512), (300, 1408), (17, 4128), (1000, 32)])
def test_quantize_rows(cuda, R_, K, dtype, kind):
    _check_quantize(_wild(R_, K, R_ + K, dtype).cuda(), kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R_,K,pad", [(2, 32, 0), (7, 64, 0), (64, 96, 0), (65, 160, 3), (129, 512, 0), (130, 1408, 6), (1, 64, 1),
                                      (2049, 32, 0), (63, 4128, 1)])
def test_quantize_columns(cuda, R_, K, pad, dtype, kind):
    """The transposed view of a [K, N] weight, at any stride."""
    w = torch.zeros((K, R_ + pad), dtype=dtype, device="cuda")
    w[:, :R_] = _wild(R_, K, R_ + K, dtype).t()
    _check_quantize(w[:, :R_].t(), kind)
    _check_quantize(w[:, pad:].t()[:R_], kind, values=False)  # (an odd address)


def test_quantize_every_bf16(cuda):
    """All 2^16 bit patterns, each alone in a block with a fixed neighbour: elements,
    scales, NaN and Inf."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    for other in (0.0, 1.0, 448.0):
        x = torch.full((2048, 32, 32), other, dtype=torch.float32).to(BF16)
        x[:, :, 5] = bits.view(2048, 32)
        for kind in ("e4m3", "e2m1"):
            _check_quantize(x.view(2048, 1024).cuda(), kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
def test_quantize_not_finite(cuda, kind):
    """A block with NaN or Inf is NaN, its neighbours are what they were."""
    x = _rnd(8, 256, seed=3).to(BF16)
    x[1, 40], x[2, 255], x[3, 0], x[4, 100], x[4, 101] = math.nan, math.inf, -math.inf, math.inf, math.nan
    q, s = _check_quantize(x.cuda(), kind)
    assert (s == 255).sum() == 4 and np.isnan(R.values(q, s, kind)).sum() == 4 * 32
    _check_quantize(x.t().contiguous().cuda().t(), kind)


# silu's error against the formula: exp2 and its correction 2^-23 + 2^-24 and 2^-26 of the
# remainder's own rounding, times e / (1 + e) < 1; the sum 2^-24, the reciprocal 2^-23, two
# products 2^-24 each: together below 2^-21
SILU_EPS = 2.0 ** -21


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("R_,K", [(1, 32), (3, 96), (300, 1408), (1025, 512)])
def test_quantize_gated(cuda, R_, K, kind):
    from npu_amd import groups
    both = torch.cat([_rnd(R_, K, seed=1, spread=3.0), _rnd(R_, K, seed=2)], 1).to(BF16).cuda()
    gate, x = both[:, :K], both[:, K:]
    q, s = _mx(R_, K, kind)
    groups.fused_mx_quantize(x, q, s, gate=gate)
    R.check_near(q, s, _np64(x) * R.silu64(_np64(gate)), SILU_EPS, kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
def test_quantize_gated_next_to_powers_of_two(cuda, kind):
    """Products that lie within f32's roundings of a power of two, where the scale takes a step: it is
    that of the formula in 64 bits."""
    from npu_amd import groups
    gate = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    g64 = _np64(gate)
    silu = R.silu64(np.where(np.isfinite(g64) & (np.abs(g64) > 1e-20) & (g64 > -60) & (g64 < 1e30), g64, 0.0))
    pairs = []
    for m in range(128):
        x = 1.0 + m / 128
        frac = np.frexp(np.abs(x * silu))[0]  # [1/2, 1): next to either end is next to a power of two
        near = (silu != 0) & ((frac - 0.5 < 2.0 ** -21) | (1.0 - frac < 2.0 ** -21)) & (frac != 0.5)
        pairs += [(x, i) for i in np.nonzero(near)[0]]
    assert len(pairs) >= 8
    xs = torch.zeros((len(pairs), 32))
    gs = torch.zeros((len(pairs), 32), dtype=BF16)
    for row, (x, i) in enumerate(pairs):
        xs[row, row % 32], gs[row, row % 32] = x, gate[i]
    q, s = _mx(len(pairs), 32, kind)
    groups.fused_mx_quantize(xs.to(BF16).cuda(), q, s, gate=gs.cuda())
    c, sc = R.quantize(xs.double().numpy() * np.where(xs.numpy() != 0, R.silu64(_np64(gs)), 0.0), kind)
    assert np.array_equal(s.cpu().numpy(), sc)


def test_quantize_gates_far_out(cuda):
    """Gates of any size: large ones pass, very negative ones close, NaN and +Inf make their
    block NaN."""
    from npu_amd import groups
    gate = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 86.0, -86.0, 88.0, -88.0, 300.0, -300.0, 1e30, -1e30, 3e38,
                         -math.inf]).to(BF16)
    x = torch.ones((16, 32), dtype=BF16)
    g = gate[:, None].expand(16, 32).contiguous()
    q, s = _mx(16, 32, "e4m3")
    groups.fused_mx_quantize(x.cuda(), q, s, gate=g.cuda())
    y = R.silu64(_np64(g))
    y[15] = 0.0
    y[np.abs(y) < 1e-35] = 0.0  # (below -87: 0)
    got = R.values(q, s, "e4m3")
    got[np.abs(got) < 1e-35] = 0.0
    assert (np.abs(got - y) <= (2.0 ** -4 + SILU_EPS) * np.abs(y)).all()
    bad = torch.zeros((2, 64), dtype=BF16)
    bad[0, 3], bad[1, 40] = math.nan, math.inf
    q, s = _mx(2, 64, "e4m3")
    groups.fused_mx_quantize(torch.ones((2, 64), dtype=BF16, device="cuda"), q, s, gate=bad.cuda())
    assert s.tolist() == [[255, 0], [0, 255]]


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
def test_quantize_strides_and_streams(cuda, kind):
    """Rows inside wider buffers; what lies beside them stays."""
    from npu_amd import groups
    wide = _wild(9, 192, 4)[:, :184].contiguous().cuda()
    x = wide[:, 8:168]
    w = 160 if kind == "e4m3" else 80
    q = torch.full((9, w + 32), 0x33, dtype=U8, device="cuda")
    s = torch.full((9, 8), 0x33, dtype=U8, device="cuda")
    v = torch.full((9, 176), 5.0, dtype=BF16, device="cuda")
    qv = q[:, 16:16 + w]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    groups.fused_mx_quantize(x, qv.view(torch.float8_e4m3fn) if kind == "e4m3" else qv, s[:, 2:7], values=v[:, 8:168], stream=side)
    side.synchronize()
    c, sc = R.quantize(_np64(x), kind)
    assert np.array_equal(R.codes(qv.contiguous(), kind), c) and np.array_equal(s[:, 2:7].cpu().numpy(), sc)
    assert (q[:, :16] == 0x33).all() and (q[:, 16 + w:] == 0x33).all() and (s[:, :2] == 0x33).all() and (s[:, 7:] == 0x33).all()
    assert (v[:, :8] == 5).all() and (v[:, 168:] == 5).all()


# ---- norm ------------------------------------------------------------------------------
# An entry is known to some 2^-45 of it and is rounded to odd in f32, so that the last rounding is one of
# the entry itself: blocks are those of the formula in 64 bits, and bf16 is off by half a step
NORM_EPS = 2.0 ** -44


def _check_norm(x, g, kind, delta=None, h="new", eps=1e-5, stream=None):
    from npu_amd import groups
    T, D = x.shape
    q, s = (torch.full((T, D), 9.0, dtype=BF16, device="cuda"), None) if kind == "bf16" else _mx(T, D, kind)
    hw = x.float() if delta is None else x.float() + delta.float()
    hw = hw.to(BF16).cpu()
    ho = torch.full_like(x, 3.0) if h == "new" else h
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    groups.fused_llama_add_rmsnorm(x, g, q, s, delta=delta, h=ho, eps=eps, stream=stream)
    torch.cuda.synchronize()
    if ho is not None:
        assert torch.equal(ho.cpu(), hw)
    hd = hw.double().numpy()
    y = hd / np.sqrt((hd * hd).mean(1, keepdims=True) + eps) * _np64(g)
    if kind == "bf16":
        assert (np.abs(_np64(q) - y) <= (BF16_HALF_STEP + (1 + BF16_HALF_STEP) * NORM_EPS) * np.abs(y)).all()
    else:
        c, sc = R.quantize(y, kind)
        assert np.array_equal(s.cpu().numpy(), sc) and np.array_equal(R.codes(q, kind), c)
    return q, s


@pytest.mark.parametrize("kind", ["e4m3", "e2m1", "bf16"])
@pytest.mark.parametrize("T,D", [(1, 32), (5, 64), (3, 512), (9, 544), (4, 2048), (7, 2080), (48, 4096), (3, 4128), (2, 8192),
                                 (2, 8224), (3, 16384), (2, 16416), (1, 32768), (1001, 96)])
def test_norm(cuda, T, D, kind):
    g = (torch.rand(D, generator=torch.Generator().manual_seed(D)) + 0.5).cuda()
    x = _rnd(T, D, seed=T, spread=3.0)
    x[:, ::37] *= 20.0
    x, delta = x.to(BF16).cuda(), _rnd(T, D, seed=T + 1).to(BF16).cuda()
    _check_norm(x, g, kind)
    _check_norm(x, g, kind, h=None)
    _check_norm(x, g, kind, delta=delta)
    _check_norm(x, g, kind, delta=delta, h=None)


def test_norm_in_place_strided_and_zero(cuda):
    """h over x, h over delta, rows inside a wider buffer; rows of zeros."""
    g = (torch.rand(160, generator=torch.Generator().manual_seed(1)) + 0.5).cuda()
    x, delta = _rnd(6, 160, seed=1).to(BF16).cuda(), _rnd(6, 160, seed=2).to(BF16).cuda()
    from npu_amd import groups
    for where in (0, 1):
        a, b = x.clone(), delta.clone()
        want = _check_norm(x, g, "e4m3", delta=delta)
        q, s = _mx(6, 160, "e4m3")
        groups.fused_llama_add_rmsnorm(a, g, q, s, delta=b, h=(a, b)[where])
        assert torch.equal(q.view(U8), want[0].view(U8)) and torch.equal(s, want[1])
        assert torch.equal((a, b)[where], (x.float() + delta.float()).to(BF16)) and torch.equal((b, a)[where], (delta, x)[where])
    wide = _rnd(6, 400, seed=3).to(BF16).cuda()
    keep = wide[:, 320:].clone()
    _check_norm(wide[:, 8:168], g, "e4m3", delta=wide[:, 168:328], h=wide[:, 8:168], stream=torch.cuda.Stream())
    assert torch.equal(wide[:, 328:], keep[:, 8:])
    q, s = _check_norm(torch.zeros((2, 160), dtype=BF16, device="cuda"), g, "e4m3")
    assert not s.any() and not q.view(U8).any()
    _check_norm(torch.full((1, 160), 2.0 ** -60, dtype=BF16, device="cuda"), g, "bf16", eps=0.0)


@pytest.mark.parametrize("T,D", [(64, 96), (40, 2080), (30, 4096), (6, 16416)])
def test_norm_next_to_powers_of_two(cuda, T, D):
    """Gains that put each block's largest entry within 2^-24 of a power of two: the scale is that of the
    formula in 64 bits, its roundings (2^-51 or so) far below the distances there are."""
    from npu_amd import groups
    for row in range(0, T, max(1, T // 6)):
        x = _rnd(1, D, seed=row).to(BF16)
        hd = _np64(x)
        y = hd / np.sqrt((hd * hd).mean(1, keepdims=True) + 1e-5)
        b = np.abs(y).reshape(-1, 32)
        g = np.full(b.shape, 2.0 ** -6)
        top = b.argmax(1)
        at = np.arange(len(b)), top
        g[at] = 2.0 ** (np.arange(len(b)) % 5) / b[at]
        g = torch.from_numpy(g.reshape(-1)).float()
        y = (y * g.double().numpy()).reshape(1, D)
        for kind in ("e4m3", "e2m1"):
            q, s = _mx(1, D, kind)
            groups.fused_llama_add_rmsnorm(x.cuda(), g.cuda(), q, s, eps=1e-5)
            assert np.array_equal(s.cpu().numpy(), R.quantize(y, kind)[1])


def test_norm_of_huge_and_tiny_rows(cuda):
    """Squares outside f32's range: the mean is in 64 bits."""
    g = torch.ones(512, device="cuda")
    for size in (2.0 ** 120, 2.0 ** 70, 2.0 ** -70, 2.0 ** -120):
        _check_norm((_rnd(3, 512, seed=4) * size).to(BF16).cuda(), g, "e4m3", eps=0.0)


def test_norm_not_finite(cuda):
    """A row with NaN is NaN, one with Inf NaN there and 0 elsewhere; others are as ever."""
    x = _rnd(5, 512, seed=5).to(BF16)
    x[1, 7], x[3, 100] = math.nan, math.inf
    g = torch.ones(512, device="cuda")
    from npu_amd import groups
    q, s = _mx(5, 512, "e4m3")
    groups.fused_llama_add_rmsnorm(x.cuda(), g, q, s)
    v = R.values(q, s, "e4m3")
    assert np.isnan(v[1]).all() and np.isnan(v[3, 96:128]).all() and (np.delete(v[3], range(96, 128)) == 0).all()
    good = [0, 2, 4]
    q2, s2 = _check_norm(x[good].cuda(), g, "e4m3")
    assert torch.equal(q.view(U8)[good], q2.view(U8)) and torch.equal(s[good], s2)


# ---- product ---------------------------------------------------------------------------
def _blocks(R_, K, kind, seed, small=False):
    """(q, scale) of random elements; small: few bits and scales, whose sums are exact."""
    r = np.random.default_rng(seed)
    if small:
        pick = [0x00, 0x38, 0x40, 0x44, 0xb8, 0xc0, 0x30] if kind == "e4m3" else [0, 1, 2, 3, 4, 5, 9, 10, 12]
        c = np.array(pick, np.uint8)[r.integers(0, len(pick), (R_, K))]
        s = r.integers(126, 129, (R_, K // 32))
    else:
        c = r.integers(0, 16, (R_, K)) if kind == "e2m1" else R.nearest(r.standard_normal((R_, K)) * 100, "e4m3")
        c = c.astype(np.uint8)
        s = r.integers(118, 124, (R_, K // 32))
    b = c if kind == "e4m3" else (c[:, 0::2] | c[:, 1::2] << 4)
    q = torch.from_numpy(np.ascontiguousarray(b)).cuda()
    return (q.view(torch.float8_e4m3fn) if kind == "e4m3" else q), torch.from_numpy(s.astype(np.uint8)).cuda()


def _product(a, sa, w, sw, out=None, stream=None):
    from npu_amd import groups
    out = torch.full((a.shape[0], w.shape[0]), 3.0, dtype=BF16, device="cuda") if out is None else out
    ws = groups.mx_matmul_workspace(a, w)
    ws.fill_(float("nan"))
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    groups.fused_mx_matmul(a, sa, w, sw, out, ws, stream=stream)
    torch.cuda.synchronize()
    return out


def _exact(a, sa, w, sw, kind):
    A, W = torch.from_numpy(R.values(a, sa, kind)), torch.from_numpy(R.values(w, sw, "e2m1"))
    if A.numel() * W.shape[0] > 2 ** 31:
        A, W = A.cuda(), W.cuda()
    return (A @ W.t().contiguous()).cpu(), (A.abs() @ W.abs().t().contiguous()).cpu()


def _check_product(a, sa, w, sw, kind, **kw):
    """e2m1 by e2m1: f32 sums, a rounding for each step of 128, eight waves, up to 64 parts.
    e4m3: the instruction's sums, 2^-12 of the magnitudes (npu_amd.h).  Then one rounding."""
    got = _np64(_product(a, sa, w, sw, **kw))
    exact, mag = (t.numpy() for t in _exact(a, sa, w, sw, kind))
    K = sa.shape[1] * 32
    per = 2.0 ** -12 if kind == "e4m3" else (K / 128 + 128) * 2.0 ** -23
    bad = np.abs(got - exact) > BF16_HALF_STEP * np.abs(exact) + (1 + BF16_HALF_STEP) * per * mag
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0].tolist()}"
    # of usual rows far less: 2e-5 of the result beside the rounding
    assert np.linalg.norm(got - exact) <= (BF16_HALF_STEP + 1e-4) * np.linalg.norm(exact)


PRODUCTS = [(1, 1, 32), (1, 16, 32), (1, 17, 64), (3, 5, 96), (16, 16, 128), (17, 33, 160), (15, 100, 1024), (33, 64, 1056),
            (64, 48, 512), (65, 130, 1408), (1, 1408, 512), (48, 300, 4096), (100, 257, 256), (128, 128, 128), (129, 255, 288),
            (256, 256, 512), (257, 511, 1184), (300, 1408, 768), (500, 700, 2080), (513, 96, 640), (40, 1000, 14336),
            (200, 300, 9984), (1000, 1000, 32), (777, 1, 96), (1, 5000, 224), (719, 40, 128), (6650, 1840, 192),
            (8600, 140, 128)]


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(cuda, M, N, K, kind):
    """Sums that are exact come out exact; others within the sums' bound."""
    a, sa = _blocks(M, K, kind, M + N, small=True)
    w, sw = _blocks(N, K, "e2m1", K, small=True)
    exact, _ = _exact(a, sa, w, sw, kind)
    assert torch.equal(_product(a, sa, w, sw).cpu(), exact.float().to(BF16))
    _check_product(*_blocks(M, K, kind, M + 1), *_blocks(N, K, "e2m1", N + 2), kind)


FEW, JOIN, TILES, WORDS = ["mx_matmul_few"], ["mx_join"], ["mx_matmul_tile"], ["mx_scales"]


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K,kernels,tile", [
    (33, 1030, 14336, TILES + JOIN, (32, 64)),       # K in parts, an odd width of them
    (16, 171, 10656, FEW + JOIN, None),
    (51, 265, 8352, FEW + JOIN, None),
    (300, 130, 14016, TILES + JOIN, (32, 64)),       # parts whose last is shorter
    (45, 200, 992, FEW, None),
    (500, 700, 2080, TILES, (32, 64)),
    (100, 7000, 544, TILES, (32, 64)),               # a last step of a quarter
    (1281, 1500, 1056, TILES, (64, 128)),
    (1587, 65, 7200, TILES + JOIN, (64, 128)),
    (130, 5000, 14336, TILES + JOIN, (64, 128)),
    (1025, 700, 7392, TILES, (32, 64)),
    (1400, 39, 7392, TILES + JOIN, (32, 64)),
    (1500, 4100, 2080, TILES, (128, 128)),
    (8505, 68, 12736, TILES + JOIN, (128, 128)),
    (8358, 201, 1696, TILES, (128, 128)),
    (4101, 4096, 4096, WORDS + TILES + FEW, (256, 256)),  # and the rows past whole ones
    (4096, 4030, 4000, WORDS + TILES, (256, 256)),
])
def test_product_kernels(cuda, M, N, K, kernels, tile, kind):
    from npu_amd import groups
    a, sa = _blocks(M, K, kind, M + N, small=True)
    w, sw = _blocks(N, K, "e2m1", K, small=True)
    exact, _ = _exact(a, sa, w, sw, kind)
    with groups.collect_plans() as cp:
        got = _product(a, sa, w, sw)
    assert torch.equal(got.cpu(), exact.float().to(BF16))
    assert [p.kernel.decode() for p in cp.plans] == kernels
    if tile:
        m = M // 256 * 256 if FEW[0] in kernels else M
        tiles = -(-m // tile[0]) * -(-N // tile[1])
        assert {p.kernel.decode(): p.grid for p in cp.plans}["mx_matmul_tile"] in [tiles * parts for parts in range(1, 9)]
    _check_product(*_blocks(M, K, kind, M + 1), *_blocks(N, K, "e2m1", N + 2), kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(3, 40, 96), (70, 130, 544), (300, 520, 1184), (20, 24, 160), (1030, 600, 1184), (2100, 2050, 544)])
def test_product_strides_streams_and_repeats(cuda, M, N, K, kind):
    """Operands and the output inside wider buffers (output rows at any address), a side stream;
    the same call gives the same bits, and nothing beside the output changes."""
    (a, sa), (w, sw) = _blocks(M, K, kind, 1), _blocks(N, K, "e2m1", 2)

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), 0x7f, dtype=U8, device="cuda")
        wide[:, left:left + t.shape[1]] = t.view(U8)
        return wide[:, left:left + t.shape[1]].view(t.dtype)

    want = _product(a, sa, w, sw).clone()
    wide = torch.full((M, N + 9), 7.0, dtype=BF16, device="cuda")
    args = inside(a, 16, 32), inside(sa, 3, 2), inside(w, 48, 16), inside(sw, 1, 6)
    for stream in (None, torch.cuda.Stream()):
        out = _product(*args, out=wide[:, 5:5 + N], stream=stream)
        assert torch.equal(out, want)
    assert (wide[:, :5] == 7).all() and (wide[:, 5 + N:] == 7).all()


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(5, 40, 544), (300, 300, 1184), (1030, 600, 1184), (1600, 70, 7200), (2100, 2050, 544)])
def test_product_of_nan_blocks(cuda, M, N, K, kind):
    """A NaN scale makes its row of a, or column of w, NaN, and no other; scales of the least and
    largest sizes; zero blocks."""
    (a, sa), (w, sw) = _blocks(M, K, kind, 3), _blocks(N, K, "e2m1", 4)
    want = _product(a, sa, w, sw).clone()
    sa[2, K // 32 - 1], sw[33, 0] = 255, 255
    got = _product(a, sa, w, sw)
    assert torch.isnan(got[2]).all() and torch.isnan(got[:, 33]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[2], keep[:, 33] = False, False
    assert torch.equal(got[keep], want[keep])
    sa.fill_(0), sw.fill_(254)
    sa[2, 0], sw[33, 0] = 1, 253
    _check_product(a, sa, w, sw, kind)
    a.view(U8).zero_()
    assert not _product(a, sa, w, sw).any()


# ---- log probabilities -----------------------------------------------------------------
def _check_logprobs(x, tokens, k, all_outputs=True, stream=None):
    from npu_amd import groups
    T, V = x.shape
    new = lambda *s, dtype=F32: torch.full(s, 55, dtype=dtype, device="cuda")
    lp, en, rk = new(T), new(T), new(T, dtype=torch.int32)
    tt, tl = (new(T, k, dtype=torch.int32), new(T, k)) if k else (None, None)
    ws = groups.token_logprobs_workspace(x, k)
    ws.fill_(float("nan"))
    tok = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    kw = dict(entropy=en, ranks=rk) if all_outputs else {}
    groups.fused_token_logprobs(x, tok, lp, ws, top_tokens=tt, top_logprobs=tl, stream=stream, **kw)
    torch.cuda.synchronize()
    # S: up to 65 terms of a lane in turn, 6 + 2 steps, up to 256 parts, each term's exponent 2^-24
    # of its size (whose mean, by p, is at most log2 V), exp2 2^-23, its scale twice 2^-23
    per = (65 + 8 + min(256, V // 1024 + 1) + 2 * math.log2(V) + 8) * 2.0 ** -24
    got = [None if t is None else t.cpu().double().numpy() for t in (lp, en, rk, tt, tl)]
    host = _np64(x)
    for t in range(T):
        e = R.logprobs64(host[t], tokens[t], k)
        fin = host[t][np.isfinite(host[t])]
        m = fin.max() if fin.size else 0.0
        size = lambda v: per + 2.0 ** -23 * (abs(v) + math.log(V)) if np.isfinite(v) else 0.0
        # (outputs are f32: a value past its range, -6.8e38 say, rounds to -Inf)
        f32 = lambda b: -math.inf if b < -float(np.finfo(np.float32).max) * (1 + 2.0 ** -24) else b
        near = lambda a, b: a == f32(b) or abs(a - b) <= size(b)
        assert near(got[0][t], e[0]), (t, got[0][t], e[0])
        if all_outputs:
            # W / S: each of W and S off by `per` of its magnitude, at most log V + H each
            assert abs(got[1][t] - e[1]) <= (per + 2.0 ** -22) * (2 * math.log(V) + 2) + 2.0 ** -23, (t, got[1][t], e[1])
            assert got[2][t] == e[2], (t, got[2][t], e[2])
        if k:
            assert got[3][t].tolist() == e[3], (t, got[3][t], e[3])
            assert all(near(a, b) for a, b in zip(got[4][t], e[4])), (t, got[4][t], e[4])
    return got


def _logits(T, V, seed, dtype, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, V), generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (T, 6), generator=g), torch.rand((T, 6), generator=g) * 8)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (1, 2, 3), (3, 7, 8), (2, 9, 0), (5, 33, 32), (4, 1000, 20), (1, 32000, 20), (3, 2049, 5),
                                   (40, 50257, 5), (2, 128001, 32), (700, 511, 3), (1100, 1030, 1), (300, 9001, 20), (1, 1 << 20, 32),
                                   (1100, 16385, 5), (600, 33333, 0)])
def test_logprobs(cuda, T, V, k, dtype):
    """(bf16 logits tie often)"""
    tokens = [(37 * t * t + 11) % (V + 1) - 1 if t % 3 else (V - 1 if t % 2 else 0) for t in range(T)]
    _check_logprobs(_logits(T, V, T + V, dtype), tokens, k)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_of_hard_rows(cuda, dtype):
    """Equal logits, masks of -Inf and of the type's lowest value, NaN, +Inf, both zeros, rows of one
    candidate or none, tokens that are not there, values at the type's ends."""
    V, inf = 9000, math.inf
    low = torch.finfo(dtype).min
    x = _logits(24, V, 1, torch.float32).cpu()
    x[0] = 0.5
    x[1] = -inf
    x[2] = math.nan
    x[3] = low
    x[4, :] = low
    x[4, [5, 77, 8191, 8999]] = torch.tensor([1.0, 3.0, 3.0, -2.0])
    x[5, :] = -inf
    x[5, [8, 4096, 8200]] = torch.tensor([-7.0, -7.0, 2.0])
    x[6, [100, 8000]] = inf
    x[7, ::2] = math.nan
    x[8, ::3] = -inf
    x[9] = 0.0
    x[9, ::2] = -0.0
    x[10, 17] = -low
    x[11, :] = -low
    x[12, 4000:] = low
    x[13, 0], x[13, 1] = low, -low
    x[14] *= 100
    x[15] = -1e30
    x[15, 8999] = -1e30 / 2
    x[16, 1:] = -inf
    x[17] = torch.arange(V) // 7 * -1.0
    x[18] = -3e37
    x[18, 4] = 50.0
    x[19, 5] = 1e36
    x[20] = 200.0 + x[20]
    x[21] = inf
    x[22, :8998] = -inf
    x = x.to(dtype).cuda()
    cases = [[0] * 24, [V - 1] * 24, [-1, V, 2 ** 31 - 1, -2 ** 31] * 6, [77, 4, 100, 3, 8191, 4096, 8000, 7, 9, 10, 18, 12] * 2,
             [5, 5, 8999, 4500, 5, 8, 100, 6, 3, 4001, 17, 0, 4001, 1, 1, 8999, 0, 60, 4, 5, 9, 8, 8999, 1]]
    for tokens in cases:
        for k in (0, 1, 20, 32):
            _check_logprobs(x, tokens, k)


@pytest.mark.parametrize("n", [15, 16, 17, 255, 256, 257, 300, 1000, 1024, 1025, 1500])
def test_logprobs_of_many_equal_best(cuda, n):
    """n entries of a part share the largest logit: as many candidates, past what is listed at once."""
    x = torch.full((2, 4000), -1.0)
    x[0, 7:7 + n] = 3.0
    x[1, torch.randperm(4000, generator=torch.Generator().manual_seed(n))[:n]] = 3.0
    for dtype in (F32, BF16):
        for k in (1, 15, 32):
            _check_logprobs(x.to(dtype).cuda(), [7 + n // 2, 3999], k)


def test_logprobs_strides_streams_and_repeats(cuda):
    """Rows at odd addresses, strided alternatives, outputs left out; the same call gives the same
    bits."""
    from npu_amd import groups
    for dtype in (F32, BF16):
        wide = _logits(7, 20011, 3, dtype)
        for off in (0, 1, 3, 7):
            x = wide[:, off:off + 19990]
            first = _check_logprobs(x, [5, 19989, -1, 0, 100, 7, 3], 7, stream=torch.cuda.Stream())
            again = _check_logprobs(x, [5, 19989, -1, 0, 100, 7, 3], 7, all_outputs=False)
            assert all(np.array_equal(a, b) for i, (a, b) in enumerate(zip(first, again)) if i not in (1, 2))
        big, ids = torch.full((7, 9), 4.0, device="cuda"), torch.full((7, 11), 4, dtype=torch.int32, device="cuda")
        lp, tok = torch.zeros(7, device="cuda"), torch.arange(7, dtype=torch.int32, device="cuda")
        groups.fused_token_logprobs(wide, tok, lp, groups.token_logprobs_workspace(wide, 5), top_tokens=ids[:, 3:8],
                                    top_logprobs=big[:, 1:6])
        _, _, _, tops, lps = zip(*[R.logprobs64(_np64(wide)[t], t, 5) for t in range(7)])
        assert ids[:, 3:8].tolist() == list(map(list, tops)) and np.allclose(big[:, 1:6].cpu(), lps, atol=1e-4)
        assert (big[:, 0] == 4).all() and (big[:, 6:] == 4).all() and (ids[:, :3] == 4).all() and (ids[:, 8:] == 4).all()


def test_tokens_and_their_log_probabilities_agree(cuda):
    """The rank of a drawn token is its place among the alternatives, and greedy draws have rank 0."""
    from npu_amd import groups
    x = _logits(64, 5003, 9, BF16)
    new = lambda *s, dtype=F32: torch.full(s, 55, dtype=dtype, device="cuda")
    tok, probs, lp, rk = new(64, dtype=torch.int32), new(64), new(64), new(64, dtype=torch.int32)
    tt, tl, ws = new(64, 32, dtype=torch.int32), new(64, 32), groups.token_logprobs_workspace(x, 32)
    temperature, top_k = torch.ones(64, device="cuda"), torch.full((64,), 32, dtype=torch.int32, device="cuda")
    temperature[:8] = 0
    u = torch.rand(64, generator=torch.Generator().manual_seed(4)).cuda()
    groups.fused_sample_tokens(x, u, tok, groups.sample_workspace(x), temperature=temperature, top_k=top_k, probs=probs)
    groups.fused_token_logprobs(x, tok, lp, ws, ranks=rk, top_tokens=tt, top_logprobs=tl)
    r = rk.long()[:, None]
    assert (rk[:8] == 0).all() and (rk < 32).all()
    assert torch.equal(tt.gather(1, r)[:, 0], tok) and torch.equal(tl.gather(1, r)[:, 0], lp)
    # the drawn token's share of the 32: both within a few f32 roundings of sums and exponentials
    share = (lp - tl.logsumexp(1)).exp()
    assert ((share - probs).abs()[8:] <= 1e-5 * probs[8:]).all()


# ---- captured, on two streams, together ------------------------------------------------
def test_captured(cuda):
    """Each call captured: replays, with eager work and changed inputs between, give the eager call's
    bits; two graphs in turn with a workspace each."""
    from npu_amd import groups
    x, g = _rnd(300, 512, seed=1).to(BF16).cuda(), torch.ones(512, device="cuda")
    w, sw = _blocks(700, 512, "e2m1", 2)
    w2, sw2 = _blocks(300, 9984, "e2m1", 3)
    a2, sa2 = _blocks(40, 9984, "e4m3", 4)  # (K in parts)
    a3, sa3 = _blocks(2000, 512, "e4m3", 5)  # (tiles)
    q, s = _mx(300, 512, "e4m3")
    delta, h = _rnd(300, 512, seed=6).to(BF16).cuda(), torch.empty_like(x)
    new = lambda *sh, dtype=BF16: torch.zeros(sh, dtype=dtype, device="cuda")
    out, out2, out3, v = new(300, 700), new(40, 300), new(2000, 700), new(300, 512)
    q4, s4 = _mx(300, 512, "e2m1")
    tok = torch.arange(300, dtype=torch.int32, device="cuda")
    lp, tt, tl = new(300, dtype=F32), new(300, 4, dtype=torch.int32), new(300, 4, dtype=F32)
    logits = _rnd(300, 9001, seed=7).cuda()
    ws = [[groups.mx_matmul_workspace(q, w), groups.mx_matmul_workspace(a2, w2), groups.mx_matmul_workspace(a3, w),
           groups.token_logprobs_workspace(logits, 4)] for _ in range(3)]

    def calls(ws):
        stream = torch.cuda.current_stream()
        groups.fused_llama_add_rmsnorm(x, g, q, s, delta=delta, h=h, stream=stream)
        groups.fused_mx_matmul(q, s, w, sw, out, ws[0], stream)
        groups.fused_mx_quantize(h, q4, s4, values=v, stream=stream)
        groups.fused_mx_matmul(a2, sa2, w2, sw2, out2, ws[1], stream)
        groups.fused_mx_matmul(a3, sa3, w, sw, out3, ws[2], stream)
        groups.fused_token_logprobs(logits, tok, lp, ws[3], top_tokens=tt, top_logprobs=tl, stream=stream)

    outs = (h, q.view(U8), s, out, q4, s4, v, out2, out3, lp, tt, tl)
    calls(ws[0])
    torch.cuda.synchronize()
    graphs = []
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            calls(ws[i])
    for step in range(5):
        x.copy_(_rnd(300, 512, seed=10 + step) * (step + 1))
        logits.copy_(_rnd(300, 9001, seed=20 + step) * step)
        sw2.copy_(sw2.roll(1, 0))
        a3.view(U8).copy_(a3.view(U8).roll(1, 0))
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        calls(ws[2])
        torch.cuda.synchronize()
        for i, (t, r) in enumerate(zip(outs, replayed)):
            assert torch.equal(t, r), (step, i)


def test_two_threads_on_two_streams(cuda):
    """Each call on two streams at the same time: the bits of the same calls alone."""
    import threading

    from npu_amd import groups

    def prepare(i):
        M, N, K = ((2100, 1500, 2080), (40, 900, 9984))[i]
        (a, sa), (w, sw) = _blocks(M, K, "e4m3", i), _blocks(N, K, "e2m1", i + 5)
        x, g = _rnd(500, 2048, seed=i).to(BF16).cuda(), torch.ones(2048, device="cuda")
        q, s = _mx(500, 2048, "e4m3")
        q4, s4 = _mx(2048, 512, "e2m1")
        wide = _rnd(512, 2048, seed=i + 2).to(BF16).cuda()
        logits = _logits((30, 9)[i], 70001, i, (F32, BF16)[i])
        T = logits.shape[0]
        tok, lp = torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, device="cuda")
        tt, tl = torch.zeros((T, 7), dtype=torch.int32, device="cuda"), torch.zeros((T, 7), device="cuda")
        out, ws, lws = torch.zeros((M, N), dtype=BF16, device="cuda"), groups.mx_matmul_workspace(a, w), groups.token_logprobs_workspace(logits, 7)

        def run(stream):
            groups.fused_llama_add_rmsnorm(x, g, q, s, stream=stream)
            groups.fused_mx_matmul(a, sa, w, sw, out, ws, stream)
            groups.fused_mx_quantize(wide.t(), q4, s4, stream=stream)
            groups.fused_token_logprobs(logits, tok, lp, lws, top_tokens=tt, top_logprobs=tl, stream=stream)

        return run, (q.view(U8), s, out, q4, s4, lp, tt, tl)

    prepared, alone = [prepare(i) for i in range(2)], []
    for run, outs in prepared:
        run(None)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in outs])
        for t in outs:
            t.zero_()
    torch.cuda.synchronize()
    errors, together = [], threading.Barrier(2)

    def worker(i):
        try:
            stream = torch.cuda.Stream()
            together.wait()
            for _ in range(8):
                prepared[i][0](stream)
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
    for (_, outs), want in zip(prepared, alone):
        for i, (got, w) in enumerate(zip(outs, want)):
            assert torch.equal(got, w), i


def test_python_refusals(cuda):
    """Host tensors, other types and empty tensors are refused before any launch."""
    from npu_amd import groups
    from npu_amd.groups import NpuError
    x = torch.ones((4, 64), dtype=BF16, device="cuda")
    q, s = _mx(4, 64, "e4m3")
    with pytest.raises(ValueError, match="x: expected a tensor on the GPU"):
        groups.fused_mx_quantize(x.cpu(), q, s)
    with pytest.raises(TypeError, match="scale: unsupported tensor dtype"):
        groups.fused_mx_quantize(x, q, s.double())
    with pytest.raises(TypeError, match="q: expected a tensor"):
        groups.fused_mx_quantize(x, None, s)
    with pytest.raises(NpuError, match=r"gate: size\[0\] = 0|gate: rank"):
        groups.fused_mx_quantize(x, q, s, gate=torch.empty((0, 64), dtype=BF16, device="cuda"))
    with pytest.raises(NpuError, match="q: element type"):
        groups.fused_mx_quantize(x, q.view(torch.int8), s)
    with pytest.raises(ValueError, match="no product of blocks"):
        groups.mx_matmul_workspace(q, torch.zeros((5, 17), dtype=U8, device="cuda"))
    with pytest.raises(ValueError, match="33 alternatives"):
        groups.token_logprobs_workspace(x, 33)
    # other torch types of the same bytes are taken
    q4, s4 = _mx(4, 64, "e2m1")
    groups.fused_mx_quantize(x, q4.view(torch.float4_e2m1fn_x2), s4.view(torch.float8_e8m0fnu))
    assert (R.values(q4, s4, "e2m1") == 1).all()


def test_rows_past_32_bits(cuda):
    """Operands and outputs whose last rows lie past 2^31 elements, or 2^32 bytes."""
    from npu_amd import groups
    K, far = 64, (1 << 32) // 64 + 9
    big = torch.zeros((far, K), dtype=BF16, device="cuda")  # 8.6 GB
    big[-1] = _rnd(K, seed=1).to(BF16)
    q = torch.zeros((far, K // 2), dtype=U8, device="cuda")
    s = torch.full((far, 2), 9, dtype=U8, device="cuda")
    groups.fused_mx_quantize(big, q, s)
    c, sc = R.quantize(_np64(big[-1:]), "e2m1")
    assert np.array_equal(R.codes(q[-1:], "e2m1"), c) and np.array_equal(s[-1:].cpu().numpy(), sc) and not s[:-1].any()
    del big, q, s
    T, D = 1 << 23, 288  # 4.8 GB
    x = torch.zeros((T, D), dtype=BF16, device="cuda")
    x[-1] = _rnd(D, seed=1).to(BF16)
    h, (q, s) = torch.empty_like(x), _mx(T, D, "e2m1")
    groups.fused_llama_add_rmsnorm(x, torch.ones(D, device="cuda"), q, s, delta=x, h=h)
    assert torch.equal(h[-1], x[-1] * 2) and q[-1].any() and not q[:-1].any() and not h[:-1].any()
    del x, h, q, s
    # a, then out past 2^32 bytes; tiles and few rows
    for M, N, K in ((1 << 22, 40, 1056), (1 << 21, 1100, 160), (1 << 22, 600, 96)):
        a = torch.zeros((M, K), dtype=U8, device="cuda")
        a[-1] = 0x38  # 1.0
        a = a.view(torch.float8_e4m3fn)
        w, sw = _blocks(N, K, "e2m1", 2, small=True)
        out = torch.full((M, N), 5.0, dtype=BF16, device="cuda")
        one = torch.full((M, K // 32), 127, dtype=U8, device="cuda")
        groups.fused_mx_matmul(a, one, w, sw, out, groups.mx_matmul_workspace(a, w))
        want = torch.from_numpy(R.values(w, sw, "e2m1").sum(1)).float().to(BF16)
        assert torch.equal(out[-1].cpu(), want) and not out[:-1].any(), (M, N, K)
        del a, out, one
    V = 1 << 20
    x = torch.zeros((2200, V), dtype=BF16, device="cuda")
    x[-1, 12345] = 8.0
    lp, tt, tl = torch.zeros(2200, device="cuda"), torch.zeros((2200, 1), dtype=torch.int32, device="cuda"), torch.zeros((2200, 1), device="cuda")
    tok = torch.full((2200,), 12345, dtype=torch.int32, device="cuda")
    groups.fused_token_logprobs(x, tok, lp, groups.token_logprobs_workspace(x, 1), top_tokens=tt, top_logprobs=tl)
    exact = 8.0 - math.log(V - 1 + math.exp(8.0))
    assert abs(float(lp[-1]) - exact) < 1e-5 and tt[-1] == 12345 and (tt[:-1] == 0).all()
    assert (lp[:-1] + math.log(V)).abs().max() < 1e-5


# ---- a decoder in microscaled floats ---------------------------------------------------
def _unpacked(model):
    """The model's weights as the values that quantize_model's blocks stand for, bf16 [K, N] (which
    holds them: two bits and a power of two)."""
    layers, embed, g_out, w_out = model
    back = lambda qs: torch.from_numpy(R.values(*qs, "e2m1").T).to(BF16)
    out = []
    for p in layers:
        (wq, wk, wv), (wg, wu) = back(p["wqkv"]).chunk(3, 1), back(p["wgu"]).chunk(2, 1)
        out.append({"g1": p["g1"], "g2": p["g2"], "wq": wq, "wk": wk, "wv": wv, "wo": back(p["wo"]), "wg": wg, "wu": wu,
                    "wd": back(p["wd"])})
    return out, embed, g_out, back(w_out)


def test_decoder_layer_stage_by_stage(cuda):
    """mx_decoder_layer against its operators one by one, each checked against 64 bits on what the one
    before gave it."""
    import serve_refs as S
    from npu_amd import groups, serving
    D, H, F, T = 128, 2, 192, 37
    layers, _, _, _ = serving.quantize_model(*serving.random_model(1, D, H, F, 64, seed=3))
    bt = S.Batch([30, 7], [30, 19], H, 64, 16, 0, seed=3)
    cos, sin = (t.cuda() for t in S.rope_tables(bt.max_pages * 16, 32))
    p = dict(layers[0], cos_t=cos, sin_t=sin)
    x, delta = _rnd(T, D, seed=1).to(BF16).cuda(), _rnd(T, D, seed=2).to(BF16).cuda()
    batch = {"page_table": bt.page_table, "kv_len": bt.kv_len, "q_start": bt.q_start, "prefix_table": None, "prefix_len": 0}
    e = lambda n: torch.full((T, n), 5.0, dtype=BF16, device="cuda")
    pages = (bt.k_pages.clone(), bt.v_pages.clone())
    ws = groups.paged_attention_workspace(x, pages[0], bt.page_table, 0)

    q, s = _check_norm(x, p["g1"], "e4m3", delta=delta)
    h = (x.float() + delta.float()).to(BF16)
    _check_product(q, s, *p["wqkv"], "e4m3")
    qkv = _product(q, s, *p["wqkv"])
    Q, K, V = qkv[:, :D], qkv[:, D:2 * D], qkv[:, 2 * D:]
    groups.fused_llama_rope_append(Q, K, V, cos, sin, *pages, bt.page_table, bt.kv_len, Q, q_start=bt.q_start)
    A = groups.fused_llama_paged_attention(Q, *pages, bt.page_table, bt.kv_len, e(D), 64 ** -0.5, ws, q_start=bt.q_start)
    qa, sa = _check_quantize(A, "e4m3")
    _check_product(qa, sa, *p["wo"], "e4m3")
    o = _product(qa, sa, *p["wo"])
    q2, s2 = _check_norm(h, p["g2"], "e4m3", delta=o)
    _check_product(q2, s2, *p["wgu"], "e4m3")
    gu = _product(q2, s2, *p["wgu"])
    qf, sf = _mx(T, F, "e4m3")
    groups.fused_mx_quantize(gu[:, F:], qf, sf, gate=gu[:, :F])
    R.check_near(qf, sf, _np64(gu[:, F:]) * R.silu64(_np64(gu[:, :F])), SILU_EPS, "e4m3")
    _check_product(qf, sf, *p["wd"], "e4m3")
    d = _product(qf, sf, *p["wd"])

    bufs = {"x": x.clone(), "qkv": e(3 * D), "gu": e(2 * F), "A": e(D), "o": e(D), "d": e(D), "ws": ws}
    (bufs["q"], bufs["s"]), (bufs["qf"], bufs["sf"]) = _mx(T, D, "e4m3"), _mx(T, F, "e4m3")
    bufs["mx_ws"] = groups.mx_matmul_workspace(bufs["q"], p["wgu"][0])
    cache = (bt.k_pages, bt.v_pages)
    got = serving.mx_decoder_layer(p, bufs, cache, batch, H, delta=delta)
    torch.cuda.synchronize()
    assert torch.equal(got, d) and torch.equal(bufs["x"], (h.float() + o.float()).to(BF16))
    assert torch.equal(cache[0], pages[0]) and torch.equal(cache[1], pages[1])


@pytest.mark.parametrize("prefix", [0, 37])
@pytest.mark.parametrize("mx", [True, False])
def test_serving_with_alternatives_and_scores(cuda, mx, prefix):
    """Prompts, then drawn tokens, eager and replayed: logits against the whole sequence's in f64 with
    the values of the weights; tokens, log probabilities and alternatives against those logits; and the scores of
    given tokens against the f64 model's.
    The logits are off by a rounding of 2^-8 at nine places a layer and two after, and in
    microscaled floats by one of 2^-4 at four a layer and one after: at most so many of the row's
    norm."""
    import serve_refs as S
    from npu_amd import serving
    from test_gpu_serve import _model64
    H, V, L = 2, 448, 1
    model = serving.random_model(L, 128, H, 192, V, seed=5)
    if mx:
        model = serving.quantize_model(*model)
    exact_model = _unpacked(model) if mx else model
    exact_model = tuple([{k: v.cpu() for k, v in p.items()} for p in m] if isinstance(m, list) else m.cpu() for m in exact_model)
    bound = (9 * L + 2) * BF16_HALF_STEP + ((4 * L + 1) * 2.0 ** -4 if mx else 0.0)
    s = serving.Server(*model, n_heads=H, slots=3, pages=30, page=16, max_pages=8, alternatives=5)
    g = torch.Generator().manual_seed(2)
    draw = lambda n: torch.randint(0, V, (n,), generator=g).tolist()
    pre = draw(prefix)
    if prefix:
        s.set_prefix(pre)
    live = {0: draw(5), 2: draw(40)}
    s.add(0, live[0], temperature=0.7, top_k=40)
    s.add(2, live[2], temperature=0.0)

    def check(slots):
        logits, tokens = s.logits.cpu(), s.tokens.tolist()
        for b in slots:
            exact = _model64(exact_model, H, pre + live[b])[-1]
            assert float((logits[b].double() - exact).norm()) <= bound * float(exact.norm()), b
            kw = {k: v[b].item() for k, v in s.settings.items()}
            row = logits[b].double().numpy()
            assert tokens[b] == S.sample64(row, s.u[b].item(), **kw)[0], b
            lp, entropy, rank, top, tops = R.logprobs64(row, tokens[b], 5)
            # (448 entries: a lane's one, the sums' steps, exponents up to 2^5: below 2^-17)
            assert abs(s.logprobs[b].item() - lp) <= 2.0 ** -17 * (1 + abs(lp)) and abs(s.entropy[b].item() - entropy) <= 2.0 ** -14
            assert s.ranks[b].item() == rank and s.top_tokens[b].tolist() == top
            assert all(abs(x - y) <= 2.0 ** -17 * (1 + abs(y)) for x, y in zip(s.top_logprobs[b].tolist(), tops))
            live[b].append(tokens[b])

    s.u.copy_(torch.rand(3, generator=g))
    s.prefill()
    check([0, 2])
    s.u.copy_(torch.rand(3, generator=g))
    s.step()
    check([0, 2])
    graph = s.capture()
    for _ in range(4):
        s.make_room()
        s.u.copy_(torch.rand(3, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        check([0, 2])
    free = list(s.pages.free)
    logprobs, entropy = s.score(live[2], rows=17)
    exact = _model64(exact_model, H, pre + live[2])[prefix:-1]
    lp = exact.log_softmax(1)
    want = lp.gather(1, torch.tensor(live[2][1:])[:, None])[:, 0]
    # a log probability moves by at most twice the largest change of a logit
    off = 2 * bound * exact.norm(dim=1) + 2.0 ** -8 * exact.abs().amax(1)
    assert ((logprobs.cpu().double() - want).abs() <= off).all()
    assert (entropy.cpu() >= 0).all() and (entropy.cpu() <= math.log(V) + 1e-5).all()
    assert sorted(free) == sorted(s.pages.free)
    s.make_room()
    s.u.copy_(torch.rand(3, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    check([0, 2])  # (a score leaves the sequences as they are)
    with pytest.raises(ValueError, match="the table holds 128"):
        s.score([1] * 129)
    with pytest.raises(ValueError, match="0 rows"):
        s.score([1, 2], rows=0)
    assert s.score([7])[0].numel() == 0


def test_server_without_alternatives_and_refusals(cuda):
    """alternatives=0: log probabilities alone; too many and weights that are no whole blocks are refused."""
    from npu_amd import serving
    model = serving.random_model(1, 128, 2, 192, 320, seed=3)
    s = serving.Server(*serving.quantize_model(*model), n_heads=2, slots=2, pages=8, page=16, max_pages=4, alternatives=0)
    s.add(1, [3, 4, 5], temperature=0.0)
    s.u.fill_(0.5)
    s.prefill()
    s.step()
    lp, entropy, rank, _, _ = R.logprobs64(s.logits[1].cpu().double().numpy(), s.tokens[1].item(), 1)
    assert s.top_tokens is None and s.ranks[1].item() == rank == 0
    assert abs(s.logprobs[1].item() - lp) <= 2.0 ** -17 * (1 + abs(lp)) and abs(s.entropy[1].item() - entropy) <= 2.0 ** -14
    with pytest.raises(ValueError, match="33 alternatives"):
        serving.Server(*model, n_heads=2, slots=2, pages=8, page=16, max_pages=4, alternatives=33)
    with pytest.raises(Exception, match="multiple of 32"):
        serving.mx_weight(torch.zeros((48, 64), dtype=BF16, device="cuda"))
