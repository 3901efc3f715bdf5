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
# The mean's f32 sum: 32 terms of a lane in turn, six steps over lanes, up to 16 waves, the
# squares' own rounding and the division, (32 + 6 + 16 + 2) 2^-24 of it and half of that of its
# root; root, reciprocal and two products 2^-24 (and 2^-23 for each of the first two)
NORM_EPS = (56 / 2 + 6) * 2.0 ** -24


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
        R.check_near(q, s, y, NORM_EPS, kind)
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
            (200, 300, 9984), (1000, 1000, 32), (777, 1, 96), (1, 5000, 224)]


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(cuda, M, N, K, kind):
    """Sums that are exact come out exact; others within the sums' bound."""
    a, sa = _blocks(M, K, kind, M + N, small=True)
    w, sw = _blocks(N, K, "e2m1", K, small=True)
    exact, _ = _exact(a, sa, w, sw, kind)
    assert torch.equal(_product(a, sa, w, sw).cpu(), exact.float().to(BF16))
    _check_product(*_blocks(M, K, kind, M + 1), *_blocks(N, K, "e2m1", N + 2), kind)


FEW, JOIN, TILES = ["mx_matmul_few"], ["mx_join"], ["mx_scales", "mx_matmul_tile"]


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K,kernels", [
    (64, 1030, 14336, FEW + JOIN),           # K in parts, an odd width of them
    (16, 171, 10656, FEW + JOIN),
    (300, 130, 14016, FEW + JOIN),           # parts whose last is shorter
    (1000, 1000, 4096, FEW),
    (2048, 1100, 1600, TILES),               # tiles of 128
    (1400, 39, 7392, TILES + JOIN),          # in parts
    (1281, 1500, 1056, TILES),
    (4101, 2050, 1024, TILES),
    (4101, 4096, 4096, TILES + FEW),         # tiles of 256, and the rows past whole ones
    (4096, 4030, 4000, TILES),
])
def test_product_kernels(cuda, M, N, K, kernels, kind):
    from npu_amd import groups
    a, sa = _blocks(M, K, kind, M + N, small=True)
    w, sw = _blocks(N, K, "e2m1", K, small=True)
    exact, _ = _exact(a, sa, w, sw, kind)
    with groups.collect_plans() as cp:
        got = _product(a, sa, w, sw)
    assert torch.equal(got.cpu(), exact.float().to(BF16))
    assert [p.kernel.decode() for p in cp.plans] == kernels
    _check_product(*_blocks(M, K, kind, M + 1), *_blocks(N, K, "e2m1", N + 2), kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(3, 40, 96), (70, 130, 544), (300, 520, 1184), (20, 24, 160)])
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
@pytest.mark.parametrize("M,N,K", [(5, 40, 544), (300, 300, 1184)])
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
