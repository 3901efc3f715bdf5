"""The operators in microscaled floats, and the log probabilities, on the GPU where their values
come to the ends of what the types hold, against the plain 64-bit forms (mx_refs.py)."""
import math

import numpy as np
import pytest
import torch

import mx_refs as R
from test_gpu_mx import (BF16, BF16_HALF_STEP, F32, SILU_EPS, _blocks, _check_logprobs, _check_norm, _exact, _mx, _np64, _product,
                         _rnd)

pytestmark = pytest.mark.gpu


# ---- log probabilities -----------------------------------------------------------------
# From some 1e6 on, the rounding of m log2 e is no small part of an exponent; masks are such numbers.
FAR = [9.9e5, -1.1e6, 2.0 ** 22, -1e9, -2.0 ** 31, 3e9, 3003121664.0, 4.1e9, -5e9, -1e10, 1e12, -1e20, -1e30, 1e36, -1e36, 9.9e36, -1.1e37]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [100, 4000, 50257])
def test_logprobs_of_rows_far_from_zero(cuda, V, dtype):
    """Rows of one value (log p = -ln V, entropy = ln V), and with three equal best."""
    x = torch.empty((2 * len(FAR), V))
    best = [3, V // 2, V - 1]
    for i, v in enumerate(FAR):
        x[2 * i] = v
        x[2 * i + 1] = 2 * v if v < 0 else v / 2
        x[2 * i + 1, best] = v
    x = x.to(dtype).cuda()
    got = _check_logprobs(x, [(17 * t) % V if t % 2 == 0 else best[t // 2 % 3] for t in range(len(x))], 5)
    # f32 results, their sums' error some 2^-17 at most
    assert np.abs(got[0][0::2] + math.log(V)).max() < 1e-4 and np.abs(got[1][0::2] - math.log(V)).max() < 1e-4
    assert np.abs(got[0][1::2] + math.log(3)).max() < 1e-5 and np.abs(got[1][1::2] - math.log(3)).max() < 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 50257])
def test_logprobs_of_masked_vocabularies(cuda, V, dtype):
    """All but a few tokens at a mask's value: whole parts of the row have nothing else."""
    masks = [-1e6, -1e9, -2.0 ** 31, -3e9, -4.1e9, -1e10, -1e20, -1e30, float(torch.finfo(dtype).min)]
    x = torch.tensor(masks)[:, None].repeat(2, V)
    g = torch.Generator().manual_seed(V)
    x[:len(masks), 20:31] = torch.randn((len(masks), 11), generator=g) * 3
    x[len(masks):, V - 7:] = torch.randn((len(masks), 7), generator=g) * 3
    _check_logprobs(x.to(dtype).cuda(), [25, V - 3] * len(masks), 20)


@pytest.mark.parametrize("m", [3e5, 0.999e6, 1e6, 1.001e6, 5e6, -3e5, -0.99e6, -1e6, -4e6])
def test_logprobs_of_rows_about_a_far_value(cuda, m):
    """Logits whose differences count, around a value on either side of where the sums change their form."""
    x = _spread(5, 20000, 4).double() + m
    _check_logprobs(x.float().cuda(), [0, 5, 19999, 777, 12345], 8)


def _spread(rows, cols, seed):
    return torch.randn((rows, cols), generator=torch.Generator().manual_seed(seed)) * 2


# ---- gates that close --------------------------------------------------------------------
def _check_gated(x, gate, kind):
    """Scales those of the formula in 64 bits; elements within half a step, silu's error and f32's least
    step (2^-150, which the least scale makes 2^-23)."""
    from npu_amd import groups
    q, s = _mx(*x.shape, kind)
    groups.fused_mx_quantize(x.cuda(), q, s, gate=gate.cuda())
    g = _np64(gate)
    y = _np64(x) * np.where(np.isneginf(g), 0.0, R.silu64(np.where(np.isneginf(g), 0.0, g)))
    mag = np.abs(y.reshape(len(y), -1, 32)).max(2)
    sc = R.scale_of(mag, kind)
    assert np.array_equal(s.cpu().numpy(), sc), np.argwhere(s.cpu().numpy() != sc)[:5].tolist()
    most = R.TABLE[kind][7 if kind == "e2m1" else 126]
    t = np.clip(y * np.repeat(np.ldexp(1.0, 127 - sc), 32, 1), -most, most)
    err = np.abs(np.array(R.TABLE[kind])[R.codes(q, kind)] - t)
    assert (err <= R.half_step(t * (1 + SILU_EPS), kind) + SILU_EPS * np.abs(t) + 2.0 ** -23).all()
    return q, s


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 20, 2.0 ** 100, 1.9 * 2.0 ** 126])
def test_quantize_gates_that_close(cuda, size, kind):
    """Each gate from -80 to -280, alone in a block of zeros and beside others like it, by x of any size."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    gates = bits[(bits <= -80) & (bits >= -280)]
    n = len(gates)
    assert n > 200
    gate = torch.zeros((n, 64), dtype=BF16)
    rows = torch.arange(n)
    gate[rows, rows % 32] = gates
    gate[:, 32:] = gates[(rows[:, None] + torch.arange(32)) % n]
    x = torch.zeros((n, 64))
    x[:, :32] = size
    x[:, 32:] = size * (1 + torch.rand((n, 32), generator=torch.Generator().manual_seed(3)) * 0.05)
    _check_gated(x.to(BF16), gate, kind)


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
def test_quantize_gates_of_all_sizes_together(cuda, kind):
    """Rows whose lanes take either form, x of sizes over all exponents; -Inf and the type's lowest value close."""
    x = _rnd(301, 416, seed=7) * 2.0 ** torch.randint(-60, 124, (301, 416), generator=torch.Generator().manual_seed(8))
    gate = (_rnd(301, 416, seed=9) * 60).clamp(max=8)
    gate[::3] = _rnd(101, 416, seed=10)
    gate[5, ::2], gate[6], gate[7, 40:60] = -math.inf, -math.inf, float(torch.finfo(BF16).min)
    q, s = _check_gated(x.to(BF16), gate.to(BF16), kind)
    assert not s[6].any() and (R.values(q, s, kind)[6] == 0).all()


# ---- rows of the norm at bf16's ends --------------------------------------------------------
@pytest.mark.parametrize("kind", ["e4m3", "e2m1", "bf16"])
@pytest.mark.parametrize("power", [-133, -130, -127, -126, -124, -110, 104, 112, 120, 123])
def test_norm_of_rows_of_any_size(cuda, power, kind):
    """Rows of subnormals, whose root f32 does not hold, and of the largest numbers: blocks are those of the
    formula in 64 bits, eps = 0 or not."""
    x = (_rnd(40, 544, seed=power).clamp(-8, 8) * 2.0 ** power).to(BF16).cuda()
    assert torch.isfinite(x).all() and x.any(1).all()
    g = (torch.rand(544, generator=torch.Generator().manual_seed(power)) + 0.5).cuda()
    _check_norm(x, g, kind, eps=0.0)
    _check_norm(x, g, kind, eps=1e-30)
    _check_norm(x, g, kind, delta=(x.float() * 0.5).to(BF16))


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("power", [0, 100, 120, -100, -120])
def test_norm_of_wide_rows_and_gains(cuda, power, kind):
    """Rows with entries of all exponents, gains from 2^-140 to 2^118: entries down to f32's least."""
    g = torch.Generator().manual_seed(power)
    x = _rnd(20, 4096, seed=power) * 2.0 ** torch.randint(-100, 1, (20, 4096), generator=g) * 2.0 ** min(power, 123)
    gain = (torch.rand(4096, generator=g) + 0.5) * 2.0 ** torch.randint(-140, 118, (4096 // 32,), generator=g).repeat_interleave(32)
    _check_norm(x.to(BF16).cuda(), gain.cuda(), kind, eps=0.0)


def test_norm_next_to_ties_of_huge_rows(cuda):
    """Gains that put entries within 2^-23 of half way between two elements, in rows of 2^120: the side on
    which 64 bits have them."""
    from npu_amd import groups
    x = (_rnd(1, 2048, seed=11) * 2.0 ** 120).to(BF16)
    h = _np64(x)
    y = h / np.sqrt((h * h).mean(1, keepdims=True))
    want = np.abs(y).reshape(-1, 32)
    code = np.random.default_rng(1).integers(8, 120, want.shape)  # (normal elements)
    tie = (np.array(R.E4M3)[code] + np.array(R.E4M3)[code + 1]) / 2
    tie[:, 0] = 256.0  # each block's largest, whatever the others': its scale is 1
    tie[:, 1:] = np.minimum(tie[:, 1:], 248.0)
    g = torch.from_numpy((tie / np.maximum(want, 2.0 ** -20)).reshape(-1)).float()
    g[h[0] == 0] = 1.0
    q, s = _mx(1, 2048, "e4m3")
    groups.fused_llama_add_rmsnorm(x.cuda(), g.cuda(), q, s, eps=0.0)
    y = y * g.double().numpy()
    c, sc = R.quantize(y, "e4m3")
    # (f64's own roundings, 2^-51 or so, decide where a gain gives a tie to that)
    t = np.abs(y / np.repeat(np.ldexp(1.0, sc - 127), 32, 1))
    sure = np.abs(t - tie.reshape(1, -1)) > 2.0 ** -49 * t
    assert sure.mean() > 0.9 and np.array_equal(s.cpu().numpy(), sc)
    assert np.array_equal(R.codes(q, "e4m3")[sure], c[sure])


# ---- products of terms far apart -------------------------------------------------------------
def _check_far_terms(a, sa, w, sw, kind):
    """A result is off by its rounding to bf16; by the f32 sums' roundings, one for each eight k and each wave or
    part (64 at most); and with e4m3 by what the instruction cuts off: of each eight neighbouring k
    less than 2^-13 of the largest term from each of the seven others."""
    got = _np64(_product(a, sa, w, sw))
    A, W = R.values(a, sa, kind), R.values(w, sw, "e2m1")
    exact, mag, cut = A @ W.T, np.abs(A) @ np.abs(W).T, 0.0
    if kind == "e4m3":
        for k in range(0, A.shape[1], 8):
            cut = cut + np.abs(A[:, None, k:k + 8] * W[None, :, k:k + 8]).max(2)
    off = (A.shape[1] / 8 + 64) * 2.0 ** -24 * mag + 7 * 2.0 ** -13 * cut
    bad = np.abs(got - exact) > BF16_HALF_STEP * np.abs(exact) + (1 + BF16_HALF_STEP) * off
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0].tolist()}"


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(5, 40, 544), (17, 64, 128), (48, 96, 4096), (300, 130, 1184), (1030, 100, 1056)])
def test_product_of_elements_of_all_sizes(cuda, M, N, K, kind):
    """Every finite element as likely as any other, blocks' scales up to 2^16 apart."""
    r = np.random.default_rng(M + K)
    c = r.integers(0, 127, (M, K)) | r.integers(0, 2, (M, K)) << 7 if kind == "e4m3" else r.integers(0, 16, (M, K))
    a = c.astype(np.uint8) if kind == "e4m3" else (c[:, 0::2] | c[:, 1::2] << 4).astype(np.uint8)
    a = torch.from_numpy(a).cuda()
    a = a.view(torch.float8_e4m3fn) if kind == "e4m3" else a
    sa, sw = (torch.from_numpy(r.integers(119, 136, (n, K // 32)).astype(np.uint8)).cuda() for n in (M, N))
    w = torch.from_numpy(r.integers(0, 256, (N, K // 2)).astype(np.uint8)).cuda()
    _check_far_terms(a, sa, w, sw, kind)


@pytest.mark.parametrize("M", [1, 20, 200])
@pytest.mark.parametrize("near", [True, False])
def test_product_of_small_terms_beside_large_ones(cuda, near, M):
    """Terms just below what is kept beside a largest one: seven of the same eight, or of other eights, where
    f32 sums keep them.  A second large term of a later eight takes the first away again."""
    a = np.zeros((M, 128))
    a[:, 0] = a[:, 127] = 256.0
    at = np.arange(1, 8) if near else np.arange(8, 120)
    # by w = 4 a large term is 2^10; by 1 these are from 2^-3, the least that is kept beside it, down
    a[:, at] = 1.875 * 2.0 ** -(4 + np.arange(M)[:, None] % 5)
    w = np.zeros((32, 128))
    w[:, 0], w[:, 127], w[:, at] = 4.0, -4.0, 1.0
    ca, cw = R.nearest(a, "e4m3").astype(np.uint8), R.nearest(w, "e2m1").astype(np.uint8)
    one = lambda n: torch.full((n, 4), 127, dtype=torch.uint8, device="cuda")
    qa = torch.from_numpy(ca).cuda().view(torch.float8_e4m3fn)
    qw = torch.from_numpy(cw[:, 0::2] | cw[:, 1::2] << 4).cuda()
    _check_far_terms(qa, one(M), qw, one(32), "e4m3")
    if not near:
        # 2^10 and at most 112 terms in f32: the roundings' steps are 2^-14
        got, exact = _np64(_product(qa, one(M), qw, one(32))), R.values(qa, one(M), "e4m3") @ w.T
        assert (np.abs(got - exact) <= BF16_HALF_STEP * np.abs(exact) + 16 * 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [50, 4000, 50257])
def test_logprobs_of_certain_tokens(cuda, V, dtype):
    """One token far above all others, at any logit: its log probability is 0 and the entropy 0; beside
    an equal one -ln 2.  No log probability is above 0, no entropy below."""
    from npu_amd import groups
    T = 300
    g = torch.Generator().manual_seed(V)
    x = torch.randn((T, V), generator=g) - 2000
    best = torch.randint(0, V, (T,), generator=g)
    m = torch.randn(T, generator=g) * 40
    x[torch.arange(T), best] = m
    x = x.to(dtype).cuda()
    new = lambda *s, dt=F32: torch.full(s, 55, dtype=dt, device="cuda")
    lp, en, tt, tl = new(T), new(T), new(T, 2, dt=torch.int32), new(T, 2)
    groups.fused_token_logprobs(x, best.int().cuda(), lp, groups.token_logprobs_workspace(x, 2), entropy=en, top_tokens=tt,
                                top_logprobs=tl)
    # (the others' share is below e^-1700: 0 in f32)
    assert (lp == 0).all() and (en == 0).all() and (tl[:, 0] == 0).all() and torch.equal(tt[:, 0].cpu(), best.int())
    near = (torch.randn((T, V), generator=g) * 0.01 - 17).to(dtype).cuda()
    near[torch.arange(T), best] = torch.rand(T, generator=g).to(dtype).cuda()
    groups.fused_token_logprobs(near, best.int().cuda(), lp, groups.token_logprobs_workspace(near, 2), entropy=en, top_tokens=tt,
                                top_logprobs=tl)
    assert (lp <= 0).all() and (en >= 0).all() and (tl <= 0).all()


# ---- the largest sizes ---------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N", [(3, 40), (40, 64)])
def test_product_of_the_longest_rows(cuda, M, N, kind):
    """K = 2^20: sums of few bits come out exact (below 2^24 of the least unit, 2^-4)."""
    K = 1 << 20
    (a, sa), (w, sw) = _blocks(M, K, kind, M, small=True), _blocks(N, K, "e2m1", N, small=True)
    exact, mag = _exact(a, sa, w, sw, kind)
    got = _product(a, sa, w, sw).cpu()
    # (where the terms' magnitudes together stay below 2^20 every sum on the way is exact; past it each of 2^17 sums
    # rounds by half a step of at most 2^22)
    exact_sums = mag < 2.0 ** 20
    assert torch.equal(got[exact_sums], exact[exact_sums].float().to(BF16))
    off = (2.0 ** 17 + 64) * 2.0 ** -24 * mag.clamp(max=2.0 ** 22)
    assert ((got.double() - exact).abs() <= BF16_HALF_STEP * exact.abs() + (1 + BF16_HALF_STEP) * off).all()


@pytest.mark.parametrize("kind", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(40, 33, 544), (130, 70, 1184), (256, 300, 512)])
def test_product_of_rows_far_apart(cuda, M, N, K, kind):
    """Rows nearly 2^23 bytes apart, the most there is: the same bits as side by side."""
    from npu_amd import groups
    (a, sa), (w, sw) = _blocks(M, K, kind, 1), _blocks(N, K, "e2m1", 2)
    want = _product(a, sa, w, sw).clone()
    step = (1 << 23) - 16
    wide = torch.zeros((max(M, N), step), dtype=torch.uint8, device="cuda")

    def far(t, at):
        v = wide[:t.shape[0], at:at + t.shape[1]]
        v.copy_(t.view(torch.uint8))
        return v.view(t.dtype)

    got = _product(far(a, 0), far(sa, 1 << 20), far(w, 2 << 20), far(sw, (3 << 20) + 1))
    assert torch.equal(got, want)
    with pytest.raises(groups.NpuError, match="at most 2"):
        far_rows = torch.empty((2, 1 << 23), dtype=torch.uint8, device="cuda")[:, :K // 2]
        one = torch.zeros((2, K // 32), dtype=torch.uint8, device="cuda")
        groups.fused_mx_matmul(far_rows, one, w, sw, torch.empty((2, N), dtype=BF16, device="cuda"), torch.empty(1 << 20, device="cuda"))


def test_the_most_rows(cuda):
    """2^23 rows of logits, and of w: the last are those of a call of their own."""
    from npu_amd import groups
    T, V = 1 << 23, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((T, V), generator=g, device="cuda")
    tok = torch.randint(-1, V, (T,), generator=g, device="cuda").int()
    lp, rk = torch.full((T,), 5.0, device="cuda"), torch.full((T,), 5, dtype=torch.int32, device="cuda")
    tt, tl = torch.full((T, 2), 5, dtype=torch.int32, device="cuda"), torch.full((T, 2), 5.0, device="cuda")
    groups.fused_token_logprobs(x, tok, lp, groups.token_logprobs_workspace(x, 2), ranks=rk, top_tokens=tt, top_logprobs=tl)
    want = x.double().log_softmax(1)
    at = tok.long().clamp(min=0)[:, None]
    # (f32: three terms, their exponentials and logarithm, below 2^-20)
    assert torch.where(tok < 0, lp.double(), lp.double() - want.gather(1, at)[:, 0]).abs().max() < 2.0 ** -20 * 16
    best, order = x.sort(dim=1, descending=True, stable=True)
    assert torch.equal(tt.long(), order[:, :2]) and (tl.double() - want.gather(1, order[:, :2])).abs().max() < 2.0 ** -20 * 16
    assert torch.equal(rk.long(), torch.where(tok < 0, -1, (x > x.gather(1, at)).sum(1)))
    del x, want, best, order, tt, tl
    N, K = 1 << 23, 64
    (a, sa), (few, s_few) = _blocks(5, K, "e4m3", 1), _blocks(1000, K, "e2m1", 2)
    w, sw = few.repeat(N // 1000 + 1, 1)[:N].contiguous(), s_few.repeat(N // 1000 + 1, 1)[:N].contiguous()
    out, some = _product(a, sa, w, sw), _product(a, sa, few, s_few)
    assert torch.equal(out, some.repeat(1, N // 1000 + 1)[:, :N])
