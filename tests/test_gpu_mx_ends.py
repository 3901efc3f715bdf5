"""The operators in microscaled floats, and the log probabilities, on the GPU where their values
come to the ends of what the types hold, against the plain 64-bit forms (mx_refs.py)."""
import math

import numpy as np
import pytest
import torch

import mx_refs as R
from test_gpu_mx import BF16, F32, SILU_EPS, _check_logprobs, _mx, _np64, _rnd

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
