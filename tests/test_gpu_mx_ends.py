"""The operators in microscaled floats, and the log probabilities, on the GPU where their values
come to the ends of what the types hold, against the plain 64-bit forms (mx_refs.py)."""
import math

import numpy as np
import pytest
import torch

from test_gpu_mx import BF16, F32, _check_logprobs

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
