"""Plain 64-bit forms of the operators in microscaled floats and of the log probabilities."""
import math

import numpy as np
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E2M1 = E2M1 + [-v for v in E2M1]


def _e4m3(c):
    e, m = c >> 3 & 15, c & 7
    v = math.nan if c & 127 == 127 else math.ldexp(8 + m if e else m, max(e, 1) - 10)
    return -v if c & 128 else v


E4M3 = [_e4m3(c) for c in range(256)]
TABLE = {"e2m1": E2M1, "e4m3": E4M3}
EMAX = {"e2m1": 2, "e4m3": 8}


def codes(q, kind):
    """Element codes [R, K] of a quantised tensor (host)."""
    b = q.detach().cpu().view(torch.uint8).numpy()
    return b if kind == "e4m3" else np.stack([b & 15, b >> 4], 2).reshape(b.shape[0], -1)


def values(q, scale, kind):
    """What blocks stand for, f64 [R, K]; NaN where the scale is."""
    s = scale.detach().cpu().view(torch.uint8).numpy().astype(np.float64)
    s = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(int) - 127))
    return np.array(TABLE[kind])[codes(q, kind)] * np.repeat(s, 32, 1)


def scale_of(mag, kind):
    """Scale bytes of blocks whose largest magnitudes are these (f64)."""
    out = np.full(mag.shape, 255)
    ok = np.isfinite(mag)
    e = np.frexp(np.where(ok & (mag > 0), mag, 1.0))[1] - 1 - EMAX[kind]
    out[ok] = np.where(mag > 0, np.maximum(e, -127) + 127, 0)[ok]
    return out


def nearest(y, kind):
    """Codes of the nearest elements, ties to the even code, past the largest: the
    largest; the sign kept."""
    pos = np.array(TABLE[kind][:8] if kind == "e2m1" else [v for v in E4M3[:127]])
    a = np.minimum(np.abs(y), pos[-1])
    hi = np.searchsorted(pos, a, side="left")
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - pos[lo], pos[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return pick + np.where(np.signbit(y), 8 if kind == "e2m1" else 128, 0)


def quantize(x, kind):
    """(codes [R, K], scale bytes) of f64 rows."""
    b = x.reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        s = scale_of(np.where(np.isfinite(b).all(2), np.abs(b).max(2), np.nan), kind)
        c = nearest(np.where(np.isfinite(b), b, 0.0) / np.ldexp(1.0, np.minimum(s, 254) - 127)[..., None], kind)
    c[s == 255] = 127 if kind == "e4m3" else 0
    return c.reshape(x.shape), s


def half_step(y, kind):
    """Half the distance of the elements around y (before the scale), the largest
    element and beyond excepted."""
    mant, least = (3, -6) if kind == "e4m3" else (1, 0)
    e = np.maximum(np.frexp(np.maximum(np.abs(y), 1e-300))[1] - 1, least)
    return np.ldexp(0.5, e - mant)


def check_near(got_q, got_scale, y, eps, kind):
    """A quantised tensor against f64 rows y of which the kernel had y (1 + d), |d| <= eps:
    scales those of a largest magnitude within eps, elements within half a step of such
    a value (or the largest, beyond it)."""
    s = got_scale.detach().cpu().view(torch.uint8).numpy().astype(int)
    mag = np.abs(y.reshape(y.shape[0], -1, 32)).max(2)
    lo, hi = scale_of(mag * (1 - eps), kind), scale_of(mag * (1 + eps), kind)
    assert ((s >= lo) & (s <= hi)).all()
    inv = np.repeat(np.ldexp(1.0, 127 - s), 32, 1)
    t = y * inv
    got = np.array(TABLE[kind])[codes(got_q, kind)]
    most = TABLE[kind][7 if kind == "e2m1" else 126]
    t = np.clip(t, -most, most)
    err = np.abs(got - t)
    # (a value that eps moves over a power of two has the larger step)
    bound = half_step(t * (1 + eps), kind) + eps * np.abs(t)
    assert (err <= bound).all(), f"{int((err > bound).sum())} outside"


def silu64(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def logprobs64(x, token, k):
    """(log p of token, entropy, rank, top tokens, top log p) of one row, f64 numpy."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    m = x.max()
    if m == -np.inf:
        lp = np.full(x.shape, -np.inf)
    elif m == np.inf:
        lp = np.where(x == np.inf, -math.log((x == np.inf).sum()), -np.inf)
    else:
        lp = x - m - math.log(np.exp(x - m).sum())
    p = np.exp(lp)
    entropy = -float((p[p > 0] * lp[p > 0]).sum())
    order = np.argsort(-x, kind="stable")
    top = [int(j) if np.isfinite(lp[j]) else -1 for j in order[:k]] + [-1] * max(0, k - x.size)
    tops = [float(lp[j]) if j >= 0 else -math.inf for j in top]
    if not 0 <= token < x.size:
        return 0.0, entropy, -1, top, tops
    rank = int((x > x[token]).sum() + (x[:token] == x[token]).sum())
    return float(lp[token]), entropy, rank, top, tops
