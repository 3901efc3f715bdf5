"""Plain 64-bit forms of the serving operators and batches to run them on."""
import math

import numpy as np
import torch


class Batch:
    """A cache of random pages and the arrays that say what lies where.

    ``news`` and ``lens`` are the sequences' new tokens and own keys (lens may
    be less than news, or past the table); ``extra``: rows after the last
    sequence; ``max_pages``: the table's width (None: what the lengths need)."""

    def __init__(self, news, lens, Hkv, Dh, page, prefix=0, ragged=True, extra=0, max_pages=None, seed=0,
                 device="cuda"):
        rng = np.random.default_rng(seed)
        self.news, self.lens, self.Hkv, self.Dh, self.page, self.prefix = news, lens, Hkv, Dh, page, prefix
        self.B, self.T = len(news), sum(news) + extra
        self.max_pages = max_pages or max(1, max(-(-n // page) for n in lens))
        used = [min(self.max_pages, -(-max(n, 0) // page)) for n in lens]
        npre = -(-prefix // page)
        self.P = sum(used) + npre + 2
        order = rng.permutation(self.P)
        table = np.full((self.B, self.max_pages), -1, np.int32)
        at = npre
        for b, c in enumerate(used):
            table[b, :c] = order[at:at + c]
            at += c
        self.table, self.pre = table, order[:npre].astype(np.int32)
        self.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)
        g = torch.Generator(device="cpu").manual_seed(seed + 1)
        rnd = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(device)
        self.rnd, self.dev = rnd, dev
        self.k_pages, self.v_pages = rnd(self.P, Hkv, page, Dh), rnd(self.P, Hkv, page, Dh)
        self.page_table, self.kv_len = dev(table), dev(np.asarray(lens, np.int32))
        self.q_start = dev(self.start) if ragged else None
        self.prefix_table = dev(self.pre) if npre else None

    def tokens(self):
        """(row, sequence, own key index) of every token that belongs to one."""
        for b, n in enumerate(self.news):
            for i in range(n):
                yield int(self.start[b]) + i, b, self.lens[b] - n + i


def rope_tables(positions, width):
    ang = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(width) * 2 / (2 * width))
    return torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))


def rotate64(x, cos, sin, pairs):
    """x f64 [heads, Dh], cos and sin f64 [width] -> (rotated, |a cos| + |b sin|)."""
    y, mag, w = x.clone(), x.abs(), cos.numel()
    if pairs == "interleaved":
        i, j = torch.arange(0, 2 * w, 2), torch.arange(1, 2 * w, 2)
    else:
        i, j = torch.arange(w), torch.arange(w, 2 * w)
    a, b = x[:, i], x[:, j]
    y[:, i], y[:, j] = a * cos - b * sin, a * sin + b * cos
    mag[:, i] = (a * cos).abs() + (b * sin).abs()
    mag[:, j] = (a * sin).abs() + (b * cos).abs()
    return y, mag


def append64(bt, Q, K, V, cos, sin, pairs):
    """(Qo, its magnitudes, k_pages, its magnitudes, v_pages) in f64, from host copies."""
    Q, K, V, cos, sin = (t.detach().cpu().double() for t in (Q, K, V, cos, sin))
    kp, vp = bt.k_pages.cpu().double(), bt.v_pages.cpu().double()
    km, Qo, qm = kp.abs(), torch.zeros_like(Q), torch.zeros_like(Q)
    table = bt.page_table.cpu()
    for t, b, j in bt.tokens():
        if j < 0 or j >= bt.max_pages * bt.page:
            continue
        c, s = cos[bt.prefix + j], sin[bt.prefix + j]
        y, m = rotate64(Q[t].view(-1, bt.Dh), c, s, pairs)
        Qo[t], qm[t] = y.reshape(-1), m.reshape(-1)
        pid = int(table[b, j // bt.page])
        if not 0 <= pid < bt.P:
            continue
        y, m = rotate64(K[t].view(-1, bt.Dh), c, s, pairs)
        kp[pid, :, j % bt.page], km[pid, :, j % bt.page] = y, m
        vp[pid, :, j % bt.page] = V[t].view(-1, bt.Dh)
    return Qo, qm, kp, km, vp


def attend64(bt, Q, scale):
    """(A, sum |p v|, keys seen) in f64 from host copies; a row without keys is 0."""
    Q = Q.detach().cpu().double()
    kp, vp = bt.k_pages.cpu().double(), bt.v_pages.cpu().double()
    table, pre = bt.page_table.cpu().numpy(), None if bt.prefix_table is None else bt.prefix_table.cpu().numpy()
    H = Q.shape[1] // bt.Dh
    G = H // bt.Hkv
    out, mag, seen = torch.zeros_like(Q), torch.zeros_like(Q), torch.zeros(Q.shape[0], dtype=torch.int64)

    def gather(tab, n):
        """Keys and values [Hkv, m, Dh] of the first n places, those of bad pages left out, and their places."""
        j = np.arange(n)
        pid = tab[j // bt.page] if n else np.zeros(0, np.int32)
        ok = (pid >= 0) & (pid < bt.P)
        pid, j = torch.from_numpy(pid[ok].astype(np.int64)), j[ok]
        sl = torch.from_numpy(j % bt.page)
        return kp[pid, :, sl].transpose(0, 1), vp[pid, :, sl].transpose(0, 1), torch.from_numpy(j)

    pk, pv, pj = gather(pre, bt.prefix) if bt.prefix else gather(table[0], 0)
    for b, n in enumerate(bt.news):
        if not n:
            continue
        own = min(max(bt.lens[b], 0), bt.max_pages * bt.page)
        k, v, j = gather(table[b], own)
        ks, vs = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        at = torch.cat([torch.full((pj.numel(),), -(2 ** 40)), j])
        rows = slice(int(bt.start[b]), int(bt.start[b]) + n)
        place = torch.arange(bt.lens[b] - n, bt.lens[b])
        hid = at[None, :] > place[:, None]
        seen[rows] = (~hid).sum(1)
        for h in range(H):
            c = slice(h * bt.Dh, h * bt.Dh + bt.Dh)
            s = (Q[rows, c] @ ks[h // G].T * scale).masked_fill(hid, -math.inf)
            m = s.amax(1, keepdim=True).clamp(min=-1e300) if s.shape[1] else torch.zeros(n, 1, dtype=torch.float64)
            p = (s - m).exp()
            tot = p.sum(1, keepdim=True)
            p = torch.where(tot > 0, p / tot, 0.0)
            # a hidden key's value does not count, whatever it is
            clean = torch.nan_to_num(vs[h // G], nan=0.0, posinf=0.0, neginf=0.0)
            out[rows, c], mag[rows, c] = p @ clean, p @ clean.abs()
    return out, mag, seen


def sample64(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(token, probability) of one row, numpy f64: the operator's definition."""
    x = np.asarray(x, np.float64)
    cand = np.isposinf(x) if np.isposinf(x).any() else np.isfinite(x)
    idx = np.nonzero(cand)[0]
    if not idx.size:
        return -1, 0.0
    order = idx[np.argsort(-x[idx], kind="stable")]
    t = 1.0 if temperature is None else float(temperature)
    if not t > 0:
        return int(order[0]), 1.0
    top = x[order[0]]
    w = np.ones(order.size) if np.isposinf(top) else np.exp((x[order] - top) / t)
    n = order.size
    if top_k is not None and top_k > 0:
        n = min(n, int(top_k))
    cum = np.concatenate([[0.0], np.cumsum(w)])
    if top_p is not None and top_p < 1:
        n = min(n, max(1, int((cum[:n] < float(top_p) * cum[n]).sum())))
    if min_p is not None and min_p > 0:
        n = min(n, max(1, int((w >= float(min_p)).sum())))
    pick = min(n - 1, int((cum[1:n + 1] <= float(u) * cum[n]).sum()))
    return int(order[pick]), float(w[pick] / cum[n])
