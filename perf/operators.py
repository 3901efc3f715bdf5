"""Serving operators of the Llama decoder as a program calls them: keys and
values rotated and appended to a paged cache, attention over that cache with a
prefix that the whole batch shares, and the choice of the next tokens.

`run` is one pass: with `own` the framework's entry points, without it the same
in elementary torch operations.  `exact` is the operators' definition in 64
bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32


def _groups():
    path = os.path.join(os.getcwd(), "npu-dialect_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from npu_amd import groups
    return groups


def listed():
    return [
        # ---- append: one new token of one sequence in the tests' layer (8 heads
        # of 64): the smallest call, where the launch counts.
        {"name": "append_token", "op": "append", "B": 1, "H": 8, "Hkv": 8, "Dh": 64, "page": 16,
         "new_lo": 1, "new_hi": 1, "old_lo": 300, "old_hi": 300, "prefix": 0, "pairs": "interleaved"},
        # One decoding step of a batch at different lengths, four query heads to a
        # key head.
        {"name": "append_step_b48", "op": "append", "B": 48, "H": 32, "Hkv": 8, "Dh": 128, "page": 16,
         "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 4000, "prefix": 0, "pairs": "interleaved"},
        # Three prompts of odd lengths in the benchmark's wider layer.
        {"name": "append_prompts", "op": "append", "B": 3, "H": 12, "Hkv": 12, "Dh": 64, "page": 32,
         "new_lo": 301, "new_hi": 777, "old_lo": 0, "old_hi": 50, "prefix": 0, "pairs": "interleaved"},
        # Long prompts after a shared prefix, pairs of the two halves of a head.
        {"name": "append_long_prompts", "op": "append", "B": 4, "H": 32, "Hkv": 8, "Dh": 128, "page": 64,
         "new_lo": 2500, "new_hi": 4100, "old_lo": 0, "old_hi": 0, "prefix": 500, "pairs": "halves"},
        # ---- attention: one token over a short history: latency.
        {"name": "attend_token", "op": "attend", "B": 1, "H": 8, "Hkv": 8, "Dh": 64, "page": 16,
         "new_lo": 1, "new_hi": 1, "old_lo": 500, "old_hi": 500, "prefix": 0},
        # A decoding step of a batch of very different lengths.
        {"name": "attend_step_b48", "op": "attend", "B": 48, "H": 32, "Hkv": 8, "Dh": 128, "page": 16,
         "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 8000, "prefix": 0},
        # One sequence with a very long history: the keys have to be split.
        {"name": "attend_long", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "Dh": 128, "page": 64,
         "new_lo": 1, "new_hi": 1, "old_lo": 131000, "old_hi": 131000, "prefix": 0},
        # A decoding step of a batch that answers about one shared document.
        {"name": "attend_shared_b64", "op": "attend", "B": 64, "H": 32, "Hkv": 8, "Dh": 128, "page": 32,
         "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 400, "prefix": 6001},
        # Prompts taken in pieces: many new tokens over what is cached.
        {"name": "attend_prompts", "op": "attend", "B": 4, "H": 32, "Hkv": 8, "Dh": 128, "page": 32,
         "new_lo": 800, "new_hi": 2000, "old_lo": 0, "old_hi": 900, "prefix": 77},
        # ---- sampling: one row of a small vocabulary: latency.
        {"name": "sample_row", "op": "sample", "B": 1, "V": 32000, "dtype": "f32", "mix": "both"},
        # A batch of requests, each with its own settings, an odd vocabulary in bf16.
        {"name": "sample_b96_odd", "op": "sample", "B": 96, "V": 50257, "dtype": "bf16", "mix": "all"},
        # A large batch over a large vocabulary, nucleus sampling.
        {"name": "sample_b256", "op": "sample", "B": 256, "V": 128000, "dtype": "f32", "mix": "top_p"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def _draw_batch(rng, op):
    h = rng.choice([(8, 8), (12, 12), (16, 4), (32, 8), (8, 1), (15, 5), (28, 4), (6, 2)])
    case = {"op": op, "H": h[0], "Hkv": h[1], "Dh": rng.choice([64, 128]),
            "page": rng.choice([16, 32, 64, 128, 256])}
    step = rng.random() < 0.6
    case["B"] = _log_int(rng, 1, 128 if step else 8)
    case["new_lo"] = 1 if step else _log_int(rng, 1, 500)
    case["new_hi"] = 1 if step else case["new_lo"] + _log_int(rng, 1, 1000)
    case["old_hi"] = _log_int(rng, 1, 60000 // case["B"] if step else 2000)
    case["old_lo"] = rng.choice([0, case["old_hi"] // 2, case["old_hi"]])
    case["prefix"] = 0 if rng.random() < 0.5 else _log_int(rng, 1, 6000)
    if op == "append":
        case["pairs"] = rng.choice(["interleaved", "halves"])
    return case


def _draw_sample(rng):
    return {"op": "sample", "B": _log_int(rng, 1, 256), "V": _log_int(rng, 1000, 160000),
            "dtype": rng.choice(["f32", "bf16"]),
            "mix": rng.choice(["top_k", "top_p", "min_p", "both", "all", "none"])}


_LARGEST = {"append": "append_long_prompts", "attend": "attend_prompts attend_long", "sample": "sample_b256"}


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    refs = [work(c) for c in listed() if c["name"] in _LARGEST[op].split()]
    most = {k: max(r[k] for r in refs) for k in ("bytes", "flops")}
    while True:
        case = _draw_sample(rng) if op == "sample" else _draw_batch(rng, op)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


# ---- inputs -------------------------------------------------------------------
def _lengths(case):
    """New and earlier tokens of each sequence: part of the case, so that
    `work` knows them."""
    r = random.Random("%(B)d %(new_lo)d %(new_hi)d %(old_lo)d %(old_hi)d" % case)
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    old = [r.randint(case["old_lo"], case["old_hi"]) for _ in range(case["B"])]
    return new, old


def _ragged(case):
    return case["new_hi"] > 1


def _pages(n, page):
    return -(-n // page)


def _cache_inputs(case, g, d):
    """A cache whose pages lie in any order, as an allocator leaves them; the
    table's places past a sequence's last page hold -1."""
    new, old = _lengths(case)
    page, hkv, dh = case["page"], case["Hkv"], case["Dh"]
    own_len = [n + o for n, o in zip(new, old)]
    counts = [_pages(n, page) for n in own_len]
    npre = _pages(case["prefix"], page)
    total = sum(counts) + npre
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int64).to(I32)
    table = torch.full((case["B"], max(counts)), -1, dtype=I32, device="cuda")
    at = npre
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    d["page_table"] = table
    d["prefix_table"] = order[:npre].clone() if npre else None
    d["kv_len"] = torch.tensor(own_len, dtype=I32, device="cuda")
    starts = np.concatenate([[0], np.cumsum(new)])
    d["q_start"] = torch.from_numpy(starts).to(I32).cuda() if _ragged(case) else None
    shape = (total, hkv, page, dh)
    d["k_pages"] = torch.randn(shape, generator=g, device="cuda", dtype=BF16)
    d["v_pages"] = torch.randn(shape, generator=g, device="cuda", dtype=BF16)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    d = {}
    if case["op"] == "sample":
        b, v = case["B"], case["V"]
        # a head's logits: a broad bell and a few tokens that the context asks for
        x = torch.randn((b, v), generator=g, device="cuda", dtype=F32) * 2
        at = torch.randint(0, v, (b, 12), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand((b, 12), generator=g, device="cuda", dtype=F32) * 9)
        d["logits"] = x.to(BF16) if case["dtype"] == "bf16" else x
        uni = lambda lo, hi: torch.rand((b,), generator=g, device="cuda", dtype=F32) * (hi - lo) + lo
        mix = case["mix"]
        d["u"] = uni(0, 1).clamp(max=1 - 2 ** -24)
        d["temperature"] = None if mix == "none" else uni(0.5, 1.2)
        d["top_k"] = torch.randint(1, 101, (b,), generator=g, device="cuda", dtype=I32) \
            if mix in ("top_k", "both", "all") else None
        d["top_p"] = uni(0.7, 0.98) if mix in ("top_p", "both", "all") else None
        d["min_p"] = uni(0.01, 0.2) if mix in ("min_p", "all") else None
        if mix == "all":  # requests that leave a setting out, or ask for the best token
            row = torch.arange(b, device="cuda")
            d["top_k"] = torch.where(row % 3 == 1, 0, d["top_k"]).to(I32)
            d["top_p"] = torch.where(row % 4 == 2, 1.0, d["top_p"])
            d["min_p"] = torch.where(row % 2 == 0, 0.0, d["min_p"])
            d["temperature"] = torch.where(row % 16 == 5, 0.0, d["temperature"])
        return d
    new, old = _lengths(case)
    t, h, hkv, dh = sum(new), case["H"], case["Hkv"], case["Dh"]
    rows = lambda heads: torch.randn((t, heads * dh), generator=g, device="cuda", dtype=BF16)
    d["Q"] = rows(h)
    _cache_inputs(case, g, d)
    if case["op"] == "append":
        d["K"], d["V"] = rows(hkv), rows(hkv)
        n = case["prefix"] + d["page_table"].shape[1] * case["page"]
        ang = torch.arange(n, device="cuda", dtype=F64)[:, None] * \
            10000.0 ** (-torch.arange(dh // 2, device="cuda", dtype=F64) * 2 / dh)
        d["cos_t"], d["sin_t"] = ang.cos().to(F32), ang.sin().to(F32)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    st = {"case": case, "in": d}
    if case["op"] == "sample":
        st["tokens"] = torch.empty((case["B"],), dtype=I32, device="cuda")
        st["probs"] = torch.empty((case["B"],), dtype=F32, device="cuda")
    else:
        st["out"] = torch.empty_like(d["Q"])
    return st


# ---- one pass -------------------------------------------------------------------
def _scratch(state, make):
    """The workspace that a program keeps beside its buffers."""
    if "workspace" not in state:
        state["workspace"] = make()
    return state["workspace"]


def _run_own(state):
    groups = _groups()
    case, d = state["case"], state["in"]
    if case["op"] == "append":
        groups.fused_llama_rope_append(
            d["Q"], d["K"], d["V"], d["cos_t"], d["sin_t"], d["k_pages"], d["v_pages"],
            d["page_table"], d["kv_len"], state["out"], q_start=d["q_start"],
            prefix_len=case["prefix"], pairs=case["pairs"])
        return {"Q": state["out"], "k_pages": d["k_pages"], "v_pages": d["v_pages"]}
    if case["op"] == "attend":
        ws = _scratch(state, lambda: groups.paged_attention_workspace(
            d["Q"], d["k_pages"], d["page_table"], case["prefix"]))
        return groups.fused_llama_paged_attention(
            d["Q"], d["k_pages"], d["v_pages"], d["page_table"], d["kv_len"], state["out"],
            case["Dh"] ** -0.5, ws, q_start=d["q_start"], prefix_table=d["prefix_table"],
            prefix_len=case["prefix"])
    ws = _scratch(state, lambda: groups.sample_workspace(d["logits"]))
    groups.fused_sample_tokens(d["logits"], d["u"], state["tokens"], ws, temperature=d["temperature"],
                               top_k=d["top_k"], top_p=d["top_p"], min_p=d["min_p"],
                               probs=state["probs"])
    return {"tokens": state["tokens"], "probs": state["probs"]}


def _places(case, d):
    """Of each new token: its sequence and its place among the sequence's own
    keys."""
    b = case["B"]
    kv = d["kv_len"].long()
    if d["q_start"] is None:
        return torch.arange(b, device="cuda"), kv - 1
    start = d["q_start"].long()
    n = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), n, output_size=d["Q"].shape[0])
    return seq, (kv - n)[seq] + torch.arange(seq.numel(), device="cuda") - start[seq]


def _rotated(x, heads, cos, sin, pairs):
    t, w = x.shape
    v = x.float().view(t, heads, w // heads)
    c, s = cos[:, None, :], sin[:, None, :]
    if pairs == "interleaved":
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).reshape(t, heads, w // heads)
    a, b = v.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_append(case, d, out):
    page, hkv, dh = case["page"], case["Hkv"], case["Dh"]
    seq, at = _places(case, d)
    cos, sin = d["cos_t"][case["prefix"] + at], d["sin_t"][case["prefix"] + at]
    out.copy_(_rotated(d["Q"], case["H"], cos, sin, case["pairs"]).reshape(out.shape))
    pid = d["page_table"][seq, at // page].long()
    d["k_pages"][pid, :, at % page] = _rotated(d["K"], hkv, cos, sin, case["pairs"]).to(BF16)
    d["v_pages"][pid, :, at % page] = d["V"].view(-1, hkv, dh)
    return {"Q": out, "k_pages": d["k_pages"], "v_pages": d["v_pages"]}


def _plain_attend(case, d, out):
    b, h, hkv, dh = case["B"], case["H"], case["Hkv"], case["Dh"]
    g, lp, scale = h // hkv, case["prefix"], case["Dh"] ** -0.5
    seq, at = _places(case, d)
    t = seq.numel()
    # the new tokens of a sequence side by side, padded to the most that one has
    if d["q_start"] is None:
        n, col = 1, torch.zeros_like(seq)
    else:
        n = case["new_hi"]
        col = torch.arange(t, device="cuda") - d["q_start"].long()[seq]
    q = torch.zeros((b, n, hkv, g, dh), dtype=F32, device="cuda")
    q[seq, col] = d["Q"].float().view(t, hkv, g, dh)
    last = torch.full((b, n), -1, dtype=torch.int64, device="cuda")
    last[seq, col] = at
    q = q.permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, dh)
    last = last[:, None, :, None].expand(b, 1, n, g).reshape(b, 1, n * g, 1)

    def keys(pages):  # own keys or values [B, Hkv, L, Dh]
        x = pages[d["page_table"].clamp(min=0).long()].float()
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, dh)

    s = (q @ keys(d["k_pages"]).transpose(2, 3)) * scale
    s = s.masked_fill(torch.arange(s.shape[3], device="cuda") > last, float("-inf"))
    m = s.amax(3, keepdim=True)
    if lp:
        def shared(pages):  # the prefix's [Hkv, Lp, Dh]
            x = pages[d["prefix_table"].long()].float()
            return x.permute(1, 0, 2, 3).reshape(hkv, -1, dh)[:, :lp]
        qa = q.transpose(0, 1).reshape(hkv, b * n * g, dh)
        sp = (qa @ shared(d["k_pages"]).transpose(1, 2)) * scale
        mp = sp.amax(2, keepdim=True).view(hkv, b, n * g, 1).transpose(0, 1)
        m = torch.maximum(m, mp)
    m = m.clamp(min=torch.finfo(F32).min)
    p = (s - m).exp()
    total = p.sum(3, keepdim=True)
    o = p @ keys(d["v_pages"])
    if lp:
        pp = (sp - m.transpose(0, 1).reshape(hkv, b * n * g, 1)).exp()
        total = total + pp.sum(2, keepdim=True).view(hkv, b, n * g, 1).transpose(0, 1)
        o = o + (pp @ shared(d["v_pages"])).view(hkv, b, n * g, dh).transpose(0, 1)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.view(b, hkv, n, g, dh).transpose(1, 2)[seq, col]
    out.copy_(o.reshape(t, h * dh))
    return out


def _plain_sample(case, d, state):
    b, v = case["B"], case["V"]
    x, idx = torch.sort(d["logits"].double(), dim=1, descending=True, stable=True)
    col = lambda name, off: (torch.full((b, 1), off, dtype=F64, device="cuda") if d[name] is None
                             else d[name].double()[:, None])
    temp, k, p, mp = col("temperature", 1.0), col("top_k", 0), col("top_p", 1.0), col("min_p", 0.0)
    greedy = temp <= 0
    w = ((x - x[:, :1]) / torch.where(greedy, 1.0, temp)).exp()
    rank = torch.arange(v, device="cuda", dtype=F64)
    w1 = torch.where((k <= 0) | (rank < k), w, 0.0)
    s1 = w1.sum(1, keepdim=True)
    keep = (w1 > 0) & ((p >= 1) | (w1.cumsum(1) - w1 < p * s1)) & ((mp <= 0) | (w >= mp))
    keep = torch.where(greedy, rank < 1, keep | (rank < 1))
    kept = torch.where(keep, w, 0.0)
    cum = kept.cumsum(1)
    s = kept.sum(1, keepdim=True)
    pick = (cum <= d["u"].double()[:, None] * s).sum(1, keepdim=True)
    pick = torch.minimum(pick, keep.sum(1, keepdim=True) - 1)
    state["tokens"].copy_(idx.gather(1, pick)[:, 0])
    state["probs"].copy_((kept.gather(1, pick) / s)[:, 0])
    return {"tokens": state["tokens"], "probs": state["probs"]}


def run(state):
    if own:
        return _run_own(state)
    case, d = state["case"], state["in"]
    if case["op"] == "append":
        return _plain_append(case, d, state["out"])
    if case["op"] == "attend":
        return _plain_attend(case, d, state["out"])
    return _plain_sample(case, d, state)


# ---- bytes and operations -------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 28 * case["B"], "flops": 4 * n}
    new, old = _lengths(case)
    t, h, hkv, dh = sum(new), case["H"], case["Hkv"], case["Dh"]
    if case["op"] == "append":
        places = max(max(n + o for n, o in zip(new, old)) - min(old), 1)
        tables = 4 * dh * min(t, places)
        return {"bytes": 4 * t * (h + 2 * hkv) * dh + tables, "flops": 3 * t * (h + hkv) * dh}
    keys = sum(new) + sum(old) + case["prefix"]
    pairs = sum(n * (o + case["prefix"]) + n * (n + 1) // 2 for n, o in zip(new, old))
    return {"bytes": 4 * t * h * dh + 4 * keys * hkv * dh, "flops": 4 * dh * h * pairs}


# ---- the same in 64 bits ----------------------------------------------------------
def _exact_append(case, d):
    new, old = _lengths(case)
    h, hkv, dh, page, lp = case["H"], case["Hkv"], case["Dh"], case["page"], case["prefix"]
    kc, vc = d["k_pages"].to(F64), d["v_pages"].to(F64)
    r = torch.arange(dh, device="cuda")
    if case["pairs"] == "interleaved":
        angle, mate = r // 2, r ^ 1
        sign = torch.where(r % 2 == 0, -1.0, 1.0).to(F64)
    else:
        angle, mate = r % (dh // 2), (r + dh // 2) % dh
        sign = torch.where(r < dh // 2, -1.0, 1.0).to(F64)
    outs, at = [], 0
    for b, (n, o) in enumerate(zip(new, old)):
        c = d["cos_t"][lp + o:lp + o + n].to(F64)[:, None, angle]
        s = d["sin_t"][lp + o:lp + o + n].to(F64)[:, None, angle] * sign
        turn = lambda x: x * c + x[:, :, mate] * s
        outs.append(turn(d["Q"][at:at + n].to(F64).view(n, h, dh)).reshape(n, h * dh))
        j = torch.arange(o, o + n, device="cuda")
        pid = d["page_table"][b].long()[j // page]
        kc[pid, :, j % page] = turn(d["K"][at:at + n].to(F64).view(n, hkv, dh))
        vc[pid, :, j % page] = d["V"][at:at + n].to(F64).view(n, hkv, dh)
        at += n
    return {"Q": torch.cat(outs), "k_pages": kc, "v_pages": vc}


def _exact_attend(case, d):
    new, old = _lengths(case)
    h, hkv, dh, lp = case["H"], case["Hkv"], case["Dh"], case["prefix"]
    g = h // hkv
    out = torch.zeros(d["Q"].shape, dtype=F64, device="cuda")
    pre = d["prefix_table"].long() if lp else torch.zeros(0, dtype=torch.int64, device="cuda")
    at = 0
    for b, (n, o) in enumerate(zip(new, old)):
        pid = d["page_table"][b].long()
        pid = pid[pid >= 0]
        hidden = torch.arange(n + o, device="cuda")[None, :] > torch.arange(o, o + n, device="cuda")[:, None]
        for kh in range(hkv):
            both = [torch.cat([pages[pre, kh].reshape(-1, dh)[:lp], pages[pid, kh].reshape(-1, dh)[:n + o]]).to(F64)
                    for pages in (d["k_pages"], d["v_pages"])]
            for head in range(kh * g, kh * g + g):
                c = slice(head * dh, head * dh + dh)
                s = (d["Q"][at:at + n, c].to(F64) @ both[0].t().contiguous()) / math.sqrt(dh)
                s[:, lp:].masked_fill_(hidden, float("-inf"))
                out[at:at + n, c] = torch.softmax(s, 1) @ both[1]
        at += n
    return out


def _exact_sample(case, d):
    host = {n: None if t is None else t.double().cpu().numpy() for n, t in d.items()}
    tokens, probs = [], []
    for r in range(case["B"]):
        x = host["logits"][r]
        get = lambda name, off: off if host[name] is None else float(host[name][r])
        temp, k, p, mp = get("temperature", 1.0), int(get("top_k", 0)), get("top_p", 1.0), get("min_p", 0.0)
        order = np.argsort(-x, kind="stable")
        if temp <= 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        w = np.exp((x[order] - x[order[0]]) / temp)
        n = min(k, len(w)) if k > 0 else len(w)
        before = np.concatenate([[0.0], np.cumsum(w)])
        if p < 1:
            n = min(n, max(1, int(np.searchsorted(before[:n], p * before[n], side="left"))))
        if mp > 0:
            n = min(n, max(1, int((w >= mp).sum())))
        pick = min(n - 1, int(np.searchsorted(before[1:n + 1], float(host["u"][r]) * before[n], side="right")))
        tokens.append(int(order[pick]))
        probs.append(float(w[pick] / before[n]))
    return {"tokens": torch.tensor(tokens, dtype=I32, device="cuda"),
            "probs": torch.tensor(probs, dtype=F64, device="cuda")}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, d)
