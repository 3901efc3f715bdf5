"""Operators of a Llama decoder whose weights are held in four bits, as a program
calls them: quantisation to microscaled formats (OCP Microscaling Formats v1.0:
blocks of 32 along K share a power of two), the residual's addition and norm with
an output in eight bits, the product of such operands, and the log probabilities
of tokens.

`run` is one pass: with `own` the framework's entry points, without it the same
in elementary torch operations.  `exact` is the operators' definition in 64
bits.
"""
import math
import os
import random
import sys

import torch

own = False

F32, F64, BF16, I32, U8 = torch.float32, torch.float64, torch.bfloat16, torch.int32, torch.uint8
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-5


def _groups():
    path = os.path.join(os.getcwd(), "npu-dialect_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from npu_amd import groups
    return groups


def listed():
    return [
        # ---- norm: one token in the tests' layer: the smallest call, where the
        # launch counts.
        {"name": "norm_token", "op": "norm", "T": 1, "D": 512, "delta": False},
        # A decoding step's batch between two products.
        {"name": "norm_step_t48", "op": "norm", "T": 48, "D": 4096, "delta": True},
        # Prompts, an odd number of tokens.
        {"name": "norm_prompts", "op": "norm", "T": 8191, "D": 4096, "delta": True},
        # ---- quantise: a step's gated activations in the benchmark's layer, the gate
        # and the other half in one buffer.
        {"name": "quantize_gated", "op": "quantize", "R": 300, "K": 1408, "kind": "gated"},
        # A prompt's gated activations of a wide layer.
        {"name": "quantize_gated_prompt", "op": "quantize", "R": 4099, "K": 14336, "kind": "gated"},
        # A weight [K, N] to four bits, when a model is loaded.
        {"name": "quantize_weight", "op": "quantize", "R": 14336, "K": 4096, "kind": "weight"},
        # ---- product: one token in the tests' layer.
        {"name": "product_token", "op": "product", "M": 1, "N": 1408, "K": 512, "a": "e4m3"},
        # A decoding step: the weight's bytes.
        {"name": "product_step_t48", "op": "product", "M": 48, "N": 14336, "K": 4096, "a": "e4m3"},
        # Prompts of an odd number of tokens, activations in eight bits.
        {"name": "product_prompt", "op": "product", "M": 4099, "N": 4096, "K": 14336, "a": "e4m3"},
        # A large batch of prompts, both operands in four bits.
        {"name": "product_large", "op": "product", "M": 8192, "N": 8192, "K": 8192, "a": "e2m1"},
        # ---- log probabilities: a step's answers with their alternatives, an odd
        # vocabulary.
        {"name": "logprobs_step_b48", "op": "logprobs", "T": 48, "V": 50257, "dtype": "bf16", "top": 20},
        # A prompt scored over a large vocabulary.
        {"name": "logprobs_prompt", "op": "logprobs", "T": 2000, "V": 128000, "dtype": "bf16", "top": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def _draw(rng, op):
    if op == "norm":
        return {"op": op, "T": _log_int(rng, 1, 16000), "D": 32 * _log_int(rng, 2, 512), "delta": rng.random() < 0.7}
    if op == "quantize":
        return {"op": op, "R": _log_int(rng, 1, 16000), "K": 32 * _log_int(rng, 2, 512),
                "kind": rng.choice(["gated", "plain", "f32", "weight"])}
    if op == "product":
        return {"op": op, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 16, 16384), "K": 32 * _log_int(rng, 2, 512),
                "a": rng.choice(["e4m3", "e2m1"])}
    return {"op": op, "T": _log_int(rng, 1, 2000), "V": _log_int(rng, 1000, 160000),
            "dtype": rng.choice(["f32", "bf16"]), "top": rng.choice([0, 1, 5, 20])}


_LARGEST = {"norm": "norm_prompts", "quantize": "quantize_gated_prompt quantize_weight",
            "product": "product_large product_prompt", "logprobs": "logprobs_prompt"}


def draw(rng):
    op = rng.choice(["norm", "quantize", "product", "product", "logprobs"])
    refs = [work(c) for c in listed() if c["name"] in _LARGEST[op].split()]
    most = {k: max(r[k] for r in refs) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng, op)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


# ---- inputs -------------------------------------------------------------------
def _activations(g, rows, cols):
    """Rows whose size varies, with a few channels far above the others, as a
    decoder's are."""
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=F32)
    x *= torch.rand((rows, 1), generator=g, device="cuda") * 1.5 + 0.5
    at = torch.randint(0, cols, (max(1, cols // 200),), generator=g, device="cuda")
    x[:, at] *= 20.0
    return x


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    d = {}
    if case["op"] == "norm":
        d["x"] = _activations(g, case["T"], case["D"]).to(BF16)
        d["delta"] = torch.randn(d["x"].shape, generator=g, device="cuda", dtype=BF16) if case["delta"] else None
        d["g"] = torch.rand((case["D"],), generator=g, device="cuda", dtype=F32) + 0.5
    elif case["op"] == "quantize":
        r, k = case["R"], case["K"]
        d["gate"] = None
        if case["kind"] == "gated":
            both = torch.randn((r, 2 * k), generator=g, device="cuda", dtype=BF16)
            both *= 2.0
            d["gate"], d["x"] = both[:, :k], both[:, k:]
        elif case["kind"] == "weight":
            # [K, N], its rows padded to 16 bytes; the operator takes the transposed view
            w = torch.randn((k, -(-r // 8) * 8), generator=g, device="cuda", dtype=BF16)
            w *= k ** -0.5
            d["x"] = w[:, :r].t()
        else:
            d["x"] = _activations(g, r, k).to(F32 if case["kind"] == "f32" else BF16)
    elif case["op"] == "product":
        d["a"], d["a_scale"] = _to_blocks(_activations(g, case["M"], case["K"]), case["a"])
        w = torch.randn((case["N"], case["K"]), generator=g, device="cuda", dtype=F32)
        w *= case["K"] ** -0.5
        d["w"], d["w_scale"] = _to_blocks(w, "e2m1")
    else:
        t, v = case["T"], case["V"]
        # a head's logits: a broad bell and a few tokens that the context asks for
        x = torch.randn((t, v), generator=g, device="cuda", dtype=BF16 if case["dtype"] == "bf16" else F32)
        x *= 2.0
        at = torch.randint(0, v, (t, 1), generator=g, device="cuda")
        at = (at + torch.arange(12, device="cuda") * (v // 12)) % v
        x.scatter_add_(1, at, (torch.rand((t, 12), generator=g, device="cuda") * 9).to(x.dtype))
        d["logits"] = x
        # mostly a likely token, sometimes any; some rows of a padded batch have none
        any_token = torch.randint(0, v, (t,), generator=g, device="cuda")
        row = torch.arange(t, device="cuda")
        token = torch.where(row % 5 == 4, any_token, at[:, 0])
        d["tokens"] = torch.where(row % 40 == 30, -1, token).to(I32)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    st = {"case": case, "in": d}
    new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device="cuda")
    if case["op"] == "norm":
        t, k = case["T"], case["D"]
        st["h"] = new(BF16, t, k) if case["delta"] else None
        st["q"], st["scale"] = new(E4M3, t, k), new(E8M0, t, k // 32)
    elif case["op"] == "quantize":
        r, k = case["R"], case["K"]
        four = case["kind"] == "weight"
        st["q"], st["scale"] = new(U8, r, k // 2) if four else new(E4M3, r, k), new(E8M0, r, k // 32)
        st["values"] = new(BF16, r, k) if four else None
    elif case["op"] == "product":
        st["out"] = new(BF16, case["M"], case["N"])
    else:
        t, k = case["T"], case["top"]
        st["logprobs"], st["entropy"], st["ranks"] = new(F32, t), new(F32, t), new(I32, t)
        st["top_tokens"] = new(I32, t, k) if k else None
        st["top_logprobs"] = new(F32, t, k) if k else None
    return st


# ---- one pass -------------------------------------------------------------------
def _scratch(state, make):
    """The workspace that a program keeps beside its buffers."""
    if "workspace" not in state:
        state["workspace"] = make()
    return state["workspace"]


def _outputs(state):
    """A pass's buffers; four-bit values are returned as the numbers they stand for."""
    op = state["case"]["op"]
    if op == "product":
        return state["out"]
    if op == "norm":
        return {"h": state["h"], "q": state["q"], "scale": state["scale"]}
    if op == "quantize":
        four = state["values"] is not None
        if four:
            return {"q": state["q"], "values": state["values"], "scale": state["scale"]}
        return {"values": state["q"], "scale": state["scale"]}
    return {n: state[n] for n in ("logprobs", "entropy", "ranks", "top_tokens", "top_logprobs")}


def _run_own(state):
    groups = _groups()
    case, d = state["case"], state["in"]
    if case["op"] == "norm":
        groups.fused_llama_add_rmsnorm(d["x"], d["g"], state["q"], state["scale"], delta=d["delta"], h=state["h"],
                                       eps=EPS)
    elif case["op"] == "quantize":
        groups.fused_mx_quantize(d["x"], state["q"], state["scale"], gate=d["gate"], values=state["values"])
    elif case["op"] == "product":
        ws = _scratch(state, lambda: groups.mx_matmul_workspace(d["a"], d["w"]))
        groups.fused_mx_matmul(d["a"], d["a_scale"], d["w"], d["w_scale"], state["out"], ws)
    else:
        ws = _scratch(state, lambda: groups.token_logprobs_workspace(d["logits"], case["top"]))
        groups.fused_token_logprobs(d["logits"], d["tokens"], state["logprobs"], ws, entropy=state["entropy"],
                                    ranks=state["ranks"], top_tokens=state["top_tokens"],
                                    top_logprobs=state["top_logprobs"])
    return _outputs(state)


def _scaled(x, largest):
    """Entries over their block's scale, and the scales' bytes."""
    blocks = x.reshape(x.shape[0], -1, 32)
    top = blocks.abs().amax(2)
    e = (torch.frexp(top).exponent - 1 - largest).clamp(min=-127)
    e = torch.where(top > 0, e, -127)
    power = (127 - e) << 23  # the bits of 2^-e
    return (blocks * power.to(I32).view(F32)[..., None]).reshape(x.shape), (e + 127).to(U8)


def _e2m1_code(y):
    a = y.abs()
    code = (a > 0.25).to(U8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    return code + torch.signbit(y).to(U8) * 8


def _to_blocks(x, kind):
    """(q, scale) of f32 rows."""
    y, s = _scaled(x, 8 if kind == "e4m3" else 2)
    if kind == "e4m3":
        return y.clamp(-448.0, 448.0).to(E4M3), s.view(E8M0)
    c = _e2m1_code(y)
    return c[:, 0::2] | c[:, 1::2] << 4, s.view(E8M0)


def _values_of(q, s):
    """What blocks stand for, in f32."""
    if q.dtype == E4M3:
        v = q.to(F32)
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
        c = torch.stack([q & 15, q >> 4], 2).reshape(q.shape[0], -1)
        v = table[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).to(F32))
    return (v.view(v.shape[0], -1, 32) * s.to(F32)[..., None]).view(v.shape)


def run(state):
    if own:
        return _run_own(state)
    case, d = state["case"], state["in"]
    if case["op"] == "norm":
        h = d["x"]
        if d["delta"] is not None:
            h = state["h"].copy_(d["x"].to(F32) + d["delta"].to(F32))
        h = h.to(F32)
        y = h * (h.square().mean(1, keepdim=True) + EPS).rsqrt() * d["g"]
        q, s = _to_blocks(y, "e4m3")
        state["q"].copy_(q)
        state["scale"].copy_(s)
    elif case["op"] == "quantize":
        x = d["x"].to(F32)
        if d["gate"] is not None:
            z = d["gate"].to(F32)
            x = x * (z / (1.0 + (-z).exp()))
        q, s = _to_blocks(x, "e2m1" if case["kind"] == "weight" else "e4m3")
        state["q"].copy_(q)
        state["scale"].copy_(s)
        if state["values"] is not None:
            state["values"].copy_(_values_of(q, s))
    elif case["op"] == "product":
        state["out"].copy_(_values_of(d["a"], d["a_scale"]) @ _values_of(d["w"], d["w_scale"]).t())
    else:
        x = d["logits"].to(F32)
        m = x.amax(1, keepdim=True)
        e = (x - m).exp()
        total = e.sum(1, keepdim=True)
        state["entropy"].copy_((total.log() - ((x - m) * e).sum(1, keepdim=True) / total)[:, 0])
        lse = m + total.log()
        t = d["tokens"].long()[:, None]
        xt = x.gather(1, t.clamp(min=0))
        state["logprobs"].copy_(torch.where(t < 0, 0.0, xt - lse)[:, 0])
        before = torch.arange(x.shape[1], device="cuda") < t
        rank = ((x > xt) | ((x == xt) & before)).sum(1, keepdim=True)
        state["ranks"].copy_(torch.where(t < 0, -1, rank)[:, 0])
        if case["top"]:
            best, at = torch.sort(x, dim=1, descending=True, stable=True)
            state["top_tokens"].copy_(at[:, :case["top"]])
            state["top_logprobs"].copy_(best[:, :case["top"]] - lse)
    return _outputs(state)


# ---- bytes and operations -------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n = case["T"] * case["D"]
        return {"bytes": n * ((6 if case["delta"] else 2) + 1) + n // 32 + 4 * case["D"], "flops": 8 * n}
    if case["op"] == "quantize":
        n = case["R"] * case["K"]
        each = {"gated": 4 + 1, "plain": 2 + 1, "f32": 4 + 1, "weight": 2 + 0.5 + 2}[case["kind"]]
        return {"bytes": int(n * each) + n // 32, "flops": (12 if case["kind"] == "gated" else 4) * n}
    if case["op"] == "product":
        m, n, k = case["M"], case["N"], case["K"]
        a = m * k if case["a"] == "e4m3" else m * k // 2
        return {"bytes": a + n * k // 2 + (m + n) * k // 32 + 2 * m * n,
                "flops": 2 * m * n * k}
    n = case["T"] * case["V"]
    return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + (16 + 8 * case["top"]) * case["T"], "flops": 6 * n}


# ---- the same in 64 bits ----------------------------------------------------------
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _power64(e):
    """2^e of whole e as it is (pow rounds), for normal f64 numbers."""
    return ((e.long() + 1023) << 52).view(F64)


def _floor_log2(x):
    """Of positive f64 numbers; log2 rounds next to a power of two."""
    return torch.frexp(x).exponent - 1


def _nearest64(y, mantissa, least, most):
    """The nearest number with `mantissa` bits after the point, exponents from
    `least` on and at most `most`; ties to even."""
    step = _power64(_floor_log2(y.abs().clamp(min=2.0 ** least)) - mantissa)
    return (torch.round(y / step) * step).clamp(-most, most)


def _quantize64(x, kind):
    """(numbers before the scale, scales) of f64 rows."""
    emax, mantissa, least, most = (8, 3, -6, 448.0) if kind == "e4m3" else (2, 1, 0, 6.0)
    b = x.reshape(x.shape[0], x.shape[1] // 32, 32)
    top = b.abs().max(dim=2).values
    s = _power64(torch.where(top > 0, _floor_log2(top) - emax, -127).clamp(min=-127))
    return _nearest64(b / s[:, :, None], mantissa, least, most), s


def _numbers64(q, s):
    if q.dtype == E4M3:
        v = q.to(F64)
    else:
        signed = torch.tensor(_E2M1 + [-t for t in _E2M1], dtype=F64, device="cuda")
        v = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=F64, device="cuda")
        v[:, 0::2] = signed[(q % 16).int()]
        v[:, 1::2] = signed[(q // 16).int()]
    return v * _power64(s.view(U8).long() - 127).repeat_interleave(32, 1)


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "norm":
        h = d["x"].to(F64)
        out = {"h": None}
        if d["delta"] is not None:
            h = h + d["delta"].to(F64)
            out["h"] = h
            h = h.to(F32).to(BF16).to(F64)  # (the sum of two bf16 rounds once: f32 holds it where both are near)
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["D"] + EPS) * d["g"].to(F64)
        q, s = _quantize64(y, "e4m3")
        return {**out, "q": q.reshape(y.shape), "scale": s}
    if case["op"] == "quantize":
        x = d["x"].to(F64)
        if d["gate"] is not None:
            x = x * d["gate"].to(F64) * torch.sigmoid(d["gate"].to(F64))
        four = case["kind"] == "weight"
        q, s = _quantize64(x, "e2m1" if four else "e4m3")
        out = {"values": (q * s[:, :, None] if four else q).reshape(x.shape), "scale": s}
        return {**out, "q": None} if four else out
    if case["op"] == "product":
        return _numbers64(d["a"], d["a_scale"]) @ _numbers64(d["w"], d["w_scale"]).t().contiguous()
    t, k = case["T"], case["top"]
    out = {"logprobs": torch.zeros(t, dtype=F64, device="cuda"), "entropy": torch.zeros(t, dtype=F64, device="cuda"),
           "ranks": torch.full((t,), -1, dtype=I32, device="cuda"),
           "top_tokens": torch.zeros((t, k), dtype=I32, device="cuda") if k else None,
           "top_logprobs": torch.zeros((t, k), dtype=F64, device="cuda") if k else None}
    for r0 in range(0, t, 128):
        rows = slice(r0, min(t, r0 + 128))
        lp = torch.log_softmax(d["logits"][rows].to(F64), 1)
        out["entropy"][rows] = -(lp.exp() * lp).sum(1)
        order = torch.argsort(d["logits"][rows].to(F64), dim=1, descending=True, stable=True)
        if k:
            out["top_tokens"][rows] = order[:, :k].to(I32)
            out["top_logprobs"][rows] = lp.gather(1, order[:, :k])
        for i in range(lp.shape[0]):
            token = int(d["tokens"][r0 + i])
            if token >= 0:
                out["logprobs"][r0 + i] = lp[i, token]
                out["ranks"][r0 + i] = int((order[i] == token).nonzero()[0])
    return out
