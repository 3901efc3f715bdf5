"""Refusals of the entry points in microscaled floats and of the log probabilities: each
returns before any launch (no GPU)."""
import ctypes as C

import pytest

import npu_amd
from npu_amd import _lib
from npu_amd.memref import BF16, E4M3, F32, I32, I8, U8


def mr(shape, dtype=F32, strides=None, ptr=0x10000):
    m = _lib.NpuMemref()
    m.allocated = m.aligned = ptr
    st = strides or [C.c_int64(1).value] * 0
    if not st:
        n = 1
        for s in reversed(shape):
            st.insert(0, n)
            n *= s
    for i, (s, t) in enumerate(zip(shape, st)):
        m.sizes[i], m.strides[i] = s, t
    m.rank, m.dtype = len(shape), dtype
    return m


def refused(name, args, more, status, text):
    fn = getattr(npu_amd.lib(), name)
    got = fn(*[None if a is None else C.byref(a) for a in args], *more, None)
    msg = npu_amd.lib().npu_last_error().decode()
    assert got == status and text in msg, (got, msg)


def test_workspaces():
    lib = npu_amd.lib()
    assert lib.npu_mx_matmul_workspace(1, 1, 32) > 0 and lib.npu_mx_matmul_workspace(5000, 4096, 14336) > 0
    for bad in ((0, 1, 32), (1, 0, 32), (1, 1, 0), (1, 1, 33), (-1, 1, 32), (1, 1, (1 << 20) + 32), ((1 << 23) + 1, 1, 32),
                (1, (1 << 23) + 1, 32), (1 << 17, 1 << 15, 32), (1 << 15, 1, 1 << 20)):
        assert lib.npu_mx_matmul_workspace(*bad) == -1, bad
    assert lib.npu_token_logprobs_workspace(1, 1, 0) > 0 and lib.npu_token_logprobs_workspace(8, 1 << 20, 32) > 0
    for bad in ((0, 1, 0), (1, 0, 0), (1, (1 << 20) + 1, 0), (1, 5, 33), (1, 5, -1), ((1 << 23) + 1, 5, 0), (1 << 15, 1 << 19, 0)):
        assert lib.npu_token_logprobs_workspace(*bad) == -1, bad


QUANTIZE = {"x": mr([4, 64], BF16), "gate": mr([4, 64], BF16), "q": mr([4, 64], E4M3), "scale": mr([4, 2], U8),
            "values": mr([4, 64], BF16)}


@pytest.mark.parametrize("change,status,text", [
    ({"x": None}, 1, "x: null descriptor"),
    ({"x": mr([4, 64], I32)}, 1, "x: element type"),
    ({"x": mr([4, 48], BF16)}, 2, "multiple of 32"),
    ({"x": mr([4, (1 << 20) + 32], BF16)}, 2, "2^20"),
    ({"x": mr([1 << 16, 1 << 18], BF16)}, 2, "2^34"),
    ({"x": mr([4, 64], BF16, [128, 2])}, 2, "rows or columns must be contiguous"),
    ({"x": mr([4, 64], BF16, [1, 3]), "gate": None}, 2, "columns of 4 overlap"),
    ({"x": mr([4, 64], BF16, [1, 4])}, 2, "contiguous columns"),
    ({"x": mr([4, 64], BF16, [60, 1])}, 2, "overlap"),
    ({"x": mr([4, 64], BF16, [68, 1])}, 2, "16-byte aligned"),
    ({"x": mr([4, 64], BF16, ptr=0x10002)}, 2, "16-byte aligned"),
    ({"x": mr([4, 64], F32)}, 2, "gate: given, x is f32"),
    ({"gate": mr([4, 64], F32)}, 1, "gate: element type"),
    ({"gate": mr([4, 32], BF16)}, 1, "gate: [4,32]"),
    ({"q": mr([4, 64], I8)}, 1, "q: element type"),
    ({"q": mr([4, 32], E4M3)}, 1, "q: [4,32], expected [4,64]"),
    ({"q": mr([4, 64], U8)}, 1, "q: [4,64], expected [4,32]"),
    ({"q": mr([5, 64], E4M3)}, 1, "q: [5,64]"),
    ({"q": mr([4, 64], E4M3, [72, 1])}, 2, "16-byte aligned"),
    ({"scale": None}, 1, "scale: null descriptor"),
    ({"scale": mr([4, 3], U8)}, 1, "scale: [4,3], expected [4,2]"),
    ({"scale": mr([4, 2], F32)}, 1, "scale: element type"),
    ({"values": mr([4, 64], F32)}, 1, "values: element type"),
    ({"values": mr([3, 64], BF16)}, 1, "values: [3,64]"),
    ({"x": mr([0, 64], BF16)}, 1, "size[0] = 0"),
])
def test_quantize_refuses(change, status, text):
    refused("fused_mx_quantize", list({**QUANTIZE, **change}.values()), [], status, text)


NORM = {"x": mr([4, 64], BF16), "delta": mr([4, 64], BF16), "g": mr([64]), "h": mr([4, 64], BF16), "q": mr([4, 64], E4M3),
        "scale": mr([4, 2], U8)}


@pytest.mark.parametrize("change,eps,status,text", [
    ({"x": mr([4, 64])}, 1e-5, 1, "x: element type"),
    ({"x": mr([4, 40], BF16)}, 1e-5, 2, "multiple of 32 up to 32768"),
    ({"x": mr([4, 32800], BF16)}, 1e-5, 2, "multiple of 32 up to 32768"),
    ({"x": mr([(1 << 23) + 1, 64], BF16)}, 1e-5, 2, "at most 2^23"),
    ({"delta": mr([4, 32], BF16)}, 1e-5, 1, "delta: [4,32]"),
    ({"g": mr([32])}, 1e-5, 1, "g: size 32, expected 64"),
    ({"g": mr([64], BF16)}, 1e-5, 1, "g: element type"),
    ({"g": mr([64], ptr=0x10004)}, 1e-5, 2, "g: data pointer"),
    ({"g": mr([64], strides=[2])}, 1e-5, 2, "g: stride 2"),
    ({"h": mr([4, 96], BF16)}, 1e-5, 1, "h: [4,96]"),
    ({"q": None}, 1e-5, 1, "q: null descriptor"),
    ({"q": mr([4, 64], BF16)}, 1e-5, 1, "scale: given, q is bf16"),
    ({"q": mr([4, 64], F32)}, 1e-5, 1, "q: element type"),
    ({"scale": None}, 1e-5, 1, "scale: null descriptor"),
    ({"q": mr([4, 32], U8), "scale": mr([4, 1], U8)}, 1e-5, 1, "scale: [4,1]"),
    ({}, -1.0, 1, "eps"),
    ({}, float("nan"), 1, "eps"),
    ({}, float("inf"), 1, "eps"),
])
def test_norm_refuses(change, eps, status, text):
    refused("fused_llama_add_rmsnorm", list({**NORM, **change}.values()), [eps], status, text)


PRODUCT = {"a": mr([4, 64], E4M3), "a_scale": mr([4, 2], U8), "w": mr([8, 32], U8), "w_scale": mr([8, 2], U8),
           "out": mr([4, 8], BF16), "workspace": mr([1 << 20])}


@pytest.mark.parametrize("change,status,text", [
    ({"a": None}, 1, "a: null descriptor"),
    ({"a": mr([4, 64], BF16)}, 1, "a: element type"),
    ({"a": mr([4, 48], E4M3)}, 2, "multiple of 32"),
    ({"a": mr([4, 24], U8)}, 2, "16-byte aligned"),
    ({"a": mr([1, 24], U8), "a_scale": mr([1, 1], U8)}, 2, "multiple of 32"),
    ({"a_scale": mr([4, 1], U8)}, 1, "a_scale: [4,1]"),
    ({"w": None}, 1, "w: null descriptor"),
    ({"w": mr([8, 64], E4M3)}, 2, "w: e4m3, expected e2m1"),
    ({"w": mr([8, 64], U8)}, 1, "w: [8,64], expected [8,32]"),
    ({"w": mr([8, 32], U8, ptr=0x10008)}, 2, "w: data pointer"),
    ({"w_scale": mr([7, 2], U8)}, 1, "w_scale: [7,2]"),
    ({"out": mr([4, 8])}, 1, "out: element type"),
    ({"out": mr([8, 4], BF16)}, 1, "out: [8,4]"),
    ({"out": mr([4, 8], BF16, [1, 4])}, 2, "rows must be contiguous"),
    ({"a": mr([4, 64], E4M3, [1 << 23, 1])}, 2, "at most 2^23"),
    ({"w_scale": mr([8, 2], U8, [1 << 23, 1])}, 2, "at most 2^23"),
    ({"a": mr([(1 << 23) + 1, 64], E4M3), "a_scale": mr([(1 << 23) + 1, 2], U8), "out": mr([(1 << 23) + 1, 8], BF16)}, 2,
     "at most 2^23 each"),
    ({"a": mr([1 << 20, 64], E4M3), "a_scale": mr([1 << 20, 2], U8), "w": mr([4096, 32], U8), "w_scale": mr([4096, 2], U8),
      "out": mr([1 << 20, 4096], BF16)}, 2, "2^32 entries"),
    ({"workspace": None}, 1, "workspace: null descriptor"),
    ({"workspace": mr([1])}, 1, "needed"),
    ({"workspace": mr([1 << 20], I32)}, 1, "workspace: element type"),
])
def test_product_refuses(change, status, text):
    refused("fused_mx_matmul", list({**PRODUCT, **change}.values()), [], status, text)


LOGPROBS = {"logits": mr([4, 100], BF16), "tokens": mr([4], I32), "logprobs": mr([4]), "entropy": mr([4]), "ranks": mr([4], I32),
            "top_tokens": mr([4, 5], I32), "top_logprobs": mr([4, 5]), "workspace": mr([1 << 20])}


@pytest.mark.parametrize("change,status,text", [
    ({"logits": None}, 1, "logits: null descriptor"),
    ({"logits": mr([4, 100], I32)}, 1, "logits: element type"),
    ({"logits": mr([4, (1 << 20) + 1])}, 2, "at most 2^20"),
    ({"logits": mr([(1 << 23) + 1, 4])}, 2, "at most 2^23"),
    ({"logits": mr([1 << 15, 1 << 19], BF16)}, 2, "2^34 entries"),
    ({"logits": mr([4, 100], BF16, [100, 2])}, 2, "rows must be contiguous"),
    ({"tokens": mr([4])}, 1, "tokens: element type"),
    ({"tokens": mr([3], I32)}, 1, "tokens: size 3"),
    ({"logprobs": None}, 1, "logprobs: null descriptor"),
    ({"entropy": mr([5])}, 1, "entropy: size 5"),
    ({"ranks": mr([4])}, 1, "ranks: element type"),
    ({"top_tokens": None}, 1, "one without the other"),
    ({"top_logprobs": None}, 1, "one without the other"),
    ({"top_tokens": mr([4, 33], I32)}, 2, "at most 32"),
    ({"top_tokens": mr([4, 6], I32)}, 1, "top_logprobs: [4,5]"),
    ({"top_tokens": mr([3, 5], I32)}, 1, "top_tokens: [3,5]"),
    ({"workspace": None}, 1, "workspace: null descriptor"),
    ({"workspace": mr([2])}, 1, "needed"),
])
def test_logprobs_refuse(change, status, text):
    refused("fused_token_logprobs", list({**LOGPROBS, **change}.values()), [], status, text)
