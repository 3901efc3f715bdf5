"""Descriptors where torch does not name all the element types that the operators in microscaled floats
take (no GPU)."""
import os
import re

import pytest
import torch

from npu_amd import memref

NEWER = ["float8_e8m0fnu", "float4_e2m1fn_x2", "float8_e4m3fn"]
BIND = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "npu-dialect_amd", "bind", "serve_bind.cpp")


@pytest.mark.parametrize("missing", [NEWER[:1], NEWER[:2], NEWER])
def test_an_older_torch_describes_the_others(monkeypatch, missing):
    lacking = {name: getattr(torch, name) for name in missing}
    for name in missing:
        monkeypatch.delattr(torch, name)
    monkeypatch.setattr(memref, "_DTYPE_CODES", None)
    for dtype, code in ((torch.float32, memref.F32), (torch.bfloat16, memref.BF16), (torch.uint8, memref.U8)):
        m = memref.from_tensor(torch.zeros((2, 4), dtype=dtype))
        assert (m.dtype, m.rank, list(m.sizes[:2])) == (code, 2, [2, 4])
    for dtype in lacking.values():
        with pytest.raises(TypeError, match="unsupported tensor dtype"):
            memref.tensor_dtype(torch.zeros((2, 4), dtype=torch.uint8).view(dtype))


def test_all_types_are_described():
    for name, code in zip(NEWER, (memref.U8, memref.U8, memref.E4M3)):
        assert memref.tensor_dtype(torch.zeros((2, 4), dtype=torch.uint8).view(getattr(torch, name))) == code


def test_the_binding_names_no_newer_type():
    """c10's enumerators are not there in an older torch: the binding would not build."""
    with open(BIND) as f:
        assert not re.search(r"kFloat8|kFloat4|ScalarType::Float[48]", f.read())
