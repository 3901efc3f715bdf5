"""npu_memref descriptors built from torch tensors (device memory plumbing only)."""
from __future__ import annotations

import ctypes as C
import struct

from ._lib import NpuMemref

F32, BF16, I8, I32, U8, E4M3 = 0, 1, 2, 3, 4, 5

_DTYPE_CODES = None


def _codes():
    global _DTYPE_CODES
    if _DTYPE_CODES is None:
        import torch
        _DTYPE_CODES = {torch.float32: F32, torch.bfloat16: BF16, torch.int8: I8,
                        torch.int32: I32, torch.uint8: U8}
        # (an older torch lacks some of these)
        for name, code in (("float8_e8m0fnu", U8), ("float4_e2m1fn_x2", U8), ("float8_e4m3fn", E4M3)):
            if hasattr(torch, name):
                _DTYPE_CODES[getattr(torch, name)] = code
    return _DTYPE_CODES


# NpuMemref's layout by rank, the sizes and strides past the rank left zero.
# Packing a descriptor in one call takes 1.8 us where assigning its fields one
# by one took 6.3; every group call builds four to eleven of them.
_PACK = [struct.Struct(f"<QQq{r}q{8 * (4 - r)}x{r}q{8 * (4 - r)}xii") for r in range(5)]
assert all(p.size == C.sizeof(NpuMemref) for p in _PACK)


def tensor_dtype(t) -> int:
    """The npu_dtype code of a tensor a descriptor can describe."""
    code = _codes().get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported tensor dtype {t.dtype}")
    if t.dim() > 4:
        raise ValueError("npu_memref holds at most rank 4")
    return code


def from_tensor(t) -> NpuMemref:
    """Descriptor of a torch tensor: the storage pointer, its offset and strides."""
    code, rank = tensor_dtype(t), t.dim()
    base = t.untyped_storage().data_ptr()
    return NpuMemref.from_buffer_copy(_PACK[rank].pack(base, base, t.storage_offset(), *t.shape,
                                                       *t.stride(), rank, code))


def absent() -> NpuMemref:
    """An optional operand that is not present (null data pointer)."""
    m = NpuMemref()
    m.rank = 1
    return m


def ref(m: NpuMemref):
    return C.byref(m)
