"""Checks and C-ABI arguments of the operators over rows: floats, microscaling blocks, and where they live."""

from __future__ import annotations

from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import TYPES, require_one_gpu

MX_BLOCK = 32
FP8 = torch.float8_e4m3fn
_FP4_STORED = (torch.uint8, torch.float4_e2m1fn_x2)
_SCALES = (torch.uint8, torch.float8_e8m0fnu)


def require_current_gpu(name: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """All tensors on the current HIP device: streams and launches belong to it."""
    require_one_gpu(name, first, *others)
    if first.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name}: the tensors must live on the current HIP device")


def float_rows(name: str, what: str, t: torch.Tensor) -> tuple[int, int, int, int]:
    """(rows, columns, type code, byte stride; 0 for a single row, whose stride may be anything) of dense float rows."""
    code = TYPES.get(t.dtype)
    if code is None or t.dim() != 2:
        raise ValueError(f"{name}: {what} must be float32, bfloat16 or float16 [rows, columns] with dense rows")
    rows, columns = t.shape
    stride, element = t.stride()
    if (element != 1 and columns > 1) or (stride < columns and rows > 1):
        raise ValueError(f"{name}: {what} must be float32, bfloat16 or float16 [rows, columns] with dense rows")
    return rows, columns, code, 0 if rows <= 1 else stride * (2 if code else 4)


def vector(name: str, what: str, t: torch.Tensor | None, count: int) -> int | None:
    """Address of a contiguous float32 vector, or None."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != count or (t.stride(0) != 1 and count > 1):
        raise ValueError(f"{name}: {what} must be contiguous float32 [{count}]")
    return t.data_ptr()


def _byte_rows(name: str, what: str, t: torch.Tensor, dtypes: tuple, shape: tuple[int, int] | None) -> int:
    """Byte stride (0 for a single row) of dense rows of one-byte elements."""
    if t.dtype not in dtypes or t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        kind = " or ".join(str(d).removeprefix("torch.") for d in dtypes)
        raise ValueError(f"{name}: {what} must be {kind} {'[rows, columns]' if shape is None else list(shape)} with dense rows")
    rows, columns = t.shape
    stride, element = t.stride()
    if (element != 1 and columns > 1) or (stride < columns and rows > 1):
        raise ValueError(f"{name}: {what} must have dense rows")
    return 0 if rows <= 1 else stride


def mx_format(name: str, what: str) -> int:
    if what not in ("mxfp4", "mxfp8"):
        raise ValueError(f"{name}: the block format must be 'mxfp4' or 'mxfp8', got {what!r}")
    return _lib.MX_FP8 if what == "mxfp8" else _lib.MX_FP4


def mx_rows(name: str, what: str, values: torch.Tensor, scales: torch.Tensor, formats: tuple[int, ...] = (0, 1)) -> tuple[int, int, int, bytes]:
    """(rows, columns, format, ``qxt_mx_matrix``) of stored blocks: the values' type tells the format."""
    fp8 = values.dtype is FP8
    if (_lib.MX_FP8 if fp8 else _lib.MX_FP4) not in formats:
        raise ValueError(f"{name}: {what} values must be packed 4-bit elements, uint8 [rows, columns / 2]")
    stride = _byte_rows(name, f"{what} values", values, (FP8,) if fp8 else _FP4_STORED, None)
    rows, stored = values.shape
    columns = stored if fp8 else 2 * stored
    if columns == 0 or columns % MX_BLOCK:
        raise ValueError(f"{name}: {what} must have columns in positive multiples of {MX_BLOCK}")
    scale_stride = _byte_rows(name, f"{what} scales", scales, _SCALES, (rows, columns // MX_BLOCK))
    packed = _lib.MX_MATRIX.pack(values.data_ptr(), stride, scales.data_ptr(), scale_stride)
    return rows, columns, _lib.MX_FP8 if fp8 else _lib.MX_FP4, packed


def mx_outputs(name: str, rows: int, columns: int, fp8: bool, values: torch.Tensor | None, scales: torch.Tensor | None,
               empty: Any) -> tuple[torch.Tensor, int, torch.Tensor, int]:
    """(values, byte stride, scales, byte stride) to write blocks into; ``empty(shape, dtype)`` makes what is not given."""
    if columns == 0 or columns % MX_BLOCK:
        raise ValueError(f"{name}: columns must be a positive multiple of {MX_BLOCK}")
    shape = (rows, columns if fp8 else columns // 2)
    if values is None:
        values = empty(shape, FP8 if fp8 else torch.uint8)
    if scales is None:
        scales = empty((rows, columns // MX_BLOCK), torch.uint8)
    return (values, _byte_rows(name, "values", values, (FP8,) if fp8 else _FP4_STORED, shape),
            scales, _byte_rows(name, "scales", scales, _SCALES, (rows, columns // MX_BLOCK)))
