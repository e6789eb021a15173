"""Checks and C-ABI arguments of the operators over rows: floats, microscaling blocks, and where they live.

They run at every call, and a call of few rows is bound by them: shapes and strides are read once each, devices are
compared as integers, and outputs made here are not looked at again.
"""

from __future__ import annotations

from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import TYPES, empty_for

MX_BLOCK = 32
FP8 = torch.float8_e4m3fn
_FP4_STORED = (torch.uint8, torch.float4_e2m1fn_x2)
_SCALES = (torch.uint8, torch.float8_e8m0fnu)


def require_current_gpu(name: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """All tensors on the current HIP device: streams and launches belong to it."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError(f"{name}: all tensors must live on one HIP device (no CPU fallback)")
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"{name}: the tensors must live on the current HIP device")


def new_rows(stream: Any, like: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
    """``empty_for`` on a tensor's device; on the current stream at two thirds of its time where the shapes agree."""
    if stream is None:
        if like.shape == shape:
            return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)
        return torch.empty(shape, dtype=dtype, device=like.device)
    return empty_for(stream, shape, dtype, like.device)


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
    dtype, shape, scale_shape = values.dtype, values.shape, scales.shape
    fmt = _lib.MX_FP8 if dtype is FP8 else _lib.MX_FP4
    if fmt not in formats or (fmt == _lib.MX_FP4 and dtype not in _FP4_STORED) or len(shape) != 2:
        raise ValueError(f"{name}: {what} values must be packed 4-bit elements, uint8 [rows, columns / 2]"
                         + (", or float8_e4m3fn [rows, columns]" if _lib.MX_FP8 in formats else ""))
    rows, columns = shape
    if fmt == _lib.MX_FP4:
        columns *= 2
    if columns == 0 or columns % MX_BLOCK:
        raise ValueError(f"{name}: {what} must have columns in positive multiples of {MX_BLOCK}")
    if scales.dtype not in _SCALES or len(scale_shape) != 2 or scale_shape[0] != rows or scale_shape[1] != columns // MX_BLOCK:
        raise ValueError(f"{name}: {what} scales must be uint8 or float8_e8m0fnu [{rows}, {columns // MX_BLOCK}]")
    stride, element = values.stride()
    scale_stride, scale_element = scales.stride()
    if element != 1 or (scale_element != 1 and scale_shape[1] > 1) or (rows > 1 and (
            stride < shape[1] or scale_stride < scale_shape[1])):
        raise ValueError(f"{name}: {what} must have dense rows of values and scales")
    if rows <= 1:  # torch gives a single row any stride
        stride = scale_stride = 0
    return rows, columns, fmt, _lib.MX_MATRIX.pack(values.data_ptr(), stride, scales.data_ptr(), scale_stride)


def mx_outputs(name: str, like: torch.Tensor, rows: int, columns: int, fp8: bool, values: torch.Tensor | None,
               scales: torch.Tensor | None, stream: Any) -> tuple[torch.Tensor, int, torch.Tensor, int]:
    """(values, byte stride, scales, byte stride) to write blocks into, made on ``like``'s device where not given."""
    if columns == 0 or columns % MX_BLOCK:
        raise ValueError(f"{name}: columns must be a positive multiple of {MX_BLOCK}")
    shape = (rows, columns if fp8 else columns // 2)
    if values is None:
        values, stride = new_rows(stream, like, shape, FP8 if fp8 else torch.uint8), shape[1]
    else:
        stride = _byte_rows(name, "values", values, (FP8,) if fp8 else _FP4_STORED, shape)
    if scales is None:
        scales, scale_stride = new_rows(stream, like, (rows, columns // MX_BLOCK), torch.uint8), columns // MX_BLOCK
    else:
        scale_stride = _byte_rows(name, "scales", scales, _SCALES, (rows, columns // MX_BLOCK))
    return values, stride, scales, scale_stride


def share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows of two tensors (or vectors) with dense rows share memory, as the C entries tell it.

    Tensors of one row stride may lie between each other's rows; those of different strides are taken to meet where their
    ranges do.
    """
    spans = []
    for t in (a, b):
        rows, size = (t.shape[0], t.element_size()) if t.dim() > 1 else (1, t.element_size())
        spans.append((t.data_ptr(), rows, t.stride(0) * size if rows > 1 else 0, t.shape[-1] * size))
    (at, rows, skip, size), (to, to_rows, to_skip, to_size) = spans
    if not (rows and size and to_rows and to_size) or a.get_device() != b.get_device():
        return False
    skip, to_skip = skip or to_skip, to_skip or skip
    if at + (rows - 1) * skip + size <= to or to + (to_rows - 1) * to_skip + to_size <= at:
        return False
    if skip != to_skip or not skip:
        return True
    ahead = (to - at) % skip
    return ahead < size or ahead + to_size > skip
