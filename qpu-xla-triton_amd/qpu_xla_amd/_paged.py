"""Checks and C-ABI arguments shared by the attention operators over a paged cache."""

from __future__ import annotations

import ctypes
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._tensors import ptr, stream_handle

TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
CACHE_TYPES = (torch.bfloat16, torch.float16)
UINT32_MAX = 2**32 - 1


def empty_for(stream: Any, shape: tuple[int, ...], dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A new tensor that work on ``stream`` (None: the current stream) may write at once.

    The caching allocator orders a block's reuse on the stream that it was allocated for: memory written on another
    stream is allocated there, and marked as used on the caller's.
    """
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    current = torch.cuda.current_stream(device)
    handle = stream_handle(stream)
    if handle == current.cuda_stream:
        return torch.empty(shape, dtype=dtype, device=device)
    owner = torch.cuda.default_stream(device) if handle == 0 else torch.cuda.ExternalStream(handle, device=device)
    with torch.cuda.stream(owner):
        tensor = torch.empty(shape, dtype=dtype, device=device)
    tensor.record_stream(current)
    return tensor


def byte_strides(t: torch.Tensor, dims: int) -> list[int]:
    """Byte strides of the first ``dims`` dimensions; 0 for those of one entry (torch gives them any)."""
    size = t.element_size()
    return [0 if extent == 1 else step * size for extent, step in zip(t.shape[:dims], t.stride()[:dims])]


def dense_last(t: torch.Tensor) -> bool:
    return t.shape[-1] == 1 or t.stride(-1) == 1


def check_head_rows(name: str, what: str, t: torch.Tensor) -> None:
    if t.dim() != 3 or t.dtype not in TYPES or not dense_last(t):
        raise ValueError(f"{name}: {what} must be float32, bfloat16 or float16 [tokens, heads, head_dim] with dense rows")


def check_cache(name: str, keys: torch.Tensor, values: torch.Tensor | None) -> None:
    for what, t in (("key_cache", keys), ("value_cache", values)):
        if t is None:
            continue
        if t.dim() != 4 or t.dtype not in CACHE_TYPES or not dense_last(t):
            raise ValueError(f"{name}: {what} must be bfloat16 or float16 [pages, page_size, heads, head_dim] with dense rows")
    if values is not None and (values.shape != keys.shape or values.dtype != keys.dtype):
        raise ValueError(f"{name}: key_cache and value_cache must have one shape and type")
    if min(keys.shape) == 0:
        raise ValueError(f"{name}: the cache is empty")


def check_table(name: str, table: torch.Tensor, lens: torch.Tensor) -> None:
    if table.dim() != 2 or table.dtype != torch.int32 or not dense_last(table) or table.shape[1] == 0:
        raise ValueError(f"{name}: block_table must be int32 [sequences, pages of the longest] with dense rows")
    check_index(name, "context_lens", lens, torch.int32, table.shape[0])


def check_index(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, count: int) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != count or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous {str(dtype).removeprefix('torch.')} [{count}]")


def cache_struct(keys: torch.Tensor, values: torch.Tensor | None, table: torch.Tensor | None = None,
                 lens: torch.Tensor | None = None) -> Any:
    """``qxt_paged_cache`` by reference (the operators that take no values or table leave those out)."""
    pages, page_size, heads, head_dim = keys.shape
    value_strides = (0, 0, 0) if values is None else byte_strides(values, 3)
    sequences, width = (0, 0) if table is None else table.shape
    return ctypes.byref(_lib.PagedCache(
        ptr(keys), *byte_strides(keys, 3), ptr(values), *value_strides, ptr(table),
        0 if table is None or sequences == 1 else table.stride(0) * 4, ptr(lens), pages, page_size, heads, head_dim,
        TYPES[keys.dtype], width, sequences))


def check_per_slot(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, keys: torch.Tensor, table: torch.Tensor) -> None:
    shape = (table.shape[0], keys.shape[2], table.shape[1] * keys.shape[1])
    if t.dtype != dtype or tuple(t.shape) != shape or not dense_last(t):
        raise ValueError(f"{name}: {what} must be {str(dtype).removeprefix('torch.')} [sequences, heads, slots] = {list(shape)} "
                         "with dense rows")


def check_size(name: str, what: str, value: int) -> int:
    if not 0 <= int(value) <= UINT32_MAX:
        raise ValueError(f"{name}: {what} must be non-negative (and below 2^32)")
    return int(value)
