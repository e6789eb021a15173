"""Checks and C-ABI arguments shared by the attention operators over a paged cache.

They run at every call, and a call of few tokens is bound by them: shapes and strides are read once each, devices are
compared as integers, and the cache description is packed in one go.
"""

from __future__ import annotations

from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._tensors import stream_handle

TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
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


def like_for(stream: Any, t: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``empty_for`` of a tensor's shape, type (or ``dtype``) and device (a third of its time on the current stream)."""
    if stream is None:
        return torch.empty_like(t) if dtype is None or dtype is t.dtype else torch.empty_like(t, dtype=dtype)
    return empty_for(stream, t.shape, t.dtype if dtype is None else dtype, t.device)


def workspace_for(stream: Any, size: int, device: torch.device) -> torch.Tensor | None:
    return empty_for(stream, (size,), torch.uint8, device) if size else None


def require_one_gpu(name: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError(f"{name}: all tensors must live on one HIP device (no CPU fallback)")


def head_rows(name: str, what: str, t: torch.Tensor) -> tuple[torch.Size, int, int, int]:
    """Shape, type code and byte strides (token, head; 0 for one of them: torch gives those any) of [T, H, D] rows."""
    shape = t.shape
    code = TYPES.get(t.dtype)
    if code is None or len(shape) != 3:
        raise ValueError(f"{name}: {what} must be float32, bfloat16 or float16 [tokens, heads, head_dim] with dense rows")
    tokens, heads, dim = shape
    token, head, element = t.stride()
    if element != 1 and dim != 1:
        raise ValueError(f"{name}: {what} must be float32, bfloat16 or float16 [tokens, heads, head_dim] with dense rows")
    size = 2 if code else 4
    return shape, code, 0 if tokens == 1 else token * size, 0 if heads == 1 else head * size


def _cache_strides(name: str, what: str, t: torch.Tensor) -> tuple[torch.Size, int, int, int, int]:
    shape = t.shape
    code = TYPES.get(t.dtype)
    if not code or len(shape) != 4:
        raise ValueError(f"{name}: {what} must be bfloat16 or float16 [pages, page_size, heads, head_dim] with dense rows")
    pages, page_size, heads, dim = shape
    page, slot, head, element = t.stride()
    if element != 1 and dim != 1:
        raise ValueError(f"{name}: {what} must be bfloat16 or float16 [pages, page_size, heads, head_dim] with dense rows")
    if not (pages and page_size and heads and dim):
        raise ValueError(f"{name}: the cache is empty")
    return shape, code, 0 if pages == 1 else 2 * page, 0 if page_size == 1 else 2 * slot, 0 if heads == 1 else 2 * head


def paged_cache(name: str, keys: torch.Tensor, values: torch.Tensor | None, table: torch.Tensor | None = None,
                lens: torch.Tensor | None = None) -> tuple[torch.Size, int, int, int, bytes]:
    """(cache shape, type code, sequences, table columns, ``qxt_paged_cache``) of checked tensors."""
    shape, code, *key_strides = _cache_strides(name, "key_cache", keys)
    value_at, value_strides = 0, (0, 0, 0)
    if values is not None:
        value_shape, value_code, *value_strides = _cache_strides(name, "value_cache", values)
        if value_shape != shape or value_code != code:
            raise ValueError(f"{name}: key_cache and value_cache must have one shape and type")
        value_at = values.data_ptr()
    sequences = width = table_at = table_stride = lens_at = 0
    if table is not None:
        table_shape = table.shape
        if table.dtype is not torch.int32 or len(table_shape) != 2 or table_shape[1] == 0 or not dense_last(table):
            raise ValueError(f"{name}: block_table must be int32 [sequences, pages of the longest] with dense rows")
        sequences, width = table_shape
        check_index(name, "context_lens", lens, torch.int32, sequences)
        table_at, lens_at = table.data_ptr(), lens.data_ptr()
        table_stride = 0 if sequences == 1 else 4 * table.stride(0)
    packed = _lib.PAGED_CACHE.pack(keys.data_ptr(), *key_strides, value_at, *value_strides, table_at, table_stride, lens_at,
                                   *shape, code, width, sequences)
    return shape, code, sequences, width, packed


def dense_last(t: torch.Tensor) -> bool:
    return t.stride(-1) == 1 or t.shape[-1] == 1


def check_index(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, count: int) -> None:
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous {str(dtype).removeprefix('torch.')} [{count}]")


def per_slot(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple[int, int, int]) -> tuple[int, int]:
    """Byte strides (sequence, head) of 4-byte values [sequences, heads, slots]."""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name}: {what} must be {str(dtype).removeprefix('torch.')} [sequences, heads, slots] = {list(shape)} "
                         "with dense rows")
    sequence, head, slot = t.stride()
    if slot != 1 and shape[2] != 1:
        raise ValueError(f"{name}: {what} must be {str(dtype).removeprefix('torch.')} [sequences, heads, slots] = {list(shape)} "
                         "with dense rows")
    return 0 if shape[0] == 1 else 4 * sequence, 0 if shape[1] == 1 else 4 * head


def check_size(name: str, what: str, value: int) -> int:
    if not 0 <= value <= UINT32_MAX:
        raise ValueError(f"{name}: {what} must be non-negative (and below 2^32)")
    return int(value)
