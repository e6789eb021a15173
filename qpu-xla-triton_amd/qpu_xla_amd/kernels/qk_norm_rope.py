"""Norms of queries and keys per head and the position rotation in one pass, on gfx950.

* ``qk_norm_rope`` -- queries [T, Hq, D] and keys [T, Hkv, D] to normalised, rotated ones.
* ``qk_norm_rope_cache`` -- the same, storing the keys and (unchanged) values [T, Hkv, D] into a paged cache
  [pages, page_size, Hkv, D] at flat slots ``page * page_size + offset``; returns the queries in the cache's type.

``y = x * rsqrt(mean(x^2) + epsilon) * weight`` per row (skipped where a weight is None), then the pairs
``(y[i], y[i + R/2])``, or ``(y[2i], y[2i + 1])`` with ``interleaved``, turn by ``cos[position, i]``,
``sin[position, i]`` (fp32 [P, R/2]); elements past R stay.  Everything is computed in fp32 and rounded once.  Tokens
and heads may have any stride (slices of one q/k/v projection), rows are dense.  A position outside the table gives a
NaN row, a negative slot (padding) is not stored.

The reference's rotation and norm programs (``src/qpu_xla/kernels``) are separate fp32 launches; no counterpart of
the fused form or of the paged cache exists there.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import TYPES, byte_strides, cache_struct, check_cache, check_head_rows, check_index, empty_for
from qpu_xla_amd._tensors import ptr, require_gpu, stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel


def _check(name: str, query: torch.Tensor, key: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           positions: torch.Tensor, weights: tuple[torch.Tensor | None, torch.Tensor | None]) -> None:
    check_head_rows(name, "query", query)
    check_head_rows(name, "key", key)
    if query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2] or query.dtype != key.dtype:
        raise ValueError(f"{name}: query and key must agree in tokens, head size and type")
    head_dim = query.shape[2]
    for table in (cos, sin):
        if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
            raise ValueError(f"{name}: cos and sin must be contiguous float32 [positions, rotary / 2]")
    if cos.shape != sin.shape or 2 * cos.shape[1] > head_dim:
        raise ValueError(f"{name}: cos and sin must have one shape, of at most half the head size")
    check_index(name, "positions", positions, torch.int32, query.shape[0])
    for weight in weights:
        if weight is not None and (weight.dtype != torch.float32 or tuple(weight.shape) != (head_dim,)
                                   or not weight.is_contiguous()):
            raise ValueError(f"{name}: weights must be contiguous float32 [{head_dim}]")


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    query_weight: torch.Tensor | None = None,
    key_weight: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    interleaved: bool = False,
    query_out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated (query, key), in the inputs' type unless outputs are given (which may be the inputs)."""
    name = "qk_norm_rope"
    _check(name, query, key, cos, sin, positions, (query_weight, key_weight))
    tokens, query_heads, head_dim = query.shape
    if query_out is None:
        query_out = empty_for(stream, tuple(query.shape), query.dtype if key_out is None else key_out.dtype, query.device)
    if key_out is None:
        key_out = empty_for(stream, tuple(key.shape), query_out.dtype, key.device)
    check_head_rows(name, "query_out", query_out)
    check_head_rows(name, "key_out", key_out)
    if query_out.shape != query.shape or key_out.shape != key.shape or query_out.dtype != key_out.dtype:
        raise ValueError(f"{name}: outputs must have the inputs' shapes and one type")
    require_gpu(name, query, key, cos, sin, positions, query_weight, key_weight, query_out, key_out)
    _lib.call(
        "qxt_qk_norm_rope", ptr(query), *byte_strides(query, 2), ptr(key), *byte_strides(key, 2), ptr(query_weight),
        ptr(key_weight), epsilon, ptr(cos), ptr(sin), cos.shape[1] * 4, cos.shape[0], ptr(positions), ptr(query_out),
        *byte_strides(query_out, 2), ptr(key_out), *byte_strides(key_out, 2), tokens, query_heads, key.shape[1],
        head_dim, 2 * cos.shape[1], TYPES[query.dtype], TYPES[query_out.dtype],
        _lib.ROPE_INTERLEAVED if interleaved else 0, stream_handle(stream),
    )
    return query_out, key_out


def qk_norm_rope_cache(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    query_weight: torch.Tensor | None = None,
    key_weight: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    interleaved: bool = False,
    query_out: torch.Tensor | None = None,
    stream: Any = None,
) -> torch.Tensor:
    """Normalise and rotate, store keys and values at ``slots`` (int64 [T]) of the cache; the queries in its type."""
    name = "qk_norm_rope_cache"
    _check(name, query, key, cos, sin, positions, (query_weight, key_weight))
    check_head_rows(name, "value", value)
    if value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError(f"{name}: key and value must have one shape and type")
    check_cache(name, key_cache, value_cache)
    if tuple(key_cache.shape[2:]) != tuple(key.shape[1:]):
        raise ValueError(f"{name}: the cache must hold the keys' heads and head size")
    check_index(name, "slots", slots, torch.int64, query.shape[0])
    if query_out is None:
        query_out = empty_for(stream, tuple(query.shape), key_cache.dtype, query.device)
    check_head_rows(name, "query_out", query_out)
    if query_out.shape != query.shape or query_out.dtype != key_cache.dtype:
        raise ValueError(f"{name}: query_out must have the query's shape and the cache's type")
    require_gpu(name, query, key, value, cos, sin, positions, slots, key_cache, value_cache, query_weight, key_weight,
                query_out)
    _lib.call(
        "qxt_qk_norm_rope_cache", ptr(query), *byte_strides(query, 2), ptr(key), *byte_strides(key, 2), ptr(value),
        *byte_strides(value, 2), ptr(query_weight), ptr(key_weight), epsilon, ptr(cos), ptr(sin), cos.shape[1] * 4,
        cos.shape[0], ptr(positions), ptr(slots), ptr(query_out), *byte_strides(query_out, 2),
        cache_struct(key_cache, value_cache), query.shape[0], query.shape[1], 2 * cos.shape[1], TYPES[query.dtype],
        _lib.ROPE_INTERLEAVED if interleaved else 0, stream_handle(stream),
    )
    return query_out


@dataclass(frozen=True, slots=True)
class QkNormRopeOptions:
    """Last argument of ``QK_NORM_ROPE_CACHE_KERNEL``."""

    epsilon: float = 1e-6
    interleaved: bool = False


def qk_norm_rope_grid(query: torch.Tensor) -> tuple[int, int, int]:
    """Grid of ``QK_NORM_ROPE_CACHE_KERNEL``: (query heads, tokens, 1)."""
    return (query.shape[1], query.shape[0], 1)


def _execute_qk_norm_rope_cache(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    if (len(args) != 13 or not all(isinstance(a, torch.Tensor) for a in args[:10])
            or not all(a is None or isinstance(a, torch.Tensor) for a in args[10:12])
            or not isinstance(args[12], QkNormRopeOptions)):
        raise KernelError("norm and rotation expects (query, key, value, cos, sin, positions, slots, key_cache, value_cache, "
                          "query_out, query_weight or None, key_weight or None, QkNormRopeOptions)")
    query_out, query_weight, key_weight, options = args[9:]
    if query_out.dim() != 3 or tuple(grid) != qk_norm_rope_grid(query_out):
        raise KernelError(f"norm and rotation grid must be (query heads, tokens, 1), got {tuple(grid)}")
    qk_norm_rope_cache(*args[:9], query_weight, key_weight, epsilon=options.epsilon, interleaved=options.interleaved,
                       query_out=query_out, stream=stream)


QK_NORM_ROPE_CACHE_KERNEL = Kernel("gfx950.qk_norm_rope_cache", _execute_qk_norm_rope_cache)

__all__ = ["QK_NORM_ROPE_CACHE_KERNEL", "QkNormRopeOptions", "qk_norm_rope", "qk_norm_rope_cache", "qk_norm_rope_grid"]
