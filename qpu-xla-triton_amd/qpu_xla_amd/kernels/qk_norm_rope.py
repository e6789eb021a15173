"""Norms of queries and keys per head and the position rotation in one pass, on gfx950.

* ``qk_norm_rope`` -- queries [T, Hq, D] and keys [T, Hkv, D] to normalised, rotated ones.
* ``qk_norm_rope_cache`` -- the same, storing the keys and (unchanged) values [T, Hkv, D] into a paged cache
  [pages, page_size, Hkv, D] at flat slots ``page * page_size + offset``; returns the queries in the cache's type.

``y = x * rsqrt(mean(x^2) + epsilon) * weight`` per row (skipped where a weight is None), then the pairs
``(y[i], y[i + R/2])``, or ``(y[2i], y[2i + 1])`` with ``interleaved``, turn by ``cos[position, i]``,
``sin[position, i]`` (fp32 [P, R/2]); elements past R stay.  Everything is computed in fp32 and rounded once.  Tokens
and heads may have any stride (slices of one q/k/v projection), rows are dense.  A position outside the table makes the
row's rotated part NaN, a negative slot (padding) is not stored.

The reference's rotation and norm programs (``src/qpu_xla/kernels``) are separate fp32 launches; no counterpart of
the fused form or of the paged cache exists there.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import check_index, head_rows, like_for, paged_cache, require_one_gpu
from qpu_xla_amd._tensors import ptr, stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel


def _check_tables(name: str, tokens: int, head_dim: int, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                  *weights: torch.Tensor | None) -> tuple[int, int]:
    """(positions, half the rotary size) of the tables."""
    shape = cos.shape
    if (len(shape) != 2 or sin.shape != shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32
            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"{name}: cos and sin must be contiguous float32 [positions, rotary / 2] of one shape")
    if 2 * shape[1] > head_dim:
        raise ValueError(f"{name}: cos and sin turn more than the head size")
    check_index(name, "positions", positions, torch.int32, tokens)
    for weight in weights:
        if weight is not None:
            check_index(name, "weights", weight, torch.float32, head_dim)
    return shape[0], shape[1]


def _check_rows(name: str, query: torch.Tensor, key: torch.Tensor) -> tuple[tuple, tuple]:
    q, k = head_rows(name, "query", query), head_rows(name, "key", key)
    if q[0][0] != k[0][0] or q[0][2] != k[0][2] or q[1] != k[1]:
        raise ValueError(f"{name}: query and key must agree in tokens, head size and type")
    return q, k


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
    (shape, code, *query_strides), (key_shape, _, *key_strides) = _check_rows(name, query, key)
    tokens, query_heads, head_dim = shape
    rows, half = _check_tables(name, tokens, head_dim, cos, sin, positions, query_weight, key_weight)
    if query_out is None:
        query_out = like_for(stream, query, None if key_out is None else key_out.dtype)
    if key_out is None:
        key_out = like_for(stream, key, query_out.dtype)
    query_out_shape, out_code, *query_out_strides = head_rows(name, "query_out", query_out)
    key_out_shape, key_code, *key_out_strides = head_rows(name, "key_out", key_out)
    if query_out_shape != shape or key_out_shape != key_shape or out_code != key_code:
        raise ValueError(f"{name}: outputs must have the inputs' shapes and one type")
    require_one_gpu(name, query, key, cos, sin, positions, query_weight, key_weight, query_out, key_out)
    _lib.call(
        "qxt_qk_norm_rope", query.data_ptr(), *query_strides, key.data_ptr(), *key_strides, ptr(query_weight),
        ptr(key_weight), epsilon, cos.data_ptr(), sin.data_ptr(), half * 4, rows, positions.data_ptr(),
        query_out.data_ptr(), *query_out_strides, key_out.data_ptr(), *key_out_strides, tokens, query_heads,
        key_shape[1], head_dim, 2 * half, code, out_code, _lib.ROPE_INTERLEAVED if interleaved else 0,
        stream_handle(stream),
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
    (shape, code, *query_strides), (key_shape, _, *key_strides) = _check_rows(name, query, key)
    value_shape, value_code, *value_strides = head_rows(name, "value", value)
    if value_shape != key_shape or value_code != code:
        raise ValueError(f"{name}: key and value must have one shape and type")
    tokens, query_heads, head_dim = shape
    rows, half = _check_tables(name, tokens, head_dim, cos, sin, positions, query_weight, key_weight)
    cache_shape, cache_code, _, _, cache = paged_cache(name, key_cache, value_cache)
    if cache_shape[2:] != key_shape[1:]:
        raise ValueError(f"{name}: the cache must hold the keys' heads and head size")
    check_index(name, "slots", slots, torch.int64, tokens)
    if query_out is None:
        query_out = like_for(stream, query, key_cache.dtype)
    out_shape, out_code, *out_strides = head_rows(name, "query_out", query_out)
    if out_shape != shape or out_code != cache_code:
        raise ValueError(f"{name}: query_out must have the query's shape and the cache's type")
    require_one_gpu(name, query, key, value, cos, sin, positions, slots, key_cache, value_cache, query_weight, key_weight,
                    query_out)
    _lib.call(
        "qxt_qk_norm_rope_cache", query.data_ptr(), *query_strides, key.data_ptr(), *key_strides, value.data_ptr(),
        *value_strides, ptr(query_weight), ptr(key_weight), epsilon, cos.data_ptr(), sin.data_ptr(), half * 4, rows,
        positions.data_ptr(), slots.data_ptr(), query_out.data_ptr(), *out_strides, cache, tokens, query_heads, 2 * half,
        code, _lib.ROPE_INTERLEAVED if interleaved else 0, stream_handle(stream),
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
