"""Attention of new tokens over a paged cache on gfx950.

* ``paged_attention`` -- queries [T, Hq, D] of one token a sequence, or of chunks, over keys and values in pages.
* ``paged_attention_scores`` -- the attention weight that each cached slot received, added up per key head.

Caches are [pages, page_size, Hkv, D] (bfloat16 or float16, D a multiple of 8 up to 256, any strides with 16-byte
aligned rows); ``block_table`` int32 [B, W] names each sequence's pages in order and ``context_lens`` int32 [B] its
slots in use, the new tokens' included.  ``query_starts`` int32 [B + 1] gives each sequence's tokens
(``query_starts[b]`` up to ``query_starts[b + 1]``); without it every sequence has one.  Token i of n sees the slots
``j < L``, with ``causal`` ``j <= L - n + i``, and with a window ``j > L - n + i - window``.  A token that sees none
gets 0 (and -inf as its log-sum).  Slots that a token does not see do not reach its result, whatever they hold.

``max_query`` and ``max_context`` are the host's bounds of chunk and context lengths; they size the launch (default:
what the tensors could hold).  The reference's attention programs (``src/qpu_xla/kernels/ggml_flash_attn.py``) take
one contiguous fp32 sequence; it has no paged cache.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import (
    check_index,
    check_size,
    empty_for,
    head_rows,
    like_for,
    paged_cache,
    per_slot,
    require_one_gpu,
    workspace_for,
)
from qpu_xla_amd._tensors import ptr, stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel


def _check(name: str, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor | None,
           block_table: torch.Tensor, context_lens: torch.Tensor, query_starts: torch.Tensor | None) -> tuple:
    """(query shape, its byte strides, key heads, sequences, slots a sequence, packed cache)."""
    shape, code, token_stride, head_stride = head_rows(name, "query", query)
    cache_shape, cache_code, sequences, width, cache = paged_cache(name, key_cache, value_cache, block_table, context_lens)
    _, page_size, heads, head_dim = cache_shape
    if code != cache_code or shape[2] != head_dim:
        raise ValueError(f"{name}: query must have the cache's type and head size")
    if shape[1] == 0 or shape[1] % heads:
        raise ValueError(f"{name}: query heads must be a multiple of the cache's heads")
    if head_dim % 8 or head_dim > 256:
        raise ValueError(f"{name}: head size must be a multiple of 8 up to 256")
    if query_starts is not None:
        check_index(name, "query_starts", query_starts, torch.int32, sequences + 1)
    elif shape[0] != sequences:
        raise ValueError(f"{name}: without query_starts every sequence has one token")
    return shape, (token_stride, head_stride), heads, sequences, width * page_size, cache


def _lse_stride(name: str, shape: torch.Size, lse: torch.Tensor) -> int:
    if lse.dtype is not torch.float32 or lse.shape != shape[:2] or not (lse.stride(1) == 1 or shape[1] == 1):
        raise ValueError(f"{name}: lse must be float32 [tokens, heads] with dense rows")
    return 0 if shape[0] == 1 else 4 * lse.stride(0)


def _sizes(name: str, shape: torch.Size, slots: int, query_starts: torch.Tensor | None, scale: float | None, window: int,
           max_query: int | None, max_context: int | None) -> tuple[float, int, int, int]:
    scale = 1.0 / math.sqrt(shape[2]) if scale is None else float(scale)
    if not 0.0 < scale < 3e38:
        raise ValueError(f"{name}: scale must be positive and finite")
    if query_starts is None:
        max_query = 1
    else:
        max_query = shape[0] if max_query is None else check_size(name, "max_query", max_query)
    max_context = slots if max_context is None else min(slots, check_size(name, "max_context", max_context))
    if window < 0:
        raise ValueError(f"{name}: window must not be negative")
    return scale, min(int(window), 2**31 - 1), max_query, max_context


def paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    query_starts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    max_query: int | None = None,
    max_context: int | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    stream: Any = None,
) -> torch.Tensor:
    """Attention outputs [T, Hq, D] (the query's type, or ``out``'s); ``lse`` float32 [T, Hq] receives the log-sums.

    Rows of tokens that belong to no sequence (padding outside ``query_starts``) are not written: ``out`` and ``lse`` keep
    what they held there, and without ``out`` those rows are uninitialised.  The softmax weights are rounded to the
    cache's type for the product with the values, also for a float32 ``out``.
    """
    name = "paged_attention"
    shape, strides, heads, sequences, slots, cache = _check(name, query, key_cache, value_cache, block_table, context_lens,
                                                            query_starts)
    scale, window, max_query, max_context = _sizes(name, shape, slots, query_starts, scale, window, max_query, max_context)
    tokens, query_heads, head_dim = shape
    if out is None:
        out = like_for(stream, query)
    out_shape, out_code, *out_strides = head_rows(name, "out", out)
    if out_shape != shape:
        raise ValueError(f"{name}: out must have the query's shape")
    lse_stride = 0 if lse is None else _lse_stride(name, shape, lse)
    require_one_gpu(name, query, key_cache, value_cache, block_table, context_lens, query_starts, out, lse)
    if tokens == 0 or sequences == 0:
        return out
    size = (_lib._lib or _lib.load()).qxt_paged_attention_workspace(query_heads, heads, head_dim, sequences, tokens,
                                                                    max_query, max_context)
    workspace = workspace_for(stream, size, query.device)
    _lib.call(
        "qxt_paged_attention", query.data_ptr(), *strides, cache, ptr(query_starts), out.data_ptr(), *out_strides, out_code,
        ptr(lse), lse_stride, tokens, query_heads, scale, 1 if causal else 0, window, max_query, max_context,
        ptr(workspace), size, stream_handle(stream),
    )
    return out


def paged_attention_scores(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    lse: torch.Tensor,
    query_starts: torch.Tensor | None = None,
    *,
    scores: torch.Tensor | None = None,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    max_query: int | None = None,
    max_context: int | None = None,
    out: torch.Tensor | None = None,
    stream: Any = None,
) -> torch.Tensor:
    """Weight that each slot received, float32 [B, Hkv, W * page_size], on top of ``scores`` (None: zeros).

    ``lse`` are the log-sums that ``paged_attention`` wrote for the same queries, cache and masks; a row's weights then
    add up to 1.  ``out`` may be ``scores`` itself.  A row with a NaN log-sum makes the slots that it sees NaN.  Every slot
    of the table's width is read and written.
    """
    name = "paged_attention_scores"
    shape, strides, heads, sequences, slots, cache = _check(name, query, key_cache, None, block_table, context_lens,
                                                            query_starts)
    scale, window, max_query, max_context = _sizes(name, shape, slots, query_starts, scale, window, max_query, max_context)
    tokens, query_heads, _ = shape
    lse_stride = _lse_stride(name, shape, lse)
    scores_shape = (sequences, heads, slots)
    before = (0, 0) if scores is None else per_slot(name, "scores", scores, torch.float32, scores_shape)
    if out is None:
        out = empty_for(stream, scores_shape, torch.float32, query.device) if scores is None else like_for(stream, scores)
    after = per_slot(name, "out", out, torch.float32, scores_shape)
    require_one_gpu(name, query, key_cache, block_table, context_lens, lse, query_starts, scores, out)
    if sequences == 0:
        return out
    size = (_lib._lib or _lib.load()).qxt_paged_attention_scores_workspace(query_heads, heads, sequences, tokens, slots,
                                                                           max_query, max_context)
    workspace = workspace_for(stream, size, query.device)
    _lib.call(
        "qxt_paged_attention_scores", query.data_ptr(), *strides, cache, ptr(query_starts), lse.data_ptr(), lse_stride,
        ptr(scores), *before, out.data_ptr(), *after, tokens, query_heads, scale, 1 if causal else 0, window, max_query,
        max_context, ptr(workspace), size, stream_handle(stream),
    )
    return out


@dataclass(frozen=True, slots=True)
class PagedAttentionOptions:
    """Last argument of the ``Kernel`` objects here; the keywords of the functions."""

    scale: float | None = None
    causal: bool = True
    window: int = 0
    max_query: int | None = None
    max_context: int | None = None


def paged_attention_grid(query: torch.Tensor) -> tuple[int, int, int]:
    """Grid of the ``Kernel`` objects here: (query heads, tokens, 1)."""
    return (query.shape[1], query.shape[0], 1)


def _execute_paged_attention(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    tensors = args[:5] + args[6:7]
    if (len(args) != 9 or not all(isinstance(a, torch.Tensor) for a in tensors)
            or not all(a is None or isinstance(a, torch.Tensor) for a in (args[5], args[7]))
            or not isinstance(args[8], PagedAttentionOptions)):
        raise KernelError("paged attention expects (query, key_cache, value_cache, block_table, context_lens, "
                          "query_starts or None, out, lse or None, PagedAttentionOptions)")
    if args[0].dim() != 3 or tuple(grid) != paged_attention_grid(args[0]):
        raise KernelError(f"paged attention grid must be (query heads, tokens, 1), got {tuple(grid)}")
    o = args[8]
    paged_attention(*args[:6], scale=o.scale, causal=o.causal, window=o.window, max_query=o.max_query,
                    max_context=o.max_context, out=args[6], lse=args[7], stream=stream)


PAGED_ATTENTION_KERNEL = Kernel("gfx950.paged_attention", _execute_paged_attention)


def _execute_paged_attention_scores(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    tensors = args[:5] + args[7:8]
    if (len(args) != 9 or not all(isinstance(a, torch.Tensor) for a in tensors)
            or not all(a is None or isinstance(a, torch.Tensor) for a in (args[5], args[6]))
            or not isinstance(args[8], PagedAttentionOptions)):
        raise KernelError("paged attention scores expects (query, key_cache, block_table, context_lens, lse, query_starts or "
                          "None, scores or None, out, PagedAttentionOptions)")
    if args[0].dim() != 3 or tuple(grid) != paged_attention_grid(args[0]):
        raise KernelError(f"paged attention scores grid must be (query heads, tokens, 1), got {tuple(grid)}")
    o = args[8]
    paged_attention_scores(*args[:6], scores=args[6], scale=o.scale, causal=o.causal, window=o.window,
                           max_query=o.max_query, max_context=o.max_context, out=args[7], stream=stream)


PAGED_ATTENTION_SCORES_KERNEL = Kernel("gfx950.paged_attention_scores", _execute_paged_attention_scores)

__all__ = [
    "PAGED_ATTENTION_KERNEL",
    "PAGED_ATTENTION_SCORES_KERNEL",
    "PagedAttentionOptions",
    "paged_attention",
    "paged_attention_grid",
    "paged_attention_scores",
]
