"""Eviction from a paged cache by accumulated attention weight, on gfx950.

``paged_cache_evict`` cuts every sequence of more than ``budget`` slots down to ``budget``, each head by itself.  It
keeps the slots that come first by (recent, score, lower slot): recent are those whose position is above the head's
newest minus ``recent``, scores are what ``paged_attention_scores`` added up (a NaN is the least).  Kept slots below
``budget`` stay; the i-th slot below it that is given up takes the key row, value row, score and position of the i-th
kept slot at or above it, so rows move in place and only those that must.  Slots are then in no order of age:
``positions`` (int32 [B, Hkv, W * page_size]) travel with them, and attention over an evicted cache needs none, its
keys being rotated already (a sliding window would, and is not meaningful there).  Freed slots get score 0 and
position -1, ready for new tokens.  No page may belong to two sequences.

The reference has no counterpart (its cache is one contiguous buffer that only grows).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import check_index, check_size, like_for, paged_cache, per_slot, require_one_gpu, workspace_for
from qpu_xla_amd._tensors import stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel


def paged_cache_evict(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    scores: torch.Tensor,
    positions: torch.Tensor,
    *,
    budget: int,
    recent: int = 0,
    max_context: int | None = None,
    scores_out: torch.Tensor | None = None,
    positions_out: torch.Tensor | None = None,
    lens_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Evict in the cache; returns (new lengths int32 [B], scores, positions), new tensors unless outputs are given.

    ``scores_out`` and ``positions_out`` may be the inputs themselves, and share no memory with them otherwise, nor row
    with row; ``lens_out`` lies apart from ``context_lens``.
    ``max_context`` is the host's bound of the lengths and sizes the launch.
    """
    name = "paged_cache_evict"
    cache_shape, _, sequences, width, cache = paged_cache(name, key_cache, value_cache, block_table, context_lens)
    _, page_size, heads, head_dim = cache_shape
    if head_dim % 8 or head_dim > 256:
        raise ValueError(f"{name}: head size must be a multiple of 8 up to 256")
    budget, recent = int(budget), int(recent)
    if not 0 < budget < 2**30 or not 0 <= recent <= budget:
        raise ValueError(f"{name}: budget must be positive (below 2^30) and recent between 0 and the budget")
    slots = width * page_size
    max_context = slots if max_context is None else min(slots, check_size(name, "max_context", max_context))
    shape = (sequences, heads, slots)
    if scores_out is None:
        scores_out = like_for(stream, scores)
    if positions_out is None:
        positions_out = like_for(stream, positions)
    if lens_out is None:
        lens_out = like_for(stream, context_lens)
    else:
        check_index(name, "lens_out", lens_out, torch.int32, sequences)
    strides = [per_slot(name, what, t, dtype, shape)
               for what, t, dtype in (("scores", scores, torch.float32), ("scores_out", scores_out, torch.float32),
                                      ("positions", positions, torch.int32), ("positions_out", positions_out, torch.int32))]
    require_one_gpu(name, key_cache, value_cache, block_table, context_lens, scores, positions, scores_out, positions_out,
                    lens_out)
    if sequences == 0:
        return lens_out, scores_out, positions_out
    size = (_lib._lib or _lib.load()).qxt_paged_cache_evict_workspace(heads, sequences, slots, budget)
    workspace = workspace_for(stream, size, key_cache.device)
    _lib.call(
        "qxt_paged_cache_evict", cache, scores.data_ptr(), *strides[0], scores_out.data_ptr(), *strides[1],
        positions.data_ptr(), *strides[2], positions_out.data_ptr(), *strides[3], lens_out.data_ptr(), budget, recent,
        max_context, workspace.data_ptr(), size, stream_handle(stream),
    )
    return lens_out, scores_out, positions_out


@dataclass(frozen=True, slots=True)
class PagedEvictionOptions:
    """Last argument of ``PAGED_CACHE_EVICT_KERNEL``; the keywords of ``paged_cache_evict``."""

    budget: int
    recent: int = 0
    max_context: int | None = None


def paged_cache_evict_grid(scores: torch.Tensor) -> tuple[int, int, int]:
    """Grid of ``PAGED_CACHE_EVICT_KERNEL``: (heads, sequences, 1)."""
    return (scores.shape[1], scores.shape[0], 1)


def _execute_paged_cache_evict(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    if (len(args) != 10 or not all(isinstance(a, torch.Tensor) for a in args[:9])
            or not isinstance(args[9], PagedEvictionOptions)):
        raise KernelError("paged cache eviction expects (key_cache, value_cache, block_table, context_lens, scores, positions, "
                          "lens_out, scores_out, positions_out, PagedEvictionOptions)")
    if args[4].dim() != 3 or tuple(grid) != paged_cache_evict_grid(args[4]):
        raise KernelError(f"paged cache eviction grid must be (heads, sequences, 1), got {tuple(grid)}")
    o = args[9]
    paged_cache_evict(*args[:6], budget=o.budget, recent=o.recent, max_context=o.max_context, lens_out=args[6],
                      scores_out=args[7], positions_out=args[8], stream=stream)


PAGED_CACHE_EVICT_KERNEL = Kernel("gfx950.paged_cache_evict", _execute_paged_cache_evict)

__all__ = ["PAGED_CACHE_EVICT_KERNEL", "PagedEvictionOptions", "paged_cache_evict", "paged_cache_evict_grid"]
