"""Attention whose chunks are longer than ``max_query`` says: a workgroup then goes on from one row tile to the next.

With a window the tiles of a split differ in where its slots end, upwards too, and what a wave holds of the block table
for one tile must not serve another.  Tolerances are ``Problem.check``'s.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu

# (context, new tokens, query heads, key heads, head size, page size, window, causal, max_query, max_context): more than
# 128 rows by the hint, split slots, and a later tile of a split that ends above an earlier one.
CASES = [
    (6000, 9, 32, 1, 64, 64, 4096, True, 8, 8192),
    (1184, 130, 2, 1, 64, 8, 213, True, 70, 1184),
    (1245, 60, 5, 1, 128, 16, 979, True, 51, 1245),
    (2355, 67, 8, 2, 64, 24, 1704, True, 40, 2355),
    (1711, 271, 2, 2, 128, 64, 1514, True, 241, 1711),
    (803, 65, 4, 1, 64, 7, 721, False, 37, 803),          # pages that hold no whole units of eight
    (941, 71, 5, 1, 80, 24, 727, False, 41, 941),         # a padded head size
    (5496, 358, 10, 2, 64, 16, 3859, False, 81, 5496),    # four tiles a workgroup
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_windowed_chunks_longer_than_the_hint(case, dtype) -> None:
    context, new, heads, kv_heads, dim, page_size, window, causal, max_query, max_context = CASES[case]
    problem = Problem([(context, new)], heads, kv_heads, dim, page_size, dtype, seed=case)
    out, lse = problem.run(causal=causal, window=window, max_query=max_query, max_context=max_context)
    problem.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("causal", [True, False])
def test_chunks_longer_than_the_hint_without_a_window(causal) -> None:
    problem = Problem([(1500, 300), (700, 1)], 8, 2, 128, 16, torch.bfloat16, seed=31)
    out, lse = problem.run(causal=causal, max_query=40, max_context=1500)
    problem.check(out, lse, causal=causal)
