"""Windows at the ends of their range, beside more new tokens than slots.  Tolerances as in ``test_gpu_paged_attention``."""

from __future__ import annotations

import pytest
import torch

from qpu_xla_amd.kernels import paged_attention, paged_attention_scores
from test_gpu_paged_attention import Problem, _scores_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [1, 2**30 - 1, 2**30, 2**31 - 1, 2**40])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[(5, 40), (3, 3), (60, 2)], [(20, 200)], [(400, 9)]])
def test_any_window_over_any_length(lens, causal, window) -> None:
    problem = Problem(lens, 4, 2, 64, 16, torch.bfloat16, seed=len(lens))
    out, lse = problem.run(causal=causal, window=window)
    problem.check(out, lse, causal=causal, window=window)
    query, keys, _, table, context, starts = problem.device()
    got = paged_attention_scores(query, keys, table, context, lse, starts, scale=problem.scale, causal=causal, window=window)
    assert _scores_close(problem, got, lse, causal=causal, window=window)


def test_window_at_the_end_of_a_context_of_many_slots() -> None:
    # Slots times heads of a group pass 2^31 here; what lies before the window gets nothing, and no time.
    context, window, heads, page_size = 2**25 + 4096 + 5, 100, 64, 64
    tail = 128 + 5  # the last slots, from a page's first on: a problem of their own
    problem = Problem([(tail, 1)], heads, 1, 64, page_size, torch.bfloat16, seed=1, starts=False)
    query, keys, values, table, _, _ = problem.device()
    pages = -(-context // page_size)
    whole = table[:, :1].expand(1, pages).clone()
    whole[:, -3:] = table
    context_lens = torch.tensor([context], device="cuda", dtype=torch.int32)
    lse = torch.empty(query.shape[:2], device="cuda")
    out = paged_attention(query, keys, values, whole, context_lens, scale=problem.scale, window=window, lse=lse)
    problem.check(out, lse, window=window)
    got = paged_attention_scores(query, keys, whole, context_lens, lse, scale=problem.scale, window=window)
    last = got[..., context - tail:context]
    assert _scores_close(problem, torch.cat([last, got[..., context:]], dim=2), lse, window=window)
    assert bool((got[..., :context - window] == 0).all())
