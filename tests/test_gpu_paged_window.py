"""Windows at the ends of their range, beside more new tokens than slots.  Tolerances as in ``test_gpu_paged_attention``."""

from __future__ import annotations

import pytest
import torch

from qpu_xla_amd.kernels import paged_attention_scores
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
