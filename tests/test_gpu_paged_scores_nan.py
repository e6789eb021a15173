"""Slot weights beside rows whose log-sum is NaN: only the slots that such a row sees become NaN.

``paged_attention`` writes a NaN log-sum for a row whose query, or a key that it sees, is NaN.  Tolerance: a weight errs by
its logit's error, 2^-18 of the difference and the exponential, and the sum's (rows / 16 + 8) 2^-24, all relative.
"""

from __future__ import annotations

import math

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd.kernels import paged_attention_scores
from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu

# ((context, new tokens), heads, key heads, head size, page size, window, max_query)
CASES = [
    ((130, 4), 8, 2, 128, 16, 20, 4),        # 16 rows a key head
    ((700, 1), 32, 1, 64, 16, 50, 1),        # one token
    ((130, 20), 8, 2, 64, 16, 20, 4),        # 80 rows, in rounds of 32
    ((200, 6), 4, 1, 256, 24, 33, 6),
    ((300, 100), 8, 2, 128, 16, 17, 100),    # 400 rows
    ((333, 60), 4, 1, 80, 7, 0, 60),         # no window: later slots stay unseen
    ((900, 400), 8, 1, 64, 64, 70, 400),     # 3200 rows, split
    ((260, 90), 4, 2, 256, 16, 40, 90),
]


def _check(problem, got, lse, **masks) -> torch.Tensor:
    want = reference.scores(problem.query, problem.keys, problem.table, problem.lens, lse.cpu(), problem.starts, previous=None,
                            scale=problem.scale, **masks)
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rows = problem.query.shape[0] * problem.query.shape[1] / problem.keys.shape[2]
    clean = problem.query.double().nan_to_num(0.0).norm(dim=-1).max() * problem.keys.double().nan_to_num(0.0).norm(dim=-1).max()
    logit = (problem.query.shape[2] + 2) * 2.0**-24 * problem.scale * float(clean)
    off = (got - want).abs() - (logit + 2.0**-18 + (rows / 16 + 8) * 2.0**-24) * want.abs() - 1e-30
    off = off[~torch.isnan(want)]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
    return torch.isnan(want)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_a_nan_query_reaches_only_the_slots_that_it_sees(case, dtype, causal) -> None:
    lens, heads, kv_heads, dim, page_size, window, max_query = CASES[case]
    problem = Problem([lens], heads, kv_heads, dim, page_size, dtype, seed=case)
    token = lens[1] // 2
    problem.query[token, 0] = math.nan  # of key head 0 alone
    masks = {"causal": causal, "window": window}
    _, lse = problem.run(**masks, max_query=max_query)
    assert int(torch.isnan(lse).sum()) == 1
    query, keys, _, table, context, starts = problem.device()
    got = paged_attention_scores(query, keys, table, context, lse, starts, scale=problem.scale, max_query=max_query, **masks)
    nan = _check(problem, got, lse, **masks)
    low, high = reference.visible(*lens, token, causal, window)
    assert int(nan[0, 0].sum()) == high - low and not bool(nan[0, 1:].any())


@pytest.mark.parametrize("case", [0, 2, 4, 6])
def test_a_nan_key_reaches_the_slots_of_the_rows_that_see_it(case) -> None:
    lens, heads, kv_heads, dim, page_size, window, max_query = CASES[case]
    problem = Problem([lens], heads, kv_heads, dim, page_size, torch.bfloat16, seed=case)
    slot = lens[0] - 2  # seen by the last two tokens
    problem.keys[problem.table[0, slot // page_size], slot % page_size, 0, 3] = math.nan
    masks = {"causal": True, "window": window}
    _, lse = problem.run(**masks, max_query=max_query)
    query, keys, _, table, context, starts = problem.device()
    got = paged_attention_scores(query, keys, table, context, lse, starts, scale=problem.scale, max_query=max_query, **masks)
    nan = _check(problem, got, lse, **masks)
    assert bool(nan[0, 0].any()) and not bool(nan[0, 0].all())
