"""Eviction from a paged cache against its definition: every value is moved or chosen, so results are equal."""

from __future__ import annotations

import math

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import PAGED_CACHE_EVICT_KERNEL, PagedEvictionOptions, paged_cache_evict, paged_cache_evict_grid

pytestmark = pytest.mark.gpu


def _problem(lens, heads, dim, page_size, *, seed=0, width=None, dtype=torch.bfloat16, ties=True):
    gen = torch.Generator().manual_seed(seed)
    each = [-(-c // page_size) for c in lens]
    width = max(1, max(each)) if width is None else width
    pool = torch.randperm(sum(each) + 2, generator=gen).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(each):
        table[b, :count] = pool[at:at + count]
        at += count
    shape = (sum(each) + 2, page_size, heads, dim)
    keys, values = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
    slots = width * page_size
    scores = -torch.log(torch.rand((len(lens), heads, slots), generator=gen))
    if ties:
        scores = (scores * 4).floor() / 4  # many equal scores
    positions = torch.stack([torch.randperm(max(slots, 1), generator=gen) for _ in range(len(lens) * heads)])
    return keys, values, table, torch.tensor(lens, dtype=torch.int32), scores, positions.view(len(lens), heads, slots).int()


def _check(problem, budget, recent, **options):
    keys, values, table, lens, scores, positions = problem
    want = reference.evict(*problem, budget, recent)
    device = [t.cuda() for t in problem]
    got = paged_cache_evict(*device, budget=budget, recent=recent, **options)
    for mine, theirs in zip((*got, device[0], device[1]), want):
        mine = mine.cpu()
        if mine.dtype.is_floating_point:  # NaN scores move as they are
            assert torch.equal(torch.isnan(mine), torch.isnan(theirs))
            mine, theirs = mine.nan_to_num(-5.0), theirs.nan_to_num(-5.0)
        assert torch.equal(mine, theirs)
    assert torch.equal(device[4].cpu().nan_to_num(-5.0), scores.nan_to_num(-5.0)) and torch.equal(device[5].cpu(), positions)


@pytest.mark.parametrize("lens,budget,recent", [
    ([65], 64, 8), ([300, 64, 20, 0, 1], 64, 64), ([257, 130, 129], 128, 0), ([1000], 1, 0), ([1000], 1, 1), ([2], 1, 1),
    ([1000, 999, 513], 512, 100), ([100, 90], 99, 10), ([100], 200, 10), ([4097, 5000], 4096, 512),
    ([68, 67, 66], 64, 62), ([5, 4, 3], 2, 1), ([132, 131, 130, 129], 128, 3),  # a few over: one launch, slot by slot
])
@pytest.mark.parametrize("ties", [False, True])
def test_against_the_definition(lens, budget, recent, ties) -> None:
    for heads, dim, page_size, dtype in ((2, 64, 16, torch.bfloat16), (3, 72, 7, torch.float16)):
        _check(_problem(lens, heads, dim, page_size, seed=budget, dtype=dtype, ties=ties), budget, recent)


@pytest.mark.parametrize("scores", ["zero", "equal", "special", "negative", "denormal"])
def test_scores_of_every_kind(scores) -> None:
    problem = list(_problem([400, 129], 2, 64, 16, seed=3, ties=False))
    gen = torch.Generator().manual_seed(4)
    if scores == "zero":
        problem[4] = torch.where(torch.rand(problem[4].shape, generator=gen) < 0.5, 0.0, -0.0)
    elif scores == "equal":
        problem[4] = torch.full_like(problem[4], 0.7)
    elif scores == "special":
        choice = torch.randint(0, 5, problem[4].shape, generator=gen)
        problem[4] = torch.tensor([math.nan, math.inf, -math.inf, 1.0, -1.0])[choice]
    elif scores == "negative":
        problem[4] = torch.randn(problem[4].shape, generator=gen)
    else:
        problem[4] = problem[4] * 1e-40
    for budget, recent in ((128, 16), (100, 0), (7, 7)):
        _check(tuple(problem), budget, recent)


def test_more_keys_than_lds_holds_and_positions_that_repeat() -> None:
    problem = list(_problem([40000, 33000, 700], 1, 8, 128, seed=5))
    _check(tuple(problem), 3000, 1000)
    problem = list(_problem([9000, 500], 2, 8, 64, seed=6))
    problem[5] = problem[5] // 7 - 3  # more recent slots than the budget would hold otherwise
    _check(tuple(problem), 64, 32)
    problem[5][:] = -(2**31)
    _check(tuple(problem), 64, 32)


def test_hints_lengths_past_the_table_and_pages_that_are_not_there() -> None:
    _check(_problem([5000, 300], 2, 64, 16, seed=7), 256, 32, max_context=10)   # one launch moves them all
    _check(_problem([300], 2, 64, 16, seed=7), 256, 32, max_context=10**6)
    problem = list(_problem([200, 150], 2, 64, 16, seed=8))
    problem[3] = torch.tensor([10**6, -5], dtype=torch.int32)
    problem[2][0, 1], problem[2][0, 9] = -1, 10**6
    _check(tuple(problem), 100, 20)


def test_in_place_strided_and_repeated() -> None:
    problem = _problem([700, 650], 4, 128, 16, seed=9)
    want = reference.evict(*problem, 512, 64)
    keys, values, table, lens, scores, positions = (t.cuda() for t in problem)
    joint = torch.stack([keys, values], dim=1).transpose(2, 3).contiguous().transpose(2, 3)  # heads first, joint
    keys, values = joint[:, 0], joint[:, 1]
    slots = scores.shape[2]
    wide = torch.zeros((4, 2, slots + 3), device="cuda")
    view = wide[..., :slots].transpose(0, 1)
    view.copy_(scores)
    new_lens, s, p = paged_cache_evict(keys, values, table, lens, view, positions, budget=512, recent=64, scores_out=view,
                                       positions_out=positions)
    assert s is view and p is positions
    for mine, theirs in zip((new_lens, s, p, keys, values), want):
        assert torch.equal(mine.cpu(), theirs)
    assert bool((wide[..., slots:] == 0).all())
    # Nothing is over the budget any more: a second call changes nothing.
    again = paged_cache_evict(keys, values, table, new_lens, s, p, budget=512, recent=64)
    for mine, theirs in zip((*again, keys, values), want):
        assert torch.equal(mine.cpu(), theirs)


def test_queue_submission() -> None:
    problem = _problem([100, 300], 2, 64, 16, seed=10)
    want = reference.evict(*problem, 90, 9)
    device = [t.cuda() for t in problem]
    lens_out = torch.empty_like(device[3])
    with Queue() as queue:
        queue.submit(PAGED_CACHE_EVICT_KERNEL, (*device, lens_out, device[4], device[5], PagedEvictionOptions(90, 9)),
                     grid=paged_cache_evict_grid(device[4])).wait()
    for mine, theirs in zip((lens_out, device[4], device[5], device[0], device[1]), want):
        assert torch.equal(mine.cpu(), theirs)
