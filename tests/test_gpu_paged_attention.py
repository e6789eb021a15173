"""Attention over a paged cache and the slots' weights, against the 64-bit definition.

Tolerances.  u = 2^-8 (bfloat16) or 2^-11 (float16) is a half unit of the cache's type, e the same of the output's.  The
products of a logit are exact in fp32 and their sum errs by at most (D + 2) 2^-24 scale |q||k| =: d, so weights err
by 2 d relative (numerator and sum).  Weights are rounded to the cache's type for the product with the values: u of
sum p|v|; below float16's normal range 2^-25 absolute, of a largest weight of at least 1: 2^-25 sum |v|.  Sums over L
slots in fp32, a lane adding L / 64 of them: (L / 64 + 32) 2^-24.  Outputs round once more: e |o|.
"""

from __future__ import annotations

import math

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import (
    PAGED_ATTENTION_KERNEL,
    PAGED_ATTENTION_SCORES_KERNEL,
    PagedAttentionOptions,
    paged_attention,
    paged_attention_grid,
    paged_attention_scores,
)

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


class Problem:
    """Random queries and cache for sequences of (context, new tokens); CPU copies and device tensors."""

    def __init__(self, lens, heads, kv_heads, dim, page_size, dtype, *, seed=0, sharp=2.0, starts=True, spare=2):
        gen = torch.Generator().manual_seed(seed)
        self.lens_list = lens
        tokens = sum(n for _, n in lens)
        width = max(1, max(-(-c // page_size) for c, _ in lens))
        each = [-(-c // page_size) for c, _ in lens]
        pool = torch.randperm(sum(each) + spare, generator=gen).to(torch.int32)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, count in enumerate(each):
            self.table[b, :count] = pool[at:at + count]
            at += count
        self.query = (torch.randn((tokens, heads, dim), generator=gen) * sharp).to(dtype)
        shape = (sum(each) + spare, page_size, kv_heads, dim)
        self.keys, self.values = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
        self.lens = torch.tensor([c for c, _ in lens], dtype=torch.int32)
        self.starts = torch.tensor([0] + [n for _, n in lens]).cumsum(0).to(torch.int32) if starts else None
        self.dtype, self.scale = dtype, 1.0 / math.sqrt(dim)

    def unused_slots(self):
        """Mask [pages, page_size] of slots that no sequence has in use."""
        free = torch.ones(self.keys.shape[:2], dtype=torch.bool)
        for b, (context, _) in enumerate(self.lens_list):
            for j in range(context):
                free[self.table[b, j // free.shape[1]], j % free.shape[1]] = False
        return free

    def device(self):
        starts = None if self.starts is None else self.starts.cuda()
        return self.query.cuda(), self.keys.cuda(), self.values.cuda(), self.table.cuda(), self.lens.cuda(), starts

    def logit_error(self):
        norms = self.query.double().nan_to_num(0, 0, 0).norm(dim=-1).max() * self.keys.double().nan_to_num(0, 0, 0).norm(dim=-1).max()
        return float((self.query.shape[2] + 2) * 2.0**-24 * self.scale * norms)

    def check(self, out, lse=None, *, causal=True, window=0, rows=slice(None)):
        want, want_lse, bound = reference.attention(self.query, self.keys, self.values, self.table, self.lens, self.starts,
                                                    scale=self.scale, causal=causal, window=window)
        longest = max(c for c, _ in self.lens_list)
        d, sums = self.logit_error(), (longest / 64 + 32) * 2.0**-24
        tolerance = (UNIT[self.dtype] + 2 * d + 2 * sums) * bound + UNIT[out.dtype] * want.abs() + 1e-30
        if self.dtype == torch.float16:
            tolerance += 2.0**-25 * longest * float(self.values.double().nan_to_num(0, 0, 0).abs().max())
        if out.dtype == torch.float16:
            tolerance += 2.0**-25
        got = out.cpu().double()[rows]
        want, bound, tolerance = want[rows], bound[rows], tolerance[rows]
        finite = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), finite)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        off = (got - want)[finite].abs() - tolerance[finite]
        assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
        if lse is not None:
            got_lse, want_lse = lse.cpu().double()[rows], want_lse[rows]
            empty = want_lse == -math.inf
            assert torch.equal(got_lse == -math.inf, empty)
            assert torch.equal(torch.isnan(got_lse), torch.isnan(want_lse))
            fine = torch.isfinite(want_lse)
            off = (got_lse - want_lse)[fine].abs() - (d + sums + 2.0**-21 * (1 + want_lse[fine].abs()))
            assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())

    def run(self, **options):
        lse = torch.full(self.query.shape[:2], 7.0, device="cuda")
        out = paged_attention(*self.device(), scale=self.scale, lse=lse, **options)
        return out, lse


# (sequences as (context, new), heads, key heads, head size, page size)
LAYOUTS = [
    ([(1, 1)], 4, 4, 64, 16),
    ([(37, 1), (1, 1), (64, 1), (65, 1), (500, 1)], 32, 4, 64, 16),              # one token a sequence
    ([(513, 1), (31, 1)], 8, 2, 128, 1),                                        # pages of one slot
    ([(300, 3), (7, 7), (40, 0), (129, 2), (0, 0)], 8, 2, 128, 24),             # short chunks, one empty sequence
    ([(77, 9)], 7, 1, 80, 7),                                                   # 63 rows, odd group, padded head size
    ([(200, 30), (30, 30)], 8, 2, 64, 32),                                      # 120 rows
    ([(333, 100), (100, 100), (64, 1)], 12, 4, 128, 64),                        # 300 rows, ragged
    ([(260, 130)], 2, 2, 256, 64),                                              # wide heads
    ([(150, 20), (90, 9)], 4, 2, 192, 16),
    ([(64, 3)], 3, 1, 8, 5),
    ([(90, 70)], 24, 1, 128, 128),                                              # one key head for all
    ([(5, 9), (3, 3)], 4, 2, 64, 4),                                            # more new tokens than slots: rows that see nothing
]


@pytest.mark.parametrize("mask", [(True, 0), (False, 0), (True, 17), (False, 50)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_against_the_definition(layout, dtype, mask) -> None:
    lens, heads, kv_heads, dim, page_size = LAYOUTS[layout]
    problem = Problem(lens, heads, kv_heads, dim, page_size, dtype, seed=layout)
    out, lse = problem.run(causal=mask[0], window=mask[1])
    assert out.dtype == dtype
    problem.check(out, lse, causal=mask[0], window=mask[1])


@pytest.mark.parametrize("case", [
    ([(5000, 1)], 4, 1, 128, 64, 1),         # split over workgroups, joined
    ([(4000, 1), (3, 1), (0, 1)], 8, 8, 64, 16, 1),
    ([(3000, 40)], 4, 2, 128, 48, 40),
    ([(2500, 200)], 2, 1, 256, 32, 200),
    ([(2222, 150), (1, 1)], 3, 1, 96, 16, 150),
])
@pytest.mark.parametrize("window", [0, 700])
def test_long_contexts_are_split_and_joined(case, window) -> None:
    lens, heads, kv_heads, dim, page_size, most = case
    problem = Problem(lens, heads, kv_heads, dim, page_size, torch.bfloat16, seed=heads)
    out, lse = problem.run(window=window, max_query=most)
    problem.check(out, lse, window=window)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_outputs_of_other_types_and_strides(out_dtype) -> None:
    for lens in ([(600, 1)] * 3, [(70, 40), (50, 50)], [(4000, 2)]):
        problem = Problem(lens, 8, 2, 64, 16, torch.bfloat16, seed=4)
        tokens = problem.query.shape[0]
        out = torch.full((8, tokens, 72), 5.0, device="cuda", dtype=out_dtype)
        view = out[..., :64].transpose(0, 1)
        lse = torch.full((tokens, 11), 5.0, device="cuda")
        query, keys, values, table, lens_t, starts = problem.device()
        wide = torch.zeros((tokens, 10, 64), device="cuda", dtype=torch.bfloat16)  # queries inside a wider projection
        wide[:, 1:9] = query
        assert paged_attention(wide[:, 1:9], keys, values, table, lens_t, starts, out=view, lse=lse[:, 2:10]) is view
        problem.check(view, lse[:, 2:10])
        assert bool((out[..., 64:] == 5).all()) and bool((lse[:, :2] == 5).all()) and bool((lse[:, 10:] == 5).all())


@pytest.mark.parametrize("order", ["heads_first", "joint", "wide_rows"])
def test_caches_in_other_orders(order) -> None:
    problem = Problem([(200, 1), (77, 5)], 8, 4, 64, 16, torch.float16, seed=6)
    query, keys, values, table, lens, starts = problem.device()
    if order == "heads_first":
        keys, values = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (keys, values))
    elif order == "joint":
        joint = torch.stack([keys, values], dim=1)
        keys, values = joint[:, 0], joint[:, 1]
    else:
        keys, values = (torch.cat([c, torch.full_like(c, math.nan)], dim=3)[..., :64] for c in (keys, values))
    table = torch.cat([table, table], dim=1)[:, : table.shape[1]]  # rows with a stride
    problem.check(paged_attention(query, keys, values, table, lens, starts, scale=problem.scale))


@pytest.mark.parametrize("lens", [[(130, 1), (33, 1), (1, 1)], [(100, 40), (64, 64)], [(300, 290)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_unused_slots_hold_does_not_matter(lens, dtype) -> None:
    problem = Problem(lens, 8, 2, 128, 16, dtype, seed=7)
    clean = problem.run()
    free = problem.unused_slots()
    problem.keys[free] = math.nan
    problem.values[free] = math.inf
    dirty = problem.run()
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("case", [
    ([(90, 40)], 8, 2, 128, 16, 0),     # 160 rows
    ([(50, 12), (9, 9)], 4, 2, 64, 16, 5),   # 24 rows: key parts are joined
    ([(66, 30)], 2, 1, 256, 16, 0),     # 60 rows, wide
    ([(3000, 10)], 4, 1, 128, 16, 0),   # split
    ([(75, 25)], 4, 1, 128, 16, 30),    # 100 rows with a window
    ([(90, 20)], 32, 1, 128, 16, 0),    # 640 rows: a wave's rows are one token's, the workgroup's are not
    ([(90, 20)], 32, 1, 128, 16, 11),
    ([(90, 20)], 32, 1, 64, 12, 11),    # pages that hold no whole units
    ([(200, 8)], 32, 1, 64, 16, 50),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_and_nan_slots_reach_only_rows_that_see_them(case, dtype) -> None:
    lens, heads, kv_heads, dim, page_size, window = case
    problem = Problem(lens, heads, kv_heads, dim, page_size, dtype, seed=8)
    context, new = lens[0]

    def put(cache, slot, head, value, element=slice(None)):
        cache[problem.table[0, slot // page_size], slot % page_size, head, element] = value

    put(problem.values, context - 4, 0, math.nan)                 # seen by the last four tokens
    put(problem.values, context - 6, 0, math.inf, 5)
    put(problem.values, context - 5, 0, -math.inf, 5)
    put(problem.keys, context - 2, 0, math.nan)
    out, lse = problem.run(window=window)
    problem.check(out, lse, window=window)
    before = problem.run(window=window)[0][: new - 6]
    assert bool(torch.isfinite(before).all())


def test_hints_that_are_too_small_and_lengths_past_the_table() -> None:
    problem = Problem([(900, 200), (40, 3)], 8, 2, 64, 16, torch.bfloat16, seed=9)
    out, lse = problem.run(max_query=3, max_context=10)
    problem.check(out, lse)
    # A length past the table's width counts as the width; table entries of no page are zero rows.
    query, keys, values, table, lens, starts = problem.device()
    problem.table[0, 3], problem.table[0, 5] = -1, 10**6
    problem.lens = torch.tensor([10**6, 40], dtype=torch.int32)
    out = paged_attention(query, keys, values, problem.table.cuda(), problem.lens.cuda(), starts, scale=problem.scale)
    problem.check(out)


def test_tokens_of_no_sequence_are_left_alone() -> None:
    for max_context in (64, 3000):
        problem = Problem([(2900, 5)], 4, 2, 64, 16, torch.bfloat16, seed=10)
        query, keys, values, table, lens, _ = problem.device()
        padded = torch.cat([query, query, query])
        out = torch.full_like(padded, 3.0)
        starts = torch.tensor([5, 10], device="cuda", dtype=torch.int32)
        paged_attention(padded, keys, values, table, lens, starts, scale=problem.scale, out=out, max_query=5,
                        max_context=max_context)
        problem.check(out[5:10])
        assert bool((out[:5] == 3).all()) and bool((out[10:] == 3).all())


def test_large_logits_and_growing_maxima() -> None:
    # Logits in the hundreds, the largest last: the running maximum moves at almost every step.
    problem = Problem([(700, 1), (300, 20)], 4, 2, 64, 16, torch.bfloat16, seed=11, sharp=60.0)
    problem.check(*problem.run())
    problem.keys *= torch.linspace(0.1, 2.0, problem.keys.shape[0])[:, None, None, None].to(torch.bfloat16)
    problem.check(*problem.run())


def test_offsets_past_32_bits() -> None:
    # Pages more than 2^32 bytes into the cache.
    pages, page_size, heads, dim = 34000, 64, 8, 128  # 4.45 GB each
    keys, values = (torch.empty((pages, page_size, heads, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    problem = Problem([(190, 4), (70, 1)], 16, 8, dim, page_size, torch.bfloat16, seed=12)
    places = torch.tensor([pages - 1, 5, pages - 3, 32768, 33000, 7, 9], dtype=torch.int32)[: problem.keys.shape[0]]
    keys[places.long().cuda()] = problem.keys.cuda()
    values[places.long().cuda()] = problem.values.cuda()
    table = torch.where(problem.table >= 0, places[problem.table.clamp(min=0).long()], -1).to(torch.int32)
    query, _, _, _, lens, starts = problem.device()
    lse = torch.empty(query.shape[:2], device="cuda")
    out = paged_attention(query, keys, values, table.cuda(), lens, starts, scale=problem.scale, lse=lse)
    problem.check(out, lse)
    got = paged_attention_scores(query, keys, table.cuda(), lens, lse, starts, scale=problem.scale)
    assert _scores_close(problem, got, lse)


def test_streams_queue_and_graph() -> None:
    problem = Problem([(3000, 1), (500, 1)], 8, 2, 128, 16, torch.bfloat16, seed=13)
    args = problem.device()[:5]
    want = paged_attention(*args, scale=problem.scale)
    problem.check(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = [paged_attention(*args, scale=problem.scale, stream=side) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(r, want) for r in results)
    with Queue() as queue:
        out, lse = torch.empty_like(want), torch.empty(want.shape[:2], device="cuda")
        options = PagedAttentionOptions(scale=problem.scale)
        grid = paged_attention_grid(args[0])
        queue.submit(PAGED_ATTENTION_KERNEL, (*args, None, out, lse, options), grid=grid)
        scores = torch.zeros((2, 2, args[3].shape[1] * 16), device="cuda")
        queue.submit(PAGED_ATTENTION_SCORES_KERNEL, (args[0], args[1], args[3], args[4], lse, None, scores, scores, options),
                     grid=grid).wait()
    assert torch.equal(out, want)
    assert _scores_close(problem, scores, lse)
    graph, replayed = torch.cuda.CUDAGraph(), torch.empty_like(want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged_attention(*args, scale=problem.scale, out=replayed)
    for step in range(3):
        args[0].copy_(problem.query.cuda() * (1 + step))
        eager = paged_attention(*args, scale=problem.scale)
        replayed.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)


# ------------------------------------------------------------------- scores


def _scores_close(problem, got, lse, previous=None, **masks):
    want = reference.scores(problem.query, problem.keys, problem.table, problem.lens, lse.cpu(), problem.starts,
                            previous=previous, scale=problem.scale, **masks)
    rows = problem.query.shape[0] * problem.query.shape[1] / problem.keys.shape[2]
    # A weight: its logit's error d, the difference and the exponential (|difference| under 64: 2^-18); the sum.
    relative = problem.logit_error() + 2.0**-18 + (rows / 16 + 8) * 2.0**-24
    off = (got.cpu().double() - want).abs() - relative * want.abs() - 1e-30
    return float(off.max()) <= 0


@pytest.mark.parametrize("mask", [(True, 0), (False, 0), (True, 17), (False, 50)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_scores_against_the_definition(layout, dtype, mask) -> None:
    lens, heads, kv_heads, dim, page_size = LAYOUTS[layout]
    problem = Problem(lens, heads, kv_heads, dim, page_size, dtype, seed=layout)
    masks = {"causal": mask[0], "window": mask[1]}
    _, lse = problem.run(**masks)
    query, keys, _, table, lens_t, starts = problem.device()
    got = paged_attention_scores(query, keys, table, lens_t, lse, starts, scale=problem.scale, **masks)
    assert _scores_close(problem, got, lse, **masks)
    # Every row's weights add up to 1.
    rows = (lse > -math.inf).view(lse.shape[0], kv_heads, -1).sum(dim=(0, 2))
    assert torch.allclose(got.sum(dim=(0, 2)), rows.float(), rtol=1e-3, atol=1e-6)


def test_scores_accumulate_in_place_over_strides_and_splits() -> None:
    problem = Problem([(1500, 600), (90, 1), (0, 0)], 8, 2, 128, 16, torch.bfloat16, seed=21)
    _, lse = problem.run(max_query=600)
    query, keys, _, table, lens, starts = problem.device()
    slots = table.shape[1] * 16
    gen = torch.Generator().manual_seed(1)
    previous = torch.rand((3, 2, slots), generator=gen)
    previous[1, 0, 90:] = math.nan  # past the sequence's length: kept as it is
    wide = torch.zeros((2, 3, slots + 5), device="cuda")
    view = wide[..., :slots].transpose(0, 1)
    view.copy_(previous)
    for max_query, max_context in ((600, 1500), (1, 1)):  # with and without splits, right hints and too small ones
        fresh = paged_attention_scores(query, keys, table, lens, lse, starts, scores=previous.cuda(), scale=problem.scale,
                                       max_query=max_query, max_context=max_context)
        assert torch.equal(torch.isnan(fresh).cpu(), torch.isnan(previous))
        assert torch.equal(fresh[2].cpu(), previous[2])
        assert _scores_close(problem, fresh.nan_to_num(0.0), lse, previous.nan_to_num(0.0))
    again = paged_attention_scores(query, keys, table, lens, lse, starts, scores=view, out=view, scale=problem.scale,
                                   max_query=600, max_context=1500)
    repeat = paged_attention_scores(query, keys, table, lens, lse, starts, scores=previous.cuda(), scale=problem.scale,
                                    max_query=600, max_context=1500)
    assert again is view and torch.equal(view.nan_to_num(0.0), repeat.nan_to_num(0.0))
    assert bool((wide[..., slots:] == 0).all())


def test_scores_ignore_unused_slots_and_empty_rows() -> None:
    problem = Problem([(130, 1), (100, 40)], 8, 2, 128, 16, torch.float16, seed=22)
    _, lse = problem.run()
    query, keys, _, table, lens, starts = problem.device()
    clean = paged_attention_scores(query, keys, table, lens, lse, starts, scale=problem.scale)
    free = problem.unused_slots().cuda()
    keys[free] = math.nan
    dirty = paged_attention_scores(query, keys, table, lens, lse, starts, scale=problem.scale)
    assert torch.equal(clean, dirty)
    lse[5] = -math.inf
    query[5] = math.nan
    without = paged_attention_scores(query, keys, table, lens, lse, starts, scale=problem.scale)
    problem.query[5] = 0
    assert _scores_close(problem, without, lse)
