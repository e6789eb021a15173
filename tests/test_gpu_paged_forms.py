"""Forms of the attention operators that the other tests leave out: splits in fp16, split weights of wide heads, graphs."""

from __future__ import annotations

import pytest
import torch

from qpu_xla_amd.kernels import paged_attention, paged_attention_scores, paged_cache_evict, qk_norm_rope, qk_norm_rope_cache
from test_gpu_paged_attention import Problem, _scores_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [
    ([(5000, 1)], 4, 1, 128, 64, 1),
    ([(4000, 1), (3, 1), (0, 1)], 8, 8, 64, 16, 1),
    ([(3000, 40)], 4, 2, 128, 48, 40),
    ([(2500, 200)], 2, 1, 256, 32, 200),
    ([(2222, 150), (1, 1)], 3, 1, 96, 16, 150),
])
def test_split_contexts_in_fp16(case) -> None:
    lens, heads, kv_heads, dim, page_size, most = case
    problem = Problem(lens, heads, kv_heads, dim, page_size, torch.float16, seed=heads)
    out, lse = problem.run(max_query=most)
    problem.check(out, lse)
    again, lse_again = problem.run(max_query=most)  # parts are joined in one order
    assert torch.equal(out, again) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [192, 256])
def test_split_weights_of_wide_heads(dim, dtype) -> None:
    problem = Problem([(700, 300), (64, 9)], 4, 1, dim, 16, dtype, seed=dim)
    _, lse = problem.run(max_query=300)
    query, keys, _, table, context, starts = problem.device()
    args = (query, keys, table, context, lse, starts)
    got = paged_attention_scores(*args, scale=problem.scale, max_query=300, max_context=700)
    assert _scores_close(problem, got, lse)
    assert torch.equal(got, paged_attention_scores(*args, scale=problem.scale, max_query=300, max_context=700))


@pytest.mark.parametrize("lens", [[(900, 1), (500, 1)], [(700, 300), (300, 20)]])
def test_a_step_of_all_operators_in_a_graph(lens) -> None:
    heads, kv_heads, dim, page_size, budget = 8, 2, 128, 16, 256
    problem = Problem(lens, heads, kv_heads, dim, page_size, torch.bfloat16, seed=3)
    query, keys, values, table, context, starts = problem.device()
    tokens, slots = query.shape[0], table.shape[1] * page_size
    gen = torch.Generator().manual_seed(5)
    rows = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen).cuda()
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    angle = torch.rand((1024, dim // 2), generator=gen).cuda() * 6
    cos, sin = angle.cos(), angle.sin()
    position = torch.cat([torch.arange(c - n, c) for c, n in lens]).to(torch.int32).cuda()
    flat = torch.cat([problem.table[b, torch.arange(c - n, c) // page_size].long() * page_size
                      + torch.arange(c - n, c) % page_size for b, (c, n) in enumerate(lens)]).cuda()
    weight = (1 + torch.rand((dim,), generator=gen)).cuda()
    slot_positions = torch.arange(slots, dtype=torch.int32).expand(len(lens), kv_heads, slots).contiguous().cuda()
    first = {"scores": torch.rand((len(lens), kv_heads, slots), generator=gen).cuda(), "positions": slot_positions}
    held = {name: t.clone() for name, t in first.items()}
    clean = (keys.clone(), values.clone())
    sizes = {"max_query": max(n for _, n in lens), "max_context": max(c for c, _ in lens)}
    results = {"query": torch.empty_like(query), "rotated": torch.empty_like(q), "key": torch.empty_like(k),
               "out": torch.empty_like(q, dtype=torch.float32), "lse": torch.empty((tokens, heads), device="cuda"),
               "lens": torch.empty_like(context)}

    def step():
        qk_norm_rope(q, k, cos, sin, position, weight, weight, query_out=results["rotated"], key_out=results["key"])
        qk_norm_rope_cache(q, k, v, cos, sin, position, flat, keys, values, weight, weight, query_out=results["query"])
        paged_attention(results["query"], keys, values, table, context, starts, out=results["out"], lse=results["lse"], **sizes)
        paged_attention_scores(results["query"], keys, table, context, results["lse"], starts, scores=held["scores"],
                               out=held["scores"], **sizes)
        paged_cache_evict(keys, values, table, context, held["scores"], held["positions"], budget=budget, recent=32,
                          max_context=sizes["max_context"], scores_out=held["scores"], positions_out=held["positions"],
                          lens_out=results["lens"])

    def start(turn):
        rows.copy_(torch.randn(rows.shape, generator=torch.Generator().manual_seed(turn)).cuda())
        keys.copy_(clean[0])
        values.copy_(clean[1])
        for name, t in first.items():
            held[name].copy_(t)
        for t in results.values():
            t.zero_()

    def state():
        torch.cuda.synchronize()
        return {name: t.clone() for name, t in {**results, **held, "keys": keys, "values": values}.items()}

    start(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        start(turn)
        step()
        eager = state()
        assert eager["lens"].tolist() == [min(c, budget) for c, _ in lens]
        start(turn)
        graph.replay()
        replayed = state()
        for name, t in eager.items():
            assert torch.equal(replayed[name], t), name
