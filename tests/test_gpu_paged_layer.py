"""The example layer: chunks and single tokens agree with the definition, eviction keeps to its budget."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd.quantization import w8a8_linear

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "paged_attention_layer", Path(__file__).resolve().parents[1] / "examples" / "paged_attention_layer.py")
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)

SIZES = {"hidden": 256, "heads": 8, "kv_heads": 2, "head_dim": 64, "sequences": 2, "slots": 160, "page_size": 16}


def _expected(layer, x):
    """Attention of one sequence's tokens from the layer's own projection, in 64 bits, before the output projection."""
    qkv = w8a8_linear(x, layer.qkv).cpu()
    heads, kv_heads, dim = layer.heads, layer.kv_heads, layer.head_dim
    q, k, v = (p.unflatten(1, (-1, dim)) for p in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    positions = torch.arange(len(x), dtype=torch.int32)
    rotate = lambda rows, weight: reference.rope(rows, weight.cpu(), layer.cos.cpu(), layer.sin.cpu(), positions, 1e-6, False)  # noqa: E731
    q, k = (rotate(rows, weight).to(torch.bfloat16) for rows, weight in ((q, layer.query_norm), (k, layer.key_norm)))
    page = torch.zeros((1, 1), dtype=torch.int32)
    out, _, bound = reference.attention(q, k[None], v.to(torch.bfloat16)[None], page, torch.tensor([len(x)]),
                                        torch.tensor([0, len(x)], dtype=torch.int32), scale=1 / math.sqrt(dim))
    return out, bound


def test_chunks_and_single_tokens_agree_with_the_definition() -> None:
    gen = torch.Generator(device="cuda").manual_seed(3)
    layer = example.PagedAttentionLayer(**SIZES)
    attended = []
    layer_linear = example.w8a8_linear
    example.w8a8_linear = lambda x, w: (attended.append(x) if w is layer.output else None, layer_linear(x, w))[1]
    try:
        x = [torch.randn((n, 256), generator=gen, device="cuda") for n in (120, 47)]
        at = [0, 0]
        for counts in ([64, 40], [55, 1], [1, 1], [0, 5]):
            layer.step(torch.cat([x[b][at[b]:at[b] + n] for b, n in enumerate(counts)]), counts)
            at = [a + n for a, n in zip(at, counts)]
    finally:
        example.w8a8_linear = layer_linear
    rows = [torch.cat(parts) for parts in zip(*(a.split(n) for a, n in zip(attended, ([64, 40], [55, 1], [1, 1], [0, 5]))))]
    for b in range(2):
        want, bound = _expected(layer, x[b])
        # Weights are rounded to bfloat16 (2^-8 of the bound); rows are the same bfloat16 values but where a rounding
        # falls the other way after fp32 arithmetic (rare, half a unit of one element of a logit's 64): 2^-6 covers both.
        off = (rows[b].cpu().double().view_as(want) - want).abs()
        assert bool((off <= 2.0**-6 * bound + 1e-6).all()), float((off / bound).max())


def test_eviction_keeps_every_sequence_within_its_budget() -> None:
    gen = torch.Generator(device="cuda").manual_seed(4)
    layer = example.PagedAttentionLayer(**SIZES, budget=48, recent=16)
    total = [0, 0]
    for counts in ([100, 20], [1, 60], [1, 1], [1, 1], [7, 3]):
        y = layer.step(torch.randn((sum(counts), 256), generator=gen, device="cuda"), counts)
        total = [t + n for t, n in zip(total, counts)]
        assert bool(torch.isfinite(y).all())
        assert layer.lengths == [min(48, before) for before in (total if max(total) <= 48 else [min(t, 48) for t in total])]
        for b, used in enumerate(layer.lengths):
            positions = layer.slot_positions[b].cpu()
            assert bool((positions[:, used:] == -1).all()) and bool((layer.scores[b, :, used:] == 0).all())
            for head in positions[:, :used]:
                kept = sorted(head.tolist())
                assert len(set(kept)) == used and kept[-1] == total[b] - 1
                recent = [p for p in range(max(0, total[b] - 16), total[b])]
                assert kept[-len(recent):] == recent  # the newest tokens are all there


def test_the_example_runs(capsys) -> None:
    example.main()
    assert "slots in use [256, 106, 256]" in capsys.readouterr().out
