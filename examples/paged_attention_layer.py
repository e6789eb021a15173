"""A decoder layer's attention block, as a serving loop uses it.

W8A8 q/k/v projection -> norms, rotation and storing into a paged cache -> attention over the cache -> W8A8 output
projection, for a batch of sequences that prefill in chunks and then decode token by token.  With a budget, the slots'
attention weights are added up and every sequence is cut down to the budget after each step.

    python examples/paged_attention_layer.py            # on a HIP device
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qpu-xla-triton_amd"))

from qpu_xla_amd.kernels import (  # noqa: E402
    paged_attention,
    paged_attention_scores,
    paged_cache_evict,
    qk_norm_rope_cache,
)
from qpu_xla_amd.quantization import quantize_per_output_channel_int8, w8a8_linear  # noqa: E402


class PagedAttentionLayer:
    """Weights, cache pages and per-sequence state of one layer."""

    def __init__(self, *, hidden: int, heads: int, kv_heads: int, head_dim: int, sequences: int, slots: int,
                 page_size: int = 64, budget: int | None = None, recent: int = 0, max_position: int = 4096,
                 device: str = "cuda", seed: int = 0) -> None:
        gen = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.budget, self.recent, self.page_size = budget, recent, page_size

        def linear(outputs: int, inputs: int):
            return quantize_per_output_channel_int8(
                torch.randn((outputs, inputs), generator=gen, device=device) * inputs**-0.5)

        self.qkv = linear((heads + 2 * kv_heads) * head_dim, hidden)
        self.output = linear(hidden, heads * head_dim)
        self.query_norm = 1 + 0.1 * torch.randn((head_dim,), generator=gen, device=device)
        self.key_norm = 1 + 0.1 * torch.randn((head_dim,), generator=gen, device=device)
        rate = 10000.0 ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
        angle = torch.arange(max_position, device=device, dtype=torch.float64)[:, None] * rate
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

        # Pages of a pool, here dealt out up front; a server hands them out as sequences grow.
        each = -(-slots // page_size)
        shape = (sequences * each, page_size, kv_heads, head_dim)
        self.keys, self.values = (torch.zeros(shape, device=device, dtype=torch.bfloat16) for _ in range(2))
        self.table = torch.randperm(sequences * each, generator=gen, device=device).to(torch.int32).view(sequences, each)
        self.scores = torch.zeros((sequences, kv_heads, each * page_size), device=device)
        self.slot_positions = torch.full(self.scores.shape, -1, device=device, dtype=torch.int32)
        # Lengths and positions are known to the host: it decides how many tokens a step takes.
        self.lengths = [0] * sequences
        self.positions = [0] * sequences

    def step(self, x: torch.Tensor, counts: list[int]) -> torch.Tensor:
        """fp32 activations [sum(counts), hidden] of each sequence's next tokens -> the block's output, same shape."""
        device, tokens = x.device, x.shape[0]
        owner = torch.tensor([b for b, n in enumerate(counts) for _ in range(n)], device=device)
        slot = torch.tensor([self.lengths[b] + i for b, n in enumerate(counts) for i in range(n)], device=device)
        position = torch.tensor([self.positions[b] + i for b, n in enumerate(counts) for i in range(n)], device=device,
                                dtype=torch.int32)
        starts = torch.tensor([0, *counts], device=device).cumsum(0).to(torch.int32)
        lens = torch.tensor([length + n for length, n in zip(self.lengths, counts)], device=device, dtype=torch.int32)
        flat = self.table[owner, slot // self.page_size].long() * self.page_size + slot % self.page_size

        qkv = w8a8_linear(x, self.qkv)
        query, key, value = (part.unflatten(1, (-1, self.head_dim)) for part in qkv.split(
            [self.heads * self.head_dim, self.kv_heads * self.head_dim, self.kv_heads * self.head_dim], dim=1))
        query = qk_norm_rope_cache(query, key, value, self.cos, self.sin, position, flat, self.keys, self.values,
                                   self.query_norm, self.key_norm)
        out = torch.empty((tokens, self.heads, self.head_dim), device=device)  # fp32, as the next linear takes it
        lse = torch.empty((tokens, self.heads), device=device) if self.budget else None
        sizes = {"max_query": max(counts), "max_context": max(a + n for a, n in zip(self.lengths, counts))}
        paged_attention(query, self.keys, self.values, self.table, lens, starts, out=out, lse=lse, **sizes)

        self.lengths = [length + n for length, n in zip(self.lengths, counts)]
        self.positions = [p + n for p, n in zip(self.positions, counts)]
        if self.budget:
            paged_attention_scores(query, self.keys, self.table, lens, lse, starts, scores=self.scores, out=self.scores, **sizes)
            self.slot_positions[owner, :, slot] = position[:, None]
            if max(self.lengths) > self.budget:
                paged_cache_evict(self.keys, self.values, self.table, lens, self.scores, self.slot_positions,
                                  budget=self.budget, recent=self.recent, max_context=sizes["max_context"],
                                  scores_out=self.scores, positions_out=self.slot_positions)
                self.lengths = [min(length, self.budget) for length in self.lengths]
        return w8a8_linear(out.flatten(1), self.output)


def main() -> None:
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts, hidden, chunk = [700, 90, 333], 512, 256
    layer = PagedAttentionLayer(hidden=hidden, heads=8, kv_heads=2, head_dim=64, sequences=len(prompts), slots=1024,
                                budget=256, recent=64)
    done = [0] * len(prompts)
    while any(d < p for d, p in zip(done, prompts)):  # the prompts in chunks, side by side
        counts = [min(chunk, p - d) for d, p in zip(done, prompts)]
        layer.step(torch.randn((sum(counts), hidden), generator=gen, device="cuda"), counts)
        done = [d + n for d, n in zip(done, counts)]
        print(f"prefilled {done} of {prompts}, slots in use {layer.lengths}")
    for _ in range(16):
        y = layer.step(torch.randn((len(prompts), hidden), generator=gen, device="cuda"), [1] * len(prompts))
    torch.cuda.synchronize()
    print(f"16 tokens a sequence decoded, slots in use {layer.lengths}, output {tuple(y.shape)}, rms {y.square().mean().sqrt():.4f}")


if __name__ == "__main__":
    main()
