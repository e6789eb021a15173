"""Refusals of the attention operators (no GPU: checks return before any HIP call), and their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd import KernelError, LaunchConfig, _lib
from qpu_xla_amd import kernels as k

FAKE = 1 << 20  # 16-byte aligned, never dereferenced


def _attention_args(**changes):
    args = {
        "query": torch.zeros((3, 4, 64), dtype=torch.bfloat16),
        "key_cache": torch.zeros((5, 16, 2, 64), dtype=torch.bfloat16),
        "value_cache": torch.zeros((5, 16, 2, 64), dtype=torch.bfloat16),
        "block_table": torch.zeros((3, 2), dtype=torch.int32),
        "context_lens": torch.ones(3, dtype=torch.int32),
        "query_starts": None,
    }
    args.update(changes)
    return args


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"query": torch.zeros((3, 4, 64))}, "cache's type"),
    ({"query": torch.zeros((3, 4, 32), dtype=torch.bfloat16)}, "head size"),
    ({"query": torch.zeros((3, 3, 64), dtype=torch.bfloat16)}, "multiple of the cache's heads"),
    ({"query": torch.zeros((3, 64), dtype=torch.bfloat16)}, "tokens, heads, head_dim"),
    ({"query": torch.zeros((3, 4, 128), dtype=torch.bfloat16)[..., ::2]}, "dense rows"),
    ({"query": torch.zeros((4, 4, 64), dtype=torch.bfloat16)}, "one token"),
    ({"key_cache": torch.zeros((5, 16, 2, 64))}, "key_cache must be"),
    ({"value_cache": torch.zeros((5, 16, 2, 64), dtype=torch.float16)}, "one shape and type"),
    ({"value_cache": torch.zeros((5, 8, 2, 64), dtype=torch.bfloat16)}, "one shape and type"),
    ({"key_cache": torch.zeros((0, 16, 2, 64), dtype=torch.bfloat16),
      "value_cache": torch.zeros((0, 16, 2, 64), dtype=torch.bfloat16)}, "empty"),
    ({"block_table": torch.zeros((3, 2), dtype=torch.int64)}, "block_table"),
    ({"block_table": torch.zeros((3, 0), dtype=torch.int32)}, "block_table"),
    ({"context_lens": torch.ones(2, dtype=torch.int32)}, "context_lens"),
    ({"context_lens": torch.ones(3, dtype=torch.int64)}, "context_lens"),
    ({"query_starts": torch.zeros(3, dtype=torch.int32)}, "query_starts"),
    ({"scale": 0.0}, "scale"),
    ({"scale": math.nan}, "scale"),
    ({"scale": math.inf}, "scale"),
    ({"window": -1}, "window"),
    ({"max_context": -1}, "max_context"),
    ({"max_query": 2**32, "query_starts": torch.zeros(4, dtype=torch.int32)}, "max_query"),
    ({"out": torch.zeros((3, 4, 32), dtype=torch.bfloat16)}, "out must"),
    ({"out": torch.zeros((3, 4, 64), dtype=torch.float64)}, "out must"),
    ({"lse": torch.zeros((3, 5))}, "lse"),
    ({"lse": torch.zeros((3, 4), dtype=torch.bfloat16)}, "lse"),
])
def test_attention_refuses(changes, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        k.paged_attention(**_attention_args(**changes))


@pytest.mark.parametrize("dim", [4, 12, 264])
def test_attention_refuses_head_sizes(dim) -> None:
    caches = {name: torch.zeros((5, 16, 2, dim), dtype=torch.bfloat16) for name in ("key_cache", "value_cache")}
    with pytest.raises(ValueError, match="multiple of 8"):
        k.paged_attention(**_attention_args(query=torch.zeros((3, 4, dim), dtype=torch.bfloat16), **caches))


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"lse": torch.zeros((3, 3))}, "lse"),
    ({"scores": torch.zeros((3, 2, 31))}, "scores must"),
    ({"out": torch.zeros((3, 2, 32), dtype=torch.float64)}, "out must"),
    ({"out": torch.zeros((3, 2, 64))[..., ::2]}, "dense"),
])
def test_scores_refuse(changes, fragment) -> None:
    args = _attention_args(lse=torch.zeros((3, 4)))
    del args["value_cache"]
    args.update(changes)
    with pytest.raises(ValueError, match=fragment):
        k.paged_attention_scores(**args)


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"budget": 0}, "budget"),
    ({"recent": 9}, "recent"),
    ({"recent": -1}, "recent"),
    ({"scores": torch.zeros((3, 2, 31))}, "scores must"),
    ({"positions": torch.zeros((3, 2, 32), dtype=torch.int64)}, "positions must"),
    ({"lens_out": torch.zeros(2, dtype=torch.int32)}, "lens_out"),
    ({"max_context": -5}, "max_context"),
])
def test_eviction_refuses(changes, fragment) -> None:
    args = _attention_args(scores=torch.zeros((3, 2, 32)), positions=torch.zeros((3, 2, 32), dtype=torch.int32), budget=8)
    del args["query"], args["query_starts"]
    args.update(changes)
    with pytest.raises(ValueError, match=fragment):
        k.paged_cache_evict(**args)


def _rope_args(**changes):
    args = {"query": torch.zeros((3, 4, 64)), "key": torch.zeros((3, 2, 64)), "cos": torch.ones((9, 32)),
            "sin": torch.zeros((9, 32)), "positions": torch.zeros(3, dtype=torch.int32)}
    args.update(changes)
    return args


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"query": torch.zeros((3, 4, 64), dtype=torch.float64)}, "query must"),
    ({"key": torch.zeros((2, 2, 64))}, "agree"),
    ({"key": torch.zeros((3, 2, 64), dtype=torch.float16)}, "agree"),
    ({"cos": torch.ones((9, 33)), "sin": torch.ones((9, 33))}, "head size"),
    ({"sin": torch.ones((8, 32))}, "one shape"),
    ({"cos": torch.ones((9, 64))[:, ::2]}, "contiguous"),
    ({"positions": torch.zeros(3, dtype=torch.int64)}, "positions"),
    ({"query_weight": torch.ones(63)}, "weights"),
    ({"key_weight": torch.ones(64, dtype=torch.bfloat16)}, "weights"),
    ({"query_out": torch.zeros((3, 4, 32))}, "outputs"),
    ({"query_out": torch.zeros((3, 4, 64)), "key_out": torch.zeros((3, 2, 64), dtype=torch.bfloat16)}, "one type"),
])
def test_rotation_refuses(changes, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        k.qk_norm_rope(**_rope_args(**changes))


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"value": torch.zeros((3, 3, 64))}, "key and value"),
    ({"slots": torch.zeros(3, dtype=torch.int32)}, "slots"),
    ({"key_cache": torch.zeros((5, 16, 3, 64), dtype=torch.float16),
      "value_cache": torch.zeros((5, 16, 3, 64), dtype=torch.float16)}, "heads and head size"),
    ({"query_out": torch.zeros((3, 4, 64))}, "cache's type"),
])
def test_rotation_into_the_cache_refuses(changes, fragment) -> None:
    args = _rope_args(value=torch.zeros((3, 2, 64)), slots=torch.zeros(3, dtype=torch.int64),
                      key_cache=torch.zeros((5, 16, 2, 64), dtype=torch.float16),
                      value_cache=torch.zeros((5, 16, 2, 64), dtype=torch.float16))
    args.update(changes)
    with pytest.raises(ValueError, match=fragment):
        k.qk_norm_rope_cache(**args)


@pytest.mark.parametrize("kernel", [k.QK_NORM_ROPE_CACHE_KERNEL, k.PAGED_ATTENTION_KERNEL, k.PAGED_ATTENTION_SCORES_KERNEL,
                                    k.PAGED_CACHE_EVICT_KERNEL])
def test_kernels_refuse_wrong_tuples(kernel) -> None:
    with pytest.raises(KernelError, match="expects"):
        kernel.execute(0, (torch.zeros(1),), LaunchConfig())


def test_kernel_refuses_a_wrong_grid() -> None:
    a = _attention_args()
    args = (*list(a.values())[:5], None, a["query"], None, k.PagedAttentionOptions())
    with pytest.raises(KernelError, match="grid"):
        k.PAGED_ATTENTION_KERNEL.execute(0, args, LaunchConfig((4, 2, 1)))
    with pytest.raises(KernelError, match="failed"):  # right grid, tensors not on a device
        k.PAGED_ATTENTION_KERNEL.execute(0, args, LaunchConfig(k.paged_attention_grid(a["query"])))


# ------------------------------------------------------------------------ C ABI


def _cache(**changes):
    fields = {"keys": FAKE, "key_page": 4096, "key_slot": 256, "key_head": 128, "values": FAKE, "value_page": 4096,
              "value_slot": 256, "value_head": 128, "table": FAKE, "table_stride": 8, "lens": FAKE, "pages": 5, "page_size": 16,
              "heads": 2, "head_dim": 64, "type": 1, "width": 2, "sequences": 3}
    fields.update(changes)
    return _lib.PAGED_CACHE.pack(*fields.values())


def _attend(cache, **changes):
    a = {"query": FAKE, "token": 512, "head": 128, "starts": None, "out": FAKE, "out_token": 512, "out_head": 128, "out_type": 1,
         "lse": None, "lse_stride": 0, "tokens": 3, "heads": 4, "scale": 0.1, "causal": 1, "window": 0, "max_query": 1,
         "max_context": 32, "workspace": None, "bytes": 0}
    a.update(changes)
    lib = _lib.load()
    return lib.qxt_paged_attention(a["query"], a["token"], a["head"], cache, a["starts"], a["out"], a["out_token"], a["out_head"],
                                   a["out_type"], a["lse"], a["lse_stride"], a["tokens"], a["heads"], a["scale"], a["causal"],
                                   a["window"], a["max_query"], a["max_context"], a["workspace"], a["bytes"], None)


@pytest.mark.parametrize("cache,changes,fragment", [
    ({"keys": 0}, {}, "null"), ({"values": 0}, {}, "null"), ({"table": 0}, {}, "null"), ({"lens": 0}, {}, "null"),
    ({}, {"query": None}, "null"), ({}, {"out": None}, "null"),
    ({"type": 0}, {}, "bf16 or fp16"), ({"type": 7}, {}, "bf16 or fp16"), ({"page_size": 0}, {}, "positive"),
    ({"head_dim": 20}, {}, "multiple of 8"), ({"head_dim": 512}, {}, "multiple of 8"),
    ({"page_size": 2**20, "width": 2**10}, {}, "slots"), ({"key_slot": 8}, {}, "aligned"), ({"values": FAKE + 8}, {}, "aligned"),
    ({"key_page": 2**36}, {}, "64 GiB"), ({"table_stride": 6}, {}, "misaligned"),
    ({}, {"heads": 3}, "multiple"), ({}, {"scale": 0.0}, "scale"), ({}, {"scale": math.nan}, "scale"), ({}, {"causal": 2}, "causal"),
    ({}, {"tokens": 4}, "one token"), ({}, {"token": 24}, "aligned"), ({}, {"out": FAKE + 2}, "misaligned output"),
    ({}, {"out_type": 9}, "element type"), ({}, {"tokens": 2**29, "starts": FAKE}, "rows"),
    ({"width": 4096}, {"max_context": 65536}, "workspace"),
])
def test_attention_entry_point_refuses(cache, changes, fragment) -> None:
    assert _attend(_cache(**cache), **changes) == _lib.INVALID_ARGUMENT
    assert fragment in _lib.last_error()


def test_other_entry_points_refuse() -> None:
    lib, cache = _lib.load(), _cache()
    scores = lambda c, previous=None, out=FAKE, lse=FAKE: lib.qxt_paged_attention_scores(  # noqa: E731
        FAKE, 512, 128, c, None, lse, 16, previous, 0, 0, out, 256, 128, 3, 4, 0.1, 1, 0, 1, 32, None, 0, None)
    evict = lambda c, budget, recent, out=FAKE + 64, size=4096: lib.qxt_paged_cache_evict(  # noqa: E731
        c, FAKE, 256, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE, 256, 128, out, budget, recent, 32, FAKE, size, None)
    for call, fragment in (
        (lambda: scores(_cache(keys=0)), "null"), (lambda: scores(cache, out=None), "null"), (lambda: scores(cache, lse=None), "null"),
        (lambda: scores(cache, previous=FAKE + 2), "misaligned"), (lambda: evict(cache, 0, 0), "budget"),
        (lambda: evict(cache, 8, 9), "recent"), (lambda: evict(_cache(values=0), 8, 0), "null"),
        (lambda: evict(cache, 8, 0, out=FAKE), "in place"), (lambda: evict(cache, 8, 0, size=8), "workspace"),
    ):
        assert call() == _lib.INVALID_ARGUMENT
        assert fragment in _lib.last_error()


def test_injected_failure_returns_before_any_launch() -> None:
    lib, cache = _lib.load(), _cache()
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    try:
        assert _attend(cache) == _lib.SUBMISSION_FAILED
        assert lib.qxt_paged_attention_scores(FAKE, 512, 128, cache, None, FAKE, 16, None, 0, 0, FAKE, 256, 128, 3, 4, 0.1, 1, 0, 1,
                                              32, None, 0, None) == _lib.SUBMISSION_FAILED
        assert lib.qxt_paged_cache_evict(cache, FAKE, 256, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE + 64, 8, 4, 32,
                                         FAKE, 4096, None) == _lib.SUBMISSION_FAILED
        assert lib.qxt_qk_norm_rope(FAKE, 1024, 256, FAKE, 512, 256, None, None, 1e-6, FAKE, FAKE, 128, 9, FAKE, FAKE, 1024, 256,
                                    FAKE, 512, 256, 3, 4, 2, 64, 64, 0, 0, 0, None) == _lib.SUBMISSION_FAILED
        assert lib.qxt_qk_norm_rope_cache(FAKE, 1024, 256, FAKE, 512, 256, FAKE, 512, 256, None, None, 1e-6, FAKE, FAKE, 128, 9, FAKE,
                                          FAKE, FAKE, 512, 128, cache, 3, 4, 64, 0, 0, None) == _lib.SUBMISSION_FAILED
    finally:
        _lib.set_failure_mask(_lib.FAIL_NONE)


@pytest.mark.parametrize("position,value,fragment", [
    (0, None, "null"), (25, 3, "even"), (25, 130, "even"), (24, 0, "positive"), (26, 5, "type"),
    (28, 2, "flags"), (0, FAKE + 2, "misaligned input"), (1, 1022, "misaligned input"), (14, FAKE + 2, "misaligned output"),
    (9, FAKE + 2, "misaligned table"), (11, 126, "misaligned table"), (21, 2**31 - 1, "rows"),
])
def test_rotation_entry_point_refuses(position, value, fragment) -> None:
    args = [FAKE, 1024, 256, FAKE, 512, 256, None, None, 1e-6, FAKE, FAKE, 128, 9, FAKE, FAKE, 1024, 256, FAKE, 512, 256, 3, 4, 2, 64,
            64, 0, 0, 0, None]
    # Positions count from the C signature: 20 tokens, 21 query heads, 22 key heads, 23 head size, 24 rotary size,
    # 25 input type, 26 output type, 27 flags.
    place = {21: 20, 24: 23, 25: 24, 26: 25, 28: 27}.get(position, position)
    args[place] = value
    assert _lib.load().qxt_qk_norm_rope(*args) == _lib.INVALID_ARGUMENT
    assert fragment in _lib.last_error()


def test_workspaces_follow_the_plan() -> None:
    lib = _lib.load()
    assert lib.qxt_paged_attention_workspace(32, 0, 128, 1, 1, 1, 4096) == 0
    assert lib.qxt_paged_attention_workspace(32, 8, 128, 1, 0, 1, 4096) == 0
    few = lib.qxt_paged_attention_workspace(32, 8, 128, 1, 1, 1, 32768)
    assert few > 0 and few % (32 * (128 * 4 + 8)) == 0  # parts of one token's rows
    assert lib.qxt_paged_attention_workspace(32, 32, 128, 1, 8192, 8192, 8192) == 0  # enough row tiles
    assert lib.qxt_paged_cache_evict_workspace(8, 2, 100, 100) == 8 * 2 * 2 * 4
    assert lib.qxt_paged_cache_evict_workspace(8, 2, 1000, 100) == 8 * 2 * 202 * 4


# -------------------------------------------------------------- the definitions


def test_definition_of_attention_and_scores_on_a_contiguous_cache() -> None:
    gen = torch.Generator().manual_seed(0)
    n, heads, kv_heads, dim = 9, 4, 2, 8
    query = torch.randn((n, heads, dim), generator=gen)
    keys, values = (torch.randn((3, 4, kv_heads, dim), generator=gen) for _ in range(2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    lens, starts = torch.tensor([12]), torch.tensor([0, n], dtype=torch.int32)
    out, lse, _ = reference.attention(query, keys, values, table, lens, starts, scale=0.5)
    k_flat, v_flat = (c[[2, 0, 1]].flatten(0, 1).double().repeat_interleave(2, dim=1) for c in (keys, values))
    logits = torch.einsum("thd,shd->hts", query.double(), k_flat) * 0.5
    hidden = torch.arange(12)[None] > torch.arange(3, 12)[:, None]
    weights = logits.masked_fill(hidden, -math.inf).softmax(-1)
    assert torch.allclose(out, torch.einsum("hts,shd->thd", weights, v_flat))
    assert torch.allclose(lse.T, logits.masked_fill(hidden, -math.inf).logsumexp(-1))
    got = reference.scores(query, keys, table, lens, lse, starts, previous=None, scale=0.5)
    assert torch.allclose(got[0], weights.view(2, 2, n, 12).sum(dim=(1, 2)))


def test_definition_of_eviction_by_hand() -> None:
    keys = torch.arange(6.0).view(1, 6, 1, 1).expand(1, 6, 1, 8).to(torch.bfloat16).contiguous()
    scores = torch.tensor([[[5.0, 1.0, 3.0, 2.0, 1.0, 0.0]]])
    positions = torch.tensor([[[0, 1, 2, 3, 4, 5]]], dtype=torch.int32)
    lens, s, p, moved, _ = reference.evict(keys, keys.clone(), torch.zeros((1, 1), dtype=torch.int32), torch.tensor([6]), scores,
                                           positions, 3, 1)
    # Kept: slot 5 (the newest), 0 and 2 (the heaviest); 1 is given up and takes what slot 5 held.
    assert lens.tolist() == [3] and p[0, 0].tolist() == [0, 5, 2, -1, -1, -1] and s[0, 0].tolist() == [5.0, 0.0, 3.0, 0, 0, 0]
    assert moved[0, :3, 0, 0].tolist() == [0.0, 5.0, 2.0]


def test_definition_of_rotation_keeps_lengths() -> None:
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((5, 3, 16), generator=gen)
    angle = torch.rand((7, 4), generator=gen) * 6
    positions = torch.tensor([0, 6, 3, 3, 2], dtype=torch.int32)
    for interleaved in (False, True):
        y = reference.rope(x, None, angle.cos(), angle.sin(), positions, 0.0, interleaved)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6)
        assert torch.equal(y[..., 8:], x[..., 8:].double())
