"""Norms of queries and keys with the rotation, against the 64-bit definition.

Tolerances: fp32 outputs err by a few roundings of the norm (sum of squares of D terms, reciprocal root, two
products: under D/64 + 14 units of 2^-24 of the row's values) and of the rotation, whose two products are each
rounded: the error is relative to |a| + |b| of a pair, not to the result.  Half types add half a unit of the result
(2^-8 for bfloat16, 2^-11 for float16), and 2^-25 absolute below float16's normal range.
"""

from __future__ import annotations

import pytest
import torch

import paged_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import QK_NORM_ROPE_CACHE_KERNEL, QkNormRopeOptions, qk_norm_rope, qk_norm_rope_cache, qk_norm_rope_grid

pytestmark = pytest.mark.gpu

EPSILON = 1e-5
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _tables(gen, positions, rotary):
    angle = torch.rand((positions, rotary // 2), generator=gen) * 6.3
    return angle.cos(), angle.sin()


def _errors(got, x, weight, cos, sin, positions, interleaved):
    want = reference.rope(x, weight, cos, sin, positions, EPSILON, interleaved)
    size = reference.rope(x, weight, torch.ones_like(cos), torch.zeros_like(sin), positions, EPSILON, interleaved).abs()
    half = cos.shape[1]
    pair = size.clone()
    if interleaved:
        pair[..., 0:2 * half:2] += size[..., 1:2 * half:2]
        pair[..., 1:2 * half:2] += size[..., 0:2 * half:2]
    else:
        pair[..., :half] += size[..., half:2 * half]
        pair[..., half:2 * half] += size[..., :half]
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    return (got - want).abs().nan_to_num(0.0), want.abs().nan_to_num(0.0), pair.nan_to_num(0.0)


def _check(got, x, weight, cos, sin, positions, interleaved):
    off, want, pair = _errors(got, x, weight, cos, sin, positions, interleaved)
    arithmetic = (x.shape[2] / 64 + 14) * 2.0**-24 * pair
    rounding = (UNIT[got.dtype] * (want + arithmetic) + 2.0**-25) if got.dtype != torch.float32 else 0.0
    assert bool((off <= arithmetic + rounding + 1e-30).all()), float((off - arithmetic - rounding).max())


# (tokens, query heads, key heads, head size, rotary size): aligned runs, lone rows, parts past the rotation, sizes
# that only the pairwise kernel takes (odd, not multiples of four, over 512), no rotation at all.
SHAPES = [
    (1, 32, 4, 64, 64), (7, 8, 2, 128, 128), (5, 3, 1, 128, 64), (33, 4, 4, 80, 32), (9, 2, 1, 96, 96), (3, 5, 5, 256, 64),
    (4, 2, 2, 512, 512), (6, 3, 1, 72, 40), (5, 1, 1, 20, 8), (5, 2, 1, 30, 30), (4, 2, 1, 65, 10), (3, 1, 1, 2, 2),
    (2, 2, 1, 1030, 514), (6, 2, 2, 64, 0), (5, 2, 1, 64, 12), (4, 2, 1, 7, 4), (1000, 1, 1, 8, 8),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_against_the_definition(shape, dtype, interleaved) -> None:
    tokens, query_heads, key_heads, dim, rotary = shape
    gen = torch.Generator().manual_seed(hash(shape) % 1000)
    query = (torch.randn((tokens, query_heads, dim), generator=gen) * 3).to(dtype)
    key = (torch.randn((tokens, key_heads, dim), generator=gen) * 0.2).to(dtype)
    cos, sin = _tables(gen, 50, rotary)
    positions = torch.randint(0, 50, (tokens,), generator=gen, dtype=torch.int32)
    weight = 1 + 0.3 * torch.randn((dim,), generator=gen)
    q, k = qk_norm_rope(query.cuda(), key.cuda(), cos.cuda(), sin.cuda(), positions.cuda(), weight.cuda(), None,
                        epsilon=EPSILON, interleaved=interleaved)
    assert q.dtype == k.dtype == dtype
    _check(q, query, weight, cos, sin, positions, interleaved)
    _check(k, key, None, cos, sin, positions, interleaved)


@pytest.mark.parametrize("offset", [0, 1])  # 1: rows that are not aligned to four elements
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_strided_inputs_outputs_in_place_and_other_types(out_dtype, offset) -> None:
    gen = torch.Generator().manual_seed(3)
    tokens, heads, dim = 11, 6, 64
    cos, sin = _tables(gen, 20, dim)
    positions = torch.randint(0, 20, (tokens,), generator=gen, dtype=torch.int32)
    weight = torch.rand((dim + 1,), generator=gen)[offset:offset + dim].contiguous()
    fused = torch.randn((tokens, 2 * heads * dim + 8), generator=gen)
    device = fused.cuda()
    view = device[:, offset:offset + heads * dim].unflatten(1, (heads, dim))  # token stride past the row
    other = device.flatten()[8:8 + tokens * heads * dim].view(heads, tokens, dim).transpose(0, 1)  # heads first
    out = torch.full((heads, tokens, 2 * dim + 1), 7.0, device="cuda", dtype=out_dtype)
    q_out, k_out = out[..., offset:offset + dim].transpose(0, 1), torch.empty((tokens, heads, dim), device="cuda", dtype=out_dtype)
    args = (cos.cuda(), sin.cuda(), positions.cuda(), weight.cuda(), weight.cuda())
    q, k = qk_norm_rope(view, other, *args, epsilon=EPSILON, query_out=q_out, key_out=k_out)
    assert q is q_out and k is k_out
    _check(q, view.cpu(), weight, cos, sin, positions, False)
    _check(k, other.cpu(), weight, cos, sin, positions, False)
    assert bool((out[..., offset + dim:] == 7).all()) and bool((out[..., :offset] == 7).all())
    # In place: the outputs are the inputs.
    same = view.clone()
    qk_norm_rope(same, same, *args, epsilon=EPSILON, query_out=same.clone(), key_out=same)
    _check(same, view.cpu(), weight, cos, sin, positions, False)


@pytest.mark.parametrize("layout", ["pages", "heads_first", "joint"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_rows_land_in_their_slots(dtype, layout) -> None:
    gen = torch.Generator().manual_seed(5)
    tokens, query_heads, heads, dim, pages, page_size = 37, 8, 2, 128, 9, 7
    qkv = torch.randn((tokens, (query_heads + 2 * heads) * dim), generator=gen)
    parts = [p.unflatten(1, (-1, dim)) for p in qkv.split([query_heads * dim, heads * dim, heads * dim], 1)]
    device = [p.unflatten(1, (-1, dim)) for p in qkv.cuda().split([query_heads * dim, heads * dim, heads * dim], 1)]
    cos, sin = _tables(gen, 64, dim)
    positions = torch.randint(0, 64, (tokens,), generator=gen, dtype=torch.int32)
    positions[4], positions[5] = -1, 64  # outside the table: NaN
    slots = torch.randperm(pages * page_size, generator=gen)[:tokens].contiguous()
    slots[0], slots[1], slots[2] = -1, pages * page_size, 2**40  # padding, and nothing past the end
    if layout == "pages":
        caches = [torch.full((pages, page_size, heads, dim), 9.0, device="cuda", dtype=dtype) for _ in range(2)]
    elif layout == "heads_first":
        caches = [torch.full((pages, heads, page_size, dim), 9.0, device="cuda", dtype=dtype).transpose(1, 2) for _ in range(2)]
    else:
        joint = torch.full((pages, 2, page_size, heads, dim), 9.0, device="cuda", dtype=dtype)
        caches = [joint[:, 0], joint[:, 1]]
    weight = torch.rand((dim,), generator=gen) + 0.5
    q = qk_norm_rope_cache(*device, cos.cuda(), sin.cuda(), positions.cuda(), slots.cuda(), *caches, weight.cuda(), weight.cuda(),
                           epsilon=EPSILON, interleaved=True)
    assert q.dtype == dtype
    _check(q, parts[0], weight, cos, sin, positions, True)
    stored = [c.cpu().reshape(-1, heads, dim) for c in caches]
    used = (slots >= 0) & (slots < pages * page_size)
    _check(stored[0][slots[used]], parts[1][used], weight, cos, sin, positions[used], True)
    assert torch.equal(stored[1][slots[used]], parts[2][used].to(dtype))
    rest = torch.ones(pages * page_size, dtype=torch.bool)
    rest[slots[used]] = False
    assert bool((stored[0][rest] == 9).all()) and bool((stored[1][rest] == 9).all())


def test_no_tokens_and_infinities() -> None:
    cos = torch.ones((4, 32), device="cuda")
    none = torch.empty((0, 2, 64), device="cuda")
    index = torch.empty((0,), device="cuda", dtype=torch.int32)
    q, k = qk_norm_rope(none, none, cos, cos, index)
    assert q.shape == k.shape == none.shape
    x = torch.ones((1, 2, 64), device="cuda")
    x[0, 0, 3] = float("inf")
    q, _ = qk_norm_rope(x, x, cos, torch.zeros_like(cos), torch.zeros(1, device="cuda", dtype=torch.int32))
    assert torch.isinf(q[0, 0, 3]) and bool((q[0, 1] == 1).all())  # other rows are not touched by it


def test_queue_submission_and_a_foreign_stream() -> None:
    gen = torch.Generator().manual_seed(8)
    tokens, heads, dim = 64, 4, 64
    q, k, v = (torch.randn((tokens, heads, dim), generator=gen) for _ in range(3))
    cos, sin = _tables(gen, tokens, dim)
    positions = torch.arange(tokens, dtype=torch.int32)
    caches = [torch.zeros((4, 16, heads, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    q_out = torch.empty((tokens, heads, dim), device="cuda", dtype=torch.bfloat16)
    with Queue() as queue:
        args = (q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), positions.cuda(), torch.arange(tokens, device="cuda"),
                *caches, q_out, None, None, QkNormRopeOptions(epsilon=EPSILON))
        queue.submit(QK_NORM_ROPE_CACHE_KERNEL, args, grid=qk_norm_rope_grid(q)).wait()
    _check(q_out, q, None, cos, sin, positions, False)
    _check(caches[0].reshape(tokens, heads, dim), k, None, cos, sin, positions, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, _ = qk_norm_rope(args[0], args[1], *args[3:6], epsilon=EPSILON, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    _check(out, q, None, cos, sin, positions, False)
