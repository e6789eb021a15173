"""The measured workloads of the attention operators over a paged cache, through their public entry points.

Five kinds of call: the per-head norms and rotation of new queries and keys (alone, or storing keys and values into
the cache), attention of new tokens over the cache (one token a sequence, or a chunk), the attention weights that each
cached slot received, and eviction down to a budget of slots.  Head layouts are TinyLlama-1.1B's (32 query heads on 4
key heads of 64), Llama-7B class (32 on 32 of 128) and Llama-3-8B's (32 on 8 of 128), and generic ones; ``draw``
spreads more cases over the same ranges.

With ``own`` false everything is plain torch in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "qpu-xla-triton_amd")
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPSILON = 1e-5
# A drawn case costs no more than the largest listed ones.
MOST_FLOPS = 4 * 128 * 32 * (8192 * 8193 // 2)
MOST_BYTES = 2_800_000_000


def listed():
    return [
        # One new token of a TinyLlama-1.1B stream: rotate fp32 rows from the linears and store them. Latency.
        {"name": "rope_cache_t1", "kind": "rope_cache", "tokens": 1, "heads": 32, "kv_heads": 4, "dim": 64,
         "rotary": 64, "interleaved": True, "norm": False, "input": "float32", "cache": "bfloat16", "page": 16},
        # A Llama-3-8B prefill chunk with per-head norms: the ordinary large call.
        {"name": "rope_cache_t4096", "kind": "rope_cache", "tokens": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "norm": True, "input": "float32", "cache": "bfloat16", "page": 64},
        # A ragged batch without a cache, heads of 80 rotated over their first 32 dimensions.
        {"name": "rope_t777", "kind": "rope", "tokens": 777, "heads": 20, "kv_heads": 5, "dim": 80, "rotary": 32,
         "interleaved": False, "norm": True, "input": "bfloat16"},
        # One token of one TinyLlama-1.1B stream: the smallest attention, latency.
        {"name": "attention_decode_b1", "kind": "attention", "sequences": 1, "queries": 1, "context": 1900, "spread": 0.0,
         "heads": 32, "kv_heads": 4, "dim": 64, "type": "bfloat16", "page": 16, "window": 0, "causal": True},
        # A serving batch of 64 Llama-3-8B sequences of up to 16k tokens, ragged: bound by the cache's bytes.
        {"name": "attention_decode_b64", "kind": "attention", "sequences": 64, "queries": 1, "context": 16384,
         "spread": 0.8, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64, "window": 0,
         "causal": True},
        # A 512-token chunk of one long prompt over 32k cached tokens.
        {"name": "attention_chunk_512", "kind": "attention", "sequences": 1, "queries": 512, "context": 32768,
         "spread": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64, "window": 0,
         "causal": True},
        # The whole prefill of an 8k prompt on Llama-7B class heads: the largest call.
        {"name": "attention_prefill_8k", "kind": "attention", "sequences": 1, "queries": 8192, "context": 8192,
         "spread": 0.0, "heads": 32, "kv_heads": 32, "dim": 128, "type": "bfloat16", "page": 128, "window": 0,
         "causal": True},
        # A mixed step: seven sequences, chunks from a single token to 300, a window, odd pages, wide heads, half.
        {"name": "attention_mixed", "kind": "attention", "sequences": 7, "queries": 300, "context": 5001, "spread": 1.0,
         "heads": 8, "kv_heads": 2, "dim": 256, "type": "float16", "page": 24, "window": 2000, "causal": True},
        # The weights that one decode step of 16 sequences gave to each slot.
        {"name": "scores_decode_b16", "kind": "scores", "sequences": 16, "queries": 1, "context": 8192, "spread": 0.5,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64, "window": 0, "causal": True},
        # The weights of a whole 4k prompt.
        {"name": "scores_prefill_4k", "kind": "scores", "sequences": 1, "queries": 4096, "context": 4096, "spread": 0.0,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64, "window": 0, "causal": True},
        # A decode step at the budget: every head of 32 sequences gives up one slot.
        {"name": "evict_step_b32", "kind": "evict", "sequences": 32, "context": 2049, "spread": 0.0, "budget": 2048,
         "recent": 256, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64},
        # Long prompts of 4.8k to 32k slots cut down after their prefill.
        {"name": "evict_32k_to_4k", "kind": "evict", "sequences": 4, "context": 32768, "spread": 1.0, "budget": 4096,
         "recent": 1024, "kv_heads": 8, "dim": 128, "type": "bfloat16", "page": 64},
    ]


# --------------------------------------------------------------------- drawing


def _log(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm, as a multiple of `multiple`."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / multiple)) * multiple))


def _layout(rng):
    """(query heads, key heads, head size) of the listed models or in between."""
    if rng.random() < 0.5:
        return rng.choice(((32, 4, 64), (32, 32, 128), (32, 8, 128)))
    kv_heads = rng.randint(1, 8)
    return kv_heads * rng.randint(1, 8), kv_heads, rng.choice((64, 80, 96, 112, 128, 192, 256))


def draw(rng):
    while True:
        kind = rng.choice(("rope", "rope_cache", "attention", "attention", "attention", "scores", "evict"))
        heads, kv_heads, dim = _layout(rng)
        page = rng.choice((16, 32, 64, 128, rng.randint(8, 128)))
        half = rng.choice(("bfloat16", "bfloat16", "float16"))
        if kind in ("rope", "rope_cache"):
            case = {"kind": kind, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                    "rotary": rng.choice((dim, dim, dim // 2)), "interleaved": rng.random() < 0.5,
                    "norm": rng.random() < 0.7, "input": rng.choice(("float32", "float32", "bfloat16", "float16"))}
            if kind == "rope_cache":
                case["cache"], case["page"] = half, page
        elif kind in ("attention", "scores"):
            queries = 1 if rng.random() < 0.5 else _log(rng, 2, 8192)
            case = {"kind": kind, "sequences": _log(rng, 1, 64), "queries": queries,
                    "context": max(queries, _log(rng, 64, 32768)), "spread": rng.choice((0.0, 0.5, 1.0)), "heads": heads,
                    "kv_heads": kv_heads, "dim": dim, "type": half, "page": page,
                    "window": 0 if rng.random() < 0.7 else _log(rng, 32, 8192), "causal": rng.random() < 0.8}
            # The plain form lays every sequence out to the longest's length.
            if case["sequences"] * case["context"] * max(queries * heads, 2 * kv_heads * dim) > 4_000_000_000:
                continue
        else:
            budget = _log(rng, 128, 8192)
            context = budget + 1 if rng.random() < 0.4 else _log(rng, budget, 32768)
            case = {"kind": kind, "sequences": _log(rng, 1, 32), "context": context, "spread": rng.choice((0.0, 1.0)),
                    "budget": budget, "recent": rng.randint(0, budget // 2), "kv_heads": kv_heads, "dim": dim, "type": half,
                    "page": page}
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            return case


def _lengths(case):
    """(context, new tokens) of each sequence: the first is the longest, the others lie below it by up to `spread`."""
    pairs = []
    for b in range(case["sequences"]):
        share = 1.0 - case["spread"] * ((b * 0.6180339887498949) % 1.0)
        new = max(1, int(case.get("queries", 1) * (share if b % 3 else 1.0 - case["spread"] * (b > 0))))
        pairs.append((max(new, int(case["context"] * share)), new))
    return pairs


# ----------------------------------------------------------------------- costs


def _visible(context, new, causal, window):
    """(sum over new tokens of the slots each sees, slots that any of them sees)."""
    pairs, low = 0, context
    for i in range(new):
        p = context - new + i
        high = p + 1 if causal else context
        first = max(0, p - window + 1) if window else 0
        pairs += high - first
        low = min(low, first)
    return pairs, context - low


def _moved(case, context):
    """Slots per head that eviction is expected to move for scores without order."""
    budget, recent = case["budget"], case["recent"]
    if context <= budget:
        return 0
    return budget * (context - budget) / context


def work(case):
    if case["kind"] in ("rope", "rope_cache"):
        element = 4 if case["input"] == "float32" else 2
        read = case["heads"] + case["kv_heads"] * (2 if case["kind"] == "rope_cache" else 1)
        size = case["tokens"] * case["dim"]
        out = 2 if case["kind"] == "rope_cache" else element
        rotated = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": size * read * (element + out) + case["tokens"] * (case["rotary"] * 4 + 12),
                "flops": rotated * (3 * case["rotary"] + (4 * case["dim"] if case["norm"] else 0))}
    if case["kind"] == "evict":
        row = case["kv_heads"] * case["dim"] * 2
        lens = [c for c, _ in _lengths(case)]
        moved = sum(_moved(case, c) for c in lens)
        return {"bytes": int(sum(lens) * case["kv_heads"] * 16 + moved * row * 4), "flops": sum(lens) * case["kv_heads"]}
    pairs = slots = tokens = 0
    for context, new in _lengths(case):
        seen = _visible(context, new, case["causal"], case["window"])
        pairs, slots, tokens = pairs + seen[0], slots + seen[1], tokens + new
    row = case["dim"] * 2
    if case["kind"] == "attention":
        return {"bytes": 2 * slots * case["kv_heads"] * row + 2 * tokens * case["heads"] * row,
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    return {"bytes": slots * case["kv_heads"] * (row + 8) + tokens * case["heads"] * (row + 4),
            "flops": 2 * case["dim"] * case["heads"] * pairs}


# -------------------------------------------------------------------- inputs


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _table(gen, pages_each, width):
    """int32 [sequences, width]: each sequence's pages, taken from a shuffled pool; -1 past its last."""
    pool = torch.randperm(sum(pages_each), generator=gen, device="cuda").to(torch.int32)
    counts = torch.tensor(pages_each, device="cuda")
    column = torch.arange(width, device="cuda")[None, :]
    index = (counts.cumsum(0) - counts)[:, None] + column
    return torch.where(column < counts[:, None], pool[index.clamp(max=len(pool) - 1)], -1)


def _prepare_rope(case, gen):
    t, d = case["tokens"], case["dim"]
    dtype = _TYPES[case["input"]]
    counts = [case["heads"], case["kv_heads"]] + ([case["kv_heads"]] if case["kind"] == "rope_cache" else [])
    fused = torch.randn((t, sum(counts) * d), generator=gen, device="cuda").mul_(2.0).to(dtype)  # one qkv linear's rows
    parts = [p.unflatten(1, (-1, d)) for p in fused.split([c * d for c in counts], dim=1)]
    span = max(4096, t)
    rate = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
    angle = torch.arange(span, device="cuda", dtype=torch.float64)[:, None] * rate
    state = {"query": parts[0], "key": parts[1], "cos": angle.cos().float(), "sin": angle.sin().float(),
             "interleaved": case["interleaved"],
             "positions": torch.randint(0, span, (t,), generator=gen, device="cuda", dtype=torch.int32),
             "query_weight": None, "key_weight": None}
    if case["norm"]:
        state["query_weight"] = 1.0 + 0.2 * torch.randn((d,), generator=gen, device="cuda")
        state["key_weight"] = 1.0 + 0.2 * torch.randn((d,), generator=gen, device="cuda")
    if case["kind"] == "rope_cache":
        pages = -(-t // case["page"]) + 3
        shape = (pages, case["page"], case["kv_heads"], d)
        state["value"] = parts[2]
        state["slots"] = torch.randperm(pages * case["page"], generator=gen, device="cuda")[:t].contiguous()
        state["key_cache"] = torch.zeros(shape, device="cuda", dtype=_TYPES[case["cache"]])
        state["value_cache"] = torch.zeros(shape, device="cuda", dtype=_TYPES[case["cache"]])
    return state


def _prepare_attention(case, gen):
    lens = _lengths(case)
    dtype, d, page = _TYPES[case["type"]], case["dim"], case["page"]
    pages_each = [-(-c // page) for c, _ in lens]
    tokens = sum(n for _, n in lens)
    starts = torch.tensor([0] + [n for _, n in lens], device="cuda").cumsum(0).to(torch.int32)
    shape = (sum(pages_each), page, case["kv_heads"], d)
    state = {
        # Queries a little longer than keys: some slots draw most of a row's weight.
        "query": torch.randn((tokens, case["heads"], d), generator=gen, device="cuda").mul_(2.0).to(dtype),
        "key_cache": torch.randn(shape, generator=gen, device="cuda", dtype=dtype),
        "value_cache": torch.randn(shape, generator=gen, device="cuda", dtype=dtype),
        "block_table": _table(gen, pages_each, max(pages_each)),
        "context_lens": torch.tensor([c for c, _ in lens], device="cuda", dtype=torch.int32),
        "query_starts": None if all(n == 1 for _, n in lens) else starts,
        "max_query": max(n for _, n in lens), "max_context": max(c for c, _ in lens),
        "causal": case["causal"], "window": case["window"], "scale": 1.0 / math.sqrt(d),
    }
    if case["kind"] == "scores":
        del state["value_cache"]
        state["lse"] = _plain_scores(state)[1]
        width = max(pages_each) * page
        before = torch.rand((len(lens), case["kv_heads"], width), generator=gen, device="cuda")
        state["scores"] = before * (torch.arange(width, device="cuda") < state["context_lens"][:, None, None])
    return state


def _prepare_evict(case, gen):
    lens = [c for c, _ in _lengths(case)]
    page, heads = case["page"], case["kv_heads"]
    pages_each = [-(-c // page) for c in lens]
    width = max(pages_each) * page
    shape = (sum(pages_each), page, heads, case["dim"])
    used = torch.arange(width, device="cuda") < torch.tensor(lens, device="cuda")[:, None, None]
    draws = torch.rand((len(lens), heads, width), generator=gen, device="cuda")
    # A few slots hold most of the weight, many hold none at all (ties).
    scores = torch.where(draws < 0.15, 0.0, (-torch.log1p(-draws)) ** 3) * used
    # Earlier evictions left the slots in no order of age.
    order = torch.rand((len(lens), heads, width), generator=gen, device="cuda").masked_fill_(~used, 2.0)
    positions = torch.empty((len(lens), heads, width), device="cuda", dtype=torch.int32)
    positions.scatter_(2, order.argsort(dim=2), torch.arange(width, device="cuda", dtype=torch.int32).expand_as(positions))
    return {
        "key_cache": torch.randn(shape, generator=gen, device="cuda", dtype=_TYPES[case["type"]]),
        "value_cache": torch.randn(shape, generator=gen, device="cuda", dtype=_TYPES[case["type"]]),
        "block_table": _table(gen, pages_each, max(pages_each)),
        "context_lens": torch.tensor(lens, device="cuda", dtype=torch.int32), "scores": scores,
        "positions": torch.where(used, positions, -1), "budget": case["budget"], "recent": case["recent"],
        "max_context": max(lens),
    }


def prepare(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind in ("rope", "rope_cache"):
        state = _prepare_rope(case, gen)
    elif kind == "evict":
        state = _prepare_evict(case, gen)
    else:
        state = _prepare_attention(case, gen)
    state["kind"] = kind
    return state


# ---------------------------------------------------------------- plain torch


def _plain_rotate(x, weight, state):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPSILON) * weight
    cos = state["cos"][state["positions"].long()][:, None, :]
    sin = state["sin"][state["positions"].long()][:, None, :]
    half = cos.shape[-1]
    turned = x.clone()
    if state["interleaved"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned[..., 0:2 * half:2], turned[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned[..., :half], turned[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    return turned


def _plain_rope(state):
    query = _plain_rotate(state["query"], state["query_weight"], state)
    key = _plain_rotate(state["key"], state["key_weight"], state)
    if state["kind"] == "rope":
        return query.to(state["query"].dtype), key.to(state["key"].dtype)
    key_cache, value_cache = state["key_cache"], state["value_cache"]
    key_cache.flatten(0, 1)[state["slots"]] = key.to(key_cache.dtype)
    value_cache.flatten(0, 1)[state["slots"]] = state["value"].to(value_cache.dtype)
    return query.to(key_cache.dtype), key_cache, value_cache


def _rows(cache, table):
    """The cache in the order of each sequence's slots: fp32 [sequences, kv_heads, slots, dim]."""
    rows = cache[table.long().clamp(min=0)].flatten(1, 2)
    return rows.transpose(1, 2).float().contiguous()


def _plain_logits(state):
    """(scaled logits with -inf where a token sees no slot, [sequences, kv_heads, tokens * group, slots]; token numbers)."""
    query, lens = state["query"], state["context_lens"].long()
    starts = state["query_starts"]
    if starts is None:
        starts = torch.arange(len(lens) + 1, device="cuda")
    starts = starts.long()
    new = starts[1:] - starts[:-1]
    step = torch.arange(state["max_query"], device="cuda")
    token = (starts[:-1, None] + step).clamp(max=query.shape[0] - 1)  # [sequences, tokens]
    keys = _rows(state["key_cache"], state["block_table"])[:, :, : state["max_context"]]
    kv_heads, group = keys.shape[1], query.shape[1] // keys.shape[1]
    rows = query[token].float().unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()
    logits = torch.matmul(rows, keys.transpose(2, 3).contiguous()).mul_(state["scale"])
    slot = torch.arange(keys.shape[2], device="cuda")
    at = (lens - new)[:, None, None] + step[None, :, None]
    hidden = (slot >= lens[:, None, None]) | (step[None, :, None] >= new[:, None, None])
    if state["causal"]:
        hidden = hidden | (slot > at)
    if state["window"]:
        hidden = hidden | (slot <= at - state["window"])
    logits.masked_fill_(hidden.repeat_interleave(group, dim=1)[:, None], -math.inf)
    taken = torch.arange(query.shape[0], device="cuda")
    owner = (taken[:, None] >= starts[1:]).sum(dim=1)
    return logits, owner, taken - starts[owner], group


def _by_token(rows, owner, step, group):
    """[sequences, kv_heads, tokens * group, ...] -> [tokens, heads, ...]."""
    return rows.unflatten(2, (-1, group))[owner, :, step].flatten(1, 2)


def _plain_attention(state):
    logits, owner, step, group = _plain_logits(state)
    top = logits.amax(dim=-1, keepdim=True).clamp(min=-3e38)
    weights = logits.sub_(top).exp_()
    total = weights.sum(dim=-1, keepdim=True)
    values = _rows(state["value_cache"], state["block_table"])[:, :, : state["max_context"]]
    out = torch.matmul(weights, values) / torch.where(total > 0, total, 1.0)
    lse = (torch.log(total) + top)[..., 0]
    return (_by_token(out, owner, step, group).to(state["query"].dtype), _by_token(lse, owner, step, group).contiguous())


def _plain_scores(state):
    """(scores, lse); the scores are added to the state's."""
    logits, owner, step, group = _plain_logits(state)
    if "scores" not in state:
        top = logits.amax(dim=-1, keepdim=True).clamp(min=-3e38)
        lse = (logits.sub_(top).exp_().sum(dim=-1, keepdim=True).log() + top)[..., 0]
        return None, _by_token(lse, owner, step, group).contiguous()
    scores = state["scores"].clone()
    lse = torch.zeros(logits.shape[:3], device="cuda").unflatten(2, (-1, group))
    lse[owner, :, step] = state["lse"].unflatten(1, (-1, group))
    logits = logits.sub_(lse.flatten(2, 3)[..., None]).exp_()
    scores[:, :, : logits.shape[3]] += logits.sum(dim=2)
    return scores, None


def _plain_evict(state):
    budget, lens = state["budget"], state["context_lens"].long()
    scores, positions = state["scores"].clone(), state["positions"].clone()
    heads, width = scores.shape[1], scores.shape[2]
    cut = (lens > budget)[:, None, None]
    slot = torch.arange(width, device="cuda").expand_as(scores)
    used = slot < lens[:, None, None]
    newest = positions.masked_fill(~used, -1).amax(dim=2, keepdim=True)
    first = used & (positions > newest - state["recent"])
    order = scores.masked_fill(~used, -math.inf).argsort(dim=2, descending=True, stable=True)
    order = order.gather(2, first.gather(2, order).int().argsort(dim=2, descending=True, stable=True))
    rank = torch.empty_like(order).scatter_(2, order, slot.contiguous())
    kept = used & (rank < budget)
    hole = cut & ~kept & (slot < budget)
    mover = cut & kept & (slot >= budget)
    # The i-th hole takes the i-th slot that moves.
    place = torch.where(mover, mover.cumsum(dim=2) - 1, width)
    source = torch.zeros((*scores.shape[:2], width + 1), device="cuda", dtype=torch.long).scatter_(2, place, slot.contiguous())
    b, h, s = hole.nonzero(as_tuple=True)
    src = source[b, h, (hole.cumsum(dim=2) - 1)[b, h, s]]
    scores[b, h, s], positions[b, h, s] = scores[b, h, src], positions[b, h, src]
    freed = cut & (slot >= budget) & used
    scores.masked_fill_(freed, 0.0)
    positions.masked_fill_(freed, -1)
    table, page = state["block_table"].long(), state["key_cache"].shape[1]
    to, at = (table[b, s // page], s % page, h), (table[b, src // page], src % page, h)
    state["key_cache"][to] = state["key_cache"][at]
    state["value_cache"][to] = state["value_cache"][at]
    return lens.clamp(max=budget).int(), scores, positions, state["key_cache"], state["value_cache"]


# ------------------------------------------------------------------------ run


def _run_own(state):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from qpu_xla_amd import kernels

    kind = state["kind"]
    if kind == "rope":
        return kernels.qk_norm_rope(state["query"], state["key"], state["cos"], state["sin"], state["positions"],
                                    state["query_weight"], state["key_weight"], epsilon=EPSILON,
                                    interleaved=state["interleaved"])
    if kind == "rope_cache":
        query = kernels.qk_norm_rope_cache(state["query"], state["key"], state["value"], state["cos"], state["sin"],
                                           state["positions"], state["slots"], state["key_cache"], state["value_cache"],
                                           state["query_weight"], state["key_weight"], epsilon=EPSILON,
                                           interleaved=state["interleaved"])
        return query, state["key_cache"], state["value_cache"]
    if kind == "attention":
        lse = torch.empty(state["query"].shape[:2], device="cuda", dtype=torch.float32)
        out = kernels.paged_attention(state["query"], state["key_cache"], state["value_cache"], state["block_table"],
                                      state["context_lens"], state["query_starts"], scale=state["scale"],
                                      causal=state["causal"], window=state["window"], max_query=state["max_query"],
                                      max_context=state["max_context"], lse=lse)
        return out, lse
    if kind == "scores":
        return kernels.paged_attention_scores(state["query"], state["key_cache"], state["block_table"],
                                              state["context_lens"], state["lse"], state["query_starts"],
                                              scores=state["scores"], scale=state["scale"], causal=state["causal"],
                                              window=state["window"], max_query=state["max_query"],
                                              max_context=state["max_context"])
    lens, scores, positions = kernels.paged_cache_evict(
        state["key_cache"], state["value_cache"], state["block_table"], state["context_lens"], state["scores"],
        state["positions"], budget=state["budget"], recent=state["recent"], max_context=state["max_context"])
    return lens, scores, positions, state["key_cache"], state["value_cache"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind in ("rope", "rope_cache"):
        return _plain_rope(state)
    if kind == "attention":
        return _plain_attention(state)
    if kind == "scores":
        return _plain_scores(state)[0]
    return _plain_evict(state)


# ---------------------------------------------------------------------- exact


def _exact_rope(state):
    """Rotation as a product of complex numbers, norm from the definition."""
    turn = torch.complex(state["cos"].double(), state["sin"].double())[state["positions"].long()][:, None]
    half = turn.shape[-1]

    def rotate(x, weight):
        x = x.double()
        if weight is not None:
            x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPSILON)
        head, tail = x[..., : 2 * half], x[..., 2 * half:]
        if state["interleaved"]:
            pair = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * turn
            return torch.cat([torch.view_as_real(pair).flatten(-2), tail], -1)
        pair = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
        return torch.cat([pair.real, pair.imag, tail], -1)

    query, key = rotate(state["query"], state["query_weight"]), rotate(state["key"], state["key_weight"])
    if state["kind"] == "rope":
        return query, key
    caches = []
    for cache, rows in ((state["key_cache"], key), (state["value_cache"], state["value"].double())):
        flat = cache.double().flatten(0, 1)
        flat[state["slots"]] = rows
        caches.append(flat.view(cache.shape))
    return query, caches[0], caches[1]


def _exact_attention(state, case):
    """One sequence and one key head at a time, at most 1024 rows of logits."""
    query, scale = state["query"].double(), state["scale"]
    kv_heads = case["kv_heads"]
    group = case["heads"] // kv_heads
    out, lse = torch.zeros_like(query), torch.full(query.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    scores = state["scores"].double() if case["kind"] == "scores" else None
    start = 0
    for b, (context, new) in enumerate(_lengths(case)):
        slots = torch.arange(context, device="cuda")
        pages = state["block_table"][b].long()[slots // case["page"]]
        for kv in range(kv_heads):
            keys = state["key_cache"][pages, slots % case["page"], kv].double()
            values = None if scores is not None else state["value_cache"][pages, slots % case["page"], kv].double()
            for first in range(0, new, 1024):
                last = min(new, first + 1024)
                at = torch.arange(context - new + first, context - new + last, device="cuda")[:, None]
                seen = torch.ones((last - first, context), device="cuda", dtype=torch.bool)
                if case["causal"]:
                    seen &= slots <= at
                if case["window"]:
                    seen &= slots > at - case["window"]
                for head in range(kv * group, (kv + 1) * group):
                    rows = slice(start + first, start + last)
                    logits = torch.where(seen, query[rows, head] @ keys.T * scale, -math.inf)
                    if scores is not None:
                        scores[b, kv, :context] += torch.exp(logits - state["lse"][rows, head, None].double()).sum(0)
                        continue
                    lse[rows, head] = torch.logsumexp(logits, 1)
                    out[rows, head] = torch.exp(logits - lse[rows, head, None]) @ values
        start += new
    return scores if scores is not None else (out, lse)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("rope", "rope_cache"):
        return _exact_rope(state)
    if case["kind"] == "evict":
        return None
    return _exact_attention(state, case)
