"""64-bit definitions of the attention operators over a paged cache, row by row, on the CPU."""

from __future__ import annotations

import math

import torch


def rope(x, weight, cos, sin, positions, epsilon, interleaved):
    """[T, H, D] of any type -> float64, normalised and rotated."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon) * weight.double()
    out = x.clone()
    half = cos.shape[1]
    for t, position in enumerate(positions.tolist()):
        if not 0 <= position < cos.shape[0]:
            out[t, :, : 2 * half] = math.nan
            continue
        c, s = cos[position].double(), sin[position].double()
        first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
        second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
        a, b = x[t][:, first], x[t][:, second]
        out[t][:, first] = a * c - b * s
        out[t][:, second] = b * c + a * s
    return out


def slot_rows(cache, table_row, count, head):
    """Rows of the first `count` slots, zero rows where the table names no page."""
    page_size = cache.shape[1]
    rows = torch.zeros((count, cache.shape[3]), dtype=torch.float64)
    for j in range(0, count, page_size):
        page = int(table_row[j // page_size])
        if 0 <= page < cache.shape[0]:
            n = min(page_size, count - j)
            rows[j:j + n] = cache[page, :n, head].double()
    return rows


def visible(length, new, token, causal, window):
    at = length - new + token
    high = min(length, max(at + 1, 0)) if causal else length
    low = max(0, at - window + 1) if window else 0
    return min(low, high), high


def token_ranges(starts, sequences):
    return [(b, b + 1) for b in range(sequences)] if starts is None else list(zip(starts.tolist()[:-1], starts.tolist()[1:]))


def attention(query, key_cache, value_cache, table, lens, starts=None, *, scale, causal=True, window=0):
    """(out, lse, bound): bound = sum_j p_j |v_j|, the size that rounded weights err against."""
    tokens, heads, dim = query.shape
    kv_heads, slots = key_cache.shape[2], table.shape[1] * key_cache.shape[1]
    group = heads // kv_heads
    out = torch.zeros((tokens, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    for b, (first, last) in enumerate(token_ranges(starts, len(lens))):
        length = min(max(int(lens[b]), 0), slots)
        for kv in range(kv_heads):
            keys, values = (slot_rows(c, table[b], length, kv) for c in (key_cache, value_cache))
            for token in range(last - first):
                low, high = visible(length, last - first, token, causal, window)
                if low >= high:
                    continue
                for h in range(kv * group, (kv + 1) * group):
                    logits = keys[low:high] @ query[first + token, h].double() * scale
                    lse[first + token, h] = torch.logsumexp(logits, 0)
                    p = torch.exp(logits - lse[first + token, h])
                    out[first + token, h] = p @ values[low:high]
                    bound[first + token, h] = p @ values[low:high].abs()
    return out, lse, bound


def scores(query, key_cache, table, lens, lse, starts=None, *, previous, scale, causal=True, window=0):
    heads, kv_heads = query.shape[1], key_cache.shape[2]
    group, slots = heads // kv_heads, table.shape[1] * key_cache.shape[1]
    out = torch.zeros((len(lens), kv_heads, slots), dtype=torch.float64) if previous is None else previous.double()
    for b, (first, last) in enumerate(token_ranges(starts, len(lens))):
        length = min(max(int(lens[b]), 0), slots)
        for kv in range(kv_heads):
            keys = slot_rows(key_cache, table[b], length, kv)
            for token in range(last - first):
                low, high = visible(length, last - first, token, causal, window)
                for h in range(kv * group, (kv + 1) * group):
                    if low < high and lse[first + token, h] != -math.inf:
                        logits = keys[low:high] @ query[first + token, h].double() * scale
                        out[b, kv, low:high] += torch.exp(logits - lse[first + token, h].double())
    return out


def evict(key_cache, value_cache, table, lens, scores, positions, budget, recent):
    """(new lengths, scores, positions, keys, values) after eviction: copies."""
    key_cache, value_cache, scores, positions = (t.clone() for t in (key_cache, value_cache, scores, positions))
    page_size, pages = key_cache.shape[1], key_cache.shape[0]
    slots = table.shape[1] * page_size
    new_lens = []
    for b in range(len(lens)):
        length = min(max(int(lens[b]), 0), slots)
        new_lens.append(min(length, budget))
        if length <= budget:
            continue
        for h in range(key_cache.shape[2]):
            newest = int(positions[b, h, :length].max())
            rank = []
            for s in range(length):
                score = float(scores[b, h, s])
                is_recent = int(positions[b, h, s]) > newest - recent
                # NaN below -inf; recent slots are all alike.
                odd = math.isnan(score)
                rank.append((False, False, 0.0, s) if is_recent else (True, odd, 0.0 if odd else -score, s))
            kept = {entry[3] for entry in sorted(rank)[:budget]}
            holes = [s for s in range(budget) if s not in kept]
            movers = [s for s in range(budget, length) if s in kept]
            assert len(holes) == len(movers)
            old_scores, old_positions = scores[b, h].clone(), positions[b, h].clone()
            for to, source in zip(holes, movers):
                scores[b, h, to], positions[b, h, to] = old_scores[source], old_positions[source]
                to_page, from_page = int(table[b, to // page_size]), int(table[b, source // page_size])
                for cache in (key_cache, value_cache):
                    if 0 <= to_page < pages:
                        row = cache[from_page, source % page_size, h] if 0 <= from_page < pages else 0.0
                        cache[to_page, to % page_size, h] = row
            scores[b, h, budget:length] = 0.0
            positions[b, h, budget:length] = -1
    return torch.tensor(new_lens, dtype=torch.int32), scores, positions, key_cache, value_cache
