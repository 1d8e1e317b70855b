"""Paged 8-bit key/value cache oracle -- TEST INFRASTRUCTURE ONLY.

The definitions of ``paged_block_tables_``, ``paged_cache_append_`` and
``paged_attention`` in plain loops and 64 bits, on the CPU.  The reference has
no cache; what it fixes is the attention itself (flash_attention_jvp/
original.py:6-30, restated in ``fa.attention``, against which the tests hold
``attention`` here) and the convention of rows without a key.

A cache is ``(key[blocks, H, T, D], value[blocks, H, T/16, D, 16],
key_scale[blocks, H], value_scale[blocks, H])``, codes in float8_e4m3fn or int8.
"""

from __future__ import annotations

import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def block_tables(tables, context, queries, free, used, total, T):
    """(tables, query_starts, context, slots, used) after the step, as lists."""
    tables = [list(row) for row in tables]
    starts, slots, after = [0], [], []
    for b, row in enumerate(tables):
        old = max(context[b], 0)
        n = min(max(queries[b], 0), total - starts[-1])
        starts.append(starts[-1] + n)
        after.append(old + n)
        for j in range(-(-old // T), -(-(old + n) // T)):
            block = free[used] if 0 <= used < len(free) else -1
            used += 1
            if j < len(row):
                row[j] = block
        for pos in range(old, old + n):
            block = row[pos // T] if pos // T < len(row) else -1
            slots.append(block * T + pos % T if block >= 0 else -1)
    return tables, starts, after, slots + [-1] * (total - len(slots)), used


def scale_of(largest: float, most: float) -> float:
    """The least power of two s >= 2^-126 with largest <= most * s."""
    e = -126
    while most * 2.0 ** e < largest:
        e += 1
    return 2.0 ** e


def round_code(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """float64 to the nearest code, ties to even, in float64."""
    y = y.clamp(-LARGEST[dtype], LARGEST[dtype])
    if dtype == torch.int8:
        return torch.round(y)
    # e4m3: 3 bits of mantissa, the least exponent of normal numbers -6.
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def tokens_of(value):
    """A value cache [blocks, H, T/16, D, 16] as [blocks, H, T, D]."""
    return value.transpose(-1, -2).reshape(value.shape[0], value.shape[1], -1, value.shape[3])


def append(cache, key, value, slots):
    """The cache after the call: (key codes, value codes [blocks, H, T, D], key
    scales, value scales), all float64."""
    dtype, T = cache[0].dtype, cache[0].shape[2]
    got = []
    for x, codes, scales in ((key, cache[0].double(), cache[2]), (value, tokens_of(cache[1].double()), cache[3])):
        codes, scales, x = codes.clone(), scales.double().clone(), x.double()
        winners: dict[int, dict[int, int]] = {}
        for t, slot in enumerate(slots):
            if 0 <= slot < codes.shape[0] * T:
                winners.setdefault(slot // T, {})[slot % T] = t
        for block, rows in winners.items():
            begun = 0 in rows
            for h in range(codes.shape[1]):
                new = x[list(rows.values()), h]
                finite = bool(torch.isfinite(new).all()) and (begun or math.isfinite(scales[block, h]))
                if finite:
                    s = scale_of(float(new.abs().max()), LARGEST[dtype])
                    if not begun:
                        s = max(s, float(scales[block, h]))
                    ratio = 0.0 if begun else float(scales[block, h]) / s
                    codes[block, h] = round_code(codes[block, h] * ratio, dtype)
                    codes[block, h, list(rows)] = round_code(new / s, dtype)
                else:
                    s = math.nan
                    codes[block, h] = 0.0
                scales[block, h] = s
        got.append((codes, scales))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def attention(q, cache, tables, context, starts=None, *, scale=None, causal=True):
    """(out, lse, spread, slack) in float64.

    spread [tokens, Hq, D] is sum_j p_j |v_j|, what the roundings of the
    probabilities are relative to; slack [Hq, tokens] is the largest sum of
    |q||k| scale over a row's keys, what the roundings of the scores are.
    """
    key, value, key_scale, value_scale = (t.cpu() for t in cache)
    blocks, Hkv, T, D = key.shape
    tokens, Hq = q.shape[:2]
    q = q.cpu().double()
    scale = D ** -0.5 if scale is None else scale
    starts = list(range(tokens + 1)) if starts is None else starts
    out = torch.zeros(tokens, Hq, D, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((Hq, tokens), math.inf, dtype=torch.float64)
    slack = torch.zeros_like(lse)
    values = tokens_of(value.double())
    for b, c in enumerate(context):
        n = starts[b + 1] - starts[b]
        if c <= 0 or n <= 0:
            continue
        ids = [tables[b][j] if j < len(tables[b]) else -1 for j in range(-(-c // T))]
        sound = torch.tensor([0 <= i < blocks for i in ids])
        at = torch.tensor([i if 0 <= i < blocks else 0 for i in ids])
        seen_ok = sound.repeat_interleave(T)[:c]
        for h in range(Hkv):
            k = (key[at, h].double() * key_scale[at, h].double()[:, None, None]).reshape(-1, D)[:c]
            v = (values[at, h] * value_scale[at, h].double()[:, None, None]).reshape(-1, D)[:c]
            k = torch.where(seen_ok[:, None], k, math.nan)
            for i in range(n):
                reach = c - n + i + 1 if causal else c
                if reach <= 0:
                    continue
                t = starts[b] + i
                for g in range(h * Hq // Hkv, (h + 1) * Hq // Hkv):
                    s = (k[:reach] @ q[t, g]) * scale
                    lse[g, t] = torch.logsumexp(s, 0)
                    p = torch.exp(s - lse[g, t])
                    out[t, g] = p @ v[:reach] if not torch.isnan(p).any() else math.nan
                    spread[t, g] = p @ v[:reach].abs()
                    slack[g, t] = (k[:reach].abs() @ q[t, g].abs()).max() * scale
    return out, lse, spread, slack
