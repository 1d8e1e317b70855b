"""The three paged operators together, as a serving loop runs them."""

import random

import pytest
import torch

from kernelforge_amd.flash_attention_jvp import (flash_attention, paged_attention, paged_block_tables_,
                                                 paged_cache_append_, paged_kv_cache)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def elements(cache, row, count):
    """The keys and values [1, count, H, D] that a request's blocks stand for."""
    T, (H, D) = cache.key.shape[2], cache.key.shape[1::2]
    at = torch.tensor(row[:-(-count // T)], device=DEV)
    raw = [t.view(torch.uint8)[at].view(t.dtype).float() for t in cache[:2]]
    k = raw[0] * cache.key_scale[at][..., None, None]
    v = raw[1].transpose(-1, -2).reshape(k.shape) * cache.value_scale[at][..., None, None]
    return tuple(x.transpose(1, 2).reshape(1, -1, H, D)[:, :count] for x in (k, v))


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_prompts_then_decoding(dtype):
    """Ragged prompts, then tokens one by one and by drafts, one request idle now and
    then; every step's attention is the dense one on what the cache stands for,
    and what it stands for is the appended tokens to the cache's precision."""
    rng = random.Random(7)
    B, Hq, H, D, T, width = 3, 8, 2, 64, 16, 12
    g = torch.Generator(DEV).manual_seed(1)
    cache = paged_kv_cache(40, H, D, block_tokens=T, dtype=dtype)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    context, used = ints([0] * B), ints([0])
    free = ints(rng.sample(range(40), 40))
    held = [([], []) for _ in range(B)]
    for counts in ([37, 5, 64], [1, 1, 1], [1, 0, 1], [4, 1, 3], [0, 0, 0], [1, 30, 1], [1, 1, 1]):
        n, spare = sum(counts), 2
        qkv = torch.randn(n + spare, Hq + 2 * H, D, generator=g, device=DEV).to(torch.bfloat16)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        starts, context, slots, used = paged_block_tables_(tables, context, ints(counts), free, used,
                                                           total_tokens=n + spare, block_tokens=T)
        paged_cache_append_(cache, k, v, slots)
        out = paged_attention(q, cache, tables, context, starts, max_query_len=max(1, *counts))
        at, lengths, rows = starts.tolist(), context.tolist(), tables.tolist()
        for b in range(B):
            held[b][0].append(k[at[b]:at[b + 1]])
            held[b][1].append(v[at[b]:at[b + 1]])
            if not counts[b]:
                continue
            ck, cv = elements(cache, rows[b], lengths[b])
            # A code is within a rounding of its element (e4m3 2^-4 of it, int8 half a step of 2 max / 127 at
            # most), once for each time its block's scale grew after it: three here at most are allowed for.
            for x, want in ((ck, torch.cat(held[b][0])), (cv, torch.cat(held[b][1]))):
                step = 2.0 ** -4 if dtype != torch.int8 else 0.0
                bound = 3 * (step * want.abs() + want.abs().max() * (2 / 127 / 2 if dtype == torch.int8 else 2.0 ** -16))
                assert ((x[0] - want.float()).abs() <= bound).all()
            dense = flash_attention(q[None, at[b]:at[b + 1]].contiguous(), ck.to(torch.bfloat16), cv.to(torch.bfloat16),
                                    causal=True)
            # e4m3 and int8 codes times powers of two are exact in bf16; two bf16 results and the dense
            # operator's bf16 probabilities: 2^-7 of the result and 2^-8 of the largest value.
            torch.testing.assert_close(out[at[b]:at[b + 1]].float(), dense[0].float(), rtol=2.0 ** -7,
                                       atol=2.0 ** -8 * float(cv.abs().max()))
        assert not out[n:].any()
    assert used.item() == sum(-(-c // T) for c in lengths)


def test_captured_decoding_step():
    """One step captured once and replayed token by token: lengths, tables and the
    cache advance in place, as the eager loop's do."""
    B, Hq, H, D, T, width, steps = 4, 4, 2, 64, 16, 4, 40
    g = torch.Generator(DEV).manual_seed(3)
    qkv = torch.randn(steps, B, Hq + 2 * H, D, generator=g, device=DEV).to(torch.bfloat16)

    def fresh():
        return (paged_kv_cache(16, H, D, block_tokens=T), torch.full((B, width), -1, dtype=torch.int32, device=DEV),
                ints([0] * B), ints([0]))

    free, ones = ints([5, 3, 15, 0, 1, 2, 4, 6, 7, 8, 9, 10, 11, 12, 13, 14]), ints([1] * B)

    def step(x, cache, tables, context, used):
        starts, context, slots, used = paged_block_tables_(tables, context, ones, free, used, total_tokens=B,
                                                           block_tokens=T, in_place=True)
        paged_cache_append_(cache, x[:, Hq:Hq + H], x[:, Hq + H:], slots)
        return paged_attention(x[:, :Hq], cache, tables, context, starts, max_query_len=1)

    eager = fresh()
    want = [step(qkv[i], *eager) for i in range(steps)]
    state, x = fresh(), qkv[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, *state)
    for i in range(steps):
        x.copy_(qkv[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
    for a, b in zip((*state[0], *state[1:]), (*eager[0], *eager[1:])):
        assert torch.equal(*(t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b)))
    assert state[3].item() == B * -(-steps // T)
